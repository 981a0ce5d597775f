// Beam search (sm_100a): the best continuations of each request's beams over the vocabulary, and
// the states that follow the choice.
#include <climits>

#include "cc1d_beam_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {
namespace {

// ------------------------------------------------------------------------- selection
// total[k, v] = scores[k] + logits[k, v] - log sum_w exp(logits[k, w]); the best `candidates` of
// beams x vocabulary, equal ones by the lowest place.
//
// One pass over the logits: each warp walks a strip of a row with the running maximum and sum of the
// softmax, and keeps each lane's largest element in each of up to 32 chunks of the strip.  The n-th
// largest of the threads' maxima is a floor of the best n; the few chunks that reach it (about n of a
// CTA's) are read again, and the elements above it enter a sorted list of each warp, one or two entries
// a lane.  The warps' lists are joined, and a second kernel joins those of a row's parts, then ranks
// the beams' lists.  Beams that are at their end, or not in use, are not walked.
//
// What bounds it: 512 rows of 128000 bf16 logits (131 MB, 20 us of memory) take 53 us, of which the join
// takes 11: 12.8 instructions an element in walk, second look and lists (one exponential, 15 us of all),
// and chains of exchanges; with lists kept during the walk 66 us, and with a floor from its first step
// alone 116.  Beyond the 592 CTAs that run at a time rows wait for a second wave: 592 rows take 54 us,
// 600 take 75, 1024 take 90.  Four rows of 32000 take 12 us: two kernels of which the second waits for
// the first, and in them exchanges and barriers rather than data.
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 2, kChunks = 32;
constexpr int kEmpty = INT_MIN;  // below the order of every float

// Order of floats as integers; -0 counts as 0.
__device__ __forceinline__ int order_of(float f) {
  const int b = __float_as_int(f + 0.f);
  return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float value_of(int o) { return __int_as_float(o >= 0 ? o : o ^ 0x7fffffff); }

// The `n` best of what a warp has seen, sorted by key and then by place: entry 32 q + lane in
// (key[q], at[q]); the last one that counts in (last, last_at).
template <int Q>
struct Best {
  int key[Q], at[Q], last, last_at, n;
  __device__ __forceinline__ void start(int count) {
#pragma unroll
    for (int q = 0; q < Q; ++q) key[q] = kEmpty, at[q] = INT_MAX;
    n = count;
    last = kEmpty;
    last_at = INT_MAX;
  }
  __device__ __forceinline__ bool takes(int k, int place) const { return k > last || (k == last && place < last_at); }
  __device__ __forceinline__ void insert(int k, int place, int lane) {
    int pos = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) pos += __popc(__ballot_sync(~0u, key[q] > k || (key[q] == k && at[q] < place)));
#pragma unroll
    for (int q = Q - 1; q >= 0; --q) {
      int ku = __shfl_up_sync(~0u, key[q], 1), au = __shfl_up_sync(~0u, at[q], 1);
      if (q > 0) {
        const int kl = __shfl_sync(~0u, key[q - 1], 31), al = __shfl_sync(~0u, at[q - 1], 31);
        if (lane == 0) ku = kl, au = al;
      }
      const int i = q * 32 + lane;
      if (i > pos) key[q] = ku, at[q] = au;
      else if (i == pos) key[q] = k, at[q] = place;
    }
    int l = key[0], la = at[0];
#pragma unroll
    for (int q = 1; q < Q; ++q)
      if ((n - 1) / 32 == q) l = key[q], la = at[q];
    const int nl = __shfl_sync(~0u, l, (n - 1) & 31), na = __shfl_sync(~0u, la, (n - 1) & 31);
    if (nl != kEmpty) last = nl, last_at = na;  // a floor stays until the list is full
  }
  // One entry of each lane that has one.
  __device__ __forceinline__ void offer(int k, int place, bool has, int lane) {
    unsigned todo = __ballot_sync(~0u, has && takes(k, place));
    while (todo) {
      const int from = __ffs(todo) - 1;
      insert(__shfl_sync(~0u, k, from), __shfl_sync(~0u, place, from), lane);
      todo &= todo - 1;
      todo &= __ballot_sync(~0u, takes(k, place));
    }
  }
  // The list of 32 entries that stands in `other` is joined to this one (Q = 1).  Of two descending
  // lists a and b the better of a[i] and b[31 - i] are the 32 best, in a bitonic order.
  __device__ __forceinline__ void join(const int2* other, int lane) {
    const int2 o = other[31 - lane];
    int k = key[0], place = at[0];
    if (o.x > k || (o.x == k && o.y < place)) k = o.x, place = o.y;
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
      const int ok = __shfl_xor_sync(~0u, k, step), op = __shfl_xor_sync(~0u, place, step);
      const bool mine = k > ok || (k == ok && place < op), same = k == ok && place == op;
      if (!same && mine != ((lane & step) == 0)) k = ok, place = op;
    }
    key[0] = k;
    at[0] = place;
  }
  // The first entries, one of each lane (none: kEmpty): sorted by exchanges.
  __device__ __forceinline__ void fill(int k, int place, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
      for (int step = size / 2; step > 0; step /= 2) {  // bitonic, the better ones first
        const int ok = __shfl_xor_sync(~0u, k, step), op = __shfl_xor_sync(~0u, place, step);
        const bool low = (lane & step) == 0, down = (lane & size) == 0;
        const bool mine = k > ok || (k == ok && place < op), same = k == ok && place == op;
        if (!same && mine != (low == down)) k = ok, place = op;
      }
    key[0] = k;
    at[0] = place;
    if (n <= 32) {
      last = __shfl_sync(~0u, k, n - 1);
      last_at = __shfl_sync(~0u, place, n - 1);
    }
  }
};

// The sum s + low of 2^(x L - r), L = kLog2e, of a lane or a part of a row.  m is an element that none
// exceeds by more than kRise: rows that rise would else scale their sums down hundreds of times, each
// time off by a rounding.  The reference r is m L as it is rounded, c, where |m| is at most 2^20: one
// multiply-add makes the exponent, and c is off by at most 2^-4, so that no sum leaves the normal numbers;
// log sum exp(x) = m + (log2(sum) + r - m L) log(2) puts the rounding back.  Beyond that the rounding
// would be of any size, and m L itself may overflow: there r is m L, and the exponent (x - m) L.
struct Soft {
  float m = -INFINITY, s = 0.f, low = 0.f;
};
constexpr float kRise = 4.f, kMostFused = 1048576.f;
__device__ __forceinline__ bool is_fused(float m) { return fabsf(m) <= kMostFused; }
// c, or none; rounded wherever it is used (a product is otherwise joined with the sum behind it)
__device__ __forceinline__ float scale_of(float m) { return is_fused(m) ? __fmul_rn(m, kLog2e) : 0.f; }
__device__ __forceinline__ float rest_of(float m) { return is_fused(m) ? fmaf(-m, kLog2e, scale_of(m)) : 0.f; }  // r - m L
__device__ __forceinline__ double reference_of(float m) {
  return is_fused(m) ? static_cast<double>(scale_of(m)) : static_cast<double>(m) * kLog2e;
}
__device__ __forceinline__ void raise(Soft& a, float m) {
  if (m > a.m) {
    float f = 0.f;
    if (is_fused(a.m) && is_fused(m)) f = ex2_approx(scale_of(a.m) - scale_of(m));
    else if (a.m > -INFINITY) f = ex2_approx(fmaf(a.m - m, kLog2e, rest_of(a.m) - rest_of(m)));
    a.s *= f;
    a.low *= f;
    a.m = m;
  }
}
// s + low with the rounding of the sum kept (Knuth's two-sum)
__device__ __forceinline__ void add_to(Soft& a, float v) {
  const float t = a.s + v, w = t - a.s;
  a.low += (a.s - (t - w)) + (v - w);
  a.s = t;
}

// The largest of 2 P elements, two neighbouring ones in one float2.
template <int P>
__device__ __forceinline__ float top_of(const float2 (&x)[P]) {
  float top = fmaxf(x[0].x, x[0].y);
#pragma unroll
  for (int p = 1; p < P; ++p) top = fmaxf(top, fmaxf(x[p].x, x[p].y));
  return top;
}
// Adds the exponentials of 2 P H elements, of which `top` is the largest; c = scale_of(a.m).  Steps whose
// top is not above `limit` need nothing else: the limit is kRise above m, or, where m is beyond 2^20 and
// c is 0, below everything, and the elements become their difference from m.
template <int H, int P>
__device__ __forceinline__ void add_exps(Soft& a, float& c, float& limit, float2 (&x)[H][P], float top) {
  if (top > limit) {
    if (top > a.m + kRise) {
      raise(a, top);
      c = scale_of(top);
    }
    limit = a.m + kRise;
    if (!is_fused(a.m)) {
      limit = -INFINITY;
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int p = 0; p < P; ++p) x[h][p] = fadd2(x[h][p], make_float2(-a.m, -a.m));
    }
  }
  float2 s[H * P];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float2 v = ffma2(x[h][p], make_float2(kLog2e, kLog2e), make_float2(-c, -c));
      s[h * P + p] = make_float2(ex2_approx(v.x), ex2_approx(v.y));
    }
#pragma unroll
  for (int w = H * P / 2; w > 0; w /= 2)
#pragma unroll
    for (int i = 0; i < w; ++i) s[i] = fadd2(s[i], s[i + w]);
  add_to(a, s[0].x + s[0].y);
}

// One step of a bitonic network on the lanes' keys: lanes `step` apart, the larger first where `down`.
__device__ __forceinline__ int exchange(int k, int step, bool down, int lane) {
  const int o = __shfl_xor_sync(~0u, k, step);
  return ((lane & step) == 0) == down ? max(k, o) : min(k, o);
}
__device__ __forceinline__ int sorted_down(int k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2) k = exchange(k, step, (lane & size) == 0, lane);
  return k;
}
// A beam at its end, or without a finite score, has no use for its logits.
__device__ __forceinline__ bool beam_done(const BeamSelectArgs& a, int64_t b, int64_t k, float* score) {
  *score = a.scores[b * a.scores_s0 + k * a.scores_s1];
  return a.finished && a.finished[b * a.finished_s0 + k * a.finished_s1];
}

// Four CTAs an SM leave 64 registers.  When the walk took 54 us, three with four steps on their way took 65
// (two waves), five and six, which spill, 57 and 72.
template <typename T, int Q>
__global__ void __launch_bounds__(kThreads, kBeamCtas) beam_parts_kernel(const BeamSelectArgs a) {
  constexpr int E = 16 / sizeof(T), P = E / 2;
  __shared__ int2 lists[kWarps][Q * 32];
  __shared__ Soft softs[kWarps];
  __shared__ int keys[kThreads], floor;
  __shared__ float maxima[kChunks][kThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int n = static_cast<int>(a.candidates);
  grid_dependency_wait();
  float score;
  const bool ended = beam_done(a, row / a.beams, row % a.beams, &score);
  const T* x = static_cast<const T*>(a.logits) + (row / a.beams) * a.logits_s0 + (row % a.beams) * a.logits_s1;
  const int64_t begin = part * a.part, end = begin + a.part < a.vocab ? begin + a.part : a.vocab;
  const int64_t strip = (end - begin + kWarps - 1) / kWarps;
  int64_t i = begin + warp * strip;
  const int64_t stop = i + strip < end ? i + strip : end;
  // up to the first 16-byte boundary, element by element
  const int64_t past = reinterpret_cast<uintptr_t>(x + i) % 16 / sizeof(T);
  const int64_t head = past && i < stop ? (E - past < stop - i ? E - past : stop - i) : 0, start = i;
  i += head;
  // Steps of 32 E elements; AHEAD of them are on their way, and are taken two at a time.
  constexpr int STEP = 32 * E, AHEAD = kAhead;
  const int size = i < stop ? static_cast<int>(stop - i) : 0, from = lane * E, steps = (size + STEP - 1) / STEP;
  const T* q = x + i;
  // Kept as words until they are used: taking them apart at once would wait for the load.
  uint4 next[AHEAD];
  auto fetch = [&](int n) {
    const int at = from + n * STEP;
    return at + E <= size ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
  };
  auto values = [&](int n, const uint4& u, float2 (&v)[P]) {
    unpack2<T, E>(*reinterpret_cast<const Packet<T, E>*>(&u), v);
    if ((n + 1) * STEP > size) {
      const int at = from + n * STEP;
      if (at + E > size)
#pragma unroll
        for (int p = 0; p < P; ++p)
          v[p] = make_float2(at + 2 * p < size ? to_f32(q[at + 2 * p]) : -INFINITY,
                             at + 2 * p + 1 < size ? to_f32(q[at + 2 * p + 1]) : -INFINITY);
    }
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) next[k] = fetch(k);
  if (ended || !(fabsf(score) < INFINITY)) return;
  // The sums, and the largest element of each lane in each of up to kChunks chunks of the strip.
  Soft soft;
  float c = 0.f, limit = -INFINITY, most = -INFINITY;
  const float first = lane < head ? to_f32(x[start + lane]) : -INFINITY;
  if (head) {
    float2 v[1][1] = {{make_float2(first, -INFINITY)}};
    add_exps(soft, c, limit, v, first);
  }
  const int groups = (steps + AHEAD - 1) / AHEAD, chunk = (groups + kChunks - 1) / kChunks;
  for (int g = 0, at = 0; g < groups; ++at) {
    float most_here = -INFINITY;
    for (const int till = min(g + chunk, groups); g < till; ++g) {
#pragma unroll
      for (int k = 0; k < AHEAD; k += 2) {
        const int n0 = g * AHEAD + k;
        if (n0 >= steps) break;
        float2 v[2][P];
        values(n0, next[k], v[0]);
        values(n0 + 1, next[k + 1], v[1]);
        next[k] = fetch(n0 + AHEAD);
        next[k + 1] = fetch(n0 + 1 + AHEAD);
        const float top = fmaxf(top_of(v[0]), top_of(v[1]));
        add_exps(soft, c, limit, v, top);
        most_here = fmaxf(most_here, top);
      }
    }
    maxima[at][threadIdx.x] = most_here;
    most = fmaxf(most, most_here);
  }
  // The n-th largest of the threads' maxima: n elements of the CTA's part are at least that.  A warp
  // sorts its own, and each finds its rank among all by bisection of the other warps' lists.
  const int key = sorted_down(order_of(most), lane);
  keys[threadIdx.x] = key;
  __syncthreads();
  int rank = lane;
#pragma unroll
  for (int o = 1; o < kWarps; ++o) {
    const int other = (warp + o) % kWarps;
    const int* list = keys + other * 32;
    const int least = other < warp ? key : key + 1;  // the lower warp's first
    int low = 0;  // entries that stand before
#pragma unroll
    for (int step = 16; step > 0; step /= 2)
      if (list[low + step - 1] >= least) low += step;
    rank += low + (low == 31 && list[31] >= least ? 1 : 0);
  }
  if (rank == n - 1) floor = key;
  __syncthreads();
  // The elements that may be among the n best, by places.
  Best<Q> best;
  best.start(n);
  float least;  // elements below it do not count; one that equals the list's last entry comes too late
  auto set_least = [&](int k) { least = k <= order_of(-INFINITY) ? -INFINITY : value_of(k); };
  set_least(floor);
  // `has` lanes' elements v at place + lane
  auto offer = [&](float v, int place, int has) {
    best.offer(order_of(v), place + lane, lane < has && v >= least, lane);
    set_least(max(best.last + 1, floor));
  };
  if (head) offer(first, static_cast<int>(start), static_cast<int>(head));
  for (int g = 0, at = 0; g < groups; g += chunk, ++at) {
    if (!__any_sync(~0u, maxima[at][threadIdx.x] >= least)) continue;
    const int till = min((g + chunk) * AHEAD, steps);
    for (int n0 = g * AHEAD; n0 < till; ++n0) {
      float2 v[P];
      values(n0, fetch(n0), v);
      // the lanes that have some, one after the other: its elements to the first E lanes
      unsigned todo = __ballot_sync(~0u, top_of(v) >= least);
      for (; todo; todo &= todo - 1) {
        const int of = __ffs(todo) - 1;
        float mine = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float f = __shfl_sync(~0u, e % 2 ? v[e / 2].y : v[e / 2].x, of);
          if (lane == e) mine = f;
        }
        const int here = n0 * STEP + of * E;
        offer(mine, static_cast<int>(i) + here, min(size - here, E));
      }
    }
  }
#pragma unroll
  for (int q = 0; q < Q; ++q) lists[warp][q * 32 + lane] = make_int2(best.key[q], best.at[q]);
#pragma unroll
  for (int bit = 1; bit < 32; bit *= 2) {
    Soft o;
    o.m = __shfl_xor_sync(~0u, soft.m, bit);
    o.s = __shfl_xor_sync(~0u, soft.s, bit);
    o.low = __shfl_xor_sync(~0u, soft.low, bit);
    const float m = fmaxf(soft.m, o.m);
    raise(soft, m);
    raise(o, m);
    add_to(soft, o.s);
    soft.low += o.low;
  }
  if (lane == 0) softs[warp] = soft;
  __syncthreads();
  if (warp != 0) return;
  for (int o = 1; o < kWarps; ++o) {
    if constexpr (Q == 1) {
      best.join(lists[o], lane);
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int2 c = lists[o][q * 32 + lane];
        best.offer(c.x, c.y, q * 32 + lane < n && c.x != kEmpty, lane);
      }
    }
    Soft s = softs[o];
    const float m = fmaxf(soft.m, s.m);
    raise(soft, m);
    raise(s, m);
    add_to(soft, s.s);
    soft.low += s.low;
  }
  int2* out = a.best + static_cast<int64_t>(blockIdx.x) * n;
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (q * 32 + lane < n) out[q * 32 + lane] = make_int2(best.key[q], best.at[q]);
  if (lane == 0) a.sums[blockIdx.x] = make_float2(soft.m, soft.s + soft.low);
}

// One CTA for each request.  A warp joins a beam's parts and writes the beam's best with their
// totals, in 64 bits, to shared memory; then every candidate finds its rank.
template <int Q>
__global__ void __launch_bounds__(kThreads) beam_join_kernel(const BeamSelectArgs a) {
  extern __shared__ double totals[];  // (beams, n), then the tokens
  const int n = static_cast<int>(a.candidates), beams = static_cast<int>(a.beams);
  int* tokens = reinterpret_cast<int*>(totals + beams * n);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t b = blockIdx.x;
  grid_dependency_wait();
  for (int k = warp; k < beams; k += kWarps) {
    const int64_t first = (b * beams + k) * a.parts;
    float score;
    const bool ended = beam_done(a, b, k, &score), read = !ended && fabsf(score) < INFINITY;  // the parts are there
    const int64_t parts = read ? a.parts : 0, entries = parts * n;
    Best<Q> best;
    best.start(n);
    float m = -INFINITY;
    for (int64_t p = lane; p < parts; p += 32) m = fmaxf(m, a.sums[first + p].x);
#pragma unroll
    for (int bit = 1; bit < 32; bit *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, bit));
    double s = 0.0;
    for (int64_t p = lane; p < parts; p += 32) {
      const float2 v = a.sums[first + p];
      // a part without anything above -inf has the sum 0, or NaN
      s += static_cast<double>(v.y) * (v.x > -INFINITY ? exp2(reference_of(v.x) - reference_of(m)) : 1.0);
    }
#pragma unroll
    for (int bit = 1; bit < 32; bit *= 2) s += __shfl_xor_sync(~0u, s, bit);
    // log sum exp(x) = m + above; m is taken from the logits first, since a large one would swallow the rest
    const double above = log(s) + (reference_of(m) - static_cast<double>(m) * kLog2e) * 0.69314718055994531;
    for (int64_t e = lane; e - lane < entries; e += 32) {
      const int2 c = e < entries ? a.best[first * n + e] : make_int2(kEmpty, INT_MAX);
      if (e < 32) best.fill(c.x, c.y, lane);
      else best.offer(c.x, c.y, c.x != kEmpty, lane);
    }
    // a row that is no distribution (a NaN, an infinity, nothing left) offers nothing
    const bool sound = fabsf(score) < INFINITY && (ended || fabs(above) < INFINITY);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = q * 32 + lane;
      if (i >= n) continue;
      double total = -INFINITY;
      int token = i;  // nothing offered: the lowest places
      if (sound && ended) {
        if (i == 0) total = score, token = static_cast<int>(a.end_token);
        else if (i <= a.end_token) token = i - 1;
      } else if (sound && best.key[q] != kEmpty) {
        total = static_cast<double>(score) + (static_cast<double>(value_of(best.key[q])) - m - above);
        token = best.at[q];
      }
      totals[k * n + i] = total;
      tokens[k * n + i] = i < a.vocab ? token : -1;
    }
  }
  __syncthreads();
  // Each candidate's rank: how many of its own beam stand before it, and how many of each other
  // beam are better, by bisection of that beam's descending totals.
  for (int i = threadIdx.x; i < beams * n; i += kThreads) {
    const int k = i / n, e = i - k * n;
    if (tokens[i] < 0) continue;
    const double t = totals[i];
    int rank = e;
    for (int o = 0; o < beams && rank < n; ++o) {
      if (o == k) continue;
      const double* list = totals + o * n;
      const int* names = tokens + o * n;
      int low = 0, high = n;  // entries before `low` are better, those from `high` on are not
      while (low < high) {
        const int m = (low + high) / 2;
        const bool better = names[m] >= 0 && (list[m] > t || (list[m] == t && o < k));
        if (better) low = m + 1;
        else high = m;
      }
      rank += low;
    }
    if (rank >= n) continue;
    a.out_scores[b * n + rank] = static_cast<float>(t);
    a.parents[b * n + rank] = k;
    a.tokens[b * n + rank] = tokens[i];
  }
}

template <typename T, int Q>
cudaError_t run_select(const BeamSelectArgs& a, cudaStream_t s) {
  cudaError_t e = launch_dependent(beam_parts_kernel<T, Q>, dim3(static_cast<unsigned>(a.batch * a.beams * a.parts)), dim3(kThreads), 0, s, a);
  if (e != cudaSuccess) return e;
  const size_t smem = static_cast<size_t>(a.beams * a.candidates) * 12;
  e = allow_dynamic_smem(reinterpret_cast<const void*>(beam_join_kernel<Q>), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(beam_join_kernel<Q>, dim3(static_cast<unsigned>(a.batch)), dim3(kThreads), smem, s, a);
}
template <typename T>
cudaError_t run_select(const BeamSelectArgs& a, cudaStream_t s) {
  return a.candidates <= 32 ? run_select<T, 1>(a, s) : run_select<T, 2>(a, s);
}

// ------------------------------------------------------------------------ reordering
// A thread takes one column of a request's rows: it reads it from every parent that is needed,
// then writes it to every beam whose parent is another one, so the rows change in place.  32 requests
// of 8 beams with 430 MB to move take 68 us, 66 at the copy's rate.
template <int BEAMS, typename U>
__device__ __forceinline__ void move_column(const BeamReorderArgs& a, const BeamRows& t, int64_t column, const int* source, const int* target) {
  int64_t at = column * t.step0;
  if (t.size0 < t.columns) {
    const int64_t rest = column / t.size0, outer = rest / t.size1;
    at += (rest - outer * t.size1) * t.step1 - rest * t.size0 * t.step0;
    at += outer < t.size2 ? outer * t.step2 : outer % t.size2 * t.step2 + outer / t.size2 * t.step3;
  }
  U v[BEAMS];
#pragma unroll
  for (int k = 0; k < BEAMS; ++k)
    if (k < a.beams && source[k] >= 0) v[k] = *reinterpret_cast<const U*>(t.data + source[k] * t.row_bytes + at);
#pragma unroll
  for (int k = 0; k < BEAMS; ++k)
    if (k < a.beams && source[k] >= 0) *reinterpret_cast<U*>(t.data + target[k] * t.row_bytes + at) = v[k];
}

template <int BEAMS>
__global__ void __launch_bounds__(kThreads) beam_reorder_kernel(const __grid_constant__ BeamReorderArgs a) {
  __shared__ int source[BEAMS], target[BEAMS];  // rows; source -1: the beam keeps its row
  int64_t i = blockIdx.x;
  int n = 0;
  while (i >= a.batch * a.t[n].blocks) i -= a.batch * a.t[n++].blocks;
  const BeamRows& t = a.t[n];
  const uint32_t b = static_cast<uint32_t>(i) / static_cast<uint32_t>(t.blocks);  // grids are below 2^31
  const int64_t block = i - static_cast<int64_t>(b) * t.blocks;
  grid_dependency_wait();
  if (threadIdx.x < a.beams) {
    const int64_t k = threadIdx.x, at = static_cast<int64_t>(b) * a.parents_s0 + k * a.parents_s1;
    const int64_t parent = a.wide_parents ? static_cast<const int64_t*>(a.parents)[at] : static_cast<const int32_t*>(a.parents)[at];
    int64_t from = -1, to = static_cast<int64_t>(b) * a.beams + k;
    if (parent >= 0 && parent < a.beams && parent != k) {
      from = static_cast<int64_t>(b) * a.beams + parent;
      if (a.indices) {
        from = a.indices[from * a.indices_stride];
        to = a.indices[to * a.indices_stride];
      }
      if (from < 0 || from >= t.rows || to < 0 || to >= t.rows) from = -1;
    }
    source[k] = static_cast<int>(from);
    target[k] = static_cast<int>(to);
  }
  __syncthreads();
  const int64_t column = block * kThreads + threadIdx.x;
  if (column >= t.columns) return;
  switch (t.unit) {
    case 16:
      if constexpr (BEAMS <= 16) move_column<BEAMS, uint4>(a, t, column, source, target);
      break;
    case 8:
      if constexpr (BEAMS <= 32) move_column<BEAMS, uint2>(a, t, column, source, target);
      break;
    case 4: move_column<BEAMS, uint32_t>(a, t, column, source, target); break;
    case 2: move_column<BEAMS, uint16_t>(a, t, column, source, target); break;
    default: move_column<BEAMS, uint8_t>(a, t, column, source, target); break;
  }
}

}  // namespace

int64_t beam_most_unit(int64_t beams) { return beams <= 16 ? 16 : beams <= 32 ? 8 : 4; }

cudaError_t beam_select(const BeamSelectArgs& a, int dtype, cudaStream_t s) {
  switch (dtype) {
    case CC1D_FLOAT32: return run_select<float>(a, s);
    case CC1D_FLOAT16: return run_select<__half>(a, s);
    default: return run_select<__nv_bfloat16>(a, s);
  }
}

cudaError_t beam_reorder(const BeamReorderArgs& a, int64_t ctas, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(ctas));
  if (a.beams <= 4) return launch_dependent(beam_reorder_kernel<4>, grid, dim3(kThreads), 0, s, a);
  if (a.beams <= 8) return launch_dependent(beam_reorder_kernel<8>, grid, dim3(kThreads), 0, s, a);
  if (a.beams <= 16) return launch_dependent(beam_reorder_kernel<16>, grid, dim3(kThreads), 0, s, a);
  if (a.beams <= 32) return launch_dependent(beam_reorder_kernel<32>, grid, dim3(kThreads), 0, s, a);
  return launch_dependent(beam_reorder_kernel<64>, grid, dim3(kThreads), 0, s, a);
}

}  // namespace cc1d
