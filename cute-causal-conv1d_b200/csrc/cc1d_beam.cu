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
// One pass over the logits: each warp walks a strip of a row with the running maximum and sum of
// the softmax and a sorted list of the strip's best in registers, one or two entries a lane.  An
// element is looked at one by one only if it beats the list's last entry, which becomes rare
// after the first steps; a floor from all warps of a CTA (the n-th largest of their elements' maxima,
// later of their lists) keeps out most of the others.  A second kernel joins the strips' lists, by
// beams, then over beams.
//
// What bounds it: 512 rows of 128000 bf16 logits (131 MB, 20 us of memory) take 78 us, mostly the
// instructions of the exponentials' sums and comparisons, two per element, and the insertions before
// the floors are known; without the floors 180 us, with one made once from the threads' maxima 116.
// Four rows of 32000 take 12.7 us: two kernels of which the second waits for the first, and in them
// chains of exchanges and barriers rather than data.
constexpr int kWarps = kThreads / 32;
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

// The running maximum m and sum s + low of 2^(x L - c), L = kLog2e, of a lane or a part of a row.
// c = m L as it is rounded (0 before there is an m): one multiply-add makes the exponent, and
// log sum exp(x) = m + log(sum) + (c - m L) log(2) puts the rounding back.
struct Soft {
  float m = -INFINITY, s = 0.f, low = 0.f;
};
__device__ __forceinline__ float scale_of(float m) { return m > -INFINITY ? m * kLog2e : 0.f; }
__device__ __forceinline__ void raise(Soft& a, float m) {
  if (m > a.m) {
    const float f = a.m > -INFINITY ? ex2_approx(scale_of(a.m) - scale_of(m)) : 0.f;
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

template <typename T, int Q>
struct Strip {
  Best<Q> best;
  Soft soft;
  int lane;
  int floor = kEmpty;  // n elements of the CTA's part are at least that
  // E neighbouring elements of each lane from place `at` on; `has` of them
  template <int E>
  __device__ __forceinline__ void step(const float (&x)[E], int at, int has) {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
    raise(soft, top);
    const float c = scale_of(soft.m);
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = ex2_approx(fmaf(x[e], kLog2e, -c));
#pragma unroll
    for (int w = E / 2; w > 0; w /= 2)
#pragma unroll
      for (int e = 0; e < w; ++e) s[e] += s[e + w];
    add_to(soft, s[0]);
    const int key = order_of(top);
    const int least = max(best.last, floor);
    if (!__any_sync(~0u, has > 0 && key >= least)) return;
    // the lanes' elements that may count, one after the other
    unsigned mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine |= (e < has && order_of(x[e]) >= least ? 1u : 0u) << e;
    while (true) {
      const unsigned todo = __ballot_sync(~0u, mine != 0);
      if (!todo) break;
      const int from = __ffs(todo) - 1, first = __ffs(mine) - 1;
      float v = x[0];
#pragma unroll
      for (int e = 1; e < E; ++e) v = e == first ? x[e] : v;
      const int k = __shfl_sync(~0u, order_of(v), from), place = __shfl_sync(~0u, at + first, from);
      if (best.takes(k, place)) best.insert(k, place, lane);
      if (lane == from) mine &= mine - 1;
    }
  }
};

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
// The n-th largest (n <= 32) of kWarps descending lists of 32 keys in shared memory.  Of two
// descending lists a and b the larger of a[i] and b[31 - i] are the 32 largest, in a bitonic order.
__device__ __forceinline__ int nth_of_lists(const int* keys, int n, int lane) {
  int k = keys[lane];
  for (int w = 1; w < kWarps; ++w) {
    k = max(k, keys[w * 32 + 31 - lane]);
#pragma unroll
    for (int step = 16; step > 0; step /= 2) k = exchange(k, step, true, lane);
  }
  return __shfl_sync(~0u, k, n - 1);
}

template <typename T, int Q>
__global__ void __launch_bounds__(kThreads) beam_parts_kernel(const BeamSelectArgs a) {
  constexpr int E = 16 / sizeof(T);
  __shared__ int2 lists[kWarps][Q * 32];
  __shared__ Soft softs[kWarps];
  __shared__ int keys[2][kThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int n = static_cast<int>(a.candidates);
  grid_dependency_wait();
  const T* x = static_cast<const T*>(a.logits) + (row / a.beams) * a.logits_s0 + (row % a.beams) * a.logits_s1;
  const int64_t begin = part * a.part, end = begin + a.part < a.vocab ? begin + a.part : a.vocab;
  const int64_t strip = (end - begin + kWarps - 1) / kWarps;
  int64_t i = begin + warp * strip;
  const int64_t stop = i + strip < end ? i + strip : end;
  Strip<T, Q> w;
  w.lane = lane;
  w.best.start(n);
  // up to the first 16-byte boundary, element by element
  const int64_t past = reinterpret_cast<uintptr_t>(x + i) % 16 / sizeof(T);
  const int64_t head = past ? E - past : 0;
  if (i < stop && head) {
    const int64_t count = head < stop - i ? head : stop - i;
    float v[1] = {lane < count ? to_f32(x[i + lane]) : -INFINITY};
    w.step(v, static_cast<int>(i + lane), lane < count ? 1 : 0);
    i += count;
  }
  // steps of 32 E elements, the next two on their way; the last one may be short
  constexpr int STEP = 32 * E, AHEAD = 2;
  const int size = i < stop ? static_cast<int>(stop - i) : 0, from = lane * E, steps = (size + STEP - 1) / STEP;
  const T* q = x + i;
  // Kept as words until they are used: taking them apart at once would wait for the load.
  uint4 next[AHEAD];
  auto fetch = [&](int n) {
    const int at = from + n * STEP;
    return at + E <= size ? *reinterpret_cast<const uint4*>(q + at) : make_uint4(0, 0, 0, 0);
  };
  auto count = [&](int n) { return min(max(size - from - n * STEP, 0), E); };
  auto values = [&](int n, const uint4& u, float (&v)[E]) {
    unpack<T, E>(*reinterpret_cast<const Packet<T, E>*>(&u), v);
    if ((n + 1) * STEP > size) {
      const int at = from + n * STEP;
      if (at + E > size)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at + e < size ? to_f32(q[at + e]) : -INFINITY;
    }
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) next[k] = fetch(k);
  auto run = [&](int first, int end) {  // first: a multiple of AHEAD
    for (int n0 = first; n0 < end; n0 += AHEAD) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (n0 + k >= end) break;
        float v[E];
        values(n0 + k, next[k], v);
        next[k] = fetch(n0 + k + AHEAD);
        w.step(v, static_cast<int>(i) + from + (n0 + k) * STEP, count(n0 + k));
      }
    }
  };
  // A floor before the first step: the n-th largest of the threads' maxima of it.  For long strips
  // another one after eight steps: the n-th largest of the warps' lists.
  constexpr int FIRST = 8;
  if constexpr (Q == 1) {
    int top = kEmpty;
    if (count(0) > 0) {
      float v[E];
      values(0, next[0], v);
      float m = v[0];
#pragma unroll
      for (int e = 1; e < E; ++e) m = fmaxf(m, v[e]);
      top = order_of(m);
    }
    keys[0][threadIdx.x] = sorted_down(top, lane);
    __syncthreads();
    w.floor = nth_of_lists(keys[0], n, lane);
  }
  run(0, steps < FIRST ? steps : FIRST);
  if constexpr (Q == 1)
    if (strip >= 2 * FIRST * STEP) {  // the same for all warps
      keys[1][threadIdx.x] = lane < n ? w.best.key[0] : kEmpty;
      __syncthreads();
      w.floor = max(w.floor, nth_of_lists(keys[1], n, lane));
    }
  run(FIRST, steps);
#pragma unroll
  for (int q = 0; q < Q; ++q) lists[warp][q * 32 + lane] = make_int2(w.best.key[q], w.best.at[q]);
#pragma unroll
  for (int bit = 1; bit < 32; bit *= 2) {
    Soft o;
    o.m = __shfl_xor_sync(~0u, w.soft.m, bit);
    o.s = __shfl_xor_sync(~0u, w.soft.s, bit);
    o.low = __shfl_xor_sync(~0u, w.soft.low, bit);
    const float m = fmaxf(w.soft.m, o.m);
    raise(w.soft, m);
    raise(o, m);
    add_to(w.soft, o.s);
    w.soft.low += o.low;
  }
  if (lane == 0) softs[warp] = w.soft;
  __syncthreads();
  if (warp != 0) return;
  for (int o = 1; o < kWarps; ++o) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int2 c = lists[o][q * 32 + lane];
      w.best.offer(c.x, c.y, q * 32 + lane < n && c.x != kEmpty, lane);
    }
    Soft s = softs[o];
    const float m = fmaxf(w.soft.m, s.m);
    raise(w.soft, m);
    raise(s, m);
    add_to(w.soft, s.s);
    w.soft.low += s.low;
  }
  int2* out = a.best + static_cast<int64_t>(blockIdx.x) * n;
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (q * 32 + lane < n) out[q * 32 + lane] = make_int2(w.best.key[q], w.best.at[q]);
  if (lane == 0) a.sums[blockIdx.x] = make_float2(w.soft.m, w.soft.s + w.soft.low);
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
    Best<Q> best;
    best.start(n);
    float m = -INFINITY;
    for (int64_t p = lane; p < a.parts; p += 32) m = fmaxf(m, a.sums[first + p].x);
#pragma unroll
    for (int bit = 1; bit < 32; bit *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, bit));
    double s = 0.0;
    for (int64_t p = lane; p < a.parts; p += 32) {
      const float2 v = a.sums[first + p];
      s += static_cast<double>(v.y) * exp2(static_cast<double>(scale_of(v.x)) - scale_of(m));
    }
#pragma unroll
    for (int bit = 1; bit < 32; bit *= 2) s += __shfl_xor_sync(~0u, s, bit);
    const double lse = m + log(s) + (scale_of(m) - static_cast<double>(m) * kLog2e) * 0.69314718055994531;
    const int64_t entries = a.parts * n;
    for (int64_t e = lane; e - lane < entries; e += 32) {
      const int2 c = e < entries ? a.best[first * n + e] : make_int2(kEmpty, INT_MAX);
      if (e < 32) best.fill(c.x, c.y, lane);
      else best.offer(c.x, c.y, c.x != kEmpty, lane);
    }
    const float score = a.scores[b * a.scores_s0 + k * a.scores_s1];
    const bool ended = a.finished && a.finished[b * a.finished_s0 + k * a.finished_s1];
    // a row that is no distribution (a NaN, an infinity, nothing left) offers nothing
    const bool sound = fabsf(score) < INFINITY && (ended || fabs(lse) < INFINITY);
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
        total = static_cast<double>(score) + (static_cast<double>(value_of(best.key[q])) - lse);
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
    const int64_t rest = column / t.size0;
    at += (rest % t.size1) * t.step1 + rest / t.size1 * t.step2 - rest * t.size0 * t.step0;
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
