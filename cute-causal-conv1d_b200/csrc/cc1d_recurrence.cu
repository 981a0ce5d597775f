// Gated linear recurrence along the sequence, forward and backward (sm_100a).
//
//   a = sigmoid(gate + bias), c = 1 - a = sigmoid(-(gate + bias))
//   h_t = a_t h_{t-1} + c_t x_t,  out_t = h_t silu(z_t)
//
// Backward, with g_t the gradient that reaches h_t from out_t (dout_t silu(z_t)), s_t what
// later positions send back to h_t (dfinal after a sequence's last position):
//   dh_t = g_t + s_t,  s_{t-1} = a_t dh_t
//   dx_t = dh_t c_t,  dgate_t = dh_t (h_{t-1} - x_t) a_t c_t,  dz_t = dout_t h_t silu'(z_t),
//   dinit = s before the first position,  dbias = sum of dgate.
//
// A position is the affine map h -> a h + c x, and maps compose, so a stretch of positions is
// summed up by two numbers per channel.  Each warp does that for its 8 positions of a chunk,
// from registers; the CTA's 4 warps exchange the sums through shared memory, and each then
// knows the state its positions start from and goes through them once more, still from
// registers.  The inputs are read once, into a ring of shared-memory tiles a few chunks
// ahead.  The backward does the same in both directions at once: the forward direction from
// the state that the forward pass kept for each chunk, the other from the chunk to the right.
//
// With fewer tiles of channels than the SMs can hold CTAs, a cluster shares a tile: its CTAs
// take consecutive chunks and send each other the chunks' sums, one exchange per round.  No CTA
// waits for another outside its cluster, and results do not depend on timing.
//
// Bound by HBM in the limit; at this writing by issue slots (29 and 45 instructions per
// element, with z) and latency: bf16 (8, 4096, 8192) channel-last takes 408 us forward (82%
// of the copy rate) and 718 us backward (81%), fp32 (8, 4096, 4096) 358 us (93%) and 640 us
// (91%).  Off the 16-byte alignment, with (8, 4094, 8192), 659 and 1248 us (51 and 47%).  4 warps
// and 32 positions: more CTAs fit an SM than with 8 warps and 64 (445 us forward where this took
// 405), and a warp's 8 positions amortise the exchange better than 4 (545 us).
#include <cudaTypedefs.h>

#include "cc1d_recurrence.cuh"

namespace cc1d {
namespace {

// Ring slots: the chunk in work, the one before, whose results are still being stored from its
// tiles, and one (backward) or two chunks that are being loaded.  A cluster's rounds are longer:
// one chunk ahead is enough there and leaves room for a fourth CTA.  Off their alignment strips
// have larger tiles, and channel-last none that are stored from.
template <int SKEW, int LAYOUT, bool CLUSTER> constexpr int kFwdStages = CLUSTER || (SKEW && LAYOUT != kLayoutRows) ? 3 : 4;
constexpr int kBwdStages = 3, kMostStages = 4;

// s = sigmoid(v + bias) at a warp's 8 positions, and if wanted c = 1 - s = e s, e = exp(-v - bias).
// GATE: they weight a state.  For 16-bit tensors -v log2(e) = v m + n with m = -log2(e),
// for fp32 n is added to v.
//
// 1 - s by subtraction would leave few bits of a slow channel's c, or of silu'(z) = s + z s c where
// z is large (2e-3 off at v = 10, all of them lost from 17 on); e s is relative to itself.  A slow channel multiplies its state by thousands
// of s, so the reciprocal's error is taken out with one step of Newton's iteration on the residual
// 1 - s - e s: s is then rounded as near to one as fp32 allows, about 2^-25 of it.
//
// 16-bit: four positions share one reciprocal, of the product of their 1 + e (the special
// function unit would bound the forward otherwise: 4 of its operations per element, now 2.5).
// Its three more roundings leave 2^-22, which is enough for c and for silu.  Where one of a lane's
// e is above 2^30 or NaN the product might not be finite or the NaN reach its neighbours, and where
// an fp32 exponent is beyond 87 exp leaves the normal numbers: such a lane's positions are taken
// one by one.  That shows before any e is there, from the least argument of 8 positions (clamping
// each e took more instructions, and left a sigmoid of 2^-30 where there should be none; the same
// minimum as a tree instead of a chain takes the largest forward from 409 to 422 us).
template <typename T, int V, bool GATE, bool C>
__device__ __forceinline__ void sigmoids(const Lane<V> (&v)[kRecSteps], const Lane<V>& n, Lane<V> (&s)[kRecSteps], Lane<V>* c) {
  static_assert(C || !GATE, "the residual is taken from c");
  constexpr bool kWide = std::is_same<T, float>::value;
  const Lane<V> one = splat(1.f, n);
  Lane<V> e[kRecSteps];  // fp32: the arguments; 16-bit: exp of the negated ones
  bool ordinary = true;
  if constexpr (kWide) {
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) e[j] = add(v[j], n);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float far = 0.f;  // 16-bit: the least of v, fp32: the largest magnitude
    if constexpr (!kWide) far = el(v[0], i);
#pragma unroll
    for (int j = 0; j < kRecSteps; j += 2)
      far = kWide ? max_nan(far, fabsf(el(e[j], i)), fabsf(el(e[j + 1], i))) : min_nan(far, el(v[j], i), el(v[j + 1], i));
    ordinary = ordinary && (kWide ? far <= kMostExponent : fmaf(far, -kLog2e, el(n, i)) <= kMostBits);
  }
  if (!ordinary) {
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a, b;
        if constexpr (kWide) sigmoid_pair<GATE>(el(e[j], i), a, b);
        else sigmoid_pair_of_bits(fmaf(el(v[j], i), -kLog2e, el(n, i)), a, b);
        el(s[j], i) = a;
        if constexpr (C) el(c[j], i) = b;
      }
    }
    return;
  }
  if constexpr (kWide) {
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float a, b;
        pair_of_exp<GATE>(exp_minus(el(e[j], i)), a, b);
        el(s[j], i) = a;
        if constexpr (C) el(c[j], i) = b;
      }
    }
  } else {
#pragma unroll
    for (int q = 0; q < kRecSteps; q += 4) {
      Lane<V> d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[q + j] = fma(v[q + j], splat(-kLog2e, n), n);
#pragma unroll
        for (int i = 0; i < V; ++i) el(e[q + j], i) = ex2_approx(el(e[q + j], i));
        d[j] = add(e[q + j], one);
      }
      const Lane<V> lo = mul(d[0], d[1]), hi = mul(d[2], d[3]);
      Lane<V> r = mul(lo, hi);
#pragma unroll
      for (int i = 0; i < V; ++i) el(r, i) = rcp_approx(el(r, i));
      const Lane<V> rlo = mul(r, hi), rhi = mul(r, lo);
      s[q] = mul(rlo, d[1]);
      s[q + 1] = mul(rlo, d[0]);
      s[q + 2] = mul(rhi, d[3]);
      s[q + 3] = mul(rhi, d[2]);
#pragma unroll
      for (int j = q; j < q + 4; ++j) {
        if constexpr (C) c[j] = mul(e[j], s[j]);
        if constexpr (GATE) s[j] = fma(s[j], sub(sub(one, s[j]), c[j]), s[j]);
      }
    }
  }
}

template <typename T, int LAYOUT>
__device__ __forceinline__ Lane<4 / sizeof(T)> gate_offset(const RecArgs& a, int64_t d0, int lane) {
  Lane<4 / sizeof(T)> nb;
#pragma unroll
  for (int i = 0; i < static_cast<int>(4 / sizeof(T)); ++i) {
    const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
    const float b = a.bias.data && d < a.dim ? load_any(a.bias.data, a.bias.dtype, d * a.bias.s0) : 0.f;
    el(nb, i) = std::is_same<T, float>::value ? b : -kLog2e * b;
  }
  return nb;
}

// `same`: the cover of a tensor that lies like t; with kOwn there is none.
template <typename T, int LAYOUT, int SKEW>
__device__ __forceinline__ void load_by_threads(unsigned char* tile, const Strip<T>& t, const Cover<T, LAYOUT>& same, int64_t t0, int nd, int nt) {
  if constexpr (SKEW & 1) load_strips<T, LAYOUT, true>(tile, t, Cover<T, LAYOUT>(t), t0, nd, nt);
  else if constexpr (SKEW) load_strips<T, LAYOUT, false>(tile, t, same, t0, nd, nt);
  else load_tile<T, LAYOUT>(tile, t, t0, nd, nt);
}
// The tensor whose offsets tell those of t.
template <int SKEW, typename T>
__device__ __forceinline__ const Strip<T>& like(const Strip<T>& t, const Strip<T>& x) {
  if constexpr (SKEW & 1) return t;
  else return x;
}

// Positions of a chunk or of a warp, t .. t + n - 1, that lie within the sequence (may be <= 0).
__device__ __forceinline__ int within(int64_t t, int64_t len, int n) {
  return static_cast<int>(max(static_cast<int64_t>(-1), min(len - t, static_cast<int64_t>(n))));
}
__device__ __forceinline__ unsigned below(int n) { return n >= kRecSteps ? 0xffu : n <= 0 ? 0u : (1u << n) - 1u; }

// What a CTA is: a tile of channels of a batch row, and its place in the cluster.
struct Place {
  int64_t b, d0;
  int nd, cluster, rank, rounds;
};
template <int CHANNELS, bool CLUSTER>
__device__ __forceinline__ Place place_of(const RecArgs& a) {
  Place p;
  p.cluster = CLUSTER ? a.cluster : 1;
  p.rank = CLUSTER ? static_cast<int>(cluster_rank()) : 0;
  const unsigned tile = blockIdx.x / static_cast<unsigned>(p.cluster), n = static_cast<unsigned>(a.dtiles);
  p.b = tile / n;
  p.d0 = static_cast<int64_t>(tile % n) * CHANNELS;
  p.nd = static_cast<int>(min(a.dim - p.d0, static_cast<int64_t>(CHANNELS)));
  p.rounds = static_cast<int>((a.nchunks + p.cluster - 1) / p.cluster);
  return p;
}

// What the warps of a CTA tell each other about their positions: the product A of the a's, H
// with h -> A h + H forward through them (and B with s -> A s + B back), and whether a
// sequence starts (ends) among them: the map is then constant, also for an h that is infinite
// or NaN.
template <int V> struct Sums {
  Lane<V> A[kRecWarps * 32], H[kRecWarps * 32];
  unsigned cut[kRecWarps];
};
template <int V> struct SumsBack {
  Lane<V> B[kRecWarps * 32];
  unsigned cut[kRecWarps];
};
__device__ __forceinline__ unsigned cuts_of(const unsigned* cut, int lane) {
  return __ballot_sync(0xffffffffu, lane < kRecWarps && cut[lane & (kRecWarps - 1)]);
}

// h = m h + c if p, as one predicated instruction.
__device__ __forceinline__ void fma_if(bool p, Lane<1>& h, const Lane<1>& m, const Lane<1>& c) {
  asm("{.reg .pred p;\n setp.ne.s32 p, %3, 0;\n @p fma.rn.f32 %0, %1, %0, %2;\n}" : "+f"(h.v) : "f"(m.v), "f"(c.v), "r"(static_cast<int>(p)));
}
__device__ __forceinline__ void fma_if(bool p, Lane<2>& h, const Lane<2>& m, const Lane<2>& c) {
  asm("{.reg .pred p;\n .reg .b64 h, m, c;\n setp.ne.s32 p, %6, 0;\n mov.b64 h, {%0, %1};\n mov.b64 m, {%2, %3};\n mov.b64 c, {%4, %5};\n"
      "@p fma.rn.f32x2 h, m, h, c;\n mov.b64 {%0, %1}, h;\n}"
      : "+f"(h.v.x), "+f"(h.v.y) : "f"(m.v.x), "f"(m.v.y), "f"(c.v.x), "f"(c.v.y), "r"(static_cast<int>(p)));
}

// The maps of the warps before warp w (FORWARD: lower warps first) after each other, applied to h.
template <int V, bool SEQ, bool FORWARD>
__device__ __forceinline__ Lane<V> through_warps(const Lane<V>* A, const Lane<V>* H, unsigned cuts, int w, int lane, Lane<V> h) {
  if (!SEQ || cuts == 0) {
#pragma unroll
    for (int i = 0; i < kRecWarps - 1; ++i) {
      const int q = FORWARD ? i : kRecWarps - 1 - i;
      fma_if(FORWARD ? q < w : q > w, h, A[q * 32 + lane], H[q * 32 + lane]);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < kRecWarps - 1; ++i) {
      const int q = FORWARD ? i : kRecWarps - 1 - i;
      if (FORWARD ? q >= w : q <= w) break;
      const Lane<V> c = H[q * 32 + lane];
      h = cuts >> q & 1u ? c : fma(A[q * 32 + lane], h, c);
    }
  }
  return h;
}

// A CTA of a cluster sends the composition of its maps to all of them, itself included.
template <int V, bool SEQ, bool FORWARD>
__device__ __forceinline__ void send_to_cluster(const Lane<V>* A, const Lane<V>* H, unsigned cuts, Map<V>* far, unsigned bar,
                                                const Place& p, int w, int lane) {
  if (threadIdx.x == 0) mbar_expect(bar, p.cluster * 32 * sizeof(Map<V>));
  if (w >= p.cluster) return;  // this warp sends to ranks w, w + 4, ...
  Map<V> all;
  all.A = splat(1.f, Lane<V>{});
  all.H = splat(0.f, Lane<V>{});
#pragma unroll
  for (int i = 0; i < kRecWarps; ++i) {
    const int q = FORWARD ? i : kRecWarps - 1 - i;
    const Lane<V> m = A[q * 32 + lane], c = H[q * 32 + lane];
    all.H = fma(m, all.H, c);
    if (SEQ && (cuts >> q & 1u)) all.H = c;
    all.A = mul(m, all.A);
  }
  if (SEQ && cuts) all.A = splat(-1.f, all.A);
  const unsigned slot = shared_addr(far + p.rank * 32 + lane);
  for (int r = w; r < p.cluster; r += kRecWarps) send_map<V>(slot, bar, r, all);
}

// The state that this CTA's chunk starts from.  `carry` is the state the round starts from, and
// becomes the one that the next starts from.  A partner that never answers leaves NaN in the
// results instead of a hang.
template <int V, bool SEQ, bool FORWARD>
__device__ __forceinline__ Lane<V> from_cluster(const Map<V>* far, unsigned bar, unsigned parity, const Place& p, int lane, Lane<V>& carry) {
  Lane<V> h = mbar_wait(bar, parity) ? carry : splat(__int_as_float(0x7fc00000), carry);
  Lane<V> start = h;
  const int mine = FORWARD ? p.rank : p.cluster - 1 - p.rank;  // how many come before this CTA
  for (int i = 0; i < p.cluster; i += 2) {
    const int r = FORWARD ? i : p.cluster - 1 - i;
    const bool two = i + 1 < p.cluster;
    const Map<V> m0 = far[r * 32 + lane], m1 = far[(two ? FORWARD ? r + 1 : r - 1 : r) * 32 + lane];
    if (i == mine) start = h;
    h = apply<V, SEQ>(m0, h);
    if (i + 1 == mine) start = h;
    if (two) h = apply<V, SEQ>(m1, h);
  }
  carry = h;
  return start;
}

// What else a CTA keeps in shared memory: without a cluster, the state that one round's last
// positions hand to the next round; the barriers.
// ids of positions t0 - 1 .. t0 + 32 and (backward) the state before position t0 of the chunks
// of three rounds, copied two rounds ahead.
template <int V> struct Common {
  Lane<V> handed[2][32];
  Lane<V> start[3][32];
  int ids[3][kRecChunk + 4];
  uint64_t bars[kMostStages + 2];
};

// Starts the copy of a round's ids; the caller commits.  Outside the sequence they are -1.
__device__ __forceinline__ void load_ids(const RecArgs& a, int64_t b, int64_t t0, int* ids) {
  const int i = threadIdx.x;
  if (i >= kRecChunk + 2) return;
  const int64_t t = t0 - 1 + i;
  const int* from = static_cast<const int*>(a.seq_idx.data) + b * a.seq_idx.s0 + t * a.seq_idx.s1;
  if (t >= 0 && t < a.seqlen) cp4(shared_addr(ids + i), from, 4);
  else ids[i] = -1;
}

// The barriers of the ring (one per slot) and of the cluster's exchange (two).
template <int S, bool CLUSTER>
__device__ __forceinline__ void start_barriers(unsigned bars, bool tma) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, tma ? 1 : 2 * kRecThreads);
    mbar_init(bars + 8 * S, 1);
    mbar_init(bars + 8 * S + 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (CLUSTER) cluster_sync();  // they are there before a partner's first map arrives
  else __syncthreads();
}

template <typename T, int LAYOUT, int SKEW, bool SEQ, bool Z, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads, 4) rec_fwd_kernel(const __grid_constant__ RecArgs a, const __grid_constant__ RecMaps maps) {
  using C = Tile<T, LAYOUT, SKEW>;
  constexpr int V = C::V, NT = Z ? 3 : 2, S = kFwdStages<SKEW, LAYOUT, CLUSTER>;
  using L = Lane<V>;
  extern __shared__ __align__(1024) unsigned char smem[];
  // ring of tiles (gate, x, z) | sums of the warps [2] | maps of the cluster [2][cluster][32] | common
  Sums<V>* const sums = reinterpret_cast<Sums<V>*>(smem + S * NT * C::kBytes);
  Map<V>* const far = reinterpret_cast<Map<V>*>(sums + 2);
  Common<V>& common = *reinterpret_cast<Common<V>*>(far + (CLUSTER ? 2 * a.cluster * 32 : 0));
  const unsigned ring = shared_addr(smem), bars = shared_addr(common.bars);

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const Place p = place_of<C::kChannels, CLUSTER>(a);
  const bool tma = !SKEW && a.move == kTma;
  constexpr bool kDirect = SKEW && !C::kRows;  // results are stored from registers
  start_barriers<S, CLUSTER>(bars, tma);
  grid_dependency_wait();
  const Strip<T> gt = strip_of<T>(a.gate, maps.gate, p.b, p.d0), xt = strip_of<T>(a.x, maps.x, p.b, p.d0);
  const Strip<T> zt = Z ? strip_of<T>(a.z, maps.z, p.b, p.d0) : gt, ot = strip_of<T>(a.out, maps.out, p.b, p.d0);

  const Cover<T, LAYOUT> cover(xt);
  int load_slot = 0;
  auto load = [&](int k) {  // the tiles of round k
    if (k < p.rounds) {
      const int64_t t0 = (static_cast<int64_t>(k) * p.cluster + p.rank) * kRecChunk;
      const int nt = within(t0, a.seqlen, kRecChunk), o = load_slot * NT * C::kBytes;
      const unsigned bar = bars + 8 * load_slot;
      if (tma) {
        if (threadIdx.x == 0) {
          if (nt > 0) {
            mbar_expect(bar, NT * C::kBytes);
            tma_load<LAYOUT>(ring + o, gt.map, p.d0, t0, p.b, bar);
            tma_load<LAYOUT>(ring + o + C::kBytes, xt.map, p.d0, t0, p.b, bar);
            if constexpr (Z) tma_load<LAYOUT>(ring + o + 2 * C::kBytes, zt.map, p.d0, t0, p.b, bar);
          } else {
            mbar_arrive(bar);
          }
        }
      } else {
        if (nt > 0) {
          load_by_threads<T, LAYOUT, SKEW>(smem + o, gt, cover, t0, p.nd, nt);
          load_by_threads<T, LAYOUT, SKEW>(smem + o + C::kBytes, xt, cover, t0, p.nd, nt);
          if constexpr (Z) load_by_threads<T, LAYOUT, SKEW>(smem + o + 2 * C::kBytes, zt, cover, t0, p.nd, nt);
        }
        mbar_arrive_copies(bar);  // of the asynchronous copies
        mbar_arrive(bar);         // and of the plain stores
      }
    }
    if (++load_slot == S) load_slot = 0;
  };
  auto store = [&](int k, int slot) {  // the results of round k, from the tiles of x
    const int64_t t0 = (static_cast<int64_t>(k) * p.cluster + p.rank) * kRecChunk;
    const int nt = within(t0, a.seqlen, kRecChunk), o = slot * NT * C::kBytes + C::kBytes;
    if (tma) {
      if (threadIdx.x == 0) {
        if (nt > 0) tma_store<LAYOUT>(ring + o, ot.map, p.d0, t0, p.b);
        tma_commit();
      }
    } else if (nt > 0) {
      store_tile<T, LAYOUT, SKEW>(smem + o, ot, t0, p.nd, nt);
    }
  };
#pragma unroll
  for (int k = 0; k < S - 2; ++k) load(k);
  if (tma || kDirect) load(S - 2);
  const L nb = gate_offset<T, LAYOUT>(a, p.d0, lane);
  L carry = SEQ ? splat(0.f, L{}) : load_state<T, LAYOUT>(a.init, p.b, a.nstates, p.d0, a.dim, lane);
  if (w == 0) common.handed[0][lane] = carry;
  auto copy_ids = [&](int k) {
    if constexpr (SEQ) {
      if (k < p.rounds) load_ids(a, p.b, (static_cast<int64_t>(k) * p.cluster + p.rank) * kRecChunk, common.ids[k % 3]);
      cp_async_commit();
    }
  };
  if constexpr (SEQ) {
    copy_ids(0);
    copy_ids(1);
    cp_async_wait<0>();
    __syncthreads();
  }

  int slot = 0;
  unsigned parity = 0;
  for (int k = 0; k < p.rounds; ++k) {
    const int64_t c = static_cast<int64_t>(k) * p.cluster + p.rank;
    const int64_t t0 = c * kRecChunk, tw = t0 + w * kRecSteps;
    unsigned char* const now = smem + slot * NT * C::kBytes;
    const int buf = k & 1;
    const bool there = mbar_wait(bars + 8 * slot, parity);

    Edges e;
    if constexpr (SEQ) {
      e = edges_of(common.ids[k % 3][w * kRecSteps + min(lane, kRecSteps + 1)]);
    }
    // Rare: positions without a token are cleared.  Nothing reads the state that leaves them, but
    // four positions share a reciprocal, and their roundings must not depend on what padding or
    // old tiles hold (the TMA fills up with zeros).
    const unsigned valid = SEQ ? e.valid : SKEW ? below(within(tw, a.seqlen, kRecSteps)) : 0xffu;
    if (valid != 0xffu) {
      zero_steps<T, LAYOUT, SKEW>(now, like<SKEW>(gt, xt), w, lane, ~valid);
      zero_steps<T, LAYOUT, SKEW>(now + C::kBytes, xt, w, lane, ~valid);
      if constexpr (Z) zero_steps<T, LAYOUT, SKEW>(now + 2 * C::kBytes, like<SKEW>(zt, xt), w, lane, ~valid);
      __syncwarp();
    }
    // the 8 positions' maps and their composition
    L ga[kRecSteps], gb[kRecSteps];
    read_steps<T, LAYOUT, SKEW>(now, like<SKEW>(gt, xt), w, lane, ga);
    read_steps<T, LAYOUT, SKEW>(now + C::kBytes, xt, w, lane, gb);
    {
      L gc[kRecSteps];
      sigmoids<T, V, true, true>(ga, nb, ga, gc);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) gb[j] = mul(gc[j], gb[j]);
    }
    if (!there) ga[0] = splat(__int_as_float(0x7fc00000), L{});
    L A = ga[0], H = gb[0];
#pragma unroll
    for (int j = 1; j < kRecSteps; ++j) {
      A = mul(ga[j], A);
      H = fma(ga[j], H, gb[j]);
    }
    if (SEQ && e.first) {  // a sequence starts here: H again, from its initial state
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (e.first >> j & 1u)
          H = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
        H = fma(ga[j], H, gb[j]);
      }
    }
    Sums<V>& sum = sums[buf];
    sum.A[w * 32 + lane] = A;
    sum.H[w * 32 + lane] = H;
    if (SEQ && lane == 0) sum.cut[w] = e.first;
    if (SEQ) cp_async_wait<0>();  // the ids of the next round, for all after the barrier
    __syncthreads();
    const unsigned cuts = SEQ ? cuts_of(sum.cut, lane) : 0;
    if (CLUSTER) send_to_cluster<V, SEQ, true>(sum.A, sum.H, cuts, far + buf * p.cluster * 32, bars + 8 * (S + buf), p, w, lane);
    copy_ids(k + 2);
    if (!kDirect && k > 0) store(k - 1, slot == 0 ? S - 1 : slot - 1);
    if (kDirect) load(k + S - 1);       // into the last round's slot
    else if (!tma) load(k + S - 2);     // into the slot that was stored a round ago
    L zs[kRecSteps];
    auto silu = [&] {
      L z[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now + 2 * C::kBytes, like<SKEW>(zt, xt), w, lane, z);
      sigmoids<T, V, false, false>(z, splat(0.f, L{}), zs, nullptr);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) zs[j] = mul(zs[j], z[j]);
    };
    if constexpr (Z && CLUSTER) silu();  // while the cluster's maps are on their way
    L h = !CLUSTER ? common.handed[buf][lane]
                         : from_cluster<V, SEQ, true>(far + buf * p.cluster * 32, bars + 8 * (S + buf), (k >> 1) & 1, p, lane, carry);
    h = through_warps<V, SEQ, true>(sum.A, sum.H, cuts, w, lane, h);
    if (w == 0 && a.checkpoints && c < a.nchunks) {
      float* to = a.checkpoints + (p.b * a.nchunks + c) * a.dim + p.d0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int d = lane_channel<T, LAYOUT>(lane, i);
        if (d < p.nd) to[d] = el(h, i);
      }
    }

    // the states themselves
    if (SEQ && e.first) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (e.first >> j & 1u)
          h = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
        h = fma(ga[j], h, gb[j]);
        gb[j] = h;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        h = fma(ga[j], h, gb[j]);
        gb[j] = h;
      }
    }
    if (!CLUSTER && w == kRecWarps - 1) common.handed[buf ^ 1][lane] = h;
    if (a.final_states.data && (SEQ ? e.last != 0 : tw < a.seqlen && tw + kRecSteps >= a.seqlen)) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if constexpr (SEQ) {
          if (e.last >> j & 1u)
            store_state<T, LAYOUT>(a.final_states, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane, gb[j]);
        } else {
          if (tw + j == a.seqlen - 1) store_state<T, LAYOUT>(a.final_states, p.b, a.nstates, p.d0, a.dim, lane, gb[j]);
        }
      }
    }
    if constexpr (Z) {
      if constexpr (!CLUSTER) silu();
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) gb[j] = mul(gb[j], zs[j]);
    }
    if constexpr (kDirect) {
      store_steps<T, SKEW>(ot, tw, lane, p.nd - V * lane, within(tw, a.seqlen, kRecSteps), SEQ ? ~e.valid & 0xffu : 0u, gb);
    } else {
      write_steps<T, LAYOUT, SKEW>(now + C::kBytes, w, lane, gb);
      if (SEQ && e.valid != 0xffu) clear_steps<T, LAYOUT, SKEW>(now + C::kBytes, w, lane, ~e.valid);
    }
    if (tma) {
      tma_fence();
      if (threadIdx.x == 0) tma_wait_read<0>();  // by now the last round's tiles have been stored
      load(k + S - 1);
    }
    if (++slot == S) slot = 0, parity ^= 1;
  }
  __syncthreads();
  if (!kDirect) store(p.rounds - 1, slot == 0 ? S - 1 : slot - 1);
  if (tma && threadIdx.x == 0) tma_wait_read<0>();
  if (CLUSTER) cluster_sync();  // no CTA leaves while a partner may still write to it
}

template <typename T, int LAYOUT, int SKEW, bool SEQ, bool Z, bool CLUSTER>
__global__ void __launch_bounds__(kRecThreads, 4) rec_bwd_kernel(const __grid_constant__ RecArgs a, const __grid_constant__ RecMaps maps) {
  using C = Tile<T, LAYOUT, SKEW>;
  constexpr int V = C::V, NT = Z ? 4 : 3, S = kBwdStages;
  using L = Lane<V>;
  extern __shared__ __align__(1024) unsigned char smem[];
  // ring of tiles (gate, x, dout, z) | sums of the warps, forward and back [2] | maps of the
  // cluster, back [2][cluster][32] | common
  Sums<V>* const sums = reinterpret_cast<Sums<V>*>(smem + S * NT * C::kBytes);
  SumsBack<V>* const sums_back = reinterpret_cast<SumsBack<V>*>(sums + 2);
  Map<V>* const far = reinterpret_cast<Map<V>*>(sums_back + 2);
  Common<V>& common = *reinterpret_cast<Common<V>*>(far + (CLUSTER ? 2 * a.cluster * 32 : 0));
  const unsigned ring = shared_addr(smem), bars = shared_addr(common.bars);

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const Place p = place_of<C::kChannels, CLUSTER>(a);
  const bool tma = !SKEW && a.move == kTma;
  constexpr bool kDirect = SKEW && !C::kRows;  // results are stored from registers
  start_barriers<S, CLUSTER>(bars, tma);
  grid_dependency_wait();
  const Strip<T> gt = strip_of<T>(a.gate, maps.gate, p.b, p.d0), xt = strip_of<T>(a.x, maps.x, p.b, p.d0);
  const Strip<T> yt = strip_of<T>(a.dout, maps.dout, p.b, p.d0), zt = Z ? strip_of<T>(a.z, maps.z, p.b, p.d0) : gt;
  const Strip<T> dxt = strip_of<T>(a.dx, maps.dx, p.b, p.d0), dgt = strip_of<T>(a.dgate, maps.dgate, p.b, p.d0);
  const Strip<T> dzt = Z ? strip_of<T>(a.dz, maps.dz, p.b, p.d0) : dgt;

  auto chunk_of = [&](int k) { return static_cast<int64_t>(p.rounds - 1 - k) * p.cluster + p.rank; };
  const Cover<T, LAYOUT> cover(xt);
  int load_slot = 0;
  auto load = [&](int k) {
    if (k < p.rounds) {
      const int64_t t0 = chunk_of(k) * kRecChunk;
      const int nt = within(t0, a.seqlen, kRecChunk), o = load_slot * NT * C::kBytes;
      const unsigned bar = bars + 8 * load_slot;
      if (tma) {
        if (threadIdx.x == 0) {
          if (nt > 0) {
            mbar_expect(bar, NT * C::kBytes);
            tma_load<LAYOUT>(ring + o, gt.map, p.d0, t0, p.b, bar);
            tma_load<LAYOUT>(ring + o + C::kBytes, xt.map, p.d0, t0, p.b, bar);
            tma_load<LAYOUT>(ring + o + 2 * C::kBytes, yt.map, p.d0, t0, p.b, bar);
            if constexpr (Z) tma_load<LAYOUT>(ring + o + 3 * C::kBytes, zt.map, p.d0, t0, p.b, bar);
          } else {
            mbar_arrive(bar);
          }
        }
      } else {
        if (nt > 0) {
          load_by_threads<T, LAYOUT, SKEW>(smem + o, gt, cover, t0, p.nd, nt);
          load_by_threads<T, LAYOUT, SKEW>(smem + o + C::kBytes, xt, cover, t0, p.nd, nt);
          load_by_threads<T, LAYOUT, SKEW>(smem + o + 2 * C::kBytes, yt, cover, t0, p.nd, nt);
          if constexpr (Z) load_by_threads<T, LAYOUT, SKEW>(smem + o + 3 * C::kBytes, zt, cover, t0, p.nd, nt);
        }
        mbar_arrive_copies(bar);
        mbar_arrive(bar);
      }
    }
    if (++load_slot == S) load_slot = 0;
  };
  auto store = [&](int k, int slot) {  // dgate, dx and dz of round k, from the tiles of gate, x and z
    const int64_t t0 = chunk_of(k) * kRecChunk;
    const int nt = within(t0, a.seqlen, kRecChunk), o = slot * NT * C::kBytes;
    if (tma) {
      if (threadIdx.x == 0) {
        if (nt > 0) {
          tma_store<LAYOUT>(ring + o, dgt.map, p.d0, t0, p.b);
          tma_store<LAYOUT>(ring + o + C::kBytes, dxt.map, p.d0, t0, p.b);
          if constexpr (Z) tma_store<LAYOUT>(ring + o + 3 * C::kBytes, dzt.map, p.d0, t0, p.b);
        }
        tma_commit();
      }
    } else if (nt > 0) {
      store_tile<T, LAYOUT, SKEW>(smem + o, dgt, t0, p.nd, nt);
      store_tile<T, LAYOUT, SKEW>(smem + o + C::kBytes, dxt, t0, p.nd, nt);
      if constexpr (Z) store_tile<T, LAYOUT, SKEW>(smem + o + 3 * C::kBytes, dzt, t0, p.nd, nt);
    }
  };
  auto copy_ahead = [&](int k) {  // what round k needs besides the tiles
    if (k < p.rounds) {
      const int64_t c = chunk_of(k);
      if (w == kRecWarps - 1) {
        const float* from = a.checkpoints + (p.b * a.nchunks + c) * a.dim + p.d0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int d = lane_channel<T, LAYOUT>(lane, i);
          const bool in = c < a.nchunks && d < p.nd;
          cp4(shared_addr(&common.start[k % 3][lane]) + 4 * i, in ? from + d : a.checkpoints, in ? 4 : 0);
        }
      }
      if constexpr (SEQ) load_ids(a, p.b, c * kRecChunk, common.ids[k % 3]);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < S - 2; ++k) load(k);
  if (tma || kDirect) load(S - 2);
  const L nb = gate_offset<T, LAYOUT>(a, p.d0, lane);
  L carry = SEQ ? splat(0.f, L{}) : load_state<T, LAYOUT>(a.dfinal, p.b, a.nstates, p.d0, a.dim, lane);
  if (w == 0) common.handed[0][lane] = carry;
  copy_ahead(0);
  copy_ahead(1);
  cp_async_wait<0>();
  __syncthreads();
  L bias_sum = splat(0.f, L{}), bias_lost = bias_sum;

  int slot = 0;
  unsigned parity = 0;
  for (int k = 0; k < p.rounds; ++k) {
    const int64_t t0 = chunk_of(k) * kRecChunk, tw = t0 + w * kRecSteps;
    unsigned char* const now = smem + slot * NT * C::kBytes;
    const int buf = k & 1;
    const bool there = mbar_wait(bars + 8 * slot, parity);

    Edges e;
    unsigned valid = below(within(tw, a.seqlen, kRecSteps));
    if constexpr (SEQ) {
      e = edges_of(common.ids[k % 3][w * kRecSteps + min(lane, kRecSteps + 1)]);
      valid = e.valid;
    }
    if (valid != 0xffu) {  // rare: positions without a token are cleared
      zero_steps<T, LAYOUT, SKEW>(now, like<SKEW>(gt, xt), w, lane, ~valid);
      zero_steps<T, LAYOUT, SKEW>(now + C::kBytes, xt, w, lane, ~valid);
      zero_steps<T, LAYOUT, SKEW>(now + 2 * C::kBytes, like<SKEW>(yt, xt), w, lane, ~valid);
      if constexpr (Z) zero_steps<T, LAYOUT, SKEW>(now + 3 * C::kBytes, like<SKEW>(zt, xt), w, lane, ~valid);
      __syncwarp();
    }
    L ga[kRecSteps], gc[kRecSteps], x[kRecSteps], gy[kRecSteps], dz[kRecSteps];
    {
      L g[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now, like<SKEW>(gt, xt), w, lane, g);
      sigmoids<T, V, true, true>(g, nb, ga, gc);
      if (valid != 0xffu) {  // and hand the gradient on as it is, whatever the bias
#pragma unroll
        for (int j = 0; j < kRecSteps; ++j)
          if (!(valid >> j & 1u)) {
            ga[j] = splat(1.f, L{});
            gc[j] = splat(0.f, L{});
          }
      }
      if (!there) ga[0] = splat(__int_as_float(0x7fc00000), L{});
    }
    read_steps<T, LAYOUT, SKEW>(now + C::kBytes, xt, w, lane, x);
    read_steps<T, LAYOUT, SKEW>(now + 2 * C::kBytes, like<SKEW>(yt, xt), w, lane, gy);
    if constexpr (Z) {
      L z[kRecSteps], s[kRecSteps], c[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now + 3 * C::kBytes, like<SKEW>(zt, xt), w, lane, z);
      sigmoids<T, V, false, true>(z, splat(0.f, L{}), s, c);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        // silu(z) = z s and silu'(z) = s + z s c, s = sigmoid(z), c = 1 - s
        const L zs = mul(z[j], s[j]);
        dz[j] = mul(gy[j], fma(zs, c[j], s[j]));
        gy[j] = mul(gy[j], zs);
      }
    }
    L A = ga[0], H = mul(gc[0], x[0]);
#pragma unroll
    for (int j = 1; j < kRecSteps; ++j) {
      A = mul(ga[j], A);
      H = fma(ga[j], H, mul(gc[j], x[j]));
    }
    L B = mul(ga[kRecSteps - 1], gy[kRecSteps - 1]);
#pragma unroll
    for (int j = kRecSteps - 2; j >= 0; --j) B = mul(ga[j], add(gy[j], B));
    if (SEQ && (e.first | e.last)) {  // a sequence starts or ends here
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (e.first >> j & 1u)
          H = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
        H = j == 0 && !(e.first & 1u) ? mul(gc[0], x[0]) : fma(ga[j], H, mul(gc[j], x[j]));
      }
#pragma unroll
      for (int j = kRecSteps - 1; j >= 0; --j) {
        if (e.last >> j & 1u)
          B = load_state<T, LAYOUT>(a.dfinal, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
        B = j == kRecSteps - 1 && !(e.last >> j & 1u) ? mul(ga[j], gy[j]) : mul(ga[j], add(gy[j], B));
      }
    }
    Sums<V>& sum = sums[buf];
    SumsBack<V>& sum_back = sums_back[buf];
    sum.A[w * 32 + lane] = A;
    sum.H[w * 32 + lane] = H;
    sum_back.B[w * 32 + lane] = B;
    if (SEQ && lane == 0) {
      sum.cut[w] = e.first;
      sum_back.cut[w] = e.last;
    }
    cp_async_wait<0>();  // what the next round needs, for all after the barrier
    __syncthreads();
    const unsigned cuts = SEQ ? cuts_of(sum_back.cut, lane) : 0;
    if (CLUSTER) send_to_cluster<V, SEQ, false>(sum.A, sum_back.B, cuts, far + buf * p.cluster * 32, bars + 8 * (S + buf), p, w, lane);
    copy_ahead(k + 2);
    if (!kDirect && k > 0) store(k - 1, slot == 0 ? S - 1 : slot - 1);
    if (kDirect) load(k + S - 1);
    else if (!tma) load(k + S - 2);
    L h = through_warps<V, SEQ, true>(sum.A, sum.H, SEQ ? cuts_of(sum.cut, lane) : 0, w, lane, common.start[k % 3][lane]);

    // forward through the positions: h before each, and dz
    L prev[kRecSteps];
    if (SEQ && e.first) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (e.first >> j & 1u)
          h = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
        prev[j] = h;
        h = fma(ga[j], h, mul(gc[j], x[j]));
        if constexpr (Z) dz[j] = mul(dz[j], h);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        prev[j] = h;
        h = fma(ga[j], h, mul(gc[j], x[j]));
        if constexpr (Z) dz[j] = mul(dz[j], h);
      }
    }
    // and back: dx (in gy) and dgate (in prev)
    L s = !CLUSTER ? common.handed[buf][lane]
                         : from_cluster<V, SEQ, false>(far + buf * p.cluster * 32, bars + 8 * (S + buf), (k >> 1) & 1, p, lane, carry);
    s = through_warps<V, SEQ, false>(sum.A, sum_back.B, cuts, w, lane, s);
    auto step_back = [&](int j) {
      const L dh = add(gy[j], s);
      gy[j] = mul(dh, gc[j]);
      s = mul(ga[j], dh);
      prev[j] = mul(mul(s, gc[j]), sub(prev[j], x[j]));
    };
    if (SEQ && (e.first | e.last)) {
#pragma unroll
      for (int j = kRecSteps - 1; j >= 0; --j) {
        if (e.last >> j & 1u)
          s = load_state<T, LAYOUT>(a.dfinal, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
        step_back(j);
        if (e.first >> j & 1u)
          store_state<T, LAYOUT>(a.dinit, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane, s);
      }
    } else {
#pragma unroll
      for (int j = kRecSteps - 1; j >= 0; --j) step_back(j);
    }
    if (!CLUSTER && w == 0) common.handed[buf ^ 1][lane] = s;
    // dbias, with the sum's own rounding carried along (Kahan): thousands of rounds add up
    L round_sum = prev[0];
#pragma unroll
    for (int j = 1; j < kRecSteps; ++j) round_sum = add(round_sum, prev[j]);
    round_sum = sub(round_sum, bias_lost);
    const L new_sum = add(bias_sum, round_sum);
    bias_lost = sub(sub(new_sum, bias_sum), round_sum);
    bias_sum = new_sum;
    if constexpr (kDirect) {
      const int left = within(tw, a.seqlen, kRecSteps), n = p.nd - V * lane;
      const unsigned clear = SEQ ? ~valid & 0xffu : 0u;
      store_steps<T, SKEW>(dgt, tw, lane, n, left, clear, prev);
      store_steps<T, SKEW>(dxt, tw, lane, n, left, clear, gy);
      if constexpr (Z) store_steps<T, SKEW>(dzt, tw, lane, n, left, clear, dz);
    } else {
      write_steps<T, LAYOUT, SKEW>(now, w, lane, prev);
      write_steps<T, LAYOUT, SKEW>(now + C::kBytes, w, lane, gy);
      if constexpr (Z) write_steps<T, LAYOUT, SKEW>(now + 3 * C::kBytes, w, lane, dz);
      if (SEQ && valid != 0xffu) {
        clear_steps<T, LAYOUT, SKEW>(now, w, lane, ~valid);
        clear_steps<T, LAYOUT, SKEW>(now + C::kBytes, w, lane, ~valid);
        if constexpr (Z) clear_steps<T, LAYOUT, SKEW>(now + 3 * C::kBytes, w, lane, ~valid);
      }
    }
    if (tma) {
      tma_fence();
      if (threadIdx.x == 0) tma_wait_read<0>();  // by now the last round's tiles have been stored
      load(k + S - 1);
    }
    if (++slot == S) slot = 0, parity ^= 1;
  }
  __syncthreads();
  if (!kDirect) store(p.rounds - 1, slot == 0 ? S - 1 : slot - 1);
  if (!SEQ && w == 0 && p.rank == 0)
    store_state<T, LAYOUT>(a.dinit, p.b, a.nstates, p.d0, a.dim, lane, !CLUSTER ? common.handed[p.rounds & 1][lane] : carry);
  if (a.dbias) {
    L* const sum = sums[0].A;
    sum[w * 32 + lane] = bias_sum;
    __syncthreads();
    if (w == 0) {
      L total = sum[lane];
#pragma unroll
      for (int q = 1; q < kRecWarps; ++q) total = add(total, sum[q * 32 + lane]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t d = p.d0 + lane_channel<T, LAYOUT>(lane, i);
        if (d < a.dim) a.partials[(p.b * p.cluster + p.rank) * a.dim + d] = el(total, i);
      }
    }
  }
  if (tma && threadIdx.x == 0) tma_wait_read<0>();
  if (CLUSTER) cluster_sync();
}

// The tensor map of a strip-wise aligned tensor; channel-last (dim, seqlen, batch), rows
// (seqlen, dim, batch), boxes of a tile's strips.
template <typename T, int LAYOUT>
bool make_map(CUtensorMap* map, const TensorArg& t, const RecArgs& a) {
  if (!t.data) return true;
  using C = Tile<T, LAYOUT, 0>;
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  if (!encode) return false;
  const int64_t inner = C::kRows ? a.seqlen : a.dim, outer = C::kRows ? a.dim : a.seqlen, step = C::kRows ? t.s1 : t.s2;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), static_cast<cuuint64_t>(a.batch)};
  // an extent of one never uses its stride, which may then be anything
  const cuuint64_t strides[2] = {outer > 1 ? static_cast<cuuint64_t>(step) * sizeof(T) : 16, a.batch > 1 ? static_cast<cuuint64_t>(t.s0) * sizeof(T) : 16};
  const cuuint32_t box[3] = {C::kStripBytes / sizeof(T), static_cast<cuuint32_t>(C::kStrips), 1};
  const cuuint32_t one[3] = {1, 1, 1};
  return encode(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, t.data, dims, strides, box, one,
                CU_TENSOR_MAP_INTERLEAVE_NONE, !C::kRows ? CU_TENSOR_MAP_SWIZZLE_NONE : C::kStripBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clusters (CTAs if there are none) of this launch that run at the same time on the device.
template <bool CLUSTER>
cudaError_t capacity_of(const void* kernel, const cudaLaunchConfig_t& cfg, int cluster, int64_t* out) {
  int dev = 0, n = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if constexpr (CLUSTER) {
    e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
  } else {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kRecThreads, cfg.dynamicSmemBytes);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    n *= sms;
  }
  *out = n;
  return e;
}

template <typename T, int LAYOUT, int SKEW, bool BWD, bool SEQ, bool Z, bool CLUSTER>
cudaError_t run(RecArgs& a, cudaStream_t s) {
  using C = Tile<T, LAYOUT, SKEW>;
  constexpr int NT = (BWD ? 3 : 2) + (Z ? 1 : 0);
  constexpr int stages = BWD ? kBwdStages : kFwdStages<SKEW, LAYOUT, CLUSTER>;
  RecMaps maps = {};
  if (a.move == kTma && !a.capacity) {
    const bool ok = make_map<T, LAYOUT>(&maps.gate, a.gate, a) && make_map<T, LAYOUT>(&maps.x, a.x, a) && make_map<T, LAYOUT>(&maps.z, a.z, a) &&
                    (BWD ? make_map<T, LAYOUT>(&maps.dout, a.dout, a) && make_map<T, LAYOUT>(&maps.dx, a.dx, a) &&
                               make_map<T, LAYOUT>(&maps.dgate, a.dgate, a) && make_map<T, LAYOUT>(&maps.dz, a.dz, a)
                         : make_map<T, LAYOUT>(&maps.out, a.out, a));
    if (!ok) a.move = kElements;
  }
  const size_t smem = static_cast<size_t>(stages) * NT * C::kBytes + 2 * (sizeof(Sums<C::V>) + (BWD ? sizeof(SumsBack<C::V>) : 0)) +
                      (CLUSTER ? 2 * a.cluster * 32 * sizeof(Map<C::V>) : 0) + sizeof(Common<C::V>);
  auto kernel = BWD ? rec_bwd_kernel<T, LAYOUT, SKEW, SEQ, Z, CLUSTER> : rec_fwd_kernel<T, LAYOUT, SKEW, SEQ, Z, CLUSTER>;
  const void* ptr = reinterpret_cast<const void*>(kernel);
  cudaError_t e = allow_dynamic_smem(ptr, smem);
  if (e == cudaSuccess && a.cluster > 8) e = cudaFuncSetAttribute(ptr, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch * a.dtiles * a.cluster));
  cfg.blockDim = dim3(kRecThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  if (a.capacity) return capacity_of<CLUSTER>(ptr, cfg, a.cluster, a.capacity);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const RecArgs&>(a), static_cast<const RecMaps&>(maps));
}

template <typename T, int LAYOUT, int SKEW, bool BWD, bool SEQ, bool Z>
cudaError_t pick_cluster(RecArgs& a, cudaStream_t s) {
  return a.cluster > 1 ? run<T, LAYOUT, SKEW, BWD, SEQ, Z, true>(a, s) : run<T, LAYOUT, SKEW, BWD, SEQ, Z, false>(a, s);
}
template <typename T, int LAYOUT, int SKEW, bool BWD>
cudaError_t pick_options(RecArgs& a, cudaStream_t s) {
  if (a.seq_idx.data)
    return a.z.data ? pick_cluster<T, LAYOUT, SKEW, BWD, true, true>(a, s) : pick_cluster<T, LAYOUT, SKEW, BWD, true, false>(a, s);
  return a.z.data ? pick_cluster<T, LAYOUT, SKEW, BWD, false, true>(a, s) : pick_cluster<T, LAYOUT, SKEW, BWD, false, false>(a, s);
}
template <typename T, bool BWD>
cudaError_t pick(RecArgs& a, cudaStream_t s) {
  constexpr int own = sizeof(T) == 2 ? 3 : 5;
  if constexpr (sizeof(T) == 2) {
    if (a.move == kHalves) return a.rows ? pick_options<T, kLayoutRows, 2, BWD>(a, s) : pick_options<T, kLayoutChannelLast, 2, BWD>(a, s);
  }
  if (a.move == kOwn) return a.rows ? pick_options<T, kLayoutRows, own, BWD>(a, s) : pick_options<T, kLayoutChannelLast, own, BWD>(a, s);
  if (a.move == kWords) return a.rows ? pick_options<T, kLayoutRows, 4, BWD>(a, s) : pick_options<T, kLayoutChannelLast, 4, BWD>(a, s);
  return a.rows ? pick_options<T, kLayoutRows, 0, BWD>(a, s) : pick_options<T, kLayoutChannelLast, 0, BWD>(a, s);
}

}  // namespace

using DT = CC1D_DT_TYPE;

cudaError_t CC1D_DT_NAME(rec_fwd)(RecArgs& a, cudaStream_t s) {
  return pick<DT, false>(a, s);
}
cudaError_t CC1D_DT_NAME(rec_bwd)(RecArgs& a, cudaStream_t s) {
  cudaError_t e = pick<DT, true>(a, s);
  if (a.capacity) return e;
  if (e == cudaSuccess && a.dbias) e = sum_rows(a.partials, a.batch * a.cluster, a.dim, a.dbias, s);
  return e;
}
}  // namespace cc1d
