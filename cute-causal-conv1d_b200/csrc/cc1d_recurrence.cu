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
// from registers; the CTA's 8 warps exchange the sums through shared memory, and each then
// knows the state its positions start from and goes through them once more, still from
// registers.  The inputs are read once, into a ring of shared-memory tiles a few chunks
// ahead.  The backward does the same in both directions at once: the forward direction from
// the state that the forward pass kept for each chunk, the other from the chunk to the right.
//
// With fewer tiles of channels than the SMs can hold CTAs, a cluster shares a tile: its CTAs
// take consecutive chunks and exchange the chunks' sums through distributed shared memory,
// one cluster barrier per round.  No CTA waits for another outside its cluster, and results
// do not depend on timing.
#include "cc1d_recurrence.cuh"

namespace cc1d {
namespace {

// Ring slots: chunks in flight and the one in work.
constexpr int kFwdStages = 3;
template <int LAYOUT> constexpr int kBwdStages = LAYOUT == kLayoutRows ? 2 : 3;

// exp(-(gate + bias)), at most 1e30; nb is -bias log2(e) for 16-bit tensors, else the bias.
template <typename T>
__device__ __forceinline__ float gate_exp(float gate, float nb) {
  if constexpr (std::is_same<T, float>::value) return clamp_exp(expf(-(gate + nb)));
  else return clamp_exp(ex2_approx(fmaf(gate, -kLog2e, nb)));
}

// a and c of the 8 positions from the gate's values.
template <typename T, int V>
__device__ __forceinline__ void gates(const Lane<V> (&g)[kRecSteps], const Lane<V>& nb, Lane<V> (&a)[kRecSteps], Lane<V> (&c)[kRecSteps]) {
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j) {
    Lane<V> e;
#pragma unroll
    for (int i = 0; i < V; ++i) el(e, i) = gate_exp<T>(el(g[j], i), el(nb, i));
    const Lane<V> d = add(e, splat(1.f, e));
#pragma unroll
    for (int i = 0; i < V; ++i) el(a[j], i) = reciprocal<T>(el(d, i));
    c[j] = mul(e, a[j]);
  }
}

template <typename T, int LAYOUT>
__device__ __forceinline__ Lane<Tile<T, LAYOUT>::V> gate_offset(const RecArgs& a, int64_t d0, int lane) {
  Lane<Tile<T, LAYOUT>::V> nb;
#pragma unroll
  for (int i = 0; i < Tile<T, LAYOUT>::V; ++i) {
    const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
    const float b = a.bias.data && d < a.dim ? load_any(a.bias.data, a.bias.dtype, d * a.bias.s0) : 0.f;
    el(nb, i) = std::is_same<T, float>::value ? b : -kLog2e * b;
  }
  return nb;
}

// The 8-bit mask of a warp's positions t .. t + 7 below len.
__device__ __forceinline__ unsigned below(int64_t t, int64_t len) {
  const int64_t n = len - t;
  return n >= kRecSteps ? 0xffu : n <= 0 ? 0u : (1u << n) - 1u;
}

template <typename T, int LAYOUT, bool SEQ, bool Z>
__global__ void __launch_bounds__(kRecThreads, 2) rec_fwd_kernel(const RecArgs a) {
  using C = Tile<T, LAYOUT>;
  constexpr int V = C::V, NT = Z ? 3 : 2, S = kFwdStages;
  using L = Lane<V>;
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* const ring = smem;
  L* const sumA = reinterpret_cast<L*>(smem + S * NT * C::kBytes);  // [2][warps][32]
  L* const sumH = sumA + 2 * kRecWarps * 32;
  L* const farA = sumH + 2 * kRecWarps * 32;  // [2][cluster][32]
  L* const farH = farA + 2 * a.cluster * 32;

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const unsigned cluster = a.cluster, rank = cluster > 1 ? cluster_rank() : 0;
  const int64_t tile = blockIdx.x / cluster;
  const int64_t b = tile / a.dtiles, d0 = (tile - b * a.dtiles) * C::kChannels;
  const int64_t rounds = (a.nchunks + cluster - 1) / cluster;
  grid_dependency_wait();

  const T* const xp = static_cast<const T*>(a.x.data) + b * a.x.s0;
  const T* const gp = static_cast<const T*>(a.gate.data) + b * a.gate.s0;
  const T* const zp = Z ? static_cast<const T*>(a.z.data) + b * a.z.s0 : nullptr;
  T* const op = static_cast<T*>(a.out.data) + b * a.out.s0;
  const int dl = lane_channel<T, LAYOUT>(lane, 0);
  const int nch = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(V), a.dim - d0 - dl)));

  auto load = [&](int64_t k) {
    const int64_t c = k * cluster + rank;
    if (k < rounds && c < a.nchunks) {
      unsigned char* t = ring + (k % S) * NT * C::kBytes;
      load_tile<T, LAYOUT>(t, gp, a.gate.s1, a.gate.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      load_tile<T, LAYOUT>(t + C::kBytes, xp, a.x.s1, a.x.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      if constexpr (Z) load_tile<T, LAYOUT>(t + 2 * C::kBytes, zp, a.z.s1, a.z.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) load(k);
  if (cluster > 1) {  // the others' shared memory may be written once they have all begun
    cluster_arrive();
    cluster_wait();
  }
  const L nb = gate_offset<T, LAYOUT>(a, d0, lane);
  L carry = SEQ ? splat(0.f, L{}) : load_state<T, LAYOUT>(a.init, b, a.nstates, d0, a.dim, lane);
  int ids = SEQ ? load_ids(a, b, static_cast<int64_t>(rank) * kRecChunk + w * kRecSteps, lane) : 0;

  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t c = k * cluster + rank;
    const int64_t t0 = c * kRecChunk, tw = t0 + w * kRecSteps;
    unsigned char* const now = ring + (k % S) * NT * C::kBytes;
    const int buf = static_cast<int>(k & 1);
    cp_async_wait<S - 2>();
    if constexpr (C::kRows) {
      __syncthreads();
      if (k > 0)
        store_tile<T>(ring + ((k - 1) % S) * NT * C::kBytes + C::kBytes, op, a.out.s1, a.out.s2, d0, t0 - static_cast<int64_t>(cluster) * kRecChunk,
                      a.dim, a.seqlen, a.packed);
    } else {
      __syncwarp();
    }
    load(k + S - 1);

    // the 8 positions' maps and their composition
    L ga[kRecSteps], gb[kRecSteps];
    {
      L g[kRecSteps], x[kRecSteps];
      read_steps<T, LAYOUT>(now, w, lane, g);
      read_steps<T, LAYOUT>(now + C::kBytes, w, lane, x);
      L gc[kRecSteps];
      gates<T, V>(g, nb, ga, gc);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) gb[j] = mul(gc[j], x[j]);
    }
    Edges e;
    unsigned valid = below(tw, a.seqlen);
    if constexpr (SEQ) {
      e = edges_of(ids);
      valid = e.valid;
      ids = load_ids(a, b, tw + static_cast<int64_t>(cluster) * kRecChunk, lane);
    }
    L A, H;
    const bool whole = valid == 0xffu && !(SEQ && e.first);
    if (whole) {
      A = ga[0];
      H = gb[0];
#pragma unroll
      for (int j = 1; j < kRecSteps; ++j) {
        A = mul(ga[j], A);
        H = fma(ga[j], H, gb[j]);
      }
    } else {
      A = splat(1.f, L{});
      H = splat(0.f, L{});
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (!(valid >> j & 1u)) {  // no token: the state passes
          ga[j] = splat(1.f, L{});
          gb[j] = splat(0.f, L{});
        }
        if (SEQ && (e.first >> j & 1u)) {
          H = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane);
          A = splat(-1.f, L{});
        }
        A = mul(ga[j], A);
        H = fma(ga[j], H, gb[j]);
      }
    }
    sumA[(buf * kRecWarps + w) * 32 + lane] = A;
    sumH[(buf * kRecWarps + w) * 32 + lane] = H;
    __syncthreads();

    L h = carry;
    if (cluster == 1) {
      L p = carry;
#pragma unroll
      for (int q = 0; q < kRecWarps; ++q) {
        if (q == w) h = p;
        p = apply<V, SEQ>(sumA[(buf * kRecWarps + q) * 32 + lane], sumH[(buf * kRecWarps + q) * 32 + lane], p);
      }
      carry = p;
    } else {
      L pa = splat(1.f, L{}), ph = splat(0.f, L{}), wa = pa, wh = ph;
#pragma unroll
      for (int q = 0; q < kRecWarps; ++q) {
        if (q == w) wa = pa, wh = ph;
        const L qa = sumA[(buf * kRecWarps + q) * 32 + lane];
        ph = apply<V, SEQ>(qa, sumH[(buf * kRecWarps + q) * 32 + lane], ph);
        pa = chain<V, SEQ>(qa, pa);
      }
      for (unsigned r = w; r < cluster; r += kRecWarps) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          store_remote(&el(farA[(buf * cluster + rank) * 32 + lane], i), r, el(pa, i));
          store_remote(&el(farH[(buf * cluster + rank) * 32 + lane], i), r, el(ph, i));
        }
      }
      cluster_arrive();
      cluster_wait();
      L p = carry;
      for (unsigned r = 0; r < cluster; ++r) {
        if (r == rank) h = p;
        p = apply<V, SEQ>(farA[(buf * cluster + r) * 32 + lane], farH[(buf * cluster + r) * 32 + lane], p);
      }
      carry = p;
      h = apply<V, SEQ>(wa, wh, h);
    }
    if (w == 0 && a.checkpoints && c < a.nchunks) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
        if (d < a.dim) a.checkpoints[(b * a.nchunks + c) * a.dim + d] = el(h, i);
      }
    }

    // the states themselves
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
      if (SEQ && !whole && (e.first >> j & 1u))
        h = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane);
      h = fma(ga[j], h, gb[j]);
      gb[j] = h;
    }
    if (SEQ && e.last && a.final_states.data) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j)
        if (e.last >> j & 1u)
          store_state<T, LAYOUT>(a.final_states, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane, gb[j]);
    }
    if constexpr (Z) {
      L z[kRecSteps];
      read_steps<T, LAYOUT>(now + 2 * C::kBytes, w, lane, z);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        L s;
#pragma unroll
        for (int i = 0; i < V; ++i) el(s, i) = silu_of<T>(el(z[j], i));
        gb[j] = mul(gb[j], s);
      }
    }
    if (SEQ && valid != 0xffu) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j)
        if (!(valid >> j & 1u)) gb[j] = splat(0.f, L{});
    }
    if constexpr (C::kRows) {
      write_steps<T, LAYOUT>(now + C::kBytes, w, lane, gb);
    } else {
      T* o = op + (d0 + dl) * a.out.s1 + tw * a.out.s2;
      if (tw + kRecSteps <= a.seqlen) {
#pragma unroll
        for (int j = 0; j < kRecSteps; ++j) store_step<T>(o + j * a.out.s2, a.out.s1, nch, a.packed, gb[j]);
      } else {
#pragma unroll
        for (int j = 0; j < kRecSteps; ++j)
          if (tw + j < a.seqlen) store_step<T>(o + j * a.out.s2, a.out.s1, nch, a.packed, gb[j]);
      }
    }
  }
  if constexpr (C::kRows) {
    __syncthreads();
    store_tile<T>(ring + ((rounds - 1) % S) * NT * C::kBytes + C::kBytes, op, a.out.s1, a.out.s2, d0,
                  ((rounds - 1) * cluster + rank) * kRecChunk, a.dim, a.seqlen, a.packed);
  }
  if (!SEQ && w == 0 && rank == 0) store_state<T, LAYOUT>(a.final_states, b, a.nstates, d0, a.dim, lane, carry);
}

template <typename T, int LAYOUT, bool SEQ, bool Z>
__global__ void __launch_bounds__(kRecThreads, 2) rec_bwd_kernel(const RecArgs a) {
  using C = Tile<T, LAYOUT>;
  constexpr int V = C::V, NT = Z ? 4 : 3, S = kBwdStages<LAYOUT>;
  using L = Lane<V>;
  extern __shared__ __align__(128) unsigned char smem[];
  unsigned char* const ring = smem;  // gate, x, dout, z
  L* const sumA = reinterpret_cast<L*>(smem + S * NT * C::kBytes);  // [2][warps][32], of h -> A h + H
  L* const sumH = sumA + 2 * kRecWarps * 32;
  L* const sumS = sumH + 2 * kRecWarps * 32;                 // of s -> R s + S, back through the warp's positions
  L* const sumR = SEQ ? sumS + 2 * kRecWarps * 32 : sumA;    // the same product unless a sequence ends or starts
  L* const farR = (SEQ ? sumR : sumS) + 2 * kRecWarps * 32;  // [2][cluster][32]
  L* const farS = farR + 2 * a.cluster * 32;

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const unsigned cluster = a.cluster, rank = cluster > 1 ? cluster_rank() : 0;
  const int64_t tile = blockIdx.x / cluster;
  const int64_t b = tile / a.dtiles, d0 = (tile - b * a.dtiles) * C::kChannels;
  const int64_t rounds = (a.nchunks + cluster - 1) / cluster;
  grid_dependency_wait();

  const T* const xp = static_cast<const T*>(a.x.data) + b * a.x.s0;
  const T* const gp = static_cast<const T*>(a.gate.data) + b * a.gate.s0;
  const T* const yp = static_cast<const T*>(a.dout.data) + b * a.dout.s0;
  const T* const zp = Z ? static_cast<const T*>(a.z.data) + b * a.z.s0 : nullptr;
  T* const dxp = static_cast<T*>(a.dx.data) + b * a.dx.s0;
  T* const dgp = static_cast<T*>(a.dgate.data) + b * a.dgate.s0;
  T* const dzp = Z ? static_cast<T*>(a.dz.data) + b * a.dz.s0 : nullptr;
  const int dl = lane_channel<T, LAYOUT>(lane, 0);
  const int nch = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(V), a.dim - d0 - dl)));

  auto chunk_of = [&](int64_t k) { return (rounds - 1 - k) * cluster + rank; };
  auto load = [&](int64_t k) {
    const int64_t c = chunk_of(k);
    if (k < rounds && c < a.nchunks) {
      unsigned char* t = ring + (k % S) * NT * C::kBytes;
      load_tile<T, LAYOUT>(t, gp, a.gate.s1, a.gate.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      load_tile<T, LAYOUT>(t + C::kBytes, xp, a.x.s1, a.x.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      load_tile<T, LAYOUT>(t + 2 * C::kBytes, yp, a.dout.s1, a.dout.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      if constexpr (Z) load_tile<T, LAYOUT>(t + 3 * C::kBytes, zp, a.z.s1, a.z.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
    }
    cp_async_commit();
  };
  auto store = [&](int64_t k) {  // rows: the gradients of round k, from the tiles they replaced
    const int64_t c = chunk_of(k);
    if (c >= a.nchunks) return;
    const unsigned char* t = ring + (k % S) * NT * C::kBytes;
    if constexpr (C::kRows) {
      store_tile<T>(t, dgp, a.dgate.s1, a.dgate.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      store_tile<T>(t + C::kBytes, dxp, a.dx.s1, a.dx.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
      if constexpr (Z) store_tile<T>(t + 3 * C::kBytes, dzp, a.dz.s1, a.dz.s2, d0, c * kRecChunk, a.dim, a.seqlen, a.packed);
    }
  };
  auto checkpoint = [&](int64_t k) {
    L r = splat(0.f, L{});
    const int64_t c = chunk_of(k);
    if (k < rounds && c < a.nchunks) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
        if (d < a.dim) el(r, i) = __ldg(a.checkpoints + (b * a.nchunks + c) * a.dim + d);
      }
    }
    return r;
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) load(k);
  if (cluster > 1) {  // the others' shared memory may be written once they have all begun
    cluster_arrive();
    cluster_wait();
  }
  const L nb = gate_offset<T, LAYOUT>(a, d0, lane);
  L carry = SEQ ? splat(0.f, L{}) : load_state<T, LAYOUT>(a.dfinal, b, a.nstates, d0, a.dim, lane);
  L start = checkpoint(0);
  int ids = SEQ ? load_ids(a, b, chunk_of(0) * kRecChunk + w * kRecSteps, lane) : 0;
  L bias_sum = splat(0.f, L{});

  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t t0 = chunk_of(k) * kRecChunk, tw = t0 + w * kRecSteps;
    unsigned char* const now = ring + (k % S) * NT * C::kBytes;
    const int buf = static_cast<int>(k & 1);
    cp_async_wait<S - 2>();
    if constexpr (C::kRows) {
      __syncthreads();
      if (k > 0) store(k - 1);
    } else {
      __syncwarp();
    }
    load(k + S - 1);

    L ga[kRecSteps], gc[kRecSteps], x[kRecSteps], gy[kRecSteps], dz[kRecSteps];
    {
      L g[kRecSteps];
      read_steps<T, LAYOUT>(now, w, lane, g);
      gates<T, V>(g, nb, ga, gc);
    }
    read_steps<T, LAYOUT>(now + C::kBytes, w, lane, x);
    read_steps<T, LAYOUT>(now + 2 * C::kBytes, w, lane, gy);
    if constexpr (Z) {
      L z[kRecSteps];
      read_steps<T, LAYOUT>(now + 3 * C::kBytes, w, lane, z);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        L s, d;
#pragma unroll
        for (int i = 0; i < V; ++i) silu_and_grad<T>(el(z[j], i), el(s, i), el(d, i));
        dz[j] = mul(gy[j], d);
        gy[j] = mul(gy[j], s);
      }
    }
    Edges e;
    unsigned valid = below(tw, a.seqlen);
    if constexpr (SEQ) {
      e = edges_of(ids);
      valid = e.valid;
      ids = load_ids(a, b, tw - static_cast<int64_t>(cluster) * kRecChunk, lane);
    }
    const bool whole = valid == 0xffu && !(SEQ && (e.first || e.last));
    L A, H, R, B;
    if (whole) {
      A = ga[0];
      H = mul(gc[0], x[0]);
#pragma unroll
      for (int j = 1; j < kRecSteps; ++j) {
        A = mul(ga[j], A);
        H = fma(ga[j], H, mul(gc[j], x[j]));
      }
      B = mul(ga[kRecSteps - 1], gy[kRecSteps - 1]);
#pragma unroll
      for (int j = kRecSteps - 2; j >= 0; --j) B = mul(ga[j], add(gy[j], B));
      R = A;
    } else {
      A = R = splat(1.f, L{});
      H = B = splat(0.f, L{});
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (!(valid >> j & 1u)) {
          ga[j] = splat(1.f, L{});
          gc[j] = x[j] = gy[j] = splat(0.f, L{});
        }
        if (SEQ && (e.first >> j & 1u)) {
          H = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane);
          A = splat(-1.f, L{});
        }
        A = mul(ga[j], A);
        H = fma(ga[j], H, mul(gc[j], x[j]));
      }
#pragma unroll
      for (int j = kRecSteps - 1; j >= 0; --j) {
        if (SEQ && (e.last >> j & 1u)) {
          B = load_state<T, LAYOUT>(a.dfinal, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane);
          R = splat(-1.f, L{});
        }
        R = mul(ga[j], R);
        B = mul(ga[j], add(gy[j], B));
      }
    }
    sumA[(buf * kRecWarps + w) * 32 + lane] = A;
    sumH[(buf * kRecWarps + w) * 32 + lane] = H;
    sumS[(buf * kRecWarps + w) * 32 + lane] = B;
    if constexpr (SEQ) sumR[(buf * kRecWarps + w) * 32 + lane] = R;
    __syncthreads();

    L h = start;
#pragma unroll
    for (int q = 0; q < kRecWarps - 1; ++q)
      if (q < w) h = apply<V, SEQ>(sumA[(buf * kRecWarps + q) * 32 + lane], sumH[(buf * kRecWarps + q) * 32 + lane], h);
    start = checkpoint(k + 1);
    L s = carry;
    if (cluster == 1) {
      L p = carry;
#pragma unroll
      for (int q = kRecWarps - 1; q >= 0; --q) {
        if (q == w) s = p;
        p = apply<V, SEQ>(sumR[(buf * kRecWarps + q) * 32 + lane], sumS[(buf * kRecWarps + q) * 32 + lane], p);
      }
      carry = p;
    } else {
      L pr = splat(1.f, L{}), ps = splat(0.f, L{}), wr = pr, ws = ps;
#pragma unroll
      for (int q = kRecWarps - 1; q >= 0; --q) {
        if (q == w) wr = pr, ws = ps;
        const L qr = sumR[(buf * kRecWarps + q) * 32 + lane];
        ps = apply<V, SEQ>(qr, sumS[(buf * kRecWarps + q) * 32 + lane], ps);
        pr = chain<V, SEQ>(qr, pr);
      }
      for (unsigned r = w; r < cluster; r += kRecWarps) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          store_remote(&el(farR[(buf * cluster + rank) * 32 + lane], i), r, el(pr, i));
          store_remote(&el(farS[(buf * cluster + rank) * 32 + lane], i), r, el(ps, i));
        }
      }
      cluster_arrive();
      cluster_wait();
      L p = carry;
      for (int r = static_cast<int>(cluster) - 1; r >= 0; --r) {
        if (r == static_cast<int>(rank)) s = p;
        p = apply<V, SEQ>(farR[(buf * cluster + r) * 32 + lane], farS[(buf * cluster + r) * 32 + lane], p);
      }
      carry = p;
      s = apply<V, SEQ>(wr, ws, s);
    }

    // forward through the positions: h before each, and dz
    L prev[kRecSteps];
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
      if (SEQ && !whole && (e.first >> j & 1u))
        h = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane);
      prev[j] = h;
      h = fma(ga[j], h, mul(gc[j], x[j]));
      if constexpr (Z) dz[j] = mul(dz[j], h);
    }
    // and back: dx (in gy) and dgate (in prev)
#pragma unroll
    for (int j = kRecSteps - 1; j >= 0; --j) {
      if (SEQ && !whole && (e.last >> j & 1u))
        s = load_state<T, LAYOUT>(a.dfinal, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane);
      const L dh = add(gy[j], s);
      gy[j] = mul(dh, gc[j]);
      s = mul(ga[j], dh);
      prev[j] = mul(mul(s, gc[j]), sub(prev[j], x[j]));
      if (!whole && !(valid >> j & 1u)) {
        gy[j] = prev[j] = splat(0.f, L{});
        if constexpr (Z) dz[j] = splat(0.f, L{});
      }
      bias_sum = add(bias_sum, prev[j]);
      if (SEQ && !whole && (e.first >> j & 1u))
        store_state<T, LAYOUT>(a.dinit, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, d0, a.dim, lane, s);
    }
    if constexpr (C::kRows) {
      write_steps<T, LAYOUT>(now, w, lane, prev);
      write_steps<T, LAYOUT>(now + C::kBytes, w, lane, gy);
      if constexpr (Z) write_steps<T, LAYOUT>(now + 3 * C::kBytes, w, lane, dz);
    } else {
      const int64_t d = d0 + dl;
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (tw + j >= a.seqlen) break;
        store_step<T>(dxp + d * a.dx.s1 + (tw + j) * a.dx.s2, a.dx.s1, nch, a.packed, gy[j]);
        store_step<T>(dgp + d * a.dgate.s1 + (tw + j) * a.dgate.s2, a.dgate.s1, nch, a.packed, prev[j]);
        if constexpr (Z) store_step<T>(dzp + d * a.dz.s1 + (tw + j) * a.dz.s2, a.dz.s1, nch, a.packed, dz[j]);
      }
    }
  }
  __syncthreads();
  if constexpr (C::kRows) store(rounds - 1);
  if (!SEQ && w == 0 && rank == 0) store_state<T, LAYOUT>(a.dinit, b, a.nstates, d0, a.dim, lane, carry);
  if (a.dbias) {
    sumA[w * 32 + lane] = bias_sum;
    __syncthreads();
    if (w == 0) {
      L sum = sumA[lane];
#pragma unroll
      for (int q = 1; q < kRecWarps; ++q) sum = add(sum, sumA[q * 32 + lane]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t d = d0 + lane_channel<T, LAYOUT>(lane, i);
        if (d < a.dim) a.partials[(b * cluster + rank) * a.dim + d] = el(sum, i);
      }
    }
  }
}

// dbias[d] = the tiles' partial sums added up in order.
__global__ void __launch_bounds__(kThreads) rec_bias_kernel(const RecArgs a) {
  grid_dependency_wait();
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (d >= a.dim) return;
  const int64_t n = a.batch * a.cluster;
  float s = 0.f;
#pragma unroll 8
  for (int64_t i = 0; i < n; ++i) s += a.partials[i * a.dim + d];
  a.dbias[d] = s;
}

template <typename T>
__device__ __forceinline__ float at(const TensorArg& t, int64_t b, int64_t d, int64_t l) {
  return to_f32(static_cast<const T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2]);
}
template <typename T>
__device__ __forceinline__ void put(const TensorArg& t, int64_t b, int64_t d, int64_t l, float v) {
  static_cast<T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2] = from_f32<T>(v);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rec_update_kernel(const RecUpdateArgs a) {
  grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * a.dim) return;
  const int64_t b = i / a.dim, d = i - b * a.dim;
  const int64_t row = a.indices ? a.indices[b * a.indices_stride] : b;
  if (row < 0 || row >= a.nstates) {
    for (int64_t l = 0; l < a.seqlen; ++l) put<T>(a.out, b, d, l, 0.f);
    return;
  }
  const float bias = a.bias.data ? load_any(a.bias.data, a.bias.dtype, d * a.bias.s0) : 0.f;
  float* hp = static_cast<float*>(a.state.data) + row * a.state.s0 + d * a.state.s1;
  float h = *hp;
  for (int64_t l = 0; l < a.seqlen; ++l) {
    float ga, gc;
    sigmoid_pair<T>(at<T>(a.gate, b, d, l) + bias, ga, gc);
    h = fmaf(ga, h, gc * at<T>(a.x, b, d, l));
    put<T>(a.out, b, d, l, a.z.data ? h * silu_of<T>(at<T>(a.z, b, d, l)) : h);
  }
  *hp = h;
}

unsigned blocks_for(int64_t threads) { return static_cast<unsigned>((threads + kThreads - 1) / kThreads); }

template <typename T, int LAYOUT, bool BWD, bool SEQ, bool Z>
cudaError_t run(const RecArgs& a, cudaStream_t s) {
  using C = Tile<T, LAYOUT>;
  constexpr int NT = (BWD ? 3 : 2) + (Z ? 1 : 0);
  constexpr int stages = BWD ? kBwdStages<LAYOUT> : kFwdStages;
  constexpr int sums = BWD ? (SEQ ? 4 : 3) : 2;
  const size_t smem = static_cast<size_t>(stages) * NT * C::kBytes + sizeof(Lane<C::V>) * 32 * 2 * (sums * kRecWarps + (a.cluster > 1 ? 2 * a.cluster : 0));
  auto kernel = BWD ? rec_bwd_kernel<T, LAYOUT, SEQ, Z> : rec_fwd_kernel<T, LAYOUT, SEQ, Z>;
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
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int LAYOUT, bool BWD>
cudaError_t pick(const RecArgs& a, cudaStream_t s) {
  if (a.seq_idx.data) return a.z.data ? run<T, LAYOUT, BWD, true, true>(a, s) : run<T, LAYOUT, BWD, true, false>(a, s);
  return a.z.data ? run<T, LAYOUT, BWD, false, true>(a, s) : run<T, LAYOUT, BWD, false, false>(a, s);
}

}  // namespace

using DT = CC1D_DT_TYPE;

cudaError_t CC1D_DT_NAME(rec_fwd)(const RecArgs& a, cudaStream_t s) {
  return a.rows ? pick<DT, kLayoutRows, false>(a, s) : pick<DT, kLayoutChannelLast, false>(a, s);
}
cudaError_t CC1D_DT_NAME(rec_bwd)(const RecArgs& a, cudaStream_t s) {
  cudaError_t e = a.rows ? pick<DT, kLayoutRows, true>(a, s) : pick<DT, kLayoutChannelLast, true>(a, s);
  if (e == cudaSuccess && a.dbias) e = launch_dependent(rec_bias_kernel, dim3(blocks_for(a.dim)), dim3(kThreads), 0, s, a);
  return e;
}
cudaError_t CC1D_DT_NAME(rec_update)(const RecUpdateArgs& a, cudaStream_t s) {
  return launch_dependent(rec_update_kernel<DT>, dim3(blocks_for(a.batch * a.dim)), dim3(kThreads), 0, s, a);
}

}  // namespace cc1d
