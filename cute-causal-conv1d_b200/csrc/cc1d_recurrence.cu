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
template <int CHANNELS>
__device__ __forceinline__ Place place_of(const RecArgs& a) {
  Place p;
  p.cluster = a.cluster;
  p.rank = a.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
  const unsigned tile = blockIdx.x / static_cast<unsigned>(a.cluster), n = static_cast<unsigned>(a.dtiles);
  p.b = tile / n;
  p.d0 = static_cast<int64_t>(tile % n) * CHANNELS;
  p.nd = static_cast<int>(min(a.dim - p.d0, static_cast<int64_t>(CHANNELS)));
  p.rounds = static_cast<int>((a.nchunks + a.cluster - 1) / a.cluster);
  return p;
}

// The maps of the warps before warp w (FORWARD: lower warps first) after each other, applied to h.
template <int V, bool SEQ, bool FORWARD>
__device__ __forceinline__ Lane<V> through_warps(const Map<V>* sums, int w, int lane, Lane<V> h) {
#pragma unroll
  for (int i = 0; i < kRecWarps - 1; ++i) {
    const int q = FORWARD ? i : kRecWarps - 1 - i;
    const Map<V> m = sums[q * 32 + lane];
    const Lane<V> r = apply<V, SEQ>(m.A, m.H, h);
    if (FORWARD ? q < w : q > w) h = r;
  }
  return h;
}

// The state that warp w's positions start from, for a CTA of a cluster.  Takes the CTA's maps,
// sends their composition to the cluster's CTAs and joins theirs; `carry` is the state the
// round starts from, and becomes the one that the next starts from.
template <int V, bool SEQ, bool FORWARD>
__device__ __forceinline__ Lane<V> through_cluster(const Map<V>* sums, Map<V>* far, unsigned bar, unsigned parity, const Place& p,
                                                   int w, int lane, Lane<V>& carry) {
  Map<V> all, mine;
  all.A = splat(1.f, Lane<V>{});
  all.H = splat(0.f, Lane<V>{});
  mine = all;
#pragma unroll
  for (int i = 0; i < kRecWarps; ++i) {
    const int q = FORWARD ? i : kRecWarps - 1 - i;
    if (q == w) mine = all;
    const Map<V> m = sums[q * 32 + lane];
    all.H = apply<V, SEQ>(m.A, m.H, all.H);
    all.A = chain<V, SEQ>(m.A, all.A);
  }
  if (threadIdx.x == 0) mbar_expect(bar, p.cluster * 32 * sizeof(Map<V>));
  const unsigned slot = static_cast<unsigned>(__cvta_generic_to_shared(far + p.rank * 32 + lane));
  for (int r = w; r < p.cluster; r += kRecWarps) send_map<V>(slot, bar, r, all);
  // a partner that never answers leaves NaN in the results instead of a hang
  Lane<V> h = mbar_wait(bar, parity) ? carry : splat(__int_as_float(0x7fc00000), carry);
  Lane<V> start = h;
#pragma unroll 4
  for (int i = 0; i < p.cluster; ++i) {
    const int r = FORWARD ? i : p.cluster - 1 - i;
    if (r == p.rank) start = h;
    const Map<V> m = far[r * 32 + lane];
    h = apply<V, SEQ>(m.A, m.H, h);
  }
  carry = h;
  return apply<V, SEQ>(mine.A, mine.H, start);
}

template <typename T, int LAYOUT, bool SKEW, bool SEQ, bool Z>
__global__ void __launch_bounds__(kRecThreads, 2) rec_fwd_kernel(const RecArgs a) {
  using C = Tile<T, LAYOUT, SKEW>;
  constexpr int V = C::V, NT = Z ? 3 : 2, S = kFwdStages;
  using L = Lane<V>;
  extern __shared__ __align__(128) unsigned char smem[];
  // ring of tiles (gate, x, z) | maps of the warps [2][warps][32] | maps of the cluster [2][cluster][32]
  Map<V>* const sums = reinterpret_cast<Map<V>*>(smem + S * NT * C::kBytes);
  Map<V>* const far = sums + 2 * kRecWarps * 32;
  __shared__ L handed[2][32];     // without a cluster: the state after the last warp's positions
  __shared__ uint64_t bars[2];
  const unsigned ring = static_cast<unsigned>(__cvta_generic_to_shared(smem));
  const unsigned bar = static_cast<unsigned>(__cvta_generic_to_shared(bars));

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const Place p = place_of<C::kChannels>(a);
  grid_dependency_wait();
  const Strip<T> gt = strip_of<T, LAYOUT, SKEW>(a.gate, p.b, p.d0), xt = strip_of<T, LAYOUT, SKEW>(a.x, p.b, p.d0);
  const Strip<T> zt = Z ? strip_of<T, LAYOUT, SKEW>(a.z, p.b, p.d0) : gt, ot = strip_of<T, LAYOUT, SKEW>(a.out, p.b, p.d0);
  const int nch = p.nd - lane * V;

  int load_slot = 0;
  auto load = [&](int k) {
    const int64_t t0 = (static_cast<int64_t>(k) * p.cluster + p.rank) * kRecChunk;
    const int nt = within(t0, a.seqlen, kRecChunk), o = load_slot * NT * C::kBytes;
    if (k < p.rounds && nt > 0) {
      load_tile<T, LAYOUT, SKEW>(ring + o, smem + o, gt, t0, p.nd, nt, a.packed);
      load_tile<T, LAYOUT, SKEW>(ring + o + C::kBytes, smem + o + C::kBytes, xt, t0, p.nd, nt, a.packed);
      if constexpr (Z) load_tile<T, LAYOUT, SKEW>(ring + o + 2 * C::kBytes, smem + o + 2 * C::kBytes, zt, t0, p.nd, nt, a.packed);
    }
    cp_async_commit();
    if (++load_slot == S) load_slot = 0;
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) load(k);
  if (p.cluster > 1) {
    if (threadIdx.x == 0) {
      mbar_init(bar);
      mbar_init(bar + 8);
      mbar_init_done();
    }
    cluster_sync();  // the barriers are there before a partner's first map arrives
  }
  const L nb = gate_offset<T, LAYOUT>(a, p.d0, lane);
  L carry = SEQ ? splat(0.f, L{}) : load_state<T, LAYOUT>(a.init, p.b, a.nstates, p.d0, a.dim, lane);
  if (w == 0) handed[0][lane] = carry;
  int ids = SEQ ? load_ids(a, p.b, static_cast<int64_t>(p.rank) * kRecChunk + w * kRecSteps, lane) : 0;

  int slot = 0;
  for (int k = 0; k < p.rounds; ++k) {
    const int64_t c = static_cast<int64_t>(k) * p.cluster + p.rank;
    const int64_t t0 = c * kRecChunk, tw = t0 + w * kRecSteps;
    const int left = within(tw, a.seqlen, kRecSteps);
    unsigned char* const now = smem + slot * NT * C::kBytes;
    const int buf = k & 1;
    cp_async_wait<S - 2>();
    if constexpr (C::kRows) {
      __syncthreads();
      if (k > 0) {
        const int64_t tp = t0 - static_cast<int64_t>(p.cluster) * kRecChunk;
        store_tile<T, SKEW>(smem + (slot == 0 ? S - 1 : slot - 1) * NT * C::kBytes + C::kBytes, ot, tp, p.nd, within(tp, a.seqlen, kRecChunk), a.packed);
        if constexpr (SKEW) __syncthreads();
      }
    } else {
      __syncwarp();
    }
    load(k + S - 1);

    // the 8 positions' maps and their composition
    L ga[kRecSteps], gb[kRecSteps];
    {
      L g[kRecSteps], x[kRecSteps], gc[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now, gt, t0, w, lane, g);
      gates<T, V>(g, nb, ga, gc);
      read_steps<T, LAYOUT, SKEW>(now + C::kBytes, xt, t0, w, lane, x);
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) gb[j] = mul(gc[j], x[j]);
    }
    Edges e;
    unsigned valid = below(left);
    if constexpr (SEQ) {
      e = edges_of(ids);
      valid = e.valid;
      ids = load_ids(a, p.b, tw + static_cast<int64_t>(p.cluster) * kRecChunk, lane);
    }
    Map<V> m;
    const bool whole = valid == 0xffu && !(SEQ && e.first);
    if (whole) {
      m.A = ga[0];
      m.H = gb[0];
#pragma unroll
      for (int j = 1; j < kRecSteps; ++j) {
        m.A = mul(ga[j], m.A);
        m.H = fma(ga[j], m.H, gb[j]);
      }
    } else {
      m.A = splat(1.f, L{});
      m.H = splat(0.f, L{});
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (!(valid >> j & 1u)) {  // no token: the state passes
          ga[j] = splat(1.f, L{});
          gb[j] = splat(0.f, L{});
        }
        if (SEQ && (e.first >> j & 1u)) {
          m.H = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
          m.A = splat(-1.f, L{});
        }
        m.A = mul(ga[j], m.A);
        m.H = fma(ga[j], m.H, gb[j]);
      }
    }
    Map<V>* const sum = sums + buf * kRecWarps * 32;
    sum[w * 32 + lane] = m;
    __syncthreads();
    L h = p.cluster == 1 ? through_warps<V, SEQ, true>(sum, w, lane, handed[buf][lane])
                         : through_cluster<V, SEQ, true>(sum, far + buf * p.cluster * 32, bar + 8 * buf, (k >> 1) & 1, p, w, lane, carry);
    if (w == 0 && a.checkpoints && c < a.nchunks) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t d = p.d0 + lane_channel<T, LAYOUT>(lane, i);
        if (d < a.dim) a.checkpoints[(p.b * a.nchunks + c) * a.dim + d] = el(h, i);
      }
    }

    // the states themselves
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
      if (SEQ && !whole && (e.first >> j & 1u))
        h = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
      h = fma(ga[j], h, gb[j]);
      gb[j] = h;
    }
    if (p.cluster == 1 && w == kRecWarps - 1) handed[buf ^ 1][lane] = h;
    if (SEQ && e.last && a.final_states.data) {
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j)
        if (e.last >> j & 1u)
          store_state<T, LAYOUT>(a.final_states, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane, gb[j]);
    }
    if constexpr (Z) {
      L z[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now + 2 * C::kBytes, zt, t0, w, lane, z);
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
      write_steps<T, SKEW>(now + C::kBytes, w, lane, gb);
    } else {
      store_steps<T, SKEW>(ot, tw, lane, nch, left, a.packed, gb);
    }
    if (++slot == S) slot = 0;
  }
  if constexpr (C::kRows) {
    __syncthreads();
    const int64_t tp = (static_cast<int64_t>(p.rounds - 1) * p.cluster + p.rank) * kRecChunk;
    store_tile<T, SKEW>(smem + (slot == 0 ? S - 1 : slot - 1) * NT * C::kBytes + C::kBytes, ot, tp, p.nd, within(tp, a.seqlen, kRecChunk), a.packed);
  }
  if (!SEQ && a.final_states.data && p.rank == 0) {
    if (p.cluster == 1) {
      __syncthreads();
      carry = handed[p.rounds & 1][lane];
    }
    if (w == 0) store_state<T, LAYOUT>(a.final_states, p.b, a.nstates, p.d0, a.dim, lane, carry);
  }
  if (p.cluster > 1) cluster_sync();  // no CTA leaves while a partner may still write to it
}

template <typename T, int LAYOUT, bool SKEW, bool SEQ, bool Z>
__global__ void __launch_bounds__(kRecThreads, 2) rec_bwd_kernel(const RecArgs a) {
  using C = Tile<T, LAYOUT, SKEW>;
  constexpr int V = C::V, NT = Z ? 4 : 3, S = kBwdStages<LAYOUT>;
  using L = Lane<V>;
  extern __shared__ __align__(128) unsigned char smem[];
  // ring of tiles (gate, x, dout, z) | maps of the warps, forward and back [2][2][warps][32] |
  // maps of the cluster, back [2][cluster][32]
  Map<V>* const sums = reinterpret_cast<Map<V>*>(smem + S * NT * C::kBytes);
  Map<V>* const far = sums + 4 * kRecWarps * 32;
  __shared__ L handed[2][32];
  __shared__ uint64_t bars[2];
  const unsigned ring = static_cast<unsigned>(__cvta_generic_to_shared(smem));
  const unsigned bar = static_cast<unsigned>(__cvta_generic_to_shared(bars));

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const Place p = place_of<C::kChannels>(a);
  grid_dependency_wait();
  const Strip<T> gt = strip_of<T, LAYOUT, SKEW>(a.gate, p.b, p.d0), xt = strip_of<T, LAYOUT, SKEW>(a.x, p.b, p.d0);
  const Strip<T> yt = strip_of<T, LAYOUT, SKEW>(a.dout, p.b, p.d0), zt = Z ? strip_of<T, LAYOUT, SKEW>(a.z, p.b, p.d0) : gt;
  const Strip<T> dxt = strip_of<T, LAYOUT, SKEW>(a.dx, p.b, p.d0), dgt = strip_of<T, LAYOUT, SKEW>(a.dgate, p.b, p.d0);
  const Strip<T> dzt = Z ? strip_of<T, LAYOUT, SKEW>(a.dz, p.b, p.d0) : dgt;
  const int nch = p.nd - lane * V;

  auto chunk_of = [&](int k) { return static_cast<int64_t>(p.rounds - 1 - k) * p.cluster + p.rank; };
  int load_slot = 0;
  auto load = [&](int k) {
    const int64_t t0 = chunk_of(k) * kRecChunk;
    const int nt = within(t0, a.seqlen, kRecChunk), o = load_slot * NT * C::kBytes;
    if (k < p.rounds && nt > 0) {
      load_tile<T, LAYOUT, SKEW>(ring + o, smem + o, gt, t0, p.nd, nt, a.packed);
      load_tile<T, LAYOUT, SKEW>(ring + o + C::kBytes, smem + o + C::kBytes, xt, t0, p.nd, nt, a.packed);
      load_tile<T, LAYOUT, SKEW>(ring + o + 2 * C::kBytes, smem + o + 2 * C::kBytes, yt, t0, p.nd, nt, a.packed);
      if constexpr (Z) load_tile<T, LAYOUT, SKEW>(ring + o + 3 * C::kBytes, smem + o + 3 * C::kBytes, zt, t0, p.nd, nt, a.packed);
    }
    cp_async_commit();
    if (++load_slot == S) load_slot = 0;
  };
  auto store = [&](int k, const unsigned char* t) {  // rows: the gradients of round k, from the tiles they replaced
    if constexpr (C::kRows) {
      const int64_t t0 = chunk_of(k) * kRecChunk;
      const int nt = within(t0, a.seqlen, kRecChunk);
      store_tile<T, SKEW>(t, dgt, t0, p.nd, nt, a.packed);
      store_tile<T, SKEW>(t + C::kBytes, dxt, t0, p.nd, nt, a.packed);
      if constexpr (Z) store_tile<T, SKEW>(t + 3 * C::kBytes, dzt, t0, p.nd, nt, a.packed);
    }
  };
  auto checkpoint = [&](int k) {
    L r = splat(0.f, L{});
    const int64_t c = chunk_of(k);
    if (k < p.rounds && c < a.nchunks) {
      const float* from = a.checkpoints + (p.b * a.nchunks + c) * a.dim + p.d0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int d = lane_channel<T, LAYOUT>(lane, i);
        if (d < p.nd) el(r, i) = __ldg(from + d);
      }
    }
    return r;
  };
#pragma unroll
  for (int k = 0; k < S - 1; ++k) load(k);
  if (p.cluster > 1) {
    if (threadIdx.x == 0) {
      mbar_init(bar);
      mbar_init(bar + 8);
      mbar_init_done();
    }
    cluster_sync();
  }
  const L nb = gate_offset<T, LAYOUT>(a, p.d0, lane);
  L carry = SEQ ? splat(0.f, L{}) : load_state<T, LAYOUT>(a.dfinal, p.b, a.nstates, p.d0, a.dim, lane);
  if (w == 0) handed[0][lane] = carry;
  L start = checkpoint(0);
  int ids = SEQ ? load_ids(a, p.b, chunk_of(0) * kRecChunk + w * kRecSteps, lane) : 0;
  L bias_sum = splat(0.f, L{});

  int slot = 0;
  for (int k = 0; k < p.rounds; ++k) {
    const int64_t t0 = chunk_of(k) * kRecChunk, tw = t0 + w * kRecSteps;
    const int left = within(tw, a.seqlen, kRecSteps);
    unsigned char* const now = smem + slot * NT * C::kBytes;
    const int buf = k & 1;
    cp_async_wait<S - 2>();
    if constexpr (C::kRows) {
      __syncthreads();
      if (k > 0) {
        store(k - 1, smem + (slot == 0 ? S - 1 : slot - 1) * NT * C::kBytes);
        if constexpr (SKEW) __syncthreads();
      }
    } else {
      __syncwarp();
    }
    load(k + S - 1);

    L ga[kRecSteps], gc[kRecSteps], x[kRecSteps], gy[kRecSteps], dz[kRecSteps];
    {
      L g[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now, gt, t0, w, lane, g);
      gates<T, V>(g, nb, ga, gc);
    }
    read_steps<T, LAYOUT, SKEW>(now + C::kBytes, xt, t0, w, lane, x);
    read_steps<T, LAYOUT, SKEW>(now + 2 * C::kBytes, yt, t0, w, lane, gy);
    if constexpr (Z) {
      L z[kRecSteps];
      read_steps<T, LAYOUT, SKEW>(now + 3 * C::kBytes, zt, t0, w, lane, z);
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
    unsigned valid = below(left);
    if constexpr (SEQ) {
      e = edges_of(ids);
      valid = e.valid;
      ids = load_ids(a, p.b, tw - static_cast<int64_t>(p.cluster) * kRecChunk, lane);
    }
    const bool whole = valid == 0xffu && !(SEQ && (e.first || e.last));
    Map<V> f, r;  // h -> A h + H forward through the positions, s -> A s + H back
    if (whole) {
      f.A = ga[0];
      f.H = mul(gc[0], x[0]);
#pragma unroll
      for (int j = 1; j < kRecSteps; ++j) {
        f.A = mul(ga[j], f.A);
        f.H = fma(ga[j], f.H, mul(gc[j], x[j]));
      }
      r.H = mul(ga[kRecSteps - 1], gy[kRecSteps - 1]);
#pragma unroll
      for (int j = kRecSteps - 2; j >= 0; --j) r.H = mul(ga[j], add(gy[j], r.H));
      r.A = f.A;
    } else {
      f.A = r.A = splat(1.f, L{});
      f.H = r.H = splat(0.f, L{});
#pragma unroll
      for (int j = 0; j < kRecSteps; ++j) {
        if (!(valid >> j & 1u)) {
          ga[j] = splat(1.f, L{});
          gc[j] = x[j] = gy[j] = splat(0.f, L{});
        }
        if (SEQ && (e.first >> j & 1u)) {
          f.H = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
          f.A = splat(-1.f, L{});
        }
        f.A = mul(ga[j], f.A);
        f.H = fma(ga[j], f.H, mul(gc[j], x[j]));
      }
#pragma unroll
      for (int j = kRecSteps - 1; j >= 0; --j) {
        if (SEQ && (e.last >> j & 1u)) {
          r.H = load_state<T, LAYOUT>(a.dfinal, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
          r.A = splat(-1.f, L{});
        }
        r.A = mul(ga[j], r.A);
        r.H = mul(ga[j], add(gy[j], r.H));
      }
    }
    Map<V>* const ahead = sums + 2 * buf * kRecWarps * 32;
    Map<V>* const back = ahead + kRecWarps * 32;
    ahead[w * 32 + lane] = f;
    back[w * 32 + lane] = r;
    __syncthreads();
    L h = through_warps<V, SEQ, true>(ahead, w, lane, start);
    start = checkpoint(k + 1);
    L s = p.cluster == 1 ? through_warps<V, SEQ, false>(back, w, lane, handed[buf][lane])
                         : through_cluster<V, SEQ, false>(back, far + buf * p.cluster * 32, bar + 8 * buf, (k >> 1) & 1, p, w, lane, carry);

    // forward through the positions: h before each, and dz
    L prev[kRecSteps];
#pragma unroll
    for (int j = 0; j < kRecSteps; ++j) {
      if (SEQ && !whole && (e.first >> j & 1u))
        h = load_state<T, LAYOUT>(a.init, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
      prev[j] = h;
      h = fma(ga[j], h, mul(gc[j], x[j]));
      if constexpr (Z) dz[j] = mul(dz[j], h);
    }
    // and back: dx (in gy) and dgate (in prev)
#pragma unroll
    for (int j = kRecSteps - 1; j >= 0; --j) {
      if (SEQ && !whole && (e.last >> j & 1u))
        s = load_state<T, LAYOUT>(a.dfinal, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane);
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
        store_state<T, LAYOUT>(a.dinit, __shfl_sync(0xffffffffu, e.id, j + 1), a.nstates, p.d0, a.dim, lane, s);
    }
    if (p.cluster == 1 && w == 0) handed[buf ^ 1][lane] = s;
    if constexpr (C::kRows) {
      write_steps<T, SKEW>(now, w, lane, prev);
      write_steps<T, SKEW>(now + C::kBytes, w, lane, gy);
      if constexpr (Z) write_steps<T, SKEW>(now + 3 * C::kBytes, w, lane, dz);
    } else {
      store_steps<T, SKEW>(dxt, tw, lane, nch, left, a.packed, gy);
      store_steps<T, SKEW>(dgt, tw, lane, nch, left, a.packed, prev);
      if constexpr (Z) store_steps<T, SKEW>(dzt, tw, lane, nch, left, a.packed, dz);
    }
    if (++slot == S) slot = 0;
  }
  __syncthreads();
  if constexpr (C::kRows) store(p.rounds - 1, smem + (slot == 0 ? S - 1 : slot - 1) * NT * C::kBytes);
  if (!SEQ && w == 0 && p.rank == 0)
    store_state<T, LAYOUT>(a.dinit, p.b, a.nstates, p.d0, a.dim, lane, p.cluster == 1 ? handed[p.rounds & 1][lane] : carry);
  if (a.dbias) {
    L* const sum = reinterpret_cast<L*>(sums);
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
  if (p.cluster > 1) cluster_sync();
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

template <typename T, int LAYOUT, bool SKEW, bool BWD, bool SEQ, bool Z>
cudaError_t run(const RecArgs& a, cudaStream_t s) {
  using C = Tile<T, LAYOUT, SKEW>;
  constexpr int NT = (BWD ? 3 : 2) + (Z ? 1 : 0);
  constexpr int stages = BWD ? kBwdStages<LAYOUT> : kFwdStages;
  const size_t smem = static_cast<size_t>(stages) * NT * C::kBytes +
                      sizeof(Map<C::V>) * 32 * 2 * ((BWD ? 2 : 1) * kRecWarps + (a.cluster > 1 ? a.cluster : 0));
  auto kernel = BWD ? rec_bwd_kernel<T, LAYOUT, SKEW, SEQ, Z> : rec_fwd_kernel<T, LAYOUT, SKEW, SEQ, Z>;
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

template <typename T, int LAYOUT, bool SKEW, bool BWD>
cudaError_t pick_options(const RecArgs& a, cudaStream_t s) {
  if (a.seq_idx.data)
    return a.z.data ? run<T, LAYOUT, SKEW, BWD, true, true>(a, s) : run<T, LAYOUT, SKEW, BWD, true, false>(a, s);
  return a.z.data ? run<T, LAYOUT, SKEW, BWD, false, true>(a, s) : run<T, LAYOUT, SKEW, BWD, false, false>(a, s);
}
template <typename T, bool BWD>
cudaError_t pick(const RecArgs& a, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (a.skew) return a.rows ? pick_options<T, kLayoutRows, true, BWD>(a, s) : pick_options<T, kLayoutChannelLast, true, BWD>(a, s);
  }
  return a.rows ? pick_options<T, kLayoutRows, false, BWD>(a, s) : pick_options<T, kLayoutChannelLast, false, BWD>(a, s);
}

}  // namespace

using DT = CC1D_DT_TYPE;

cudaError_t CC1D_DT_NAME(rec_fwd)(const RecArgs& a, cudaStream_t s) {
  return pick<DT, false>(a, s);
}
cudaError_t CC1D_DT_NAME(rec_bwd)(const RecArgs& a, cudaStream_t s) {
  cudaError_t e = pick<DT, true>(a, s);
  if (e == cudaSuccess && a.dbias) e = launch_dependent(rec_bias_kernel, dim3(blocks_for(a.dim)), dim3(kThreads), 0, s, a);
  return e;
}
cudaError_t CC1D_DT_NAME(rec_update)(const RecUpdateArgs& a, cudaStream_t s) {
  return launch_dependent(rec_update_kernel<DT>, dim3(blocks_for(a.batch * a.dim)), dim3(kThreads), 0, s, a);
}

}  // namespace cc1d
