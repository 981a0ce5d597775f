// Selective recurrence, forward, over whole or packed sequences (sm_100a).
//
//     s_t = softplus(delta_t + bias)         h_t[n] = exp(s_t A[n]) h_{t-1}[n] + s_t x_t B_t[n]
//     y_t = sum_n C_t[n] h_t[n] + D x_t      out_t = y_t silu(z_t)
//
// A CTA of 128 threads walks the sequence of a batch row in tiles of 32 positions (8 for at most 4
// states, 16 for at most 8).  A thread holds four states of a channel in registers; LN = 1 to 16
// threads share a channel, a CTA owns 128 / LN channels, and more than 64 states take several passes
// over a tile.  The step sizes of a tile are made once, by all threads, and with B and C lie in
// shared memory as fp32; the next tile's inputs are on their way to registers, as the words that
// they arrive in, meanwhile.
//
// What bounds it: an element of h takes one exponential (MUFU, 16 a cycle and SM) and about eleven
// instructions in all, a third of them for what is done once per position and channel.  4 x 4096 x
// 2048 x 16 bf16 with z (537 M elements, 268 MB without the checkpoints) takes 318 us: its
// exponentials alone 119, its memory 41.  Its 512 CTAs are 3.5 an SM, so the longest wait is a
// thread's chain of dependent positions; a scheduler issues .55 a cycle, the MUFU is busy 48 % of it.
//
// Eight positions are unrolled, with their loads first.  Two channels a thread took 502 us (half the
// warps), three tiles in flight in one unrolled loop 420 to 550 (the instruction cache), 64 or 96
// registers a thread 360 to 450.
#include "cc1d_selective.cuh"

namespace cc1d {
namespace {

// CTAs of an SM, which bounds the registers: three took 449 us above, four 318, five 364 (spills).
constexpr int kFwdCtas = 4;
constexpr int kSelThreads = 128;

// Shared memory: flags; (s, s x) by position and channel; y by position and channel; B and C; with
// several passes the states between two tiles.
template <int LN>
struct FwdSmem {
  static constexpr int T = sel_tile(LN), CH = kSelChannels / LN, PITCH = CH + 2;
  static constexpr int kFlags = 256, kIo = T * PITCH * 8, kY = (T * PITCH * 4 + 15) / 16 * 16;
  static int64_t bytes(const SelArgs& a) {
    return kFlags + kIo + kY + T * 8 * LN * a.blocks * 4 + (a.blocks > 1 ? a.blocks * kSelThreads * 16 : 0);
  }
};

// ENDS: only what each segment carries out of itself, for the segments behind it.
template <typename T, int LN, bool ROWS, bool MULTI, bool ENDS>
__global__ void __launch_bounds__(kSelThreads, kFwdCtas) sel_fwd_kernel(const __grid_constant__ SelArgs a) {
  using Smem = FwdSmem<LN>;
  using Where = Tile<kSelThreads, LN, ROWS>;
  constexpr int K = Where::K, PITCH = Smem::PITCH, TT = Where::T;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float biases[Smem::CH], skips[Smem::CH];
  SelFlags& flags = *reinterpret_cast<SelFlags*>(smem);
  float2* io = reinterpret_cast<float2*>(smem + Smem::kFlags);
  float* ys = reinterpret_cast<float*>(smem + Smem::kFlags + Smem::kIo);
  float* bc = reinterpret_cast<float*>(smem + Smem::kFlags + Smem::kIo + Smem::kY);
  const int np = static_cast<int>(a.padded), blocks = MULTI ? a.blocks : 1, wide = 4 * LN * blocks;
  float* held = bc + TT * 2 * wide;

  const SelPlace p = sel_place<LN>(a);
  if (ENDS && p.seg + 1 == a.segments) return;  // nothing is behind it
  const int tid = threadIdx.x, sl = tid % LN, c = tid / LN;
  const int mine = c < p.channels ? 1 : 0;
  const int64_t ch = p.ch0 + (mine ? c : 0);
  grid_dependency_wait();
  for (int i = tid; i < Smem::CH; i += kSelThreads) {
    const bool is = i < p.channels;
    biases[i] = is && a.bias.data ? load_any(a.bias.data, a.bias.dtype, (p.ch0 + i) * a.bias.s0) : 0.f;
    skips[i] = is && a.D.data ? load_any(a.D.data, a.D.dtype, (p.ch0 + i) * a.D.s0) : 0.f;
  }
  __syncthreads();
  auto of_pair = [](const float* v, int k) { return make_float2(v[2 * Where::c(k)], v[2 * Where::c(k) + 1]); };
  const float2 bias = of_pair(biases, 0), skip = of_pair(skips, 0);  // unless along the sequence

  Four h = zero4(), rate = zero4();
  float total = 0.f;  // ENDS: the sum of step sizes since the segment's start
  auto rates = [&](int n0) { return mine && n0 < np ? of4(load_rates(a.A, ch, n0, a.dstate)) : zero4(); };
  for (int nb = 0; nb < blocks; ++nb) {
    const int n0 = nb * 4 * LN + sl * kSelStates;
    rate = rates(n0);
    h = zero4();
    if (!ENDS && mine && n0 < np)
      for (int64_t s = 0; s < p.seg; ++s) {
        const int64_t at = (p.b * a.segments + s) * a.dim + ch;
        const float sum = a.steps[at];
        const float4 e = *reinterpret_cast<const float4*>(a.ends + at * np + n0);
        h.lo = make_float2(handed_on(h.lo.x, rate.lo.x, sum, e.x), handed_on(h.lo.y, rate.lo.y, sum, e.y));
        h.hi = make_float2(handed_on(h.hi.x, rate.hi.x, sum, e.z), handed_on(h.hi.y, rate.hi.y, sum, e.w));
      }
    if constexpr (MULTI) store4(held + (nb * kSelThreads + tid) * 4, h);
  }

  const Walk<T, Where> xs(a.x, p), deltas(a.delta, p), zs(a.z.data ? a.z : a.x, p), outs(a.out, p);
  const bool all_channels = p.channels == Smem::CH, packed = a.seq_idx.data != nullptr;
  Raw x[K], next_x[K], next_delta[K], z[K];
  FlagFeed<TT> feed;
  Coefficients<T, kSelThreads, LN, MULTI> next_bc(a, p);
  auto inside = [&](int64_t i) { return all_channels && (i + 1) * TT <= a.seqlen; };
  auto fetch = [&](int64_t i) {
    const bool whole = inside(i);
    xs.load(a, a.x, p, i, whole, next_x);
    deltas.load(a, a.delta, p, i, whole, next_delta);
    feed.load(a, p.b, i * TT);
    next_bc.load(a, i * TT, whole);
  };
  fetch(p.chunk0);
  for (int64_t i = p.chunk0; i < p.chunk1; ++i) {
    const int64_t t0 = i * TT;
    const bool whole = inside(i), checked = packed || !whole;
    feed.store(a, p.b, t0, flags);
    if (checked || MULTI) __syncthreads();  // flags are there
#pragma unroll
    for (int k = 0; k < K; ++k) {
      x[k] = next_x[k];
      const float2 u = fadd2(pair_of<T>(next_delta[k], a.pairs), ROWS ? of_pair(biases, k) : bias);
      const float2 s = a.softplus ? step_size<T>(u) : u, sx = fmul2(s, pair_of<T>(x[k], a.pairs));
      float4 v = make_float4(s.x, sx.x, s.y, sx.y);
      if (checked) {
        const int has = flags.valid(Where::t(k)) ? p.channels - 2 * Where::c(k) : 0;
        if (has < 1) v.x = v.y = 0.f;
        if (has < 2) v.z = v.w = 0.f;
      }
      *reinterpret_cast<float4*>(&io[Where::t(k) * PITCH + 2 * Where::c(k)]) = v;
    }
    next_bc.store(a, p, t0, checked, flags, bc);
    __syncthreads();
    if (!ENDS && a.z.data) zs.load(a, a.z, p, i, whole, z);
    if (i + 1 < p.chunk1) fetch(i + 1);

    for (int nb = 0; nb < blocks; ++nb) {
      const int n0 = nb * 4 * LN + sl * kSelStates;
      const bool has = n0 < np && mine;
      if constexpr (MULTI) {
        h = load4(held + (nb * kSelThreads + tid) * 4);
        rate = rates(n0);
      }
      if (!ENDS && a.checkpoints && has)
        store4(a.checkpoints + ((p.b * a.nchunks + i) * a.dim + ch) * np + n0, h);
      const float* row = bc + nb * 4 * LN + sl * 4;
      // y of four positions from q * 4 on: over the states' threads, then to shared memory
      auto keep = [&](int q, float (&y)[4]) {
        sum_lanes<LN>(y, sl);
#pragma unroll
        for (int j = 0; j < kSums<LN>; ++j) {
          float* o = ys + (q * 4 + first_sum<LN>(sl) + j) * PITCH + c;
          if (sl < 4) *o = MULTI && nb > 0 ? *o + y[j] : y[j];
        }
      };
#pragma unroll 1
      for (int q = 0; q < TT / 4; q += 2) {
        if (flags.word[q] == kAllInside && flags.word[q + 1] == kAllInside) {
          // eight positions: all that does not wait for h first
          Four decay[8], add[8], C[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int t = q * 4 + j;
            const float2 v = io[t * PITCH + c];
            decay[j] = decays4(make_float2(v.x, v.x), rate);
            add[j] = mul4(load4(row + t * 2 * wide), make_float2(v.y, v.y));
            if (ENDS && nb == 0) total += v.x;
            if (!ENDS) C[j] = load4(row + t * 2 * wide + wide);
          }
          float y[2][4];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            h = fma4(decay[j], h, add[j]);
            if (!ENDS) y[j / 4][j % 4] = dot4(C[j], h);
          }
          if constexpr (!ENDS) {
            keep(q, y[0]);
            keep(q + 1, y[1]);
          }
          continue;
        }
#pragma unroll 1
        for (int half = q; half < q + 2; ++half) {
          const uint32_t f = flags.word[half];
          float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
          for (int j = 0; j < 4; ++j) {
            const int t = half * 4 + j, r = flags.row[t];
            const uint32_t fj = f >> (8 * j);
            float yj = 0.f;
            if (fj & kValid) {
              if (fj & kFirst) {
                h = a.init.data && r >= 0 && has ? of4(load_state(a.init, r, ch, n0, a.dstate)) : zero4();
                if (ENDS) total = INFINITY;
              }
              const float2 v = io[t * PITCH + c];
              h = fma4(decays4(make_float2(v.x, v.x), rate), h, mul4(load4(row + t * 2 * wide), make_float2(v.y, v.y)));
              if (ENDS && nb == 0) total += v.x;
              if (!ENDS) yj = dot4(load4(row + t * 2 * wide + wide), h);
              if (!ENDS && (fj & kLast) && a.final_states.data && r >= 0 && has)
                store_state(a.final_states, r, ch, n0, a.dstate, to4(h));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e == j) y[e] = yj;
          }
          if constexpr (!ENDS) keep(half, y);
        }
      }
      if constexpr (MULTI) store4(held + (nb * kSelThreads + tid) * 4, h);
    }
    __syncthreads();
    if constexpr (!ENDS) {
      float2 out[K];
#pragma unroll
      for (int k = 0; k < K; ++k) out[k] = *reinterpret_cast<const float2*>(&ys[Where::t(k) * PITCH + 2 * Where::c(k)]);
      if (a.D.data)
#pragma unroll
        for (int k = 0; k < K; ++k) out[k] = ffma2(ROWS ? of_pair(skips, k) : skip, pair_of<T>(x[k], a.pairs), out[k]);
      if (a.z.data)
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float2 v = pair_of<T>(z[k], a.pairs);
          out[k] = fmul2(out[k], make_float2(silu_of<T>(v.x), silu_of<T>(v.y)));
        }
      if (packed) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (!flags.valid(Where::t(k))) out[k] = both(0.f);
        __syncthreads();  // flags have been read
      }
      outs.store(a, a.out, p, i, whole, out);
    }
  }
  if (ENDS && mine) {
    for (int nb = 0; nb < blocks; ++nb) {
      const int n0 = nb * 4 * LN + sl * kSelStates;
      if (n0 >= np) continue;
      if constexpr (MULTI) h = load4(held + (nb * kSelThreads + tid) * 4);
      store4(a.ends + ((p.b * a.segments + p.seg) * a.dim + ch) * np + n0, h);
    }
    if (sl == 0) a.steps[(p.b * a.segments + p.seg) * a.dim + ch] = total;
  }
}

template <typename T, int LN, bool ROWS, bool MULTI, bool ENDS>
cudaError_t launch(const SelArgs& a, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(FwdSmem<LN>::bytes(a));
  const auto kernel = sel_fwd_kernel<T, LN, ROWS, MULTI, ENDS>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(a.launch_rows * a.segments * a.tiles)), dim3(kSelThreads), smem, s, a);
}

template <typename T, int LN, bool ROWS, bool MULTI = false>
cudaError_t run(const SelArgs& a, cudaStream_t s) {
  if (a.segments > 1) {
    const cudaError_t e = launch<T, LN, ROWS, MULTI, true>(a, s);
    if (e != cudaSuccess) return e;
  }
  return launch<T, LN, ROWS, MULTI, false>(a, s);
}

template <typename T>
cudaError_t run(const SelArgs& a, cudaStream_t s) {
  if (a.blocks > 1) return a.rows ? run<T, kSelLanes, true, true>(a, s) : run<T, kSelLanes, false, true>(a, s);
  switch (a.lanes) {
    case 1: return a.rows ? run<T, 1, true>(a, s) : run<T, 1, false>(a, s);
    case 2: return a.rows ? run<T, 2, true>(a, s) : run<T, 2, false>(a, s);
    case 4: return a.rows ? run<T, 4, true>(a, s) : run<T, 4, false>(a, s);
    case 8: return a.rows ? run<T, 8, true>(a, s) : run<T, 8, false>(a, s);
    default: return a.rows ? run<T, 16, true>(a, s) : run<T, 16, false>(a, s);
  }
}

}  // namespace

cudaError_t CC1D_DT_NAME(sel_fwd)(const SelArgs& a, cudaStream_t s) { return run<CC1D_DT_TYPE>(a, s); }

}  // namespace cc1d
