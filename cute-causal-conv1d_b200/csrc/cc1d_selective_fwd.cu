// Selective recurrence, forward, over whole or packed sequences (sm_100a).
//
//     s_t = softplus(delta_t + bias)         h_t[n] = exp(s_t A[n]) h_{t-1}[n] + s_t x_t B_t[n]
//     y_t = sum_n C_t[n] h_t[n] + D x_t      out_t = y_t silu(z_t)
//
// A CTA of 128 threads owns up to 32 channels (64 or 128 for at most 8 or 4 states) of one batch
// row and walks the sequence in tiles of 32 positions.  A thread holds four states of a channel
// in registers; the step sizes of a tile are made once, by all threads, and with B and C lie in
// shared memory as fp32.
#include "cc1d_selective.cuh"

namespace cc1d {
namespace {

// Shared memory: flags; (s, s x) by position and channel; B and C; y by position and channel; with
// several passes the states between two tiles.
template <int LN>
struct FwdSmem {
  static constexpr int CH = kSelThreads / LN;
  static constexpr int kFlags = 256;
  static constexpr int kIo = kSelChunk * (CH + 1) * 8;
  static constexpr int kY = (kSelChunk * (CH + 1) * 4 + 15) / 16 * 16;
  static __host__ __device__ int64_t bytes(const SelArgs& a) {
    return kFlags + kIo + kY + kSelChunk * 2 * a.padded * 4 + (a.blocks > 1 ? a.blocks * kSelThreads * 16 : 0);
  }
};

// ENDS: only what each segment carries out of itself, for the segments behind it.
template <typename T, int LN, bool ENDS>
__global__ void __launch_bounds__(kSelThreads) sel_fwd_kernel(const SelArgs a) {
  constexpr int CH = kSelThreads / LN;
  constexpr int PITCH = CH + 1;
  extern __shared__ __align__(16) unsigned char smem[];
  SelFlags& flags = *reinterpret_cast<SelFlags*>(smem);
  float2* io = reinterpret_cast<float2*>(smem + FwdSmem<LN>::kFlags);
  float* ys = reinterpret_cast<float*>(smem + FwdSmem<LN>::kFlags + FwdSmem<LN>::kIo);
  float* bc = reinterpret_cast<float*>(smem + FwdSmem<LN>::kFlags + FwdSmem<LN>::kIo + FwdSmem<LN>::kY);
  const int np = static_cast<int>(a.padded);
  float* held = bc + kSelChunk * 2 * np;

  const SelPlace p = sel_place<LN>(a);
  const int tid = threadIdx.x, sl = tid % LN, c = tid / LN;
  const bool mine = c < p.channels;
  const int64_t ch = p.ch0 + (mine ? c : 0);
  grid_dependency_wait();

  Four h = zero4(), rate = zero4();
  float total = 0.f;  // ENDS: the sum of step sizes since the segment's start
  const int64_t ends_at = (p.b * a.segments * a.dim + ch) * np;  // of segment 0
  for (int nb = 0; nb < a.blocks; ++nb) {
    const int n0 = nb * kSelBlock + sl * kSelStates;
    const bool has = n0 < np;
    h = zero4();
    rate = mine && has ? load_rates(a, ch, n0) : zero4();
    if (!ENDS && mine && has)
      for (int64_t s = 0; s < p.seg; ++s) {
        const Four e = load4(a.ends + ends_at + s * a.dim * np + n0);
        const float sum = a.steps[(p.b * a.segments + s) * a.dim + ch];
#pragma unroll
        for (int i = 0; i < 4; ++i) h.v[i] = sum < INFINITY && h.v[i] != 0.f ? fmaf(exp2f(rate.v[i] * sum), h.v[i], e.v[i]) : e.v[i];
      }
    if (a.blocks > 1) store4(held + (nb * kSelThreads + tid) * 4, h);
  }

  for (int64_t chunk = p.chunk0; chunk < p.chunk1; ++chunk) {
    const int64_t t0 = chunk * kSelChunk;
    __syncthreads();  // the last tile's results have been read
    load_flags(a, p.b, t0, flags);
    __syncthreads();
#pragma unroll 4
    for (int e = tid; e < kSelChunk * CH; e += kSelThreads) {
      int t, cc;
      tile_place<CH>(a.rows, e, t, cc);
      float2 v = make_float2(0.f, 0.f);
      if (cc < p.channels && (reinterpret_cast<const uint8_t*>(flags.word)[t] & kValid)) {
        const int64_t d = p.ch0 + cc;
        float u = load_el<T>(a.delta, p.b, d, t0 + t);
        const float x = load_el<T>(a.x, p.b, d, t0 + t);
        if (a.bias.data) u += load_any(a.bias.data, a.bias.dtype, d * a.bias.s0);
        float slope;
        v.x = a.softplus ? step_size(u, &slope) : u;
        v.y = v.x * x;
      }
      io[t * PITCH + cc] = v;
    }
    load_bc<T>(a, p, t0, np, flags, bc);
    __syncthreads();

    for (int nb = 0; nb < a.blocks; ++nb) {
      const int n0 = nb * kSelBlock + sl * kSelStates;
      const bool has = n0 < np;
      if (a.blocks > 1) {
        h = load4(held + (nb * kSelThreads + tid) * 4);
        rate = mine && has ? load_rates(a, ch, n0) : zero4();
      }
      if (!ENDS && a.checkpoints && mine && has) store4(a.checkpoints + ((p.b * a.nchunks + chunk) * a.dim + ch) * np + n0, h);
      const float* row = bc + (has ? n0 : 0);
#pragma unroll 1
      for (int q = 0; q < kSelChunk / 4; ++q) {
        const uint32_t f = flags.word[q];
        const bool inside = f == kAllInside;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = q * 4 + j;
          const uint32_t fj = f >> (8 * j);
          y[j] = 0.f;
          if (!inside) {
            if (!(fj & kValid)) continue;
            if (fj & kFirst) {
              const int r = flags.row[t];
              h = a.init.data && r >= 0 && mine && has ? load_state(a.init, r, ch, n0, a.dstate) : zero4();
              if (ENDS) total = INFINITY;
            }
          }
          const float2 v = io[t * PITCH + c];
          const Four B = load4(row + t * 2 * np), C = load4(row + t * 2 * np + np);
          if (ENDS && nb == 0) total += v.x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            h.v[i] = fmaf(ex2_approx(v.x * rate.v[i]), h.v[i], v.y * B.v[i]);
            if (!ENDS) y[j] = fmaf(C.v[i], h.v[i], y[j]);
          }
          if (!inside && !ENDS && (fj & kLast) && a.final_states.data && flags.row[t] >= 0 && mine && has)
            store_state(a.final_states, flags.row[t], ch, n0, a.dstate, h);
        }
        if (!ENDS) {
          if (!has) y[0] = y[1] = y[2] = y[3] = 0.f;
          sum_lanes<LN>(y, sl);
#pragma unroll
          for (int j = 0; j < 4 / LN; ++j) {
            float* o = ys + (q * 4 + sl * (4 / LN) + j) * PITCH + c;
            *o = nb == 0 ? y[j] : *o + y[j];
          }
        }
      }
      if (a.blocks > 1) store4(held + (nb * kSelThreads + tid) * 4, h);
    }
    if (ENDS) continue;
    __syncthreads();
#pragma unroll 4
    for (int e = tid; e < kSelChunk * CH; e += kSelThreads) {
      int t, cc;
      tile_place<CH>(a.rows, e, t, cc);
      if (cc >= p.channels || t0 + t >= a.seqlen) continue;
      const int64_t d = p.ch0 + cc;
      float y = 0.f;
      if (reinterpret_cast<const uint8_t*>(flags.word)[t] & kValid) {
        y = ys[t * PITCH + cc];
        if (a.D.data) y = fmaf(load_any(a.D.data, a.D.dtype, d * a.D.s0), load_el<T>(a.x, p.b, d, t0 + t), y);
        if (a.z.data) y *= silu_of<T>(load_el<T>(a.z, p.b, d, t0 + t));
      }
      store_el<T>(a.out, p.b, d, t0 + t, y);
    }
  }
  if (ENDS && mine) {
    for (int nb = 0; nb < a.blocks; ++nb) {
      const int n0 = nb * kSelBlock + sl * kSelStates;
      if (n0 >= np) continue;
      if (a.blocks > 1) h = load4(held + (nb * kSelThreads + tid) * 4);
      store4(a.ends + ends_at + p.seg * a.dim * np + n0, h);
    }
    if (sl == 0) a.steps[(p.b * a.segments + p.seg) * a.dim + ch] = total;
  }
}

template <typename T, int LN, bool ENDS>
cudaError_t launch(const SelArgs& a, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(FwdSmem<LN>::bytes(a));
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(sel_fwd_kernel<T, LN, ENDS>), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(sel_fwd_kernel<T, LN, ENDS>, dim3(static_cast<unsigned>(a.batch * a.segments * a.tiles)), dim3(kSelThreads), smem, s, a);
}

template <typename T, int LN>
cudaError_t run(const SelArgs& a, cudaStream_t s) {
  if (a.segments > 1) {
    const cudaError_t e = launch<T, LN, true>(a, s);
    if (e != cudaSuccess) return e;
  }
  return launch<T, LN, false>(a, s);
}

}  // namespace

cudaError_t CC1D_DT_NAME(sel_fwd)(const SelArgs& a, cudaStream_t s) {
  switch (a.lanes) {
    case 1: return run<CC1D_DT_TYPE, 1>(a, s);
    case 2: return run<CC1D_DT_TYPE, 2>(a, s);
    default: return run<CC1D_DT_TYPE, 4>(a, s);
  }
}

}  // namespace cc1d
