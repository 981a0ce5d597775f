// Selective recurrence, backward (sm_100a).
//
// With dy = dout silu(z) and g_t the gradient of h_t,
//     g_t[n] = C_t[n] dy_t + a_{t+1}[n] g_{t+1}[n]             a = exp(s A)
//     dC_t[n] = sum_d dy_t h_t[n]        dB_t[n] = sum_d g_t[n] s_t x_t
//     dx_t = s_t sum_n g_t[n] B_t[n] + D dy_t
//     ds_t = sum_n g_t[n] a_t[n] h_{t-1}[n] A[n] + x_t sum_n g_t[n] B_t[n]
//     dA[n] = sum_t g_t[n] a_t[n] h_{t-1}[n] s_t
// and ddelta = ds sigmoid(delta + bias), dz = dout y silu'(z).
//
// CTAs, threads and tiles are the forward's; a CTA goes through its tiles from the last one back.
// From the state that the forward kept before a tile it runs forward, keeping the state before
// every fourth position, then takes the groups of four positions from the last one back: states
// again, then gradients.  dB and dC are summed over the warp's channels by exchanges between
// lanes, over the CTA's warps in shared memory and over CTAs by a second kernel, all in a fixed
// order.
#include "cc1d_selective.cuh"

namespace cc1d {
namespace {

constexpr int kWarps = kSelThreads / 32;

template <int LN>
struct BwdSmem {
  static constexpr int CH = kSelThreads / LN;
  static constexpr int kFlags = 256;
  static constexpr int kIo = kSelChunk * (CH + 1) * 16;
  static constexpr int kSums = (kSelChunk * (CH + 1) * 12 + 15) / 16 * 16;  // several passes only
  static constexpr int kSub = kSelChunk / 4 * kSelThreads * 16;
  static constexpr int kSlab = kSelChunk * 8 * LN * 4;                       // one warp's sums of dB and dC
  static __host__ __device__ int64_t bytes(const SelArgs& a) {
    return kFlags + kIo + kSub + kWarps * kSlab + kSelChunk * 2 * a.padded * 4 +
           (a.blocks > 1 ? kSums + 3ll * a.blocks * kSelThreads * 16 : 0);
  }
};

// Adds v to the sum hi + lo, which together hold twice the bits (Knuth's two-sum).
__device__ __forceinline__ void add_to(float& hi, float& lo, float v) {
  const float s = hi + v;
  const float w = s - hi;
  lo += (hi - (s - w)) + (v - w);
  hi = s;
}

// The sums of v[0 .. 8) over the channels of a warp; a lane ends with one of them, the number of
// which it returns (in v[0]); lanes that differ in further bits hold the same sums.
template <int LN>
__device__ __forceinline__ int sum_channels(float (&v)[8], int lane) {
  int which = 0;
#pragma unroll
  for (int half = 4; half >= 1; half /= 2) {
    const int bit = half == 4 ? 16 : half == 2 ? 8 : 4;
    const bool hi = lane & bit;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = hi ? v[i] : v[half + i];
      v[i] = (hi ? v[half + i] : v[i]) + __shfl_xor_sync(~0u, send, bit);
    }
    which = which * 2 + (hi ? 1 : 0);
  }
#pragma unroll
  for (int bit = 2; bit >= LN; bit /= 2) v[0] += __shfl_xor_sync(~0u, v[0], bit);
  return which;
}

// ENDS: only the gradient that each segment hands to the one before it.
template <typename T, int LN, bool ENDS>
__global__ void __launch_bounds__(kSelThreads) sel_bwd_kernel(const SelArgs a) {
  constexpr int CH = kSelThreads / LN;
  constexpr int PITCH = CH + 1;
  using Smem = BwdSmem<LN>;
  extern __shared__ __align__(16) unsigned char smem[];
  SelFlags& flags = *reinterpret_cast<SelFlags*>(smem);
  float4* io = reinterpret_cast<float4*>(smem + Smem::kFlags);  // in: s, x, dy, sigmoid; out: dx, ddelta, y
  float* sub = reinterpret_cast<float*>(smem + Smem::kFlags + Smem::kIo);
  float* slabs = reinterpret_cast<float*>(smem + Smem::kFlags + Smem::kIo + Smem::kSub);
  float* bc = slabs + kWarps * Smem::kSlab / 4;
  const int np = static_cast<int>(a.padded);
  float* held = bc + kSelChunk * 2 * np;  // several passes: g carried, dA and its low part
  float* sums = held + 3 * a.blocks * kSelThreads * 4;

  const SelPlace p = sel_place<LN>(a);
  const int tid = threadIdx.x, sl = tid % LN, c = tid / LN, lane = tid & 31, warp = tid >> 5;
  const bool mine = c < p.channels;
  const int64_t ch = p.ch0 + (mine ? c : 0);
  grid_dependency_wait();

  const float skip = a.D.data && mine ? load_any(a.D.data, a.D.dtype, ch * a.D.s0) : 0.f;
  Four rate = zero4(), carry = zero4(), da = zero4(), da_low = zero4();
  float dbias = 0.f, dbias_low = 0.f, dskip = 0.f, dskip_low = 0.f;
  float total = 0.f;
  const int64_t ends_at = (p.b * a.segments * a.dim + ch) * np;
  for (int nb = 0; nb < a.blocks; ++nb) {
    const int n0 = nb * kSelBlock + sl * kSelStates;
    const bool has = n0 < np;
    rate = mine && has ? load_rates(a, ch, n0) : zero4();
    carry = zero4();
    if (!ENDS && mine && has)
      for (int64_t s = a.segments - 1; s > p.seg; --s) {
        const Four e = load4(a.ends + ends_at + s * a.dim * np + n0);
        const float sum = a.steps[(p.b * a.segments + s) * a.dim + ch];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          carry.v[i] = sum < INFINITY && carry.v[i] != 0.f ? fmaf(exp2f(rate.v[i] * sum), carry.v[i], e.v[i]) : e.v[i];
      }
    if (a.blocks > 1) {
      store4(held + (nb * 3 * kSelThreads + tid) * 4, carry);
      store4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4, zero4());
      store4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4, zero4());
    }
  }

  for (int64_t chunk = p.chunk1 - 1; chunk >= p.chunk0; --chunk) {
    const int64_t t0 = chunk * kSelChunk;
    __syncthreads();
    load_flags(a, p.b, t0, flags);
    __syncthreads();
#pragma unroll 4
    for (int e = tid; e < kSelChunk * CH; e += kSelThreads) {
      int t, cc;
      tile_place<CH>(a.rows, e, t, cc);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (cc < p.channels && (reinterpret_cast<const uint8_t*>(flags.word)[t] & kValid)) {
        const int64_t d = p.ch0 + cc;
        float u = load_el<T>(a.delta, p.b, d, t0 + t);
        v.y = load_el<T>(a.x, p.b, d, t0 + t);
        v.z = load_el<T>(a.dout, p.b, d, t0 + t);
        if (a.z.data) v.z *= silu_of<T>(load_el<T>(a.z, p.b, d, t0 + t));
        if (a.bias.data) u += load_any(a.bias.data, a.bias.dtype, d * a.bias.s0);
        v.x = u;
        v.w = 1.f;
        if (a.softplus) v.x = step_size(u, &v.w);
      }
      io[t * PITCH + cc] = v;
    }
    load_bc<T>(a, p, t0, np, flags, bc);
    __syncthreads();

    for (int nb = 0; nb < a.blocks; ++nb) {
      const int n0 = nb * kSelBlock + sl * kSelStates;
      const bool has = n0 < np;
      if (a.blocks > 1) {
        carry = load4(held + (nb * 3 * kSelThreads + tid) * 4);
        rate = mine && has ? load_rates(a, ch, n0) : zero4();
      }
      const float* row = bc + (has ? n0 : 0);
      Four h = zero4();
      if (!ENDS) {
        if (mine && has) h = load4(a.checkpoints + ((p.b * a.nchunks + chunk) * a.dim + ch) * np + n0);
#pragma unroll 1
        for (int q = 0; q < kSelChunk / 4; ++q) {
          store4(sub + (q * kSelThreads + tid) * 4, h);
          const uint32_t f = flags.word[q];
          const bool inside = f == kAllInside;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = q * 4 + j;
            const uint32_t fj = f >> (8 * j);
            if (!inside) {
              if (!(fj & kValid)) continue;
              if (fj & kFirst) {
                const int r = flags.row[t];
                h = a.init.data && r >= 0 && mine && has ? load_state(a.init, r, ch, n0, a.dstate) : zero4();
              }
            }
            const float4 v = io[t * PITCH + c];
            const float sx = v.x * v.y;
            const Four B = load4(row + t * 2 * np);
#pragma unroll
            for (int i = 0; i < 4; ++i) h.v[i] = fmaf(ex2_approx(v.x * rate.v[i]), h.v[i], sx * B.v[i]);
          }
        }
      }
      Four da_tile = zero4();
#pragma unroll 1
      for (int q = kSelChunk / 4 - 1; q >= 0; --q) {
        const uint32_t f = flags.word[q];
        const bool inside = f == kAllInside;
        float decay[4][4], kept[4][4], now[4][4];  // a, a h_{t-1} and h of the four positions
        if (!ENDS) h = load4(sub + (q * kSelThreads + tid) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = q * 4 + j;
          const uint32_t fj = f >> (8 * j);
          if (!inside && !ENDS && (fj & kFirst)) {
            const int r = flags.row[t];
            h = a.init.data && r >= 0 && mine && has ? load_state(a.init, r, ch, n0, a.dstate) : zero4();
          }
          const float4 v = io[t * PITCH + c];
          const float sx = v.x * v.y;
          const Four B = load4(row + t * 2 * np);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            decay[j][i] = ex2_approx(v.x * rate.v[i]);
            if (ENDS) continue;
            kept[j][i] = decay[j][i] * h.v[i];
            h.v[i] = fmaf(sx, B.v[i], kept[j][i]);
            now[j][i] = h.v[i];
          }
        }
        float y[4], sa[4], sb[4];  // sums over the states of C h, g a h_{t-1} A and g B
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const int t = q * 4 + j;
          const uint32_t fj = f >> (8 * j);
          y[j] = sa[j] = sb[j] = 0.f;
          float bcs[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) bcs[i] = 0.f;
          if (inside || (fj & kValid)) {
            if (!inside && (fj & kLast)) {
              const int r = flags.row[t];
              carry = a.dfinal.data && r >= 0 && mine && has ? load_state(a.dfinal, r, ch, n0, a.dstate) : zero4();
            }
            const float4 v = io[t * PITCH + c];
            const float sx = v.x * v.y;
            const Four B = load4(row + t * 2 * np), C = load4(row + t * 2 * np + np);
            if (ENDS && nb == 0) total += v.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float g = fmaf(C.v[i], v.z, carry.v[i]);
              carry.v[i] = decay[j][i] * g;
              if (ENDS) continue;
              bcs[i] = g * sx;
              bcs[4 + i] = v.z * now[j][i];
              y[j] = fmaf(C.v[i], now[j][i], y[j]);
              sb[j] = fmaf(g, B.v[i], sb[j]);
              const float w = g * kept[j][i];
              sa[j] = fmaf(w, rate.v[i], sa[j]);
              da_tile.v[i] = fmaf(w, v.x, da_tile.v[i]);
            }
            if (!inside && (fj & kFirst)) {
              const int r = flags.row[t];
              if (!ENDS && a.dinit.data && r >= 0 && mine && has) store_state(a.dinit, r, ch, n0, a.dstate, carry);
              carry = zero4();
              if (ENDS) total = INFINITY;
            }
          }
          if (!ENDS) {
            if (p.channels < CH && !mine)  // so that 0 * infinity of no channel does not count
#pragma unroll
              for (int i = 0; i < 8; ++i) bcs[i] = 0.f;
            const int which = sum_channels<LN>(bcs, lane);
            if ((lane & 3) < LN) slabs[warp * (Smem::kSlab / 4) + t * 8 * LN + (which >> 2) * 4 * LN + sl * 4 + (which & 3)] = bcs[0];
          }
        }
        if (ENDS) continue;
        if (!has)
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = sa[j] = sb[j] = 0.f;
        sum_lanes<LN>(y, sl);
        sum_lanes<LN>(sa, sl);
        sum_lanes<LN>(sb, sl);
#pragma unroll
        for (int j = 0; j < 4 / LN; ++j) {
          const int t = q * 4 + sl * (4 / LN) + j;
          float* s = sums + (t * PITCH + c) * 3;
          if (nb > 0) {
            y[j] += s[0];
            sa[j] += s[1];
            sb[j] += s[2];
          }
          if (nb + 1 < a.blocks) {
            s[0] = y[j];
            s[1] = sa[j];
            s[2] = sb[j];
            continue;
          }
          const float4 v = io[t * PITCH + c];
          const float du = fmaf(sa[j], 0.693147181f, v.y * sb[j]) * v.w;
          __syncwarp();  // the channel's other lanes have read theirs
          io[t * PITCH + c] = make_float4(fmaf(v.x, sb[j], skip * v.z), du, fmaf(skip, v.y, y[j]), 0.f);
          add_to(dbias, dbias_low, du);
          add_to(dskip, dskip_low, v.z * v.y);
        }
      }
      if (a.blocks > 1) store4(held + (nb * 3 * kSelThreads + tid) * 4, carry);
      if (ENDS) continue;
      if (a.blocks > 1) {
        da = load4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4);
        da_low = load4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) add_to(da.v[i], da_low.v[i], da_tile.v[i]);
      if (a.blocks > 1) {
        store4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4, da);
        store4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4, da_low);
      }
      __syncthreads();
      // this pass's states of dB and dC: the warps' sums to the CTA's
      for (int e = tid; e < kSelChunk * 8 * LN; e += kSelThreads) {
        const int t = e / (8 * LN), v = e % (8 * LN), n = nb * kSelBlock + v % (4 * LN);
        if (t0 + t >= a.seqlen || n >= np) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s += slabs[w * (Smem::kSlab / 4) + e];
        a.parts_bc[(((p.b * a.seqlen + t0 + t) * a.tiles + p.tile) * 2 + v / (4 * LN)) * np + n] = s;
      }
      if (nb + 1 < a.blocks) __syncthreads();
    }
    if (ENDS) continue;
#pragma unroll 4
    for (int e = tid; e < kSelChunk * CH; e += kSelThreads) {
      int t, cc;
      tile_place<CH>(a.rows, e, t, cc);
      if (cc >= p.channels || t0 + t >= a.seqlen) continue;
      const int64_t d = p.ch0 + cc;
      const bool valid = reinterpret_cast<const uint8_t*>(flags.word)[t] & kValid;
      const float4 v = valid ? io[t * PITCH + cc] : make_float4(0.f, 0.f, 0.f, 0.f);
      store_el<T>(a.dx, p.b, d, t0 + t, v.x);
      store_el<T>(a.ddelta, p.b, d, t0 + t, v.y);
      if (a.z.data) {
        float dz = 0.f;
        if (valid) {
          // silu'(z) = s + z s (1 - s)
          const float z = load_el<T>(a.z, p.b, d, t0 + t);
          float s, less;
          sigmoid_pair_of<T>(z, s, less);
          dz = load_el<T>(a.dout, p.b, d, t0 + t) * v.z * fmaf(z * s, less, s);
        }
        store_el<T>(a.dz, p.b, d, t0 + t, dz);
      }
    }
  }

  for (int nb = 0; nb < a.blocks; ++nb) {
    const int n0 = nb * kSelBlock + sl * kSelStates;
    if (n0 >= np || !mine) continue;
    if (ENDS) {
      if (a.blocks > 1) carry = load4(held + (nb * 3 * kSelThreads + tid) * 4);
      store4(a.ends + ends_at + p.seg * a.dim * np + n0, carry);
    } else {
      if (a.blocks > 1) {
        da = load4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4);
        da_low = load4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) da.v[i] += da_low.v[i];
      store4(a.parts_a + ((p.b * a.segments + p.seg) * a.dim + ch) * np + n0, da);
    }
  }
  if (ENDS) {
    if (mine && sl == 0) a.steps[(p.b * a.segments + p.seg) * a.dim + ch] = total;
    return;
  }
  dskip += dskip_low;
  dbias += dbias_low;
#pragma unroll
  for (int bit = 1; bit < LN; bit *= 2) {
    dskip += __shfl_xor_sync(~0u, dskip, bit);
    dbias += __shfl_xor_sync(~0u, dbias, bit);
  }
  if (mine && sl == 0) {
    float* d = a.parts_d + (p.b * a.segments + p.seg) * 2 * a.dim + ch;
    d[0] = dskip;
    d[a.dim] = dbias;
  }
}

// dB and dC: the sums over a group's CTAs.  A thread takes one state of one position.
template <typename T>
__global__ void __launch_bounds__(kThreads) sel_sum_bc_kernel(const SelArgs a) {
  grid_dependency_wait();
  const int64_t per = 2 * a.padded;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * a.seqlen * a.groups * per) return;
  const int64_t v = i % per, r = i / per, g = r % a.groups, bt = r / a.groups;
  const float* part = a.parts_bc + (bt * a.tiles + g * a.group_tiles) * per + v;
  float s = 0.f;
#pragma unroll 4
  for (int64_t k = 0; k < a.group_tiles; ++k) s += part[k * per];
  const bool is_c = v >= a.padded;
  const int64_t n = is_c ? v - a.padded : v;
  if (n >= a.dstate) return;
  const TensorArg& t = is_c ? a.dC : a.dB;
  static_cast<T*>(t.data)[(bt / a.seqlen) * t.s0 + g * (is_c ? a.dC_group : a.dB_group) + n * t.s1 + (bt % a.seqlen) * t.s2] = from_f32<T>(s);
}

// dA, dD and dbias: the sums over batch rows and segments.
__global__ void __launch_bounds__(kThreads) sel_sum_params_kernel(const SelArgs a) {
  grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t na = a.dim * a.padded, rows = a.batch * a.segments;
  if (i >= na + 2 * a.dim) return;
  const bool is_a = i < na;
  const float* part = is_a ? a.parts_a + i : a.parts_d + (i - na);
  const int64_t step = is_a ? na : 2 * a.dim;
  float s = 0.f, low = 0.f;
#pragma unroll 4
  for (int64_t k = 0; k < rows; ++k) add_to(s, low, part[k * step]);
  s += low;
  if (is_a) {
    const int64_t d = i / a.padded, n = i - d * a.padded;
    if (a.dA && n < a.dstate) a.dA[d * a.dstate + n] = s;
  } else if (i - na < a.dim) {
    if (a.dD) a.dD[i - na] = s;
  } else if (a.dbias) {
    a.dbias[i - na - a.dim] = s;
  }
}

template <typename T, int LN, bool ENDS>
cudaError_t launch(const SelArgs& a, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(BwdSmem<LN>::bytes(a));
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(sel_bwd_kernel<T, LN, ENDS>), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(sel_bwd_kernel<T, LN, ENDS>, dim3(static_cast<unsigned>(a.batch * a.segments * a.tiles)), dim3(kSelThreads), smem, s, a);
}

template <typename T, int LN>
cudaError_t run(const SelArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (a.segments > 1) e = launch<T, LN, true>(a, s);
  if (e == cudaSuccess) e = launch<T, LN, false>(a, s);
  const int64_t bc = a.batch * a.seqlen * a.groups * 2 * a.padded, params = a.dim * (a.padded + 2);
  if (e == cudaSuccess)
    e = launch_dependent(sel_sum_bc_kernel<T>, dim3(static_cast<unsigned>((bc + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
  if (e == cudaSuccess)
    e = launch_dependent(sel_sum_params_kernel, dim3(static_cast<unsigned>((params + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
  return e;
}

}  // namespace

cudaError_t CC1D_DT_NAME(sel_bwd)(const SelArgs& a, cudaStream_t s) {
  switch (a.lanes) {
    case 1: return run<CC1D_DT_TYPE, 1>(a, s);
    case 2: return run<CC1D_DT_TYPE, 2>(a, s);
    default: return run<CC1D_DT_TYPE, 4>(a, s);
  }
}

}  // namespace cc1d
