// Dropout + residual add + RMSNorm over the rows of a matrix (sm_100a).
//
//   r = residual + keep x / (1 - p), stored;  n = r rstd, rstd = 1 / sqrt(mean(r^2) + eps)
//   out = n w
// Backward, with q = dout w:
//   dr = dresidual_out + rstd (q - n mean(q n)),  dresidual = dr,  dx = keep dr / (1 - p),
//   dw = sum over the rows of dout n.
//
// One CTA per row, element by element.
#include "cc1d_block_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {
namespace {

constexpr int kRowsPerPartial = 64;

__device__ __forceinline__ float cta_sum(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) s += scratch[i];
  return s;
}

__device__ __forceinline__ float kept(const AddNormArgs& a, int64_t row, int64_t c) {
  if (!a.rng) return 1.f;
  const uint4 w = philox(static_cast<uint64_t>(a.rng[0]), static_cast<uint64_t>(row * ((a.dim + 3) / 4) + c / 4),
                         static_cast<uint64_t>(a.rng[a.rng_stride]));
  const unsigned v = (c & 3) == 0 ? w.x : (c & 3) == 1 ? w.y : (c & 3) == 2 ? w.z : w.w;
  return v >= a.keep_from ? a.keep_scale : 0.f;
}

template <typename T, typename R>
__global__ void __launch_bounds__(kThreads) add_norm_fwd_kernel(const AddNormArgs a) {
  grid_dependency_wait();
  __shared__ float scratch[kThreads / 32];
  const int64_t row = blockIdx.x;
  R* ro = static_cast<R*>(a.residual_out.data) + row * a.residual_out.s0;
  float sum = 0.f;
  for (int64_t c = threadIdx.x; c < a.dim; c += kThreads) {
    const float m = kept(a, row, c);
    float r = m == 0.f ? 0.f : m * to_f32(static_cast<const T*>(a.x.data)[row * a.x.s0 + c]);
    if (a.residual.data) r += to_f32(static_cast<const R*>(a.residual.data)[row * a.residual.s0 + c]);
    const R stored = from_f32<R>(r);
    ro[c] = stored;
    r = to_f32(stored);
    sum = fmaf(r, r, sum);
  }
  const float rstd = 1.f / sqrtf(cta_sum(sum, scratch) / static_cast<float>(a.dim) + a.eps);
  for (int64_t c = threadIdx.x; c < a.dim; c += kThreads)
    static_cast<T*>(a.out.data)[row * a.out.s0 + c] =
        from_f32<T>(to_f32(ro[c]) * rstd * load_any(a.weight.data, a.weight.dtype, c * a.weight.s0));
}

template <typename T, typename R>
__global__ void __launch_bounds__(kThreads) add_norm_bwd_kernel(const AddNormArgs a) {
  grid_dependency_wait();
  __shared__ float scratch[kThreads / 32];
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRowsPerPartial;
  float* part = a.dweight ? a.partials + blockIdx.x * a.dim : nullptr;
  if (part)
    for (int64_t c = threadIdx.x; c < a.dim; c += kThreads) part[c] = 0.f;
  for (int64_t row = row0; row < min(a.rows, row0 + kRowsPerPartial); ++row) {
    const R* rp = static_cast<const R*>(a.residual_out.data) + row * a.residual_out.s0;
    const T* dy = a.dout.data ? static_cast<const T*>(a.dout.data) + row * a.dout.s0 : nullptr;
    const R* dro = a.dresidual_out.data ? static_cast<const R*>(a.dresidual_out.data) + row * a.dresidual_out.s0 : nullptr;
    float sum = 0.f, dot = 0.f;
    for (int64_t c = threadIdx.x; c < a.dim; c += kThreads) {
      const float r = to_f32(rp[c]);
      sum = fmaf(r, r, sum);
      if (dy) dot = fmaf(r, to_f32(dy[c]) * load_any(a.weight.data, a.weight.dtype, c * a.weight.s0), dot);
    }
    const float inv = 1.f / static_cast<float>(a.dim);
    const float rstd = 1.f / sqrtf(cta_sum(sum, scratch) * inv + a.eps);
    const float k = cta_sum(dot, scratch) * inv * rstd;  // mean(q n)
    for (int64_t c = threadIdx.x; c < a.dim; c += kThreads) {
      const float n = to_f32(rp[c]) * rstd;
      const float g = dy ? to_f32(dy[c]) : 0.f;
      const float q = dy ? g * load_any(a.weight.data, a.weight.dtype, c * a.weight.s0) : 0.f;
      const float dr = (dro ? to_f32(dro[c]) : 0.f) + rstd * (q - n * k);
      if (a.dresidual.data) static_cast<R*>(a.dresidual.data)[row * a.dresidual.s0 + c] = from_f32<R>(dr);
      if (a.dx.data) {
        const float m = kept(a, row, c);
        static_cast<T*>(a.dx.data)[row * a.dx.s0 + c] = from_f32<T>(m == 0.f ? 0.f : m * dr);
      }
      if (part) part[c] += g * n;
    }
  }
}

__global__ void __launch_bounds__(kThreads) add_norm_weight_kernel(const AddNormArgs a, int64_t parts) {
  grid_dependency_wait();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (c >= a.dim) return;
  float s = 0.f;
  for (int64_t i = 0; i < parts; ++i) s += a.partials[i * a.dim + c];
  a.dweight[c] = s;
}

template <typename T, typename R>
cudaError_t fwd(const AddNormArgs& a, cudaStream_t s) {
  return launch_dependent(add_norm_fwd_kernel<T, R>, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, s, a);
}
int64_t parts_of(const AddNormArgs& a) { return (a.rows + kRowsPerPartial - 1) / kRowsPerPartial; }
template <typename T, typename R>
cudaError_t bwd(const AddNormArgs& a, cudaStream_t s) {
  cudaError_t e = launch_dependent(add_norm_bwd_kernel<T, R>, dim3(static_cast<unsigned>(parts_of(a))), dim3(kThreads), 0, s, a);
  if (e != cudaSuccess || !a.dweight) return e;
  add_norm_weight_kernel<<<static_cast<unsigned>((a.dim + kThreads - 1) / kThreads), kThreads, 0, s>>>(a, parts_of(a));
  return cudaGetLastError();
}

}  // namespace

using DT = CC1D_DT_TYPE;

cudaError_t CC1D_DT_NAME(add_norm_fwd)(const AddNormArgs& a, cudaStream_t s) {
  return a.residual_out.dtype == CC1D_FLOAT32 ? fwd<DT, float>(a, s) : fwd<DT, DT>(a, s);
}
cudaError_t CC1D_DT_NAME(add_norm_bwd)(const AddNormArgs& a, cudaStream_t s) {
  return a.residual_out.dtype == CC1D_FLOAT32 ? bwd<DT, float>(a, s) : bwd<DT, DT>(a, s);
}

#if CC1D_DT == 0
int64_t add_norm_bwd_partial_floats(const AddNormArgs& a) { return parts_of(a) * a.dim; }
#endif

}  // namespace cc1d
