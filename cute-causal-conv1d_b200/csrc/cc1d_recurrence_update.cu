// The gated recurrence for a few tokens of each row against a pool of fp32 states (sm_100a).
//
// One thread takes VEC neighbouring channels of one batch row through its tokens, from the
// state it reads to the one it writes back, so a state is read and written once.  Bound by
// HBM for many rows and by the launch for few.  VEC = 4 (8 or 16 bytes of each tensor, 16 of
// the state) where every tensor has unit channel stride and that alignment: (128, 8192) bf16
// in a pool of 160 rows takes 4.4 us (60% of the copy rate, launches back to back), channel by
// channel (8191 of them) 10.6 us; else VEC = 1.
#include "cc1d_block_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {
namespace {

template <typename T, int VEC>
__device__ __forceinline__ void load_at(const TensorArg& t, int64_t b, int64_t d, int64_t l, float (&f)[VEC]) {
  const T* p = static_cast<const T*>(t.data) + b * t.s0 + d * t.s1 + l * t.s2;
  if constexpr (VEC == 1) f[0] = to_f32(*p);
  else unpack<T, VEC>(ld_packet<T, VEC>(p), f);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_at(const TensorArg& t, int64_t b, int64_t d, int64_t l, const float (&f)[VEC]) {
  T* p = static_cast<T*>(t.data) + b * t.s0 + d * t.s1 + l * t.s2;
  if constexpr (VEC == 1) *p = from_f32<T>(f[0]);
  else st_packet<T, VEC>(p, pack<T, VEC>(f));
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rec_update_kernel(const RecUpdateArgs a) {
  const int64_t nv = a.dim / VEC;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  grid_dependency_wait();
  if (i >= a.batch * nv) return;
  const int64_t b = i / nv, d = (i - b * nv) * VEC;
  const int64_t row = a.indices ? a.indices[b * a.indices_stride] : b;
  float x[VEC], g[VEC], z[VEC], y[VEC], h[VEC], bias[VEC];
  if (row < 0 || row >= a.nstates) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) y[v] = 0.f;
    for (int64_t l = 0; l < a.seqlen; ++l) store_at<T, VEC>(a.out, b, d, l, y);
    return;
  }
  // all loads of the first token before anything is used
  load_at<float, VEC>(a.state, row, d, 0, h);
  load_at<T, VEC>(a.gate, b, d, 0, g);
  load_at<T, VEC>(a.x, b, d, 0, x);
  if (a.z.data) load_at<T, VEC>(a.z, b, d, 0, z);
#pragma unroll
  for (int v = 0; v < VEC; ++v) bias[v] = a.bias.data ? load_any(a.bias.data, a.bias.dtype, (d + v) * a.bias.s0) : 0.f;
  for (int64_t l = 0;;) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float ga, gc;
      sigmoid_pair_of<T>(g[v] + bias[v], ga, gc);
      h[v] = fmaf(ga, h[v], gc * x[v]);
      y[v] = a.z.data ? h[v] * silu_of<T>(z[v]) : h[v];
    }
    store_at<T, VEC>(a.out, b, d, l, y);
    if (++l == a.seqlen) break;
    load_at<T, VEC>(a.gate, b, d, l, g);
    load_at<T, VEC>(a.x, b, d, l, x);
    if (a.z.data) load_at<T, VEC>(a.z, b, d, l, z);
  }
  store_at<float, VEC>(a.state, row, d, 0, h);
}

// Packets of 4 channels are legal.
bool packets_of_four(const RecUpdateArgs& a) {
  const struct { const TensorArg& t; int64_t rows; bool tokens; } all[] = {
      {a.x, a.batch, true}, {a.gate, a.batch, true}, {a.z, a.batch, true}, {a.out, a.batch, true}, {a.state, a.nstates, false}};
  if (a.dim % 4) return false;
  for (const auto& e : all) {
    if (!e.t.data) continue;
    const uintptr_t bytes = e.t.dtype == CC1D_FLOAT32 ? 16 : 8;
    if (e.t.s1 != 1 || (reinterpret_cast<uintptr_t>(e.t.data) % bytes) || (e.rows > 1 && e.t.s0 % 4) ||
        (e.tokens && a.seqlen > 1 && e.t.s2 % 4))
      return false;
  }
  return true;
}

template <typename T, int VEC>
cudaError_t run(const RecUpdateArgs& a, cudaStream_t s) {
  const int64_t threads = a.batch * (a.dim / VEC);
  return launch_dependent(rec_update_kernel<T, VEC>, dim3(static_cast<unsigned>((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
}

}  // namespace

cudaError_t CC1D_DT_NAME(rec_update)(RecUpdateArgs& a, cudaStream_t s) {
  return packets_of_four(a) ? run<CC1D_DT_TYPE, 4>(a, s) : run<CC1D_DT_TYPE, 1>(a, s);
}

}  // namespace cc1d
