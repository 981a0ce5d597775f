// Gated linear recurrence along the sequence, forward and backward (sm_100a).
//
//   a = sigmoid(gate + bias), c = 1 - a = sigmoid(-(gate + bias))
//   h_t = a_t h_{t-1} + c_t x_t,  out_t = h_t silu(z_t)
//
// Backward, with g_t the gradient of h_t (dout_t silu(z_t), plus dfinal at a sequence's last
// position) and s_t = a_{t+1} (g_{t+1} + s_{t+1}) what later positions send back:
//   dx_t = (g_t + s_t) c_t,  dgate_t = (g_t + s_t) (h_{t-1} - x_t) a_t c_t,
//   dz_t = dout_t h_t silu'(z_t),  dinit = s before the first position.
//
// One thread walks one channel of one batch row.
#include "cc1d_block_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {
namespace {

template <typename T>
__device__ __forceinline__ float at(const TensorArg& t, int64_t b, int64_t d, int64_t l) {
  return to_f32(static_cast<const T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2]);
}
template <typename T>
__device__ __forceinline__ void put(const TensorArg& t, int64_t b, int64_t d, int64_t l, float v) {
  static_cast<T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2] = from_f32<T>(v);
}
__device__ __forceinline__ int seq_at(const RecArgs& a, int64_t b, int64_t l) {
  if (l < 0 || l >= a.seqlen) return -1;
  return static_cast<const int*>(a.seq_idx.data)[b * a.seq_idx.s0 + l * a.seq_idx.s1];
}
__device__ __forceinline__ float state_at(const TensorArg& t, int64_t n, int64_t d) {
  return static_cast<const float*>(t.data)[n * t.s0 + d * t.s1];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rec_fwd_kernel(const RecArgs a) {
  grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * a.dim) return;
  const int64_t b = i / a.dim, d = i - b * a.dim;
  const float bias = a.bias.data ? load_any(a.bias.data, a.bias.dtype, d * a.bias.s0) : 0.f;
  const bool seq = a.seq_idx.data != nullptr;
  float h = !seq && a.init.data ? state_at(a.init, b, d) : 0.f;
  for (int64_t l = 0; l < a.seqlen; ++l) {
    if (a.checkpoints && l % kRecChunk == 0) a.checkpoints[(b * a.nchunks + l / kRecChunk) * a.dim + d] = h;
    float x = 0.f;
    bool last = l == a.seqlen - 1;
    int64_t row = b;
    if (seq) {
      const int id = seq_at(a, b, l);
      if (id < 0) {
        put<T>(a.out, b, d, l, 0.f);
        continue;
      }
      row = id;
      if (id != seq_at(a, b, l - 1)) h = a.init.data && id < a.nstates ? state_at(a.init, id, d) : 0.f;
      last = id != seq_at(a, b, l + 1);
    }
    float ga, gc;
    sigmoid_pair<T>(at<T>(a.gate, b, d, l) + bias, ga, gc);
    x = at<T>(a.x, b, d, l);
    h = fmaf(ga, h, gc * x);
    float y = h;
    if (a.z.data) y *= silu_of<T>(at<T>(a.z, b, d, l));
    put<T>(a.out, b, d, l, y);
    if (last && a.final_states.data && row < a.nstates)
      static_cast<float*>(a.final_states.data)[row * a.final_states.s0 + d * a.final_states.s1] = h;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) rec_bwd_kernel(const RecArgs a) {
  grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * a.dim) return;
  const int64_t b = i / a.dim, d = i - b * a.dim;
  const float bias = a.bias.data ? load_any(a.bias.data, a.bias.dtype, d * a.bias.s0) : 0.f;
  const bool seq = a.seq_idx.data != nullptr;
  float s = 0.f, sum = 0.f;
  for (int64_t k = a.nchunks - 1; k >= 0; --k) {
    float hs[kRecChunk + 1];  // h before each position of the chunk
    const int64_t l0 = k * kRecChunk;
    const int n = static_cast<int>(min(static_cast<int64_t>(kRecChunk), a.seqlen - l0));
    float h = a.checkpoints[(b * a.nchunks + k) * a.dim + d];
    for (int j = 0; j < n; ++j) {
      const int64_t l = l0 + j;
      const int id = seq ? seq_at(a, b, l) : 0;
      if (seq && id >= 0 && id != seq_at(a, b, l - 1)) h = a.init.data && id < a.nstates ? state_at(a.init, id, d) : 0.f;
      hs[j] = h;
      if (id < 0) continue;
      float ga, gc;
      sigmoid_pair<T>(at<T>(a.gate, b, d, l) + bias, ga, gc);
      h = fmaf(ga, h, gc * at<T>(a.x, b, d, l));
    }
    for (int j = n - 1; j >= 0; --j) {
      const int64_t l = l0 + j;
      int64_t row = b;
      bool first = l == 0, last = l == a.seqlen - 1;
      if (seq) {
        const int id = seq_at(a, b, l);
        if (id < 0) {
          put<T>(a.dx, b, d, l, 0.f);
          put<T>(a.dgate, b, d, l, 0.f);
          if (a.z.data) put<T>(a.dz, b, d, l, 0.f);
          continue;
        }
        row = id;
        first = id != seq_at(a, b, l - 1);
        last = id != seq_at(a, b, l + 1);
      }
      if (last) s = a.dfinal.data && row < a.nstates ? state_at(a.dfinal, row, d) : 0.f;
      float ga, gc;
      sigmoid_pair<T>(at<T>(a.gate, b, d, l) + bias, ga, gc);
      const float x = at<T>(a.x, b, d, l);
      const float dy = at<T>(a.dout, b, d, l);
      float g = dy;
      if (a.z.data) {
        float si, ds;
        silu_and_grad<T>(at<T>(a.z, b, d, l), si, ds);
        g = dy * si;
        put<T>(a.dz, b, d, l, dy * fmaf(ga, hs[j], gc * x) * ds);
      }
      g += s;
      put<T>(a.dx, b, d, l, g * gc);
      s = ga * g;
      const float du = s * gc * (hs[j] - x);
      put<T>(a.dgate, b, d, l, du);
      sum += du;
      if (first && a.dinit.data && row < a.nstates)
        static_cast<float*>(a.dinit.data)[row * a.dinit.s0 + d * a.dinit.s1] = s;
    }
  }
  if (a.dbias) a.partials[b * a.dim + d] = sum;
}

// dbias[d] = sum over the batch rows' partial sums, in order.
__global__ void __launch_bounds__(kThreads) rec_bias_kernel(const RecArgs a) {
  grid_dependency_wait();
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (d >= a.dim) return;
  float s = 0.f;
  for (int64_t b = 0; b < a.batch; ++b) s += a.partials[b * a.dim + d];
  a.dbias[d] = s;
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

}  // namespace

using DT = CC1D_DT_TYPE;

cudaError_t CC1D_DT_NAME(rec_fwd)(const RecArgs& a, cudaStream_t s) {
  return launch_dependent(rec_fwd_kernel<DT>, dim3(blocks_for(a.batch * a.dim)), dim3(kThreads), 0, s, a);
}
cudaError_t CC1D_DT_NAME(rec_bwd)(const RecArgs& a, cudaStream_t s) {
  cudaError_t e = launch_dependent(rec_bwd_kernel<DT>, dim3(blocks_for(a.batch * a.dim)), dim3(kThreads), 0, s, a);
  if (e == cudaSuccess && a.dbias) e = launch_dependent(rec_bias_kernel, dim3(blocks_for(a.dim)), dim3(kThreads), 0, s, a);
  return e;
}
cudaError_t CC1D_DT_NAME(rec_update)(const RecUpdateArgs& a, cudaStream_t s) {
  return launch_dependent(rec_update_kernel<DT>, dim3(blocks_for(a.batch * a.dim)), dim3(kThreads), 0, s, a);
}

#if CC1D_DT == 0
int64_t rec_bwd_partial_floats(const RecArgs& a) { return a.batch * a.dim; }
#endif

}  // namespace cc1d
