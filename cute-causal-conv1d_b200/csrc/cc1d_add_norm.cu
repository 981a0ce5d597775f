// Dropout + residual add + RMSNorm over the rows of a matrix (sm_100a).
//
//   r = residual + keep x / (1 - p), stored;  n = r rstd, rstd = 1 / sqrt(mean(r^2) + eps)
//   out = n w
// Backward, with q = dout w:
//   dr = dresidual_out + rstd (q - n mean(q n)),  dresidual = dr,  dx = keep dr / (1 - p),
//   dw = sum over the rows of dout n.
//
// G threads take a row and hold it in registers between its sum and its use, so every element
// is read and written once: a warp up to 1024 columns (512 in fp32), which needs no barrier,
// else the whole CTA.  Each thread has E neighbouring columns per step, a multiple of the 4
// that one Philox block decides: the mask costs about 20 integer instructions per element,
// computed where it is used, forward and backward.  CTAs stay (a few per SM) and load their
// next row before they work on the present one.
//
// Bound by HBM without dropout (65536 x 4096 bf16: forward 334 us, 99% of the copy rate; backward
// 362 us, 92%, with dx and dresidual one tensor as the Python function makes them), by the mask's
// integer arithmetic with it (419 and 562 us).  Rows too wide for the registers (more than 16384
// columns, backward 8192, and 8192 in fp32 or off the 16-byte alignment) are read a second time,
// from L2, and move element by element whatever their alignment: 8192 x 20480 bf16 forward 442 us
// (47%), 8192 x 16384 backward 843 us (20%).
#include "cc1d_block_launch.h"
#include "cc1d_block_math.cuh"

namespace cc1d {
namespace {

constexpr int kWideElements = 4;  // columns of a thread per step, rows read twice

// E neighbouring elements as they lie in memory.
template <typename T, int E> struct alignas(16) Cols { T v[E]; };

// The widest access, up to 16 bytes, to elements of rows that start on multiples of A of them.
// Known at compile time: bf16 8192 x 4092, without dropout, forward 49 us with A = 4 and 111 us
// element by element (115 us with a branch on the address); x 4094 (A = 2) 64 us; fp32 x 4094
// forward 100 and backward 113 us against 121 and 159.
template <int BYTES> struct Access;
template <> struct Access<16> { using Type = uint4; };
template <> struct Access<8> { using Type = uint2; };
template <> struct Access<4> { using Type = uint32_t; };
template <> struct Access<2> { using Type = uint16_t; };
template <typename T, int A> struct Piece {
  static constexpr int kBytes = A * sizeof(T) < 16 ? A * sizeof(T) : 16, kElements = kBytes / sizeof(T);
  using Type = typename Access<kBytes>::Type;
};

// n of E elements from p, zero beyond, in pieces where all are there.
template <typename T, int E, int A>
__device__ __forceinline__ void load_cols(const T* p, int n, Cols<T, E>& r) {
  using P = Piece<T, A>;
  if (P::kElements > 1 && n >= E) {
#pragma unroll
    for (int i = 0; i < E; i += P::kElements)
      *reinterpret_cast<typename P::Type*>(&r.v[i]) = __ldg(reinterpret_cast<const typename P::Type*>(p + i));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) r.v[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
}
template <typename T, int E>
__device__ __forceinline__ void widen(const Cols<T, E>& r, float (&f)[E]) {
  unpack<T, E>(*reinterpret_cast<const Packet<T, E>*>(&r), f);
}
template <typename T, int E, int A>
__device__ __forceinline__ void load_cols(const T* p, int n, float (&f)[E]) {
  Cols<T, E> r;
  load_cols<T, E, A>(p, n, r);
  widen<T, E>(r, f);
}
template <typename T, int E>
__device__ __forceinline__ void narrow(const float (&f)[E], Cols<T, E>& r) {
  *reinterpret_cast<Packet<T, E>*>(&r) = pack<T, E>(f);
}
template <typename T, int E, int A>
__device__ __forceinline__ void store_cols(T* p, int n, const Cols<T, E>& r) {
  using P = Piece<T, A>;
  if (P::kElements > 1 && n >= E) {
#pragma unroll
    for (int i = 0; i < E; i += P::kElements)
      *reinterpret_cast<typename P::Type*>(p + i) = *reinterpret_cast<const typename P::Type*>(&r.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) p[i] = r.v[i];
  }
}
template <typename T, int E, int A>
__device__ __forceinline__ void store_cols(T* p, int n, const float (&f)[E]) {
  Cols<T, E> r;
  narrow<T, E>(f, r);
  store_cols<T, E, A>(p, n, r);
}
// The weight's columns: contiguous and aligned in packets, else one by one.
template <int E>
__device__ __forceinline__ void load_weight(const TensorArg& w, int64_t c, int n, float (&f)[E]) {
  if (n >= E && w.s0 == 1 && (reinterpret_cast<uintptr_t>(w.data) & 15) == 0) {
    if (w.dtype == CC1D_FLOAT32) return load_cols<float, E, 4>(static_cast<const float*>(w.data) + c, E, f);
    if constexpr (E == 8) {
      if (w.dtype == CC1D_FLOAT16) return load_cols<__half, E, 8>(static_cast<const __half*>(w.data) + c, E, f);
      return load_cols<__nv_bfloat16, E, 8>(static_cast<const __nv_bfloat16*>(w.data) + c, E, f);
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = i < n ? load_any(w.data, w.dtype, (c + i) * w.s0) : 0.f;
}

// Dropout of N vectors of E columns; c[n] (a multiple of 4) is the first column of vector n.
// What is dropped is not used, NaN or not.
template <int N, int E>
__device__ __forceinline__ void drop_cols(const AddNormArgs& a, uint64_t key, uint64_t stream, int64_t row, const int64_t (&c)[N], float (&f)[N][E]) {
  constexpr int B = E / 4;
  const uint64_t first = static_cast<uint64_t>(row) * static_cast<uint64_t>((a.dim + 3) / 4);
  uint64_t block[N * B];
  uint32_t u[N * B][4];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < B; ++i) block[n * B + i] = first + static_cast<uint64_t>(c[n] / 4 + i);
  philox<N * B>(key, block, stream, u);
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < E; ++i) f[n][i] = u[n * B + i / 4][i & 3] >= a.keep_from ? f[n][i] * a.keep_scale : 0.f;
}
// All VPT vectors of a thread, as many at a time as make 4 Philox blocks.
template <int VPT, int E, int G>
__device__ __forceinline__ void drop_row(const AddNormArgs& a, uint64_t key, uint64_t stream, int64_t row, int g, float (&f)[VPT][E]) {
  constexpr int N = VPT * E <= 16 ? VPT : 16 / E;
#pragma unroll
  for (int v = 0; v < VPT; v += N) {
    int64_t c[N];
    float h[N][E];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      c[n] = static_cast<int64_t>((v + n) * G + g) * E;
#pragma unroll
      for (int i = 0; i < E; ++i) h[n][i] = f[v + n][i];
    }
    if (c[0] >= a.dim) break;
    drop_cols<N, E>(a, key, stream, row, c, h);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < E; ++i) f[v + n][i] = h[n][i];
  }
}

// Sums over the G threads of a row: a warp, or the CTA through shared memory (two buffers, so
// that one barrier is enough).
template <int G, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*scratch)[N][kThreads / 32], int turn) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) scratch[turn & 1][i][threadIdx.x >> 5] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) v[i] += scratch[turn & 1][i][k];
    }
  }
}

template <typename T>
__device__ __forceinline__ T* row_of(const TensorArg& t, int64_t row) { return static_cast<T*>(t.data) + row * t.s0; }

__device__ __forceinline__ int cols_left(int64_t dim, int64_t c) {
  return static_cast<int>(max(static_cast<int64_t>(0), min(dim - c, static_cast<int64_t>(1 << 20))));
}

// CTAs of a kernel that holds `elements` columns in a thread that fit an SM (its registers).
constexpr int fwd_ctas(int elements) { return elements <= 8 ? 5 : elements <= 16 ? 3 : elements <= 32 ? 2 : 1; }
constexpr int bwd_ctas(int elements) { return elements <= 8 ? 3 : elements <= 16 ? 2 : 1; }

template <typename T, typename R, int G, int VPT, int E, int A>
__global__ void __launch_bounds__(kThreads, fwd_ctas(VPT * E)) add_norm_fwd_kernel(const AddNormArgs a) {
  __shared__ float scratch[2][1][kThreads / 32];
  constexpr bool kHeld = VPT * E <= 16;  // the weight stays in registers
  const int g = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / G);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  grid_dependency_wait();
  const uint64_t key = a.rng ? static_cast<uint64_t>(a.rng[0]) : 0, stream = a.rng ? static_cast<uint64_t>(a.rng[a.rng_stride]) : 0;
  Cols<T, E> x[VPT];
  Cols<R, E> res[VPT];
  auto load = [&](int64_t at) {
    if (at >= a.rows) return;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      const int n = cols_left(a.dim, c);
      load_cols<T, E, A>(row_of<T>(a.x, at) + c, n, x[v]);
      if (a.residual.data) load_cols<R, E, A>(row_of<R>(a.residual, at) + c, n, res[v]);
    }
  };
  load(row);
  float held[kHeld ? VPT : 1][E];
  if constexpr (kHeld) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      load_weight<E>(a.weight, c, cols_left(a.dim, c), held[v]);
    }
  }
  for (int turn = 0; row < a.rows; row += step, ++turn) {
    float r[VPT][E];
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      widen<T, E>(x[v], r[v]);
    }
    if (a.rng) drop_row<VPT, E, G>(a, key, stream, row, g, r);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      if (a.residual.data) {
        float f[E];
        widen<R, E>(res[v], f);
#pragma unroll
        for (int i = 0; i < E; ++i) r[v][i] += f[i];
      }
    }
    load(row + step);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      Cols<R, E> stored;
      narrow<R, E>(r[v], stored);
      store_cols<R, E, A>(row_of<R>(a.residual_out, row) + c, cols_left(a.dim, c), stored);
      widen<R, E>(stored, r[v]);
#pragma unroll
      for (int i = 0; i < E; ++i) sum[0] = fmaf(r[v][i], r[v][i], sum[0]);  // columns beyond the row are zero
    }
    row_sum<G, 1>(sum, scratch, turn);
    const float rstd = 1.f / sqrtf(sum[0] / static_cast<float>(a.dim) + a.eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      const int n = cols_left(a.dim, c);
      float w[E];
      if constexpr (kHeld) {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = held[v][i];
      } else {
        load_weight<E>(a.weight, c, n, w);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) w[i] *= r[v][i] * rstd;
      store_cols<T, E, A>(row_of<T>(a.out, row) + c, n, w);
    }
  }
}

// Rows that do not fit the registers: the stored stream is read again for the output.
template <typename T, typename R>
__global__ void __launch_bounds__(kThreads) add_norm_fwd_wide_kernel(const AddNormArgs a) {
  constexpr int E = kWideElements;
  __shared__ float scratch[2][1][kThreads / 32];
  const int64_t row = blockIdx.x;
  grid_dependency_wait();
  const uint64_t key = a.rng ? static_cast<uint64_t>(a.rng[0]) : 0, stream = a.rng ? static_cast<uint64_t>(a.rng[a.rng_stride]) : 0;
  R* const ro = row_of<R>(a.residual_out, row);
  float sum[1] = {0.f};
  for (int64_t c = threadIdx.x * E; c < a.dim; c += kThreads * E) {
    const int n = cols_left(a.dim, c);
    float r[E], res[E];
    load_cols<T, E, 1>(row_of<T>(a.x, row) + c, n, r);
    if (a.rng) drop_cols<1, E>(a, key, stream, row, {c}, reinterpret_cast<float(&)[1][E]>(r));
    if (a.residual.data) load_cols<R, E, 1>(row_of<R>(a.residual, row) + c, n, res);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (a.residual.data) r[i] += res[i];
      r[i] = to_f32(from_f32<R>(r[i]));
      if (i < n) sum[0] = fmaf(r[i], r[i], sum[0]);
    }
    store_cols<R, E, 1>(ro + c, n, r);
  }
  row_sum<kThreads, 1>(sum, scratch, 0);
  const float rstd = 1.f / sqrtf(sum[0] / static_cast<float>(a.dim) + a.eps);
  for (int64_t c = threadIdx.x * E; c < a.dim; c += kThreads * E) {
    const int n = cols_left(a.dim, c);
    float w[E];
    load_weight<E>(a.weight, c, n, w);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) w[i] *= to_f32(ro[c + i]) * rstd;  // this thread's own stores
    store_cols<T, E, 1>(row_of<T>(a.out, row) + c, n, w);
  }
}

// Backward: a CTA takes rows blockIdx.x * rows per CTA + k * rows of the grid and adds up its
// share of dw in registers; the shares go to `partials`, one row of (dim) for each CTA.
template <typename T, typename R, int G, int VPT, int E, int A>
__global__ void __launch_bounds__(kThreads, bwd_ctas(VPT * E)) add_norm_bwd_kernel(const AddNormArgs a) {
  extern __shared__ float shares[];  // G == 32: [warps][columns]
  __shared__ float scratch[2][2][kThreads / 32];
  // dresidual_out, which the sums do not need, is loaded with its own row where two rows of
  // fp32 of it would not fit the registers
  constexpr bool kAhead = sizeof(R) == 2;
  const int g = threadIdx.x % G;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / G);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  grid_dependency_wait();
  const uint64_t key = a.rng ? static_cast<uint64_t>(a.rng[0]) : 0, stream = a.rng ? static_cast<uint64_t>(a.rng[a.rng_stride]) : 0;
  const float inv = 1.f / static_cast<float>(a.dim);
  Cols<R, E> r[VPT], dres[kAhead ? VPT : 1];
  Cols<T, E> dy[VPT];
  auto load = [&](int64_t at) {
    if (at >= a.rows) return;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      const int n = cols_left(a.dim, c);
      load_cols<R, E, A>(row_of<R>(a.residual_out, at) + c, n, r[v]);
      load_cols<T, E, A>(row_of<T>(a.dout, at) + c, a.dout.data ? n : 0, dy[v]);
      if constexpr (kAhead) load_cols<R, E, A>(row_of<R>(a.dresidual_out, at) + c, a.dresidual_out.data ? n : 0, dres[v]);
    }
  };
  load(row);
  float w[VPT][E], dw[VPT][E];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int64_t c = static_cast<int64_t>(v * G + g) * E;
    load_weight<E>(a.weight, c, cols_left(a.dim, c), w[v]);
#pragma unroll
    for (int i = 0; i < E; ++i) dw[v][i] = 0.f;
  }
  for (int turn = 0; row < a.rows; row += step, ++turn) {
    float sum[2] = {0.f, 0.f};  // of r^2 and of q r
    Cols<R, E> rn[VPT], dresn[VPT];
    Cols<T, E> dyn[VPT];
    if constexpr (!kAhead) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int64_t c = static_cast<int64_t>(v * G + g) * E;
        load_cols<R, E, A>(row_of<R>(a.dresidual_out, row) + c, a.dresidual_out.data ? cols_left(a.dim, c) : 0, dresn[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float rf[E], df[E];
      widen<R, E>(rn[v] = r[v], rf);
      widen<T, E>(dyn[v] = dy[v], df);
      if constexpr (kAhead) dresn[v] = dres[v];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        sum[0] = fmaf(rf[i], rf[i], sum[0]);
        sum[1] = fmaf(df[i] * w[v][i], rf[i], sum[1]);
      }
    }
    load(row + step);
    row_sum<G, 2>(sum, scratch, turn);
    const float rstd = 1.f / sqrtf(sum[0] * inv + a.eps);
    const float k = sum[1] * inv * rstd;  // mean(q n)
    float dr[VPT][E];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      float rf[E], df[E];
      widen<R, E>(rn[v], rf);
      widen<T, E>(dyn[v], df);
      widen<R, E>(dresn[v], dr[v]);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float nv = rf[i] * rstd;
        dw[v][i] = fmaf(df[i], nv, dw[v][i]);
        dr[v][i] = fmaf(rstd, fmaf(-nv, k, df[i] * w[v][i]), dr[v][i]);
      }
      if (a.dresidual.data) store_cols<R, E, A>(row_of<R>(a.dresidual, row) + c, cols_left(a.dim, c), dr[v]);
    }
    if (!a.dx.data) continue;
    if (a.rng) drop_row<VPT, E, G>(a, key, stream, row, g, dr);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      store_cols<T, E, A>(row_of<T>(a.dx, row) + c, cols_left(a.dim, c), dr[v]);
    }
  }
  if (!a.dweight) return;
  float* const part = a.partials + static_cast<int64_t>(blockIdx.x) * a.dim;
  if constexpr (G == 32) {
    constexpr int D = 32 * VPT * E;
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < E; ++i) shares[warp * D + (v * 32 + g) * E + i] = dw[v][i];
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < kThreads / 32; ++q) s += shares[q * D + c];
      part[c] = s;
    }
  } else {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int64_t c = static_cast<int64_t>(v * G + g) * E;
      store_cols<float, E, 1>(part + c, cols_left(a.dim, c), dw[v]);
    }
  }
}

// Rows that do not fit the registers: read twice, the share of dw kept in `partials`.
template <typename T, typename R>
__global__ void __launch_bounds__(kThreads) add_norm_bwd_wide_kernel(const AddNormArgs a) {
  constexpr int E = kWideElements;
  __shared__ float scratch[2][2][kThreads / 32];
  grid_dependency_wait();
  const uint64_t key = a.rng ? static_cast<uint64_t>(a.rng[0]) : 0, stream = a.rng ? static_cast<uint64_t>(a.rng[a.rng_stride]) : 0;
  const float inv = 1.f / static_cast<float>(a.dim);
  float* const part = a.dweight ? a.partials + static_cast<int64_t>(blockIdx.x) * a.dim : nullptr;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, ++turn) {
    float sum[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x * E; c < a.dim; c += kThreads * E) {
      const int n = cols_left(a.dim, c);
      float r[E], dy[E], w[E];
      load_cols<R, E, 1>(row_of<R>(a.residual_out, row) + c, n, r);
      load_cols<T, E, 1>(row_of<T>(a.dout, row) + c, a.dout.data ? n : 0, dy);
      load_weight<E>(a.weight, c, n, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        sum[0] = fmaf(r[i], r[i], sum[0]);
        sum[1] = fmaf(dy[i] * w[i], r[i], sum[1]);
      }
    }
    row_sum<kThreads, 2>(sum, scratch, turn);
    const float rstd = 1.f / sqrtf(sum[0] * inv + a.eps);
    const float k = sum[1] * inv * rstd;
    for (int64_t c = threadIdx.x * E; c < a.dim; c += kThreads * E) {
      const int n = cols_left(a.dim, c);
      float r[E], dy[E], w[E], dr[E];
      load_cols<R, E, 1>(row_of<R>(a.residual_out, row) + c, n, r);
      load_cols<T, E, 1>(row_of<T>(a.dout, row) + c, a.dout.data ? n : 0, dy);
      load_cols<R, E, 1>(row_of<R>(a.dresidual_out, row) + c, a.dresidual_out.data ? n : 0, dr);
      load_weight<E>(a.weight, c, n, w);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float nv = r[i] * rstd;
        if (part && i < n) part[c + i] = turn ? fmaf(dy[i], nv, part[c + i]) : dy[i] * nv;
        dr[i] = fmaf(rstd, fmaf(-nv, k, dy[i] * w[i]), dr[i]);
      }
      if (a.dresidual.data) store_cols<R, E, 1>(row_of<R>(a.dresidual, row) + c, n, dr);
      if (a.rng) drop_cols<1, E>(a, key, stream, row, {c}, reinterpret_cast<float(&)[1][E]>(dr));
      if (a.dx.data) store_cols<T, E, 1>(row_of<T>(a.dx, row) + c, n, dr);
    }
  }
}

// Every row of every tensor starts on a multiple of n elements (16 bytes if that is less).
bool rows_start_on(int n, const AddNormArgs& a) {
  const TensorArg* const all[] = {&a.x, &a.residual, &a.out, &a.residual_out, &a.dout, &a.dresidual_out, &a.dx, &a.dresidual};
  for (const TensorArg* t : all) {
    const int64_t size = t->dtype == CC1D_FLOAT32 ? 4 : 2, bytes = n * size < 16 ? n * size : 16;
    if (t->data && (reinterpret_cast<uintptr_t>(t->data) % bytes || (a.rows > 1 && t->s0 * size % bytes))) return false;
  }
  return true;
}

template <typename T, typename R, bool BWD, int G, int VPT, int E, int A>
cudaError_t run(const AddNormArgs& a, cudaStream_t s) {
  if constexpr (BWD) {
    const size_t smem = G == 32 && a.dweight ? kThreads / 32 * 32 * VPT * E * sizeof(float) : 0;
    cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(add_norm_bwd_kernel<T, R, G, VPT, E, A>), smem);
    if (e != cudaSuccess) return e;
    return launch_dependent(add_norm_bwd_kernel<T, R, G, VPT, E, A>, dim3(static_cast<unsigned>(a.ctas)), dim3(kThreads), smem, s, a);
  } else {
    return launch_dependent(add_norm_fwd_kernel<T, R, G, VPT, E, A>, dim3(static_cast<unsigned>(a.ctas)), dim3(kThreads), 0, s, a);
  }
}

template <typename T, typename R, bool BWD, int E, int A>
cudaError_t pick_width(const AddNormArgs& a, cudaStream_t s) {
  constexpr int N = kThreads;
  if (a.group == 32) {
    if (a.held == E) return run<T, R, BWD, 32, 1, E, A>(a, s);
    if (a.held == 2 * E) return run<T, R, BWD, 32, 2, E, A>(a, s);
    return run<T, R, BWD, 32, 4, E, A>(a, s);
  }
  if (a.held == E) return run<T, R, BWD, N, 1, E, A>(a, s);
  if (a.held == 2 * E) return run<T, R, BWD, N, 2, E, A>(a, s);
  if constexpr (!BWD || E == 4) {
    if (a.held == 8 * E) return run<T, R, BWD, N, 8, E, A>(a, s);
  }
  return run<T, R, BWD, N, 4, E, A>(a, s);
}

template <typename T, typename R, bool BWD>
cudaError_t pick(AddNormArgs& a, cudaStream_t s) {
  if (a.group == 0)
    return BWD ? launch_dependent(add_norm_bwd_wide_kernel<T, R>, dim3(static_cast<unsigned>(a.ctas)), dim3(kThreads), 0, s, static_cast<const AddNormArgs&>(a))
               : launch_dependent(add_norm_fwd_wide_kernel<T, R>, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, s, static_cast<const AddNormArgs&>(a));
  if constexpr (sizeof(T) == 2) {
    if (a.aligned == 8) return pick_width<T, R, BWD, 8, 8>(a, s);
  }
  switch (a.aligned) {
    case 4: return pick_width<T, R, BWD, 4, 4>(a, s);
    case 2: return pick_width<T, R, BWD, 4, 2>(a, s);
    default: return pick_width<T, R, BWD, 4, 1>(a, s);
  }
}

}  // namespace

using DT = CC1D_DT_TYPE;

cudaError_t CC1D_DT_NAME(add_norm_fwd)(AddNormArgs& a, cudaStream_t s) {
  return a.residual_out.dtype == CC1D_FLOAT32 ? pick<DT, float, false>(a, s) : pick<DT, DT, false>(a, s);
}
cudaError_t CC1D_DT_NAME(add_norm_bwd)(AddNormArgs& a, cudaStream_t s) {
  cudaError_t e = a.residual_out.dtype == CC1D_FLOAT32 ? pick<DT, float, true>(a, s) : pick<DT, DT, true>(a, s);
  if (e == cudaSuccess && a.dweight) e = sum_rows(a.partials, a.ctas, a.dim, a.dweight, s);
  return e;
}

#if CC1D_DT == 0
void add_norm_plan(AddNormArgs* a, int dtype, int sms, bool bwd) {
  a->aligned = dtype == CC1D_FLOAT32 ? 4 : 8;
  while (a->aligned > 1 && !rows_start_on(a->aligned, *a)) a->aligned /= 2;
  const int e = a->aligned == 8 ? 8 : 4;
  const int64_t steps = (a->dim + e - 1) / e;
  // 64 elements of a thread are too many for the backward's arrays of them
  const int64_t most = (bwd && e == 8 ? 4 : 8) * kThreads;
  a->group = steps <= 128 ? 32 : steps <= most ? kThreads : 0;
  a->held = e;
  while (a->group && a->held / e * a->group < steps) a->held *= 2;
  const int64_t per = a->group == 32 ? kThreads / 32 : 1, need = (a->rows + per - 1) / per;
  const int64_t fit = static_cast<int64_t>(sms) * (a->group == 0 ? 2 : bwd ? bwd_ctas(a->held) : fwd_ctas(a->held));
  a->ctas = need < fit ? need : fit;
}

namespace {
// out[d] = the partial sums of column d added up in a fixed order: 32 columns by 8 warps.
__global__ void __launch_bounds__(kThreads) sum_rows_kernel(const float* __restrict__ partials, int64_t n, int64_t dim, float* out) {
  __shared__ float part[kThreads / 32][32];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t d = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (d < dim) {
#pragma unroll 8
    for (int64_t i = w; i < n; i += kThreads / 32) s += partials[i * dim + d];
  }
  part[w][lane] = s;
  __syncthreads();
  if (w == 0 && d < dim) {
#pragma unroll
    for (int q = 1; q < kThreads / 32; ++q) s += part[q][lane];
    out[d] = s;
  }
}
}  // namespace

cudaError_t sum_rows(const float* partials, int64_t n, int64_t dim, float* out, cudaStream_t s) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((dim + 31) / 32));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sum_rows_kernel, partials, n, dim, out);
}
#endif

}  // namespace cc1d
