// The selective recurrence for a few tokens of each row against a pool of fp32 states (sm_100a).
//
// LANES threads share a channel of one batch row; each takes VEC * 4 of its states through the
// row's tokens, from the state it reads to the one it writes back, and the output is summed over
// the threads by exchanges.  A state is read and written once; it is most of what moves.
#include "cc1d_selective.cuh"

namespace cc1d {
namespace {

// PACKED: states, A, B and C lie densely along dstate, a multiple of 4, and on 16 bytes (16-bit: 8).
template <typename T, bool PACKED>
__device__ __forceinline__ Four load_inputs(const TensorArg& t, int64_t group_stride, int64_t b, int64_t g, int64_t n0, int64_t l, int64_t dstate) {
  const T* p = static_cast<const T*>(t.data) + b * t.s0 + g * group_stride + l * t.s2;
  float f[4];
  if constexpr (PACKED) {
    unpack<T, 4>(ld_packet<T, 4>(p + n0), f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = n0 + i < dstate ? to_f32(p[(n0 + i) * t.s1]) : 0.f;
  }
  return Four{make_float2(f[0], f[1]), make_float2(f[2], f[3])};
}

// Channel d of batch row b.  Every thread of a warp comes here.
template <typename T, int LANES, int VEC, bool PACKED>
__device__ __forceinline__ void update_row(const SelUpdateArgs& a, int64_t b, int64_t d, int sl) {
  const bool mine = d < a.dim;
  const int64_t row = !mine ? -1 : a.indices ? a.indices[b * a.indices_stride] : b;
  const int64_t g = a.groups == 1 ? 0 : static_cast<uint32_t>(d) / static_cast<uint32_t>(a.dim / a.groups);
  const bool live = row >= 0 && row < a.nstates;
  Four h[VEC], rate[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const int64_t n0 = (v * LANES + sl) * 4;
    h[v] = rate[v] = zero4();
    if (!live || n0 >= a.dstate) continue;
    if constexpr (PACKED) {
      h[v] = of4(*reinterpret_cast<const float4*>(static_cast<const float*>(a.state.data) + row * a.state.s0 + d * a.state.s1 + n0));
      rate[v] = of4(*reinterpret_cast<const float4*>(static_cast<const float*>(a.A.data) + d * a.A.s0 + n0));
      rate[v].lo = fmul2(rate[v].lo, both(kLog2e));
      rate[v].hi = fmul2(rate[v].hi, both(kLog2e));
    } else {
      h[v] = of4(load_state(a.state, row, d, n0, a.dstate));
      rate[v] = of4(load_rates(a.A, d, n0, a.dstate));
    }
  }
  const float bias = live && a.bias.data ? load_any(a.bias.data, a.bias.dtype, d * a.bias.s0) : 0.f;
  const float skip = live && a.D.data ? load_any(a.D.data, a.D.dtype, d * a.D.s0) : 0.f;
  for (int64_t l = 0; l < a.seqlen; ++l) {
    float y = 0.f, x = 0.f;
    if (live) {
      x = load_el<T>(a.x, b, d, l);
      float step = load_el<T>(a.delta, b, d, l) + bias;
      if (a.softplus) step = step_size<T>(step);
      const float2 s = both(step), sx = both(step * x);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const int64_t n0 = (v * LANES + sl) * 4;
        if (n0 >= a.dstate) continue;
        const Four B = load_inputs<T, PACKED>(a.B, a.B_group, b, g, n0, l, a.dstate);
        const Four C = load_inputs<T, PACKED>(a.C, a.C_group, b, g, n0, l, a.dstate);
        h[v].lo = ffma2(decays(s, rate[v].lo), h[v].lo, fmul2(B.lo, sx));
        h[v].hi = ffma2(decays(s, rate[v].hi), h[v].hi, fmul2(B.hi, sx));
        const float2 sum = ffma2(C.hi, h[v].hi, fmul2(C.lo, h[v].lo));
        y += sum.x + sum.y;
      }
    }
#pragma unroll
    for (int bit = 1; bit < LANES; bit *= 2) y += __shfl_xor_sync(~0u, y, bit);
    if (!mine || sl != 0) continue;
    if (live) {
      y = fmaf(skip, x, y);
      if (a.z.data) y *= silu_of<T>(load_el<T>(a.z, b, d, l));
    }
    store_el<T>(a.out, b, d, l, live ? y : 0.f);
  }
  if (!live) return;
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const int64_t n0 = (v * LANES + sl) * 4;
    if (n0 >= a.dstate) continue;
    if constexpr (PACKED) *reinterpret_cast<float4*>(static_cast<float*>(a.state.data) + row * a.state.s0 + d * a.state.s1 + n0) = to4(h[v]);
    else store_state(a.state, row, d, n0, a.dstate, to4(h[v]));
  }
}

template <typename T, int LANES, int VEC, bool PACKED>
__global__ void __launch_bounds__(kThreads) sel_update_kernel(const __grid_constant__ SelUpdateArgs a) {
  const int sl = threadIdx.x % LANES;
  const int64_t d = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  grid_dependency_wait();
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) update_row<T, LANES, VEC, PACKED>(a, b, d, sl);
}

// One token of rows whose states are packed: the threads of a channel take it through four batch
// rows.  All loads of states, B and C come first; what belongs to a row and channel (step size, output
// gate, output) is one thread's work for each row, and goes to the others by exchanges.
// (128, 8192, 16) bf16 in a pool of 160 rows moves 143 MB (22 us at the copy's rate) in 34 us where no state
// lies in L2: a thread's loads are on their way once, and DRAM is busy a third of the time.  Again and again
// on the same states, part of which L2 holds, it takes 25 us; there, with the step sizes, gates and outputs
// made by every thread it took 40 us, bound by its instructions, and without the packets and rows in
// flight 66 us.  In that form two rows a thread took 42 us with cold
// states, four 43, eight 49; four rows give each thread of four (16 states) one row's scalars.
constexpr int kRows = 4;

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads) sel_step_kernel(const __grid_constant__ SelUpdateArgs a) {
  constexpr int OWN = kSums<LANES>;  // rows of a thread
  const int sl = threadIdx.x % LANES, own = first_sum<LANES>(sl), quad0 = (threadIdx.x & 31) - sl;
  const uint32_t d = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int n0 = sl * 4;
  const bool mine = d < a.dim, has = mine && n0 < a.dstate;
  grid_dependency_wait();
  auto times = [](uint32_t n, int64_t stride) { return static_cast<int64_t>(static_cast<uint64_t>(n) * static_cast<uint32_t>(stride)); };
  const uint32_t g = a.groups == 1 ? 0 : d / static_cast<uint32_t>(a.dim / a.groups);
  const int64_t b0 = static_cast<int64_t>(blockIdx.y) * kRows;
  const int rows = a.batch - b0 < kRows ? static_cast<int>(a.batch - b0) : kRows;
  int row[kRows];
  float4 h[kRows];
  uint2 B[kRows][sizeof(T) / 2], C[kRows][sizeof(T) / 2];  // words until they are used
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    row[r] = r >= rows ? -1 : a.indices ? a.indices[(b0 + r) * a.indices_stride] : static_cast<int>(b0 + r);
    if (row[r] >= a.nstates) row[r] = -1;
  }
  float* const state = static_cast<float*>(a.state.data) + times(d, a.state.s1) + n0;
  const T* const pb = static_cast<const T*>(a.B.data) + b0 * a.B.s0 + g * a.B_group + n0;
  const T* const pc = static_cast<const T*>(a.C.data) + b0 * a.C.s0 + g * a.C_group + n0;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (row[r] < 0 || !has) continue;
    h[r] = *reinterpret_cast<const float4*>(state + times(row[r], a.state.s0));
#pragma unroll
    for (int w = 0; w < sizeof(T) / 2; ++w) {
      B[r][w] = reinterpret_cast<const uint2*>(pb + r * a.B.s0)[w];
      C[r][w] = reinterpret_cast<const uint2*>(pc + r * a.C.s0)[w];
    }
  }
  float x[OWN], z[OWN], s[OWN], sx[OWN];
  float bias = 0.f, skip = 0.f;
  if (mine && a.bias.data) bias = load_any(a.bias.data, a.bias.dtype, d * a.bias.s0);
  if (mine && a.D.data) skip = load_any(a.D.data, a.D.dtype, d * a.D.s0);
#pragma unroll
  for (int j = 0; j < OWN; ++j) {
    const int64_t b = b0 + own + j;
    x[j] = z[j] = s[j] = 0.f;
    if (mine && own + j < rows) {
      x[j] = to_f32((static_cast<const T*>(a.x.data) + b * a.x.s0)[times(d, a.x.s1)]);
      s[j] = to_f32((static_cast<const T*>(a.delta.data) + b * a.delta.s0)[times(d, a.delta.s1)]) + bias;
      if (a.z.data) z[j] = to_f32((static_cast<const T*>(a.z.data) + b * a.z.s0)[times(d, a.z.s1)]);
    }
    if (a.softplus) s[j] = step_size<T>(s[j]);
    sx[j] = s[j] * x[j];
  }
  Four rate = zero4();
  if (has) {
    rate = of4(*reinterpret_cast<const float4*>(static_cast<const float*>(a.A.data) + times(d, a.A.s0) + n0));
    rate.lo = fmul2(rate.lo, both(kLog2e));
    rate.hi = fmul2(rate.hi, both(kLog2e));
  }
  float y[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int from = quad0 + (LANES >= 4 ? r : r / OWN);
    const float2 sr = both(__shfl_sync(~0u, s[r % OWN], from)), sxr = both(__shfl_sync(~0u, sx[r % OWN], from));
    y[r] = 0.f;
    if (row[r] < 0 || !has) continue;
    float vb[4], vc[4];
    unpack<T, 4>(*reinterpret_cast<const Packet<T, 4>*>(&B[r]), vb);
    unpack<T, 4>(*reinterpret_cast<const Packet<T, 4>*>(&C[r]), vc);
    Four f = of4(h[r]);
    f.lo = ffma2(decays(sr, rate.lo), f.lo, fmul2(make_float2(vb[0], vb[1]), sxr));
    f.hi = ffma2(decays(sr, rate.hi), f.hi, fmul2(make_float2(vb[2], vb[3]), sxr));
    *reinterpret_cast<float4*>(state + times(row[r], a.state.s0)) = to4(f);
    const float2 sum = ffma2(make_float2(vc[2], vc[3]), f.hi, fmul2(make_float2(vc[0], vc[1]), f.lo));
    y[r] = sum.x + sum.y;
  }
  sum_lanes<LANES>(y, sl);
#pragma unroll
  for (int j = 0; j < OWN; ++j) {
    if (!mine || sl >= 4 || own + j >= rows) continue;
    bool live = false;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (r == own + j) live = row[r] >= 0;
    float o = fmaf(skip, x[j], y[j]);
    if (a.z.data) o *= silu_of<T>(z[j]);
    (static_cast<T*>(a.out.data) + (b0 + own + j) * a.out.s0)[times(d, a.out.s1)] = from_f32<T>(live ? o : 0.f);
  }
}

// Strides that are multiplied by a channel or a state's row, which 32 bits hold.
bool thin(const SelUpdateArgs& a) {
  for (int64_t s : {a.x.s1, a.delta.s1, a.z.s1, a.out.s1, a.state.s1, a.state.s0, a.A.s0})
    if (s < 0 || s >= int64_t{1} << 32) return false;
  return true;
}

// Packets of four states are legal.
bool packed(const SelUpdateArgs& a) {
  if (a.dstate % 4) return false;
  auto on = [](const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
  auto step = [](int64_t s, int64_t extent) { return extent <= 1 || s % 4 == 0; };
  if (a.state.s2 != 1 || !on(a.state.data, 16) || !step(a.state.s0, a.nstates) || !step(a.state.s1, a.dim)) return false;
  if (a.A.dtype != CC1D_FLOAT32 || a.A.s1 != 1 || !on(a.A.data, 16) || !step(a.A.s0, a.dim)) return false;
  const uintptr_t bytes = a.x.dtype == CC1D_FLOAT32 ? 16 : 8;
  const struct { const TensorArg& t; int64_t group; } both[] = {{a.B, a.B_group}, {a.C, a.C_group}};
  for (const auto& e : both)
    if (e.t.s1 != 1 || !on(e.t.data, bytes) || !step(e.t.s0, a.batch) || !step(e.group, a.groups) || !step(e.t.s2, a.seqlen)) return false;
  return true;
}

template <typename T, int LANES, int VEC>
cudaError_t run(const SelUpdateArgs& a, cudaStream_t s) {
  const int64_t per = kThreads / LANES;
  const dim3 grid(static_cast<unsigned>((a.dim + per - 1) / per), static_cast<unsigned>(a.batch < 65535 ? a.batch : 65535));
  if constexpr (VEC == 1)
    if (a.seqlen == 1 && packed(a) && thin(a) && a.batch <= 65535 * kRows)
      return launch_dependent(sel_step_kernel<T, LANES>, dim3(grid.x, static_cast<unsigned>((a.batch + kRows - 1) / kRows)), dim3(kThreads), 0, s, a);
  return packed(a) ? launch_dependent(sel_update_kernel<T, LANES, VEC, true>, grid, dim3(kThreads), 0, s, a)
                   : launch_dependent(sel_update_kernel<T, LANES, VEC, false>, grid, dim3(kThreads), 0, s, a);
}

}  // namespace

cudaError_t CC1D_DT_NAME(sel_update)(const SelUpdateArgs& a, cudaStream_t s) {
  using T = CC1D_DT_TYPE;
  return a.dstate <= 4    ? run<T, 1, 1>(a, s)
         : a.dstate <= 8  ? run<T, 2, 1>(a, s)
         : a.dstate <= 16 ? run<T, 4, 1>(a, s)
         : a.dstate <= 32 ? run<T, 8, 1>(a, s)
         : a.dstate <= 64 ? run<T, 16, 1>(a, s)
         : a.dstate <= 128 ? run<T, 32, 1>(a, s)
                           : run<T, 32, 2>(a, s);
}

}  // namespace cc1d
