// extern "C" launchers of the recurrent-block operators: the gated recurrence, its token
// update, and dropout + residual add + RMSNorm.  Argument checks happen here, before any
// launch; include/causal_conv1d_b200.h states the contract.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "cc1d_block_launch.h"

namespace cc1d {
namespace {

cc1d_status fail(cc1d_status code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
cc1d_status fail(cc1d_status code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  try {
    set_last_error(buf);
  } catch (...) {  // out of memory for the message: the status alone has to do
  }
  return code;
}

cc1d_status launched(cudaError_t e, const char* what, int kernels) {
  if (e != cudaSuccess)
    return fail(CC1D_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  count_launches(kernels);
  return CC1D_OK;
}

bool is_float(int dt) { return dt == CC1D_FLOAT32 || dt == CC1D_FLOAT16 || dt == CC1D_BFLOAT16; }
constexpr int64_t kMax31 = (int64_t{1} << 31) - 1;

// Sizes whose products stay far inside 64 bits, so that the launchers' own arithmetic cannot wrap.
bool sizes_ok(int64_t a, int64_t b, int64_t c) {
  return a >= 0 && b >= 0 && c >= 0 && a <= kMax31 && b <= kMax31 && c <= kMax31 &&
         static_cast<double>(a) * static_cast<double>(b) * static_cast<double>(c) < 4e18;
}

template <typename Args, typename Fn>
cudaError_t by_type(int dtype, Args& a, cudaStream_t s, Fn f32, Fn f16, Fn bf16) {
  switch (dtype) {
    case CC1D_FLOAT32: return f32(a, s);
    case CC1D_FLOAT16: return f16(a, s);
    default: return bf16(a, s);
  }
}

// ------------------------------------------------------------------ recurrence plan
// Unit stride along the layout's dimension, the other strides not negative.
bool strips_ok(const TensorArg& t, const RecArgs& a) {
  if (!t.data) return true;
  const int64_t unit = a.rows ? t.s2 : t.s1, step = a.rows ? t.s1 : t.s2;
  return (unit == 1 || (a.rows ? a.seqlen : a.dim) == 1) && t.s0 >= 0 && ((a.rows ? a.dim : a.seqlen) <= 1 || step >= 0);
}
// Every strip of it starts on a multiple of `bytes`.
bool strips_start_on(int bytes, const TensorArg& t, const RecArgs& a) {
  if (!t.data) return true;
  const int64_t n = bytes / (t.dtype == CC1D_FLOAT32 ? 4 : 2);
  auto step_ok = [&](int64_t s, int64_t extent) { return extent <= 1 || s % n == 0; };
  return reinterpret_cast<uintptr_t>(t.data) % bytes == 0 && step_ok(t.s0, a.batch) &&
         (a.rows ? step_ok(t.s1, a.dim) : step_ok(t.s2, a.seqlen));
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

// How many clusters of a.cluster CTAs (CTAs for 1) of this recurrence's kernel run at a time: the
// driver's answer, asked once per kernel, size and device.
int64_t clusters_at_a_time(RecArgs a, bool bwd) {
  static std::atomic<int> known[64][2][3][5][2][2][2][17];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  const int dt = a.x.dtype;
  std::atomic<int>& slot = known[dev][bwd][dt][a.move][a.rows][a.seq_idx.data != nullptr][a.z.data != nullptr][a.cluster];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    int64_t count = 0;
    a.capacity = &count;
    const cudaError_t e = bwd ? by_type(dt, a, nullptr, rec_bwd_f32, rec_bwd_f16, rec_bwd_bf16) : by_type(dt, a, nullptr, rec_fwd_f32, rec_fwd_f16, rec_fwd_bf16);
    if (e != cudaSuccess) cudaGetLastError();
    n = e == cudaSuccess && count > 0 ? static_cast<int>(count) : -1;
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

// CTAs that share a tile.  Each takes 1/cluster of the chunks, so a long sequence of few
// channels fills the GPU, but the cluster's exchange lengthens every chunk, and clusters that
// do not all run at once take a second wave.  Measured on a B200 with n CTAs on an SM, a chunk
// takes (microseconds, 16-bit, with z)
//
//   forward  .75 + .21 n alone, .74 + .045 cluster + .34 n      backward  .75 + .52 n,
//   .95 + .08 cluster + .42 n
//
// and a CTA about 6 to start.  One sequence of 32768 positions and 5120 channels (80 tiles):
// forward 1010 us alone, 684 in twos, 434 in fours, 363 in fives, 359 in sixes, 424 in eights;
// backward 517 us in fives, 626 in fours, 714 in sixes.  The constants are those of the aligned
// channel-last kernels of 16-bit tensors with z, but serve all.  Swept over every size, packed,
// without z, off 16 bytes and with 16 to 256 tiles, the choice was the fastest or within 1% of it;
// fp32 (1, 2560, 32768) backward takes 435 us in sixes and would take 409 in fives.
int choose_cluster(RecArgs* a, int64_t tiles, bool bwd) {
  const double sms = sm_count();
  double best = 0;
  int pick = 1;
  for (int c = 1; c <= 16 && (c == 1 || c <= a->nchunks); c += c < 8 ? 1 : 8) {
    a->cluster = c;
    const int64_t fit = clusters_at_a_time(*a, bwd);
    if (fit <= 0) {
      if (c == 1) return 1;
      continue;
    }
    const double rounds = static_cast<double>((a->nchunks + c - 1) / c);
    auto wave = [&](int64_t clusters) {
      const double n = std::max(1.0, static_cast<double>(clusters * c) / sms);
      const double t = c == 1 ? .75 + (bwd ? .52 : .21) * n : bwd ? .95 + .08 * c + .42 * n : .74 + .045 * c + .34 * n;
      return 6.0 + rounds * t;
    };
    const double cost = static_cast<double>(tiles / fit) * wave(fit) + (tiles % fit ? wave(tiles % fit) : 0.0);
    if (c == 1 || cost < best) {
      best = cost;
      pick = c;
    }
  }
  return pick;
}

// Layout, way of moving and cluster of a recurrence.  Rows: every tensor has unit stride along
// the sequence; all others take the channel-last kernel.  The first of the ways that the tensors
// allow is the fastest; bf16, 8 sequences of 8192, forward and backward: 408 and 718 us for
// 4096 channels (kTma), 659 and 1248 us for 4094 (kWords), 752 and 1400 us for 4095 (kHalves),
// 768 and 1586 us with an offset for each input (kOwn).
cc1d_status rec_plan(RecArgs* a, bool bwd) {
  TensorArg* const all[] = {&a->x, &a->gate, &a->z, bwd ? &a->dout : &a->out, bwd ? &a->dx : nullptr,
                            bwd ? &a->dgate : nullptr, bwd ? &a->dz : nullptr};
  bool last = true, rows = true;
  for (const TensorArg* t : all) {
    if (!t || !t->data) continue;
    last = last && (t->s1 == 1 || a->dim == 1);
    rows = rows && (t->s2 == 1 || a->seqlen == 1);
  }
  a->rows = rows && (!last || a->dim == 1);
  bool strips = true, packets = true, words = true, alike = true;
  for (TensorArg* t : all) {
    if (!t) continue;
    // The stride of an extent of one may be anything, also one that is not checked below; tiles
    // reach past such an extent, and where their strips start has to keep to the same rule.
    if (a->batch <= 1) t->s0 = 0;
    if (a->dim <= 1) t->s1 = 0;
    if (a->seqlen <= 1) t->s2 = 0;
    strips = strips && strips_ok(*t, *a);
    packets = packets && strips_start_on(16, *t, *a);
    words = words && strips_start_on(4, *t, *a);
    if (t->data && (t == &a->gate || t == &a->z || t == &a->dout))
      alike = alike && t->s0 == a->x.s0 && t->s1 == a->x.s1 && t->s2 == a->x.s2;
    if (t->data && (t == &a->x || t == &a->gate || t == &a->z || t == &a->dout))
      alike = alike && reinterpret_cast<uintptr_t>(t->data) % 16 == 0;
  }
  a->move = !strips ? kElements : packets ? kTma : !alike ? kOwn : words ? kWords : kHalves;
  const int64_t channels = a->x.dtype == CC1D_FLOAT32 ? 32 : 64;
  a->dtiles = (a->dim + channels - 1) / channels;
  const int64_t tiles = a->batch * a->dtiles;
  a->cluster = choose_cluster(a, tiles, bwd);
  if (tiles * a->cluster > kMax31) return fail(CC1D_ERR_VALUE, "batch * dim is too large");
  return CC1D_OK;
}

int64_t rec_partial_bytes(const RecArgs& a) {
  return a.batch * a.cluster * a.dim * static_cast<int64_t>(sizeof(float));
}

#define CC1D_REQUIRE(t, name) \
  if (!(t).data) return fail(CC1D_ERR_VALUE, "%s is required", name)
#define CC1D_SAME_TYPE(t, name)                            \
  if ((t).data && (t).dtype != p->x.dtype) return fail(CC1D_ERR_TYPE, "%s must have x's dtype", name)
#define CC1D_FP32(t, name) \
  if ((t).data && (t).dtype != CC1D_FLOAT32) return fail(CC1D_ERR_TYPE, "%s must be float32", name)

cc1d_status rec_check(const cc1d_recurrence_params* p, bool bwd, RecArgs* a) {
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  const int64_t B = p->batch, D = p->dim, L = p->seqlen, N = p->nstates;
  if (!sizes_ok(B, D, L) || !sizes_ok(N, D, 1))
    return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  if (!is_float(p->x.dtype)) return fail(CC1D_ERR_TYPE, "x must be float32, float16 or bfloat16");
  CC1D_SAME_TYPE(p->gate, "gate");
  CC1D_SAME_TYPE(p->z, "z");
  if (p->bias.data && !is_float(p->bias.dtype)) return fail(CC1D_ERR_TYPE, "bias must be a float tensor");
  if (p->seq_idx.data && p->seq_idx.dtype != CC1D_INT32) return fail(CC1D_ERR_TYPE, "seq_idx must be int32");
  CC1D_FP32(p->initial_states, "initial_states");
  if (!p->seq_idx.data && (p->initial_states.data || p->final_states.data || p->dfinal_states.data ||
                           p->dinitial_states.data) && N != B)
    return fail(CC1D_ERR_VALUE, "without seq_idx there is one state for each batch row");
  if (!bwd) {
    CC1D_SAME_TYPE(p->out, "out");
    CC1D_FP32(p->final_states, "final_states");
  } else {
    CC1D_SAME_TYPE(p->dout, "dout");
    CC1D_SAME_TYPE(p->dx, "dx");
    CC1D_SAME_TYPE(p->dgate, "dgate");
    CC1D_SAME_TYPE(p->dz, "dz");
    CC1D_FP32(p->dfinal_states, "dfinal_states");
    CC1D_FP32(p->dinitial_states, "dinitial_states");
  }
  if (B > 0 && D > 0 && L > 0) {
    CC1D_REQUIRE(p->x, "x");
    CC1D_REQUIRE(p->gate, "gate");
    if (!bwd) {
      CC1D_REQUIRE(p->out, "out");
    } else {
      CC1D_REQUIRE(p->dout, "dout");
      CC1D_REQUIRE(p->dx, "dx");
      CC1D_REQUIRE(p->dgate, "dgate");
      if (p->z.data) CC1D_REQUIRE(p->dz, "dz");
      if (!p->checkpoints) return fail(CC1D_ERR_VALUE, "checkpoints are required");
    }
  }
  a->batch = B;
  a->dim = D;
  a->seqlen = L;
  a->nstates = N;
  a->nchunks = (L + kRecChunk - 1) / kRecChunk;
  a->x = tensor_arg(p->x);
  a->gate = tensor_arg(p->gate);
  a->z = tensor_arg(p->z);
  a->bias = tensor_arg(p->bias);
  a->seq_idx = tensor_arg(p->seq_idx);
  a->init = tensor_arg(p->initial_states);
  a->final_states = bwd ? TensorArg{} : tensor_arg(p->final_states);
  a->out = tensor_arg(p->out);
  a->dout = tensor_arg(p->dout);
  a->dfinal = tensor_arg(p->dfinal_states);
  a->dx = tensor_arg(p->dx);
  a->dgate = tensor_arg(p->dgate);
  a->dz = tensor_arg(p->dz);
  a->dinit = tensor_arg(p->dinitial_states);
  a->dbias = bwd ? p->dbias : nullptr;
  a->checkpoints = p->checkpoints;
  a->partials = static_cast<float*>(p->workspace);
  return CC1D_OK;
}

cc1d_status add_norm_check(const cc1d_add_norm_params* p, bool bwd, AddNormArgs* a) {
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  if (!sizes_ok(p->rows, p->dim, 1)) return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  if (!is_float(p->x.dtype)) return fail(CC1D_ERR_TYPE, "x must be float32, float16 or bfloat16");
  const int rt = p->residual_out.dtype;
  if (rt != p->x.dtype && rt != CC1D_FLOAT32)
    return fail(CC1D_ERR_TYPE, "residual_out must have x's dtype or be float32");
  if (!is_float(p->weight.dtype)) return fail(CC1D_ERR_TYPE, "weight must be a float tensor");
  if (!(p->dropout_p >= 0.0 && p->dropout_p < 1.0)) return fail(CC1D_ERR_VALUE, "dropout_p must be in [0, 1)");
  if (!(p->eps >= 0.0)) return fail(CC1D_ERR_VALUE, "eps must be >= 0");
  if (p->rng_state.data && p->rng_state.dtype != CC1D_INT64) return fail(CC1D_ERR_TYPE, "rng_state must be int64");
  if (p->dropout_p > 0.0) CC1D_REQUIRE(p->rng_state, "rng_state");
  const struct { const cc1d_tensor& t; const char* name; bool stream; } all[] = {
      {p->x, "x", false},       {p->residual, "residual", true},           {p->out, "out", false},
      {p->residual_out, "residual_out", true}, {p->dout, "dout", false}, {p->dresidual_out, "dresidual_out", true},
      {p->dx, "dx", false},     {p->dresidual, "dresidual", true}};
  for (const auto& e : all) {
    if (!e.t.data) continue;
    if (e.t.dtype != (e.stream ? rt : p->x.dtype))
      return fail(CC1D_ERR_TYPE, "%s must have %s dtype", e.name, e.stream ? "residual_out's" : "x's");
    if (p->dim > 1 && e.t.stride[1] != 1) return fail(CC1D_ERR_VALUE, "%s must have channel stride 1", e.name);
  }
  if (p->rows > 0 && p->dim > 0) {
    CC1D_REQUIRE(p->weight, "weight");
    CC1D_REQUIRE(p->residual_out, "residual_out");
    if (!bwd) {
      CC1D_REQUIRE(p->x, "x");
      CC1D_REQUIRE(p->out, "out");
    }
  }
  a->rows = p->rows;
  a->dim = p->dim;
  a->x = tensor_arg(p->x);
  a->residual = tensor_arg(p->residual);
  a->weight = tensor_arg(p->weight);
  a->out = tensor_arg(p->out);
  a->residual_out = tensor_arg(p->residual_out);
  a->dout = tensor_arg(p->dout);
  a->dresidual_out = tensor_arg(p->dresidual_out);
  a->dx = tensor_arg(p->dx);
  a->dresidual = tensor_arg(p->dresidual);
  a->rng = p->dropout_p > 0.0 ? static_cast<const int64_t*>(p->rng_state.data) : nullptr;
  a->rng_stride = p->rng_state.stride[0];
  a->dweight = p->dweight;
  a->partials = static_cast<float*>(p->workspace);
  a->eps = static_cast<float>(p->eps);
  a->keep_scale = static_cast<float>(1.0 / (1.0 - p->dropout_p));
  a->keep_from = static_cast<unsigned>(p->dropout_p * 4294967296.0);
  if (p->rows > 0 && p->dim > 0) add_norm_plan(a, p->x.dtype, sm_count(), bwd);
  return CC1D_OK;
}

cc1d_status workspace_ok(const void* ws, int64_t bytes, int64_t need) {
  if (need > 0 && (!ws || bytes < need))
    return fail(CC1D_ERR_VALUE, "workspace too small: %lld bytes needed", (long long)need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & 15u)) return fail(CC1D_ERR_VALUE, "workspace must be 16-byte aligned");
  return CC1D_OK;
}

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

cc1d_status cc1d_recurrence_fwd_launch(const cc1d_recurrence_params* p, void* stream) {
  set_last_error("");
  RecArgs a;
  cc1d_status st = rec_check(p, false, &a);
  if (st != CC1D_OK || a.batch == 0 || a.dim == 0 || a.seqlen == 0) return st;
  if ((st = rec_plan(&a, false)) != CC1D_OK) return st;
  return launched(by_type(p->x.dtype, a, static_cast<cudaStream_t>(stream), rec_fwd_f32, rec_fwd_f16, rec_fwd_bf16),
                  "gated recurrence forward launch", 1);
}

int64_t cc1d_recurrence_bwd_workspace_bytes(const cc1d_recurrence_params* p) {
  set_last_error("");
  RecArgs a;
  if (rec_check(p, true, &a) != CC1D_OK) return -1;
  if (a.batch == 0 || a.dim == 0 || a.seqlen == 0 || !a.dbias) return 0;
  return rec_plan(&a, true) == CC1D_OK ? rec_partial_bytes(a) : -1;
}

cc1d_status cc1d_recurrence_bwd_launch(const cc1d_recurrence_params* p, void* stream) {
  set_last_error("");
  RecArgs a;
  cc1d_status st = rec_check(p, true, &a);
  if (st != CC1D_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.batch == 0 || a.dim == 0 || a.seqlen == 0) {
    if (!a.dbias || a.dim == 0) return CC1D_OK;
    return launched(cudaMemsetAsync(a.dbias, 0, a.dim * sizeof(float), s), "gated recurrence zero fill", 0);
  }
  if ((st = rec_plan(&a, true)) != CC1D_OK) return st;
  if (a.dbias && (st = workspace_ok(p->workspace, p->workspace_bytes, rec_partial_bytes(a))) != CC1D_OK) return st;
  return launched(by_type(p->x.dtype, a, s, rec_bwd_f32, rec_bwd_f16, rec_bwd_bf16), "gated recurrence backward launch",
                  a.dbias ? 2 : 1);
}

cc1d_status cc1d_recurrence_update_launch(const cc1d_recurrence_update_params* p, void* stream) {
  set_last_error("");
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  const int64_t B = p->batch, D = p->dim, T = p->seqlen, N = p->nstates;
  if (!sizes_ok(B, D, T) || !sizes_ok(N, D, 1)) return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  if (!is_float(p->x.dtype)) return fail(CC1D_ERR_TYPE, "x must be float32, float16 or bfloat16");
  CC1D_SAME_TYPE(p->gate, "gate");
  CC1D_SAME_TYPE(p->z, "z");
  CC1D_SAME_TYPE(p->out, "out");
  if (p->bias.data && !is_float(p->bias.dtype)) return fail(CC1D_ERR_TYPE, "bias must be a float tensor");
  CC1D_FP32(p->state, "state");
  if (p->state_indices.data && p->state_indices.dtype != CC1D_INT32)
    return fail(CC1D_ERR_TYPE, "state_indices must be int32");
  if (!p->state_indices.data && N != B) return fail(CC1D_ERR_VALUE, "without state_indices there is one state for each batch row");
  if (B == 0 || D == 0 || T == 0) return CC1D_OK;
  CC1D_REQUIRE(p->x, "x");
  CC1D_REQUIRE(p->gate, "gate");
  CC1D_REQUIRE(p->out, "out");
  if (N > 0) CC1D_REQUIRE(p->state, "state");
  if (B * D > kMax31 * 256) return fail(CC1D_ERR_VALUE, "batch * dim is too large");
  RecUpdateArgs a;
  a.batch = B;
  a.dim = D;
  a.seqlen = T;
  a.nstates = N;
  a.x = tensor_arg(p->x);
  a.gate = tensor_arg(p->gate);
  a.z = tensor_arg(p->z);
  a.bias = tensor_arg(p->bias);
  a.state = tensor_arg(p->state);
  a.out = tensor_arg(p->out);
  a.indices = static_cast<const int32_t*>(p->state_indices.data);
  a.indices_stride = p->state_indices.stride[0];
  return launched(by_type(p->x.dtype, a, static_cast<cudaStream_t>(stream), rec_update_f32, rec_update_f16, rec_update_bf16),
                  "gated recurrence update launch", 1);
}

cc1d_status cc1d_add_norm_fwd_launch(const cc1d_add_norm_params* p, void* stream) {
  set_last_error("");
  AddNormArgs a;
  const cc1d_status st = add_norm_check(p, false, &a);
  if (st != CC1D_OK || a.rows == 0 || a.dim == 0) return st;
  return launched(by_type(p->x.dtype, a, static_cast<cudaStream_t>(stream), add_norm_fwd_f32, add_norm_fwd_f16, add_norm_fwd_bf16),
                  "dropout_add_rms_norm forward launch", 1);
}

int64_t cc1d_add_norm_bwd_workspace_bytes(const cc1d_add_norm_params* p) {
  set_last_error("");
  AddNormArgs a;
  if (add_norm_check(p, true, &a) != CC1D_OK) return -1;
  if (a.rows == 0 || a.dim == 0 || !a.dweight) return 0;
  return a.ctas * a.dim * static_cast<int64_t>(sizeof(float));
}

cc1d_status cc1d_add_norm_bwd_launch(const cc1d_add_norm_params* p, void* stream) {
  set_last_error("");
  AddNormArgs a;
  cc1d_status st = add_norm_check(p, true, &a);
  if (st != CC1D_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.rows == 0 || a.dim == 0) {
    if (!a.dweight || a.dim == 0) return CC1D_OK;
    return launched(cudaMemsetAsync(a.dweight, 0, a.dim * sizeof(float), s), "dropout_add_rms_norm zero fill", 0);
  }
  if (a.dweight) {
    st = workspace_ok(p->workspace, p->workspace_bytes, a.ctas * a.dim * static_cast<int64_t>(sizeof(float)));
    if (st != CC1D_OK) return st;
  }
  return launched(by_type(p->x.dtype, a, s, add_norm_bwd_f32, add_norm_bwd_f16, add_norm_bwd_bf16),
                  "dropout_add_rms_norm backward launch", a.dweight ? 2 : 1);
}

}  // extern "C"
