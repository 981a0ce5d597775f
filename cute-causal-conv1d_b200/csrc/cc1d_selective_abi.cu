// extern "C" launchers of the selective recurrence and of its token update.  Argument checks
// happen here, before any launch; include/causal_conv1d_b200.h states the contract.
#include <algorithm>

#include "cc1d_check.h"
#include "cc1d_selective_launch.h"

namespace cc1d {
namespace {

template <typename Args, typename Fn>
cudaError_t by_type(int dtype, const Args& a, cudaStream_t s, Fn f32, Fn f16, Fn bf16) {
  switch (dtype) {
    case CC1D_FLOAT32: return f32(a, s);
    case CC1D_FLOAT16: return f16(a, s);
    default: return bf16(a, s);
  }
}

constexpr int64_t kMostStates = CC1D_SELECTIVE_MAX_STATES;

// What the sequence and the token form have in common.  p: either params struct.
template <typename P>
cc1d_status check_common(const P* p) {
  const int64_t B = p->batch, D = p->dim, L = p->seqlen, N = p->dstate, G = p->groups;
  if (!sizes_ok(B, D, L) || !sizes_ok(p->nstates, D, N) || !sizes_ok(B, L, N) || !sizes_ok(B, G, 1))
    return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  if (N < 1 || N > kMostStates) return fail(CC1D_ERR_VALUE, "dstate must be in [1, %lld]", (long long)kMostStates);
  if (G < 1 || D % G) return fail(CC1D_ERR_VALUE, "dim must be a multiple of groups");
  if (!is_float(p->x.dtype)) return fail(CC1D_ERR_TYPE, "x must be float32, float16 or bfloat16");
  CC1D_SAME_TYPE(p->delta, "delta");
  CC1D_SAME_TYPE(p->B, "B");
  CC1D_SAME_TYPE(p->C, "C");
  CC1D_SAME_TYPE(p->z, "z");
  CC1D_FLOAT(p->A, "A");
  CC1D_FLOAT(p->D, "D");
  CC1D_FLOAT(p->bias, "delta_bias");
  return CC1D_OK;
}

// The elements of a tensor that is written lie at places of their own, each dimension beyond the reach
// of those with smaller strides.
bool apart(const cc1d_tensor& t, int64_t n0, int64_t n1, int64_t n2) {
  struct { int64_t size, step; } d[3] = {{n0, t.stride[0]}, {n1, t.stride[1]}, {n2, t.stride[2]}};
  std::sort(d, d + 3, [](const auto& a, const auto& b) { return a.step < b.step; });
  int64_t reach = 1;
  for (const auto& e : d) {
    if (e.size <= 1) continue;
    if (e.step < reach) return false;
    reach += e.step * (e.size - 1);  // up to the last element
  }
  return true;
}

cc1d_status check(const cc1d_selective_params* p, bool bwd, SelArgs* a) {
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  const cc1d_status st = check_common(p);
  if (st != CC1D_OK) return st;
  if (p->seq_idx.data && p->seq_idx.dtype != CC1D_INT32) return fail(CC1D_ERR_TYPE, "seq_idx must be int32");
  CC1D_FP32(p->initial_states, "initial_states");
  if (!p->seq_idx.data && (p->initial_states.data || p->final_states.data || p->dfinal_states.data ||
                           p->dinitial_states.data) && p->nstates != p->batch)
    return fail(CC1D_ERR_VALUE, "without seq_idx there is one state for each batch row");
  if (!bwd) {
    CC1D_SAME_TYPE(p->out, "out");
    CC1D_FP32(p->final_states, "final_states");
  } else {
    CC1D_SAME_TYPE(p->dout, "dout");
    CC1D_SAME_TYPE(p->dx, "dx");
    CC1D_SAME_TYPE(p->ddelta, "ddelta");
    CC1D_SAME_TYPE(p->dB, "dB");
    CC1D_SAME_TYPE(p->dC, "dC");
    CC1D_SAME_TYPE(p->dz, "dz");
    CC1D_FP32(p->dfinal_states, "dfinal_states");
    CC1D_FP32(p->dinitial_states, "dinitial_states");
  }
  if (p->batch > 0 && p->dim > 0 && p->seqlen > 0) {
    CC1D_REQUIRE(p->x, "x");
    CC1D_REQUIRE(p->delta, "delta");
    CC1D_REQUIRE(p->A, "A");
    CC1D_REQUIRE(p->B, "B");
    CC1D_REQUIRE(p->C, "C");
    if (!bwd) {
      CC1D_REQUIRE(p->out, "out");
    } else {
      CC1D_REQUIRE(p->dout, "dout");
      CC1D_REQUIRE(p->dx, "dx");
      CC1D_REQUIRE(p->ddelta, "ddelta");
      CC1D_REQUIRE(p->dB, "dB");
      CC1D_REQUIRE(p->dC, "dC");
      if (p->z.data) CC1D_REQUIRE(p->dz, "dz");
      if (!p->checkpoints) return fail(CC1D_ERR_VALUE, "checkpoints are required");
    }
    if (reinterpret_cast<uintptr_t>(p->checkpoints) & 15u) return fail(CC1D_ERR_VALUE, "checkpoints must be 16-byte aligned");
  }
  *a = SelArgs{};
  a->batch = p->batch;
  a->dim = p->dim;
  a->seqlen = p->seqlen;
  a->dstate = p->dstate;
  a->groups = p->groups;
  a->nstates = p->nstates;
  a->x = tensor_arg(p->x);
  a->delta = tensor_arg(p->delta);
  a->A = tensor_arg(p->A);
  a->B = tensor_arg(p->B);
  a->C = tensor_arg(p->C);
  a->D = tensor_arg(p->D);
  a->z = tensor_arg(p->z);
  a->bias = tensor_arg(p->bias);
  a->seq_idx = tensor_arg(p->seq_idx);
  a->init = tensor_arg(p->initial_states);
  a->final_states = bwd ? TensorArg{} : tensor_arg(p->final_states);
  a->out = tensor_arg(p->out);
  a->dout = tensor_arg(p->dout);
  a->dfinal = tensor_arg(p->dfinal_states);
  a->dx = tensor_arg(p->dx);
  a->ddelta = tensor_arg(p->ddelta);
  a->dB = tensor_arg(p->dB);
  a->dC = tensor_arg(p->dC);
  a->dz = tensor_arg(p->dz);
  a->dinit = tensor_arg(p->dinitial_states);
  a->B_group = p->B_group_stride;
  a->C_group = p->C_group_stride;
  a->dB_group = p->dB_group_stride;
  a->dC_group = p->dC_group_stride;
  a->dA = p->dA;
  a->dD = p->dD;
  a->dbias = p->dbias;
  a->checkpoints = p->checkpoints;
  a->softplus = p->softplus != 0;
  return CC1D_OK;
}

// Neighbouring channels of it move two at a time.
bool pairs_ok(const TensorArg& t, const SelArgs& a) {
  const uintptr_t bytes = t.dtype == CC1D_FLOAT32 ? 8 : 4;
  return t.s1 == 1 && reinterpret_cast<uintptr_t>(t.data) % bytes == 0 && (a.batch <= 1 || t.s0 % 2 == 0) &&
         (a.seqlen <= 1 || t.s2 % 2 == 0);
}

// Parts of the sequence that run side by side.  One part needs no first pass over it; with more,
// that pass finds what each part hands to the next one.  Up to 16 states four CTAs run on an SM
// (registers), and a tile takes long because a thread's work is one chain: with n CTAs on an SM its time
// is about (microseconds, 32 positions, 16 states, bf16 with z)
//
//   forward  3.0 + .55 n, the first pass .66 of it      backward  13.7 + 1.2 n, .43
//
// and a part about two tiles' time to start.  The same rule stands for other types and numbers of states.  It is
// off where the backward's shared memory lets fewer CTAs run (59 KB and three of them at 32 states, 78 and
// 105 KB and two at 64 and 128, 150 KB and one at 256), as the last line shows.  Measured on a B200, bf16 with z, 16 states, microseconds
// in one part, in the parts chosen, and in the best of thirteen counts from 1 to 64:
//
//   batch x dim x seqlen   forward              backward
//   1 x 1024 x 16384       1543, 253, 253       7700, 742, 742
//   1 x 64 x 16384         1521, 58, 58         7032, 193, 193
//   1 x 4096 x 2048        197, 131, 130        1017, 431, 431
//   2 x 4096 x 2048        235, 235, 235        1026, 819, 768
//   4 x 4096 x 2048        322, 322, 322        1197, 1197, 1197
//   8 x 8192 x 128         85, 85, 85           346, 346, 346
//   1 x 5120 x 8192        915, 584, 581        3986, 1819, 1819
//   1 x 1024 x 4096 x 64   356, 255, 243        1648, 1153, 1055    (64 states)
int64_t choose_segments(const SelArgs& a, bool bwd) {
  constexpr int kFit = 4;
  const double sms = sm_count();
  const int64_t ctas = a.launch_rows * a.tiles, fit = static_cast<int64_t>(sms) * kFit;
  const double base = bwd ? 13.7 : 3.0, more = bwd ? 1.2 : .55, first = bwd ? .43 : .66;
  double best = 0;
  int64_t pick = 1;
  for (int64_t n = 1; n <= 64 && n <= a.nchunks; ++n) {
    const double tiles = static_cast<double>((a.nchunks + n - 1) / n) + 2;
    const int64_t waves = ctas * n / fit, rest = ctas * n % fit;
    const auto tile = [&](int64_t running) { return base + more * std::max(1.0, static_cast<double>(running) / sms); };
    const double cost = tiles * (n > 1 ? 1 + first : 1) * (static_cast<double>(waves) * tile(fit) + (rest ? tile(rest) : 0.0));
    if (n == 1 || cost < best) best = cost, pick = n;
  }
  return pick;
}

// Threads per channel, passes, tiles of channels, segments of the sequence, and which way the
// threads go through a tile.
cc1d_status plan(SelArgs* a, bool bwd) {
  a->padded = (a->dstate + 3) / 4 * 4;
  for (a->lanes = 1; a->lanes < kSelLanes && a->lanes * kSelStates < a->dstate;) a->lanes *= 2;
  a->blocks = static_cast<int>((a->dstate + a->lanes * kSelStates - 1) / (a->lanes * kSelStates));
  const int64_t chunk = CC1D_SELECTIVE_CHUNK(a->dstate);
  a->nchunks = (a->seqlen + chunk - 1) / chunk;
  a->gdim = a->dim / a->groups;
  const int64_t channels = kSelChannels / a->lanes;
  a->group_tiles = (a->gdim + channels - 1) / channels;
  a->tiles = a->group_tiles * a->groups;
  a->rows = a->x.s2 == 1 && a->x.s1 != 1 && a->seqlen > 1;
  a->pairs = !a->rows && a->gdim % 2 == 0;
  const TensorArg* const moved[] = {&a->x, &a->delta, &a->z, bwd ? &a->dout : &a->out, bwd ? &a->dx : nullptr,
                                    bwd ? &a->ddelta : nullptr, bwd ? &a->dz : nullptr};
  for (const TensorArg* t : moved)
    if (t && t->data) a->pairs = a->pairs && pairs_ok(*t, *a);
  // The backward's sums of dB and dC take 8 padded bytes for each position and CTA, which has 128 / lanes
  // channels: 4 bytes for each position and channel at 16 states, 16 at 32, 64 at 64, 256 at 256.  So that a
  // large batch does not take more than its tensors, as many rows go at a time as 2 GB hold.  One row always
  // goes as a whole, and may take more: 8.6 GB for 8192 channels x 16384 positions x 64 states.
  const double row_bytes = 8.0 * a->seqlen * a->tiles * a->padded;
  a->row0 = 0;
  a->launch_rows = bwd && row_bytes * a->batch > 2e9 ? std::max<int64_t>(1, static_cast<int64_t>(2e9 / row_bytes)) : a->batch;
  a->segments = choose_segments(*a, bwd);
  a->segment_chunks = (a->nchunks + a->segments - 1) / a->segments;
  a->segments = (a->nchunks + a->segment_chunks - 1) / a->segment_chunks;
  if (a->launch_rows * a->segments * a->tiles > kMax31 ||
      static_cast<double>(a->launch_rows) * a->seqlen * a->groups * 2 * a->padded / kThreads > kMax31)
    return fail(CC1D_ERR_VALUE, "the problem is too large for one launch");
  if (bwd && row_bytes * a->launch_rows > 1e17)
    return fail(CC1D_ERR_VALUE, "the workspace would be too large");
  return CC1D_OK;
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// Lays the workspace out from `base` on and returns its size.
int64_t lay_out(SelArgs* a, bool bwd, void* base) {
  int64_t at = 0;
  auto take = [&](float*& p, int64_t floats) {
    p = base ? reinterpret_cast<float*>(static_cast<char*>(base) + at) : nullptr;
    at += round16(floats * static_cast<int64_t>(sizeof(float)));
  };
  const int64_t parts = a->batch * a->segments * a->dim;
  if (a->segments > 1) {
    take(a->ends, parts * a->padded);
    take(a->steps, parts);
  }
  if (bwd) {
    take(a->parts_bc, a->launch_rows * a->seqlen * a->tiles * 2 * a->padded);
    take(a->parts_a, parts * a->padded);
    take(a->parts_d, 2 * parts);
  }
  return at;
}

bool empty(const SelArgs& a) { return a.batch == 0 || a.dim == 0 || a.seqlen == 0; }

int64_t workspace_bytes(const cc1d_selective_params* p, bool bwd) {
  set_last_error("");
  SelArgs a;
  if (check(p, bwd, &a) != CC1D_OK) return -1;
  if (empty(a)) return 0;
  return plan(&a, bwd) == CC1D_OK ? lay_out(&a, bwd, nullptr) : -1;
}

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

int64_t cc1d_selective_fwd_workspace_bytes(const cc1d_selective_params* p) { return workspace_bytes(p, false); }
int64_t cc1d_selective_bwd_workspace_bytes(const cc1d_selective_params* p) { return workspace_bytes(p, true); }

cc1d_status cc1d_selective_fwd_launch(const cc1d_selective_params* p, void* stream) {
  set_last_error("");
  SelArgs a;
  cc1d_status st = check(p, false, &a);
  if (st != CC1D_OK || empty(a)) return st;
  if ((st = plan(&a, false)) != CC1D_OK) return st;
  if ((st = workspace_ok(p->workspace, p->workspace_bytes, lay_out(&a, false, p->workspace))) != CC1D_OK) return st;
  return launched(by_type(p->x.dtype, a, static_cast<cudaStream_t>(stream), sel_fwd_f32, sel_fwd_f16, sel_fwd_bf16),
                  "selective recurrence forward launch", a.segments > 1 ? 2 : 1);
}

cc1d_status cc1d_selective_bwd_launch(const cc1d_selective_params* p, void* stream) {
  set_last_error("");
  SelArgs a;
  cc1d_status st = check(p, true, &a);
  if (st != CC1D_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (empty(a)) {
    cudaError_t e = cudaSuccess;
    if (a.dA && a.dim > 0) e = cudaMemsetAsync(a.dA, 0, a.dim * a.dstate * sizeof(float), s);
    if (e == cudaSuccess && a.dD && a.dim > 0) e = cudaMemsetAsync(a.dD, 0, a.dim * sizeof(float), s);
    if (e == cudaSuccess && a.dbias && a.dim > 0) e = cudaMemsetAsync(a.dbias, 0, a.dim * sizeof(float), s);
    // without channels B and C reach nothing: the sums over no CTA
    const bool sums = a.dim == 0 && a.batch > 0 && a.seqlen > 0 && a.dB.data && a.dC.data;
    if (e == cudaSuccess && sums) {
      if ((st = plan(&a, true)) != CC1D_OK) return st;
      e = by_type(p->x.dtype, a, s, sel_bwd_f32, sel_bwd_f16, sel_bwd_bf16);
    }
    return launched(e, "selective recurrence zero fill", sums);
  }
  if ((st = plan(&a, true)) != CC1D_OK) return st;
  if ((st = workspace_ok(p->workspace, p->workspace_bytes, lay_out(&a, true, p->workspace))) != CC1D_OK) return st;
  const int64_t times = (a.batch + a.launch_rows - 1) / a.launch_rows;
  return launched(by_type(p->x.dtype, a, s, sel_bwd_f32, sel_bwd_f16, sel_bwd_bf16), "selective recurrence backward launch",
                  static_cast<int>(times * (a.segments > 1 ? 3 : 2) + 1));
}

cc1d_status cc1d_selective_update_launch(const cc1d_selective_update_params* p, void* stream) {
  set_last_error("");
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  const cc1d_status st = check_common(p);
  if (st != CC1D_OK) return st;
  CC1D_SAME_TYPE(p->out, "out");
  CC1D_FP32(p->state, "state");
  if (p->state_indices.data && p->state_indices.dtype != CC1D_INT32)
    return fail(CC1D_ERR_TYPE, "state_indices must be int32");
  if (!p->state_indices.data && p->nstates != p->batch)
    return fail(CC1D_ERR_VALUE, "without state_indices there is one state for each batch row");
  if (p->batch == 0 || p->dim == 0 || p->seqlen == 0) return CC1D_OK;
  CC1D_REQUIRE(p->x, "x");
  CC1D_REQUIRE(p->delta, "delta");
  CC1D_REQUIRE(p->A, "A");
  CC1D_REQUIRE(p->B, "B");
  CC1D_REQUIRE(p->C, "C");
  CC1D_REQUIRE(p->out, "out");
  if (p->nstates > 0) CC1D_REQUIRE(p->state, "state");
  if (!apart(p->state, p->nstates, p->dim, p->dstate)) return fail(CC1D_ERR_VALUE, "the state's elements must not overlap");
  if (static_cast<double>(p->batch) * p->dim * 32 / kThreads > kMax31)
    return fail(CC1D_ERR_VALUE, "batch * dim is too large");
  SelUpdateArgs a;
  a.batch = p->batch;
  a.dim = p->dim;
  a.seqlen = p->seqlen;
  a.dstate = p->dstate;
  a.groups = p->groups;
  a.nstates = p->nstates;
  a.x = tensor_arg(p->x);
  a.delta = tensor_arg(p->delta);
  a.A = tensor_arg(p->A);
  a.B = tensor_arg(p->B);
  a.C = tensor_arg(p->C);
  a.D = tensor_arg(p->D);
  a.z = tensor_arg(p->z);
  a.bias = tensor_arg(p->bias);
  a.state = tensor_arg(p->state);
  a.out = tensor_arg(p->out);
  a.B_group = p->B_group_stride;
  a.C_group = p->C_group_stride;
  a.indices = static_cast<const int32_t*>(p->state_indices.data);
  a.indices_stride = p->state_indices.stride[0];
  a.softplus = p->softplus != 0;
  return launched(by_type(p->x.dtype, a, static_cast<cudaStream_t>(stream), sel_update_f32, sel_update_f16, sel_update_bf16),
                  "selective recurrence update launch", 1);
}

}  // extern "C"
