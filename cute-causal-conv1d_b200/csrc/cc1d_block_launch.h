// Host-side interface between the launchers of the recurrent-block operators
// (cc1d_block_abi.cu) and their per-element-type kernel files.
#pragma once

#include "cc1d_launch.h"

namespace cc1d {

constexpr int kRecChunk = CC1D_RECURRENCE_CHUNK;  // positions between two checkpoints

struct RecArgs {
  int64_t batch, dim, seqlen, nstates, nchunks;
  TensorArg x, gate, z, bias, seq_idx, init, final_states, out;
  TensorArg dout, dfinal, dx, dgate, dz, dinit;
  float* dbias;
  float* checkpoints;
  float* partials;  // backward: (batch * cluster, dim) sums of dgate to add up for dbias
  // the plan (rec_plan): tiles of channels, CTAs that share one, memory layout, and how the
  // tensors move
  int64_t dtiles;
  int cluster, move;
  bool rows;
};

// How the recurrence's tensors move (RecArgs::move).  kTma: the TMA copies whole tiles both
// ways (strips aligned to 16 bytes).  kPackets: strips of 16-bit elements that may start
// anywhere, by the 16-byte packets that cover them.  kElements: one by one, any strides.
constexpr int kTma = 0, kPackets = 1, kElements = 2;

struct RecUpdateArgs {
  int64_t batch, dim, seqlen, nstates;
  TensorArg x, gate, z, bias, state, out;
  const int32_t* indices;
  int64_t indices_stride;
};

struct AddNormArgs {
  int64_t rows, dim;
  TensorArg x, residual, weight, out, residual_out;
  TensorArg dout, dresidual_out, dx, dresidual;
  const int64_t* rng;
  int64_t rng_stride;
  float* dweight;
  float* partials;
  float eps, keep_scale;     // keep_scale = 1 / (1 - p)
  unsigned keep_from;        // a word below it is dropped
};

#define CC1D_DECLARE(name, Args)                       \
  cudaError_t name##_f32(const Args&, cudaStream_t);   \
  cudaError_t name##_f16(const Args&, cudaStream_t);   \
  cudaError_t name##_bf16(const Args&, cudaStream_t);

// (RecArgs is changed only where a tensor turns out not to be one that the TMA can describe)
cudaError_t rec_fwd_f32(RecArgs&, cudaStream_t);
cudaError_t rec_fwd_f16(RecArgs&, cudaStream_t);
cudaError_t rec_fwd_bf16(RecArgs&, cudaStream_t);
cudaError_t rec_bwd_f32(RecArgs&, cudaStream_t);
cudaError_t rec_bwd_f16(RecArgs&, cudaStream_t);
cudaError_t rec_bwd_bf16(RecArgs&, cudaStream_t);
CC1D_DECLARE(rec_update, RecUpdateArgs)
CC1D_DECLARE(add_norm_fwd, AddNormArgs)
CC1D_DECLARE(add_norm_bwd, AddNormArgs)
#undef CC1D_DECLARE

// fp32 values of workspace the backward kernels need.
int64_t add_norm_bwd_partial_floats(const AddNormArgs& a);

}  // namespace cc1d
