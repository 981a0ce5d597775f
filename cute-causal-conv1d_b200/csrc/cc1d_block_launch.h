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
  int64_t* capacity = nullptr;  // if set nothing is launched: how many clusters run at a time
};

// How the recurrence's tensors move (RecArgs::move).  kTma: the TMA copies whole tiles both
// ways (strips aligned to 16 bytes).  By the 16-byte packets that cover a strip: kWords and kHalves
// (strips on 4 bytes, or anywhere for 16-bit elements) where the inputs lie alike, so that one
// offset serves them all; kOwn where each has its own.  kElements: one by one, any strides.
constexpr int kTma = 0, kWords = 1, kHalves = 2, kOwn = 3, kElements = 4;

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
  // the plan (add_norm_plan): threads that share a row (0: rows too wide for the registers),
  // columns that each of them holds, CTAs, and the elements that every row starts on a multiple
  // of: 8 (16-bit types), 4, 2 or 1
  int group, held, aligned;
  int64_t ctas;
};

// The launches of one element type.  Args& is changed only where a recurrence's tensor turns
// out not to be one that the TMA can describe.
#define CC1D_DECLARE(name, Args)                 \
  cudaError_t name##_f32(Args&, cudaStream_t);   \
  cudaError_t name##_f16(Args&, cudaStream_t);   \
  cudaError_t name##_bf16(Args&, cudaStream_t);

CC1D_DECLARE(rec_fwd, RecArgs)
CC1D_DECLARE(rec_bwd, RecArgs)
CC1D_DECLARE(rec_update, RecUpdateArgs)
CC1D_DECLARE(add_norm_fwd, AddNormArgs)
CC1D_DECLARE(add_norm_bwd, AddNormArgs)
#undef CC1D_DECLARE

void add_norm_plan(AddNormArgs* a, int dtype, int sms, bool bwd);
// out[d] = sum over n rows of partials (n, dim), in a fixed order.
cudaError_t sum_rows(const float* partials, int64_t n, int64_t dim, float* out, cudaStream_t s);

}  // namespace cc1d
