// Host-side interface between the launchers of beam search (cc1d_beam_abi.cu) and its kernels
// (cc1d_beam.cu).
#pragma once

#include "cc1d_launch.h"

namespace cc1d {

struct BeamSelectArgs {
  int64_t batch, beams, vocab, candidates;
  const void* logits;
  int64_t logits_s0, logits_s1;
  const float* scores;
  int64_t scores_s0, scores_s1;
  const uint8_t* finished;
  int64_t finished_s0, finished_s1;
  int64_t end_token;
  float* out_scores;
  int64_t *parents, *tokens;  // (batch, candidates) dense, as out_scores
  // the plan: parts of a row that CTAs take side by side, and the elements of one
  int64_t parts, part;
  // workspace: (batch * beams * parts, candidates) of the parts' best and (.., 2) of their sums
  int2* best;
  float2* sums;
};

constexpr int kBeamCtas = 4;      // CTAs of the selection's first kernel on an SM
constexpr int kBeamTensors = 24;  // tensors of one reordering launch

// Rows that follow the beams.  Row r starts at data + r * row_bytes.  A row is `columns` units of
// `unit` bytes in up to four dimensions: unit u = ((i3 size2 + i2) size1 + i1) size0 + i0 lies at
// i0 step0 + i1 step1 + i2 step2 + i3 step3.
struct BeamRows {
  char* data;
  int64_t rows, row_bytes, columns, size0, size1, size2, step0, step1, step2, step3;
  int32_t unit, blocks;  // blocks: CTAs of one request
};

struct BeamReorderArgs {
  int64_t batch, beams;
  const void* parents;
  int64_t parents_s0, parents_s1;
  const int32_t* indices;
  int64_t indices_stride;
  int32_t wide_parents;  // int64 instead of int32
  int32_t count;
  BeamRows t[kBeamTensors];
};

cudaError_t beam_select(const BeamSelectArgs& a, int dtype, cudaStream_t s);
cudaError_t beam_reorder(const BeamReorderArgs& a, int64_t ctas, cudaStream_t s);
int64_t beam_most_unit(int64_t beams);  // the most bytes that a thread of beam_reorder moves per beam

}  // namespace cc1d
