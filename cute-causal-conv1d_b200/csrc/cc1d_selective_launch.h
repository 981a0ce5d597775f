// Host-side interface between the launchers of the selective recurrence (cc1d_selective_abi.cu)
// and its per-element-type kernel files.
#pragma once

#include "cc1d_launch.h"

namespace cc1d {

constexpr int kSelChunk = 32;                    // the most positions of a tile, and between two checkpoints
constexpr int kSelChannels = 128;                // channels of a CTA times the threads that share one state vector
constexpr int kSelStates = 4;                    // states of a channel that a thread holds
constexpr int kSelLanes = 16;                    // the most threads that share a channel's states
constexpr int sel_tile(int lanes) { return lanes < 4 ? 8 * lanes : 32; }  // positions of a tile

struct SelArgs {
  int64_t batch, dim, seqlen, dstate, groups, nstates;
  TensorArg x, delta, A, B, C, D, z, bias, seq_idx, init, final_states, out;
  TensorArg dout, dfinal, dx, ddelta, dB, dC, dz, dinit;
  int64_t B_group, C_group, dB_group, dC_group;  // strides between groups
  float *dA, *dD, *dbias;
  float* checkpoints;
  bool softplus;
  // the plan (sel_plan)
  int lanes;                             // threads that share a channel's states: 1, 2, 4, 8 or 16
  int blocks;                            // passes over a tile: ceil(dstate / (4 lanes))
  int64_t padded;                        // dstate rounded up to a multiple of 4
  int64_t nchunks;                       // tiles along the sequence: ceil(seqlen / sel_tile(lanes))
  int64_t gdim, group_tiles, tiles;      // channels of a group, CTAs that they take, CTAs of all groups
  int64_t segments, segment_chunks;      // parts of the sequence that run side by side, chunks of one
  bool rows;                             // unit stride along the sequence: threads go along it
  bool pairs;                            // two neighbouring channels move as one word, in every tensor
  int64_t row0, launch_rows;             // batch rows of a launch; the backward takes some at a time
  // workspace
  float* ends;      // (batch, segments, dim, padded): what a segment alone carries out of itself
  float* steps;     // (batch, segments, dim): the sum of its step sizes, or infinity if it is cut
  float* parts_bc;  // backward: (launch_rows, seqlen, tiles, 2, padded) sums of dB and dC over a tile's channels
  float* parts_a;   // backward: (batch * segments, dim, padded) sums of dA over a segment
  float* parts_d;   // backward: (batch * segments, 2, dim), of dD and dbias
};

struct SelUpdateArgs {
  int64_t batch, dim, seqlen, dstate, groups, nstates;
  TensorArg x, delta, A, B, C, D, z, bias, state, out;
  int64_t B_group, C_group;
  const int32_t* indices;
  int64_t indices_stride;
  bool softplus;
};

#define CC1D_DECLARE(name, Args)                       \
  cudaError_t name##_f32(const Args&, cudaStream_t);   \
  cudaError_t name##_f16(const Args&, cudaStream_t);   \
  cudaError_t name##_bf16(const Args&, cudaStream_t);

CC1D_DECLARE(sel_fwd, SelArgs)
CC1D_DECLARE(sel_bwd, SelArgs)
CC1D_DECLARE(sel_update, SelUpdateArgs)
#undef CC1D_DECLARE

}  // namespace cc1d
