// What the sequence kernels of the selective recurrence share.
#pragma once

#include "cc1d_block_math.cuh"
#include "cc1d_selective_launch.h"

namespace cc1d {

// softplus(u) = max(u, 0) + log(1 + exp(-|u|)) and its derivative sigmoid(u), both to full
// relative precision for u of any size.
__device__ __forceinline__ float step_size(float u, float* slope) {
  const float e = expf(-fabsf(u));
  const float r = 1.f / (1.f + e);
  *slope = u >= 0.f ? r : e * r;
  return fmaxf(u, 0.f) + log1pf(e) + (u != u ? u : 0.f);
}

// Where a position stands: kValid unless it is padding or past the end; the ends of its sequence.
constexpr uint32_t kValid = 1, kFirst = 2, kLast = 4;
constexpr uint32_t kAllInside = 0x01010101;  // four positions inside one sequence

struct SelPlace {
  int64_t b, seg, tile, group, ch0;
  int channels;        // of this CTA
  int64_t chunk0, chunk1;
};

template <int LN>
__device__ __forceinline__ SelPlace sel_place(const SelArgs& a) {
  constexpr int CH = kSelThreads / LN;
  SelPlace p;
  int64_t i = blockIdx.x;
  p.tile = i % a.tiles;
  i /= a.tiles;
  p.seg = i % a.segments;
  p.b = i / a.segments;
  p.group = p.tile / a.group_tiles;
  const int64_t in_group = (p.tile - p.group * a.group_tiles) * CH;
  p.ch0 = p.group * a.gdim + in_group;
  p.channels = static_cast<int>(a.gdim - in_group < CH ? a.gdim - in_group : CH);
  p.chunk0 = p.seg * a.segment_chunks;
  p.chunk1 = p.chunk0 + a.segment_chunks < a.nchunks ? p.chunk0 + a.segment_chunks : a.nchunks;
  return p;
}

// The flags and state rows (-1: none) of a tile's positions.
struct SelFlags {
  uint32_t word[kSelChunk / 4];
  int row[kSelChunk];
};

__device__ __forceinline__ void load_flags(const SelArgs& a, int64_t b, int64_t t0, SelFlags& s) {
  if (threadIdx.x >= kSelChunk) return;
  const int64_t t = t0 + threadIdx.x;
  uint32_t f = 0;
  int row = -1;
  if (t < a.seqlen) {
    if (a.seq_idx.data) {
      const int* ids = static_cast<const int*>(a.seq_idx.data) + b * a.seq_idx.s0;
      const int id = ids[t * a.seq_idx.s1];
      if (id >= 0) {
        f = kValid;
        if (t == 0 || ids[(t - 1) * a.seq_idx.s1] != id) f |= kFirst;
        if (t == a.seqlen - 1 || ids[(t + 1) * a.seq_idx.s1] != id) f |= kLast;
        row = id < a.nstates ? id : -1;
      }
    } else {
      f = kValid | (t == 0 ? kFirst : 0) | (t == a.seqlen - 1 ? kLast : 0);
      row = b < a.nstates ? static_cast<int>(b) : -1;
    }
  }
  reinterpret_cast<uint8_t*>(s.word)[threadIdx.x] = static_cast<uint8_t>(f);
  s.row[threadIdx.x] = row;
}

// Element e of a tile as the threads go through it: along the dimension of unit stride.
template <int CH>
__device__ __forceinline__ void tile_place(bool rows, int e, int& t, int& c) {
  if (rows) {
    t = e % kSelChunk;
    c = e / kSelChunk;
  } else {
    c = e % CH;
    t = e / CH;
  }
}

template <typename T>
__device__ __forceinline__ float load_el(const TensorArg& t, int64_t b, int64_t d, int64_t l) {
  return to_f32(static_cast<const T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2]);
}
template <typename T>
__device__ __forceinline__ void store_el(const TensorArg& t, int64_t b, int64_t d, int64_t l, float v) {
  static_cast<T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2] = from_f32<T>(v);
}

// B and C of a tile's positions as fp32 [position][B, C][padded]; zero past dstate and where a
// position is not valid, so that whatever stands there is not used.
template <typename T>
__device__ __forceinline__ void load_bc(const SelArgs& a, const SelPlace& p, int64_t t0, int np, const SelFlags& s, float* bc) {
  const T* pb = static_cast<const T*>(a.B.data) + p.b * a.B.s0 + p.group * a.B_group;
  const T* pc = static_cast<const T*>(a.C.data) + p.b * a.C.s0 + p.group * a.C_group;
  for (int e = threadIdx.x; e < kSelChunk * 2 * np; e += kSelThreads) {
    // along the states, or along the sequence where that is the unit stride
    int t, v;
    if (a.B.s1 == 1) {
      t = e / (2 * np);
      v = e - t * 2 * np;
    } else {
      t = e % kSelChunk;
      v = e / kSelChunk;
    }
    const int n = v < np ? v : v - np;
    float f = 0.f;
    if (n < a.dstate && (reinterpret_cast<const uint8_t*>(s.word)[t] & kValid))
      f = v < np ? to_f32(pb[n * a.B.s1 + (t0 + t) * a.B.s2]) : to_f32(pc[n * a.C.s1 + (t0 + t) * a.C.s2]);
    bc[t * 2 * np + v] = f;
  }
}

// Four states of a channel.  ch: the channel of all, < 0 where the thread has none.
struct Four {
  float v[4];
};
__device__ __forceinline__ Four zero4() { return Four{{0.f, 0.f, 0.f, 0.f}}; }
__device__ __forceinline__ Four load4(const float* p) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  return Four{{f.x, f.y, f.z, f.w}};
}
__device__ __forceinline__ void store4(float* p, const Four& f) {
  *reinterpret_cast<float4*>(p) = make_float4(f.v[0], f.v[1], f.v[2], f.v[3]);
}
// A row of the states (rows, dim, dstate) at channel ch, states n0 .. n0 + 3.
__device__ __forceinline__ Four load_state(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate) {
  const float* p = static_cast<const float*>(t.data) + row * t.s0 + ch * t.s1;
  Four f;
#pragma unroll
  for (int i = 0; i < 4; ++i) f.v[i] = n0 + i < dstate ? p[(n0 + i) * t.s2] : 0.f;
  return f;
}
__device__ __forceinline__ void store_state(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate, const Four& f) {
  float* p = static_cast<float*>(t.data) + row * t.s0 + ch * t.s1;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < dstate) p[(n0 + i) * t.s2] = f.v[i];
}
// A[ch, n0 .. n0 + 3] log2(e), so that exp(s A) = 2^(s A log2(e)).
__device__ __forceinline__ Four load_rates(const SelArgs& a, int64_t ch, int64_t n0) {
  Four f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f.v[i] = n0 + i < a.dstate ? kLog2e * load_any(a.A.data, a.A.dtype, ch * a.A.s0 + (n0 + i) * a.A.s1) : 0.f;
  return f;
}

// The sums over the LN threads of a channel of four positions' values; afterwards thread sl has
// those of positions sl * 4 / LN on, in v[0 .. 4 / LN).
template <int LN>
__device__ __forceinline__ void sum_lanes(float (&v)[4], int sl) {
  if constexpr (LN == 4) {
    const bool hi = sl & 2;
    const float s0 = hi ? v[0] : v[2], s1 = hi ? v[1] : v[3];
    v[0] = (hi ? v[2] : v[0]) + __shfl_xor_sync(~0u, s0, 2);
    v[1] = (hi ? v[3] : v[1]) + __shfl_xor_sync(~0u, s1, 2);
    const bool odd = sl & 1;
    const float s = odd ? v[0] : v[1];
    v[0] = (odd ? v[1] : v[0]) + __shfl_xor_sync(~0u, s, 1);
  } else if constexpr (LN == 2) {
    const bool hi = sl & 1;
    const float s0 = hi ? v[0] : v[2], s1 = hi ? v[1] : v[3];
    v[0] = (hi ? v[2] : v[0]) + __shfl_xor_sync(~0u, s0, 1);
    v[1] = (hi ? v[3] : v[1]) + __shfl_xor_sync(~0u, s1, 1);
  }
}

}  // namespace cc1d
