// What the sequence kernels of the selective recurrence share.
#pragma once

#include "cc1d_block_math.cuh"
#include "cc1d_selective_launch.h"

namespace cc1d {

// softplus(u) = max(u, 0) + log(1 + e) with e = exp(-|u|), to full relative precision for u of any
// size, NaN included.  log(1 + e) = 2 atanh(s) with s = e / (2 + e) <= 1/3, and 2 atanh(s) / s in
// w = s^2 <= 1/9 by the polynomial that interpolates it at five Chebyshev points (off by 4e-9).
__device__ __forceinline__ float softplus_of_exp(float u, float e) {
  const float s = e * rcp_approx(2.f + e);
  const float w = s * s;
  float q = fmaf(0.281577796f, w, 0.279651582f);
  q = fmaf(q, w, 0.400245965f);
  q = fmaf(q, w, 0.666663229f);
  q = fmaf(q, w, 2.f);
  return fmaf(s, q, fmaxf(u, 0.f));
}
// exp(-|u|); for 16-bit tensors the rounding of the exponent is left in it (|u| 2^-24 of it).
template <typename T>
__device__ __forceinline__ float exp_of_size(float u) {
  if constexpr (std::is_same<T, float>::value) return exp_minus(min_nan(fabsf(u), 88.f));
  else return ex2_approx(-kLog2e * fabsf(u));
}
template <typename T>
__device__ __forceinline__ float step_size(float u) { return softplus_of_exp(u, exp_of_size<T>(u)); }
// The same, and its derivative sigmoid(u).
template <typename T>
__device__ __forceinline__ float step_size(float u, float* slope) {
  const float e = exp_of_size<T>(u);
  const float r = rcp_approx(1.f + e);
  *slope = u < 0.f ? e * r : r;
  return softplus_of_exp(u, e);
}

// exp(s A) as 2^(s A log2(e)) by the hardware's approximation, for two states.  Between -0.5 and 0
// its results are 0.3 units of 2^-24 too small on the average (measured over 16 million arguments,
// mean errors of -0.29 to -0.33 units from -0.001 to -0.5), which a slow state multiplies up a
// thousand times and more: the argument is raised by as much.
constexpr float kNudge = 0.3f * 5.96046448e-8f * kLog2e;
__device__ __forceinline__ float2 decays(float2 s, float2 rate) {
  const float2 v = ffma2(s, rate, make_float2(kNudge, kNudge));
  return make_float2(ex2_approx(v.x), ex2_approx(v.y));
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

// A tile: T positions of CH channels of a batch row, and how the threads go through it, eight
// elements each, along the dimension of unit stride: element k of a thread is position t + k DT,
// channel c + k DC.
template <int LN, bool ROWS>
struct Tile {
  static constexpr int CH = kSelThreads / LN, T = 8 * LN, PITCH = CH + 1;
  static constexpr int DT = ROWS ? 0 : LN, DC = ROWS ? kSelThreads / T : 0;
  static __device__ __forceinline__ int t() { return ROWS ? threadIdx.x % T : threadIdx.x / CH; }
  static __device__ __forceinline__ int c() { return ROWS ? threadIdx.x / T : threadIdx.x % CH; }
};

// The flags and state rows (-1: none) of a tile's positions.
struct SelFlags {
  uint32_t word[kSelChunk / 4];
  int row[kSelChunk];
  __device__ __forceinline__ bool valid(int t) const { return reinterpret_cast<const uint8_t*>(word)[t] & kValid; }
};

// A position's flag and state row, one thread each.  The ids are loaded a tile ahead.
template <int T>
struct FlagFeed {
  int before, id, after;
  __device__ __forceinline__ void load(const SelArgs& a, int64_t b, int64_t t0) {
    const int64_t t = t0 + threadIdx.x;
    if (threadIdx.x >= T || !a.seq_idx.data || t < 0 || t >= a.seqlen) return;
    const int* ids = static_cast<const int*>(a.seq_idx.data) + b * a.seq_idx.s0;
    id = ids[t * a.seq_idx.s1];
    before = t > 0 ? ids[(t - 1) * a.seq_idx.s1] : -1;
    after = t + 1 < a.seqlen ? ids[(t + 1) * a.seq_idx.s1] : -1;
  }
  __device__ __forceinline__ void store(const SelArgs& a, int64_t b, int64_t t0, SelFlags& s) const {
    if (threadIdx.x >= T) return;
    const int64_t t = t0 + threadIdx.x;
    uint32_t f = 0;
    int row = -1;
    if (t < a.seqlen) {
      if (!a.seq_idx.data) {
        f = kValid | (t == 0 ? kFirst : 0) | (t == a.seqlen - 1 ? kLast : 0);
        row = b < a.nstates ? static_cast<int>(b) : -1;
      } else if (id >= 0) {
        f = kValid | (t == 0 || before != id ? kFirst : 0) | (t == a.seqlen - 1 || after != id ? kLast : 0);
        row = id < a.nstates ? id : -1;
      }
    }
    reinterpret_cast<uint8_t*>(s.word)[threadIdx.x] = static_cast<uint8_t>(f);
    s.row[threadIdx.x] = row;
  }
};

// A thread's eight elements of one tensor, walked tile by tile.
template <typename T, int LN, bool ROWS>
struct Walk {
  using Where = Tile<LN, ROWS>;
  T* p;  // of the thread's first element in tile 0
  __device__ __forceinline__ Walk(const TensorArg& t, const SelPlace& at) {
    p = static_cast<T*>(t.data) + at.b * t.s0 + (at.ch0 + Where::c()) * t.s1 + Where::t() * t.s2;
  }
  // Whether element k of the tile at t0 exists.
  static __device__ __forceinline__ bool has(const SelArgs& a, const SelPlace& at, int64_t t0, int k) {
    return t0 + Where::t() + k * Where::DT < a.seqlen && Where::c() + k * Where::DC < at.channels;
  }
  static __device__ __forceinline__ int64_t step(const TensorArg& t) { return ROWS ? Where::DC * t.s1 : Where::DT * t.s2; }
  __device__ __forceinline__ void load(const SelArgs& a, const TensorArg& t, const SelPlace& at, int64_t index, bool whole, T (&v)[8]) const {
    const T* q = p + index * (Where::T * t.s2);
    if (whole) {
#pragma unroll
      for (int k = 0; k < 8; ++k, q += step(t)) v[k] = *q;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k, q += step(t)) v[k] = has(a, at, index * Where::T, k) ? *q : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(const SelArgs& a, const TensorArg& t, const SelPlace& at, int64_t index, bool whole, const float (&v)[8]) const {
    T* q = p + index * (Where::T * t.s2);
    if (whole) {
#pragma unroll
      for (int k = 0; k < 8; ++k, q += step(t)) *q = from_f32<T>(v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k, q += step(t))
        if (has(a, at, index * Where::T, k)) *q = from_f32<T>(v[k]);
    }
  }
};

// B and C of a tile's positions in shared memory, in their own type, since what a load from there
// brings to registers is what it costs: [position][B, C][wide], wide = 4 LN per pass; zero past
// dstate and where a position is not valid, so that whatever stands there is not used.  The threads
// go along the states or, where that is B's unit stride, along the sequence; the eight elements
// of a thread for a single pass are loaded a tile ahead.
template <typename T, int LN, bool MULTI>
struct Coefficients {
  static constexpr int TT = 8 * LN, ALL = TT * 8 * LN, HELD = MULTI || ALL < kSelThreads ? 1 : ALL / kSelThreads;
  static constexpr int DT = kSelThreads / (8 * LN), DN = kSelThreads / TT, HALF = HELD > 1 ? HELD / 2 : 1;
  T v[HELD];
  const T *p, *pc;  // along the states: the thread's tensor; else B and C
  int n, t;
  bool along, is_c;
  __device__ __forceinline__ Coefficients(const SelArgs& a, const SelPlace& at) {
    along = a.B.s1 == 1 || a.B.s2 != 1;
    const int e = threadIdx.x;
    int s;
    if (along) t = e / (8 * LN), s = e % (8 * LN);
    else t = e % TT, s = e / TT;
    is_c = s >= 4 * LN;
    n = is_c ? s - 4 * LN : s;
    const T* b = static_cast<const T*>(a.B.data) + at.b * a.B.s0 + at.group * a.B_group;
    const T* c = static_cast<const T*>(a.C.data) + at.b * a.C.s0 + at.group * a.C_group;
    p = is_c ? c + n * a.C.s1 + t * a.C.s2 : b + n * a.B.s1 + t * a.B.s2;
    pc = c + n * a.C.s1 + t * a.C.s2;
  }
  __device__ __forceinline__ void load(const SelArgs& a, int64_t t0, bool whole) {
    if constexpr (MULTI) return;
    if (ALL < kSelThreads && threadIdx.x >= ALL) return;
    if (along) {
      const int64_t s2 = is_c ? a.C.s2 : a.B.s2;
      const T* q = p + t0 * s2;
      if (n >= a.dstate) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) v[k] = from_f32<T>(0.f);
      } else if (whole) {
#pragma unroll
        for (int k = 0; k < HELD; ++k, q += DT * s2) v[k] = *q;
      } else {
#pragma unroll
        for (int k = 0; k < HELD; ++k, q += DT * s2) v[k] = t0 + t + k * DT < a.seqlen ? *q : from_f32<T>(0.f);
      }
    } else {
      const bool in = t0 + t < a.seqlen;
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const bool c = k >= HALF || is_c;
        const T* q = (k >= HALF ? pc : p) + t0 * (c ? a.C.s2 : a.B.s2) + k % HALF * DN * (c ? a.C.s1 : a.B.s1);
        v[k] = in && n + k % HALF * DN < a.dstate ? *q : from_f32<T>(0.f);
      }
    }
  }
  // checked: a position may not be valid
  __device__ __forceinline__ void store(const SelArgs& a, const SelPlace& at, int64_t t0, bool checked, const SelFlags& f, T* bc) const {
    if constexpr (MULTI) {
      const int wide = 4 * LN * a.blocks;
      for (int e = threadIdx.x; e < TT * 2 * wide; e += kSelThreads) {
        const int tt = along ? e / (2 * wide) : e % TT, s = along ? e - tt * 2 * wide : e / TT;
        const bool c = s >= wide;
        const int nn = c ? s - wide : s;
        const TensorArg& x = c ? a.C : a.B;
        T r = from_f32<T>(0.f);
        if (nn < a.dstate && f.valid(tt))
          r = static_cast<const T*>(x.data)[at.b * x.s0 + at.group * (c ? a.C_group : a.B_group) + nn * x.s1 + (t0 + tt) * x.s2];
        bc[(tt * 2 + c) * wide + nn] = r;
      }
    } else {
      if (ALL < kSelThreads && threadIdx.x >= ALL) return;
      T* o = bc + (t * 2 + is_c) * 4 * LN + n;
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const int at_k = along ? k * DT * 8 * LN : (k >= HALF) * 4 * LN + k % HALF * DN;
        o[at_k] = checked && !f.valid(along ? t + k * DT : t) ? from_f32<T>(0.f) : v[k];
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ float load_el(const TensorArg& t, int64_t b, int64_t d, int64_t l) {
  return to_f32(static_cast<const T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2]);
}
template <typename T>
__device__ __forceinline__ void store_el(const TensorArg& t, int64_t b, int64_t d, int64_t l, float v) {
  static_cast<T*>(t.data)[b * t.s0 + d * t.s1 + l * t.s2] = from_f32<T>(v);
}

// Four states of a channel, in pairs: sm_100a multiplies and adds two fp32 values in one instruction.
struct Four {
  float2 lo, hi;
};
__device__ __forceinline__ Four zero4() { return Four{make_float2(0.f, 0.f), make_float2(0.f, 0.f)}; }
__device__ __forceinline__ Four load4(const float* p) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  return Four{make_float2(f.x, f.y), make_float2(f.z, f.w)};
}
__device__ __forceinline__ void store4(float* p, const Four& f) {
  *reinterpret_cast<float4*>(p) = make_float4(f.lo.x, f.lo.y, f.hi.x, f.hi.y);
}
// Four neighbouring elements, on their alignment.
template <typename T>
__device__ __forceinline__ Four load4_of(const T* p) {
  float v[4];
  unpack<T, 4>(*reinterpret_cast<const Packet<T, 4>*>(p), v);
  return Four{make_float2(v[0], v[1]), make_float2(v[2], v[3])};
}
__device__ __forceinline__ Four fma4(const Four& a, const Four& b, const Four& c) { return Four{ffma2(a.lo, b.lo, c.lo), ffma2(a.hi, b.hi, c.hi)}; }
__device__ __forceinline__ Four mul4(const Four& a, const Four& b) { return Four{fmul2(a.lo, b.lo), fmul2(a.hi, b.hi)}; }
__device__ __forceinline__ Four mul4(const Four& a, float2 b) { return Four{fmul2(a.lo, b), fmul2(a.hi, b)}; }
__device__ __forceinline__ Four fma4(const Four& a, float2 b, const Four& c) { return Four{ffma2(a.lo, b, c.lo), ffma2(a.hi, b, c.hi)}; }
__device__ __forceinline__ float sum4(const Four& a) {
  const float2 s = fadd2(a.lo, a.hi);
  return s.x + s.y;
}
__device__ __forceinline__ float dot4(const Four& a, const Four& b) {
  const float2 s = ffma2(a.hi, b.hi, fmul2(a.lo, b.lo));
  return s.x + s.y;
}
__device__ __forceinline__ Four decays4(float2 s, const Four& rate) { return Four{decays(s, rate.lo), decays(s, rate.hi)}; }
// A row of the states (rows, dim, dstate) at channel ch, states n0 .. n0 + 3.
__device__ __forceinline__ Four load_state(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate) {
  const float* p = static_cast<const float*>(t.data) + row * t.s0 + ch * t.s1;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = n0 + i < dstate ? p[(n0 + i) * t.s2] : 0.f;
  return Four{make_float2(v[0], v[1]), make_float2(v[2], v[3])};
}
__device__ __forceinline__ void store_state(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate, const Four& f) {
  float* p = static_cast<float*>(t.data) + row * t.s0 + ch * t.s1;
  const float v[4] = {f.lo.x, f.lo.y, f.hi.x, f.hi.y};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < dstate) p[(n0 + i) * t.s2] = v[i];
}
// A[ch, n0 .. n0 + 3] log2(e), so that exp(s A) = 2^(s A log2(e)).
__device__ __forceinline__ Four load_rates(const TensorArg& A, int64_t ch, int64_t n0, int64_t dstate) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = n0 + i < dstate ? kLog2e * load_any(A.data, A.dtype, ch * A.s0 + (n0 + i) * A.s1) : 0.f;
  return Four{make_float2(v[0], v[1]), make_float2(v[2], v[3])};
}
__device__ __forceinline__ Four load_rates(const SelArgs& a, int64_t ch, int64_t n0) { return load_rates(a.A, ch, n0, a.dstate); }
// What a segment's neighbour and those beyond it hand on: x exp(A sum) + e, and e alone where the
// sequence is cut between them (sum infinite) or nothing comes.
__device__ __forceinline__ float handed_on(float x, float rate, float sum, float e) {
  return sum < INFINITY && x != 0.f ? fmaf(exp2f(rate * sum), x, e) : e;
}
__device__ __forceinline__ Four handed_on(const Four& x, const Four& rate, float sum, const Four& e) {
  return Four{make_float2(handed_on(x.lo.x, rate.lo.x, sum, e.lo.x), handed_on(x.lo.y, rate.lo.y, sum, e.lo.y)),
              make_float2(handed_on(x.hi.x, rate.hi.x, sum, e.hi.x), handed_on(x.hi.y, rate.hi.y, sum, e.hi.y))};
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
