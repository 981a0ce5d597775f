// What the sequence kernels of the selective recurrence share.
#pragma once

#include "cc1d_block_math.cuh"
#include "cc1d_selective_launch.h"

namespace cc1d {

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// softplus(u) = max(u, 0) + log(1 + e) with e = exp(-|u|), for two values of any size, NaN included: within
// 2^-20 of itself (e 2^-22, the reciprocal 2^-23, five roundings), and (2^-24 + 2^-26) |u| more for 16-bit
// tensors, whose e keeps the rounding of its exponent.  Below 2^-126, u < -87.3, it is zero, as is e.
// log(1 + e) = 2 atanh(s) with s = e / (2 + e) <= 1/3, and
// 2 atanh(s) / s in w = s^2 <= 1/9 by the polynomial that interpolates it at five Chebyshev points
// (off by 4e-9).
__device__ __forceinline__ float2 softplus_of_exp(float2 u, float2 e) {
  const float2 d = fadd2(both(2.f), e);
  const float2 s = fmul2(e, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
  const float2 w = fmul2(s, s);
  float2 q = ffma2(both(0.281577796f), w, both(0.279651582f));
  q = ffma2(q, w, both(0.400245965f));
  q = ffma2(q, w, both(0.666663229f));
  q = ffma2(q, w, both(2.f));
  return ffma2(s, q, make_float2(fmaxf(u.x, 0.f), fmaxf(u.y, 0.f)));
}
// exp(-|u|); for 16-bit tensors the roundings of the exponent and of log2(e) are left in it, (2^-24 + 2^-26) |u| of it.
template <typename T>
__device__ __forceinline__ float2 exp_of_size(float2 u) {
  if constexpr (std::is_same<T, float>::value)
    return make_float2(exp_minus(min_nan(fabsf(u.x), 88.f)), exp_minus(min_nan(fabsf(u.y), 88.f)));
  const float2 v = fmul2(both(-kLog2e), make_float2(fabsf(u.x), fabsf(u.y)));
  return make_float2(ex2_approx(v.x), ex2_approx(v.y));
}
template <typename T>
__device__ __forceinline__ float2 step_size(float2 u) { return softplus_of_exp(u, exp_of_size<T>(u)); }
// The same of one.
template <typename T>
__device__ __forceinline__ float step_size(float u) {
  float e;
  if constexpr (std::is_same<T, float>::value) e = exp_minus(min_nan(fabsf(u), 88.f));
  else e = ex2_approx(-kLog2e * fabsf(u));
  const float s = e * rcp_approx(2.f + e), w = s * s;
  float q = fmaf(0.281577796f, w, 0.279651582f);
  q = fmaf(q, w, 0.400245965f);
  q = fmaf(q, w, 0.666663229f);
  q = fmaf(q, w, 2.f);
  return fmaf(s, q, fmaxf(u, 0.f));
}
// The same of two, and the derivative sigmoid(u).
template <typename T>
__device__ __forceinline__ float2 step_size(float2 u, float2* slope) {
  const float2 e = exp_of_size<T>(u), d = fadd2(both(1.f), e);
  const float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  const float2 less = fmul2(e, r);
  *slope = make_float2(u.x < 0.f ? less.x : r.x, u.y < 0.f ? less.y : r.y);
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
  constexpr int CH = kSelChannels / LN;
  SelPlace p;
  int64_t i = blockIdx.x;
  p.tile = i % a.tiles;
  i /= a.tiles;
  p.seg = i % a.segments;
  p.b = a.row0 + i / a.segments;
  p.group = p.tile / a.group_tiles;
  const int64_t in_group = (p.tile - p.group * a.group_tiles) * CH;
  p.ch0 = p.group * a.gdim + in_group;
  p.channels = static_cast<int>(a.gdim - in_group < CH ? a.gdim - in_group : CH);
  p.chunk0 = p.seg * a.segment_chunks;
  p.chunk1 = p.chunk0 + a.segment_chunks < a.nchunks ? p.chunk0 + a.segment_chunks : a.nchunks;
  return p;
}

// A tile: T positions of PAIRS pairs of channels of a batch row, and how the threads go through it,
// K pairs each, along the dimension of unit stride: the k-th of a thread is position t + k DT,
// pair c + k DC.  NT: threads of the CTA.
template <int NT, int LN, bool ROWS>
struct Tile {
  static constexpr int T = sel_tile(LN), PAIRS = kSelChannels / 2 / LN, K = T * PAIRS / NT;
  static constexpr int DT = ROWS ? 0 : NT / PAIRS, DC = ROWS ? NT / T : 0;
  static __device__ __forceinline__ int t() { return ROWS ? threadIdx.x % T : threadIdx.x / PAIRS; }
  static __device__ __forceinline__ int c() { return ROWS ? threadIdx.x / T : threadIdx.x % PAIRS; }
  static __device__ __forceinline__ int t(int k) { return t() + k * DT; }
  static __device__ __forceinline__ int c(int k) { return c() + k * DC; }
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

// Two channels of a position as they were loaded.  Kept as words until they are used: taking them
// apart at once would wait for the load.  16-bit: both in lo where they came as one word.
struct Raw {
  uint32_t lo, hi;
};
template <typename T>
__device__ __forceinline__ float2 pair_of(const Raw& r, bool pairs) {
  if constexpr (std::is_same<T, float>::value) return make_float2(__uint_as_float(r.lo), __uint_as_float(r.hi));
  const uint32_t word = pairs ? r.lo : __byte_perm(r.lo, r.hi, 0x5410);
  float f[2];
  unpack<T, 2>(*reinterpret_cast<const Packet<T, 2>*>(&word), f);
  return make_float2(f[0], f[1]);
}

// A thread's pairs of one tensor, walked tile by tile.
template <typename T, typename Where>
struct Walk {
  T* p;  // of the thread's first element in tile 0
  __device__ __forceinline__ Walk(const TensorArg& t, const SelPlace& at) {
    p = static_cast<T*>(t.data) + at.b * t.s0 + (at.ch0 + 2 * Where::c()) * t.s1 + Where::t() * t.s2;
  }
  // How many channels of pair k of the tile at t0 exist.
  static __device__ __forceinline__ int has(const SelArgs& a, const SelPlace& at, int64_t t0, int k) {
    return t0 + Where::t(k) < a.seqlen ? at.channels - 2 * Where::c(k) : 0;
  }
  static __device__ __forceinline__ int64_t step(const TensorArg& t) { return Where::DC ? 2 * Where::DC * t.s1 : Where::DT * t.s2; }
  static __device__ __forceinline__ uint32_t word(const T* q) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t*>(q);
    else return *reinterpret_cast<const uint16_t*>(q);
  }
  __device__ __forceinline__ void load(const SelArgs& a, const TensorArg& t, const SelPlace& at, int64_t index, bool whole, Raw (&v)[Where::K]) const {
    const T* q = p + index * (Where::T * t.s2);
    if (whole && a.pairs) {
#pragma unroll
      for (int k = 0; k < Where::K; ++k, q += step(t)) {
        if constexpr (sizeof(T) == 4) {
          const uint2 u = *reinterpret_cast<const uint2*>(q);
          v[k].lo = u.x, v[k].hi = u.y;
        } else {
          v[k].lo = *reinterpret_cast<const uint32_t*>(q);
        }
      }
    } else if (whole) {
#pragma unroll
      for (int k = 0; k < Where::K; ++k, q += step(t)) v[k].lo = word(q), v[k].hi = word(q + t.s1);
    } else {
#pragma unroll
      for (int k = 0; k < Where::K; ++k, q += step(t)) {
        const int n = has(a, at, index * Where::T, k);
        if (a.pairs && sizeof(T) == 2) {  // both or none
          v[k].lo = n > 0 ? *reinterpret_cast<const uint32_t*>(q) : 0;
        } else {
          v[k].lo = n > 0 ? word(q) : 0;
          v[k].hi = n > 1 ? word(q + t.s1) : 0;
        }
      }
    }
  }
  __device__ __forceinline__ void store_one(const SelArgs& a, const TensorArg& t, const SelPlace& at, int64_t index, int k, bool whole, float2 v) const {
    T* q = p + index * (Where::T * t.s2) + k * step(t);
    const float f[2] = {v.x, v.y};
    const Packet<T, 2> r = pack<T, 2>(f);
    if (whole && a.pairs) {
      *reinterpret_cast<Packet<T, 2>*>(q) = r;
    } else {
      const int n = whole ? 2 : has(a, at, index * Where::T, k);
      if (n > 0) q[0] = r.v[0];
      if (n > 1) q[t.s1] = r.v[1];
    }
  }
  __device__ __forceinline__ void store(const SelArgs& a, const TensorArg& t, const SelPlace& at, int64_t index, bool whole, const float2 (&v)[Where::K]) const {
#pragma unroll
    for (int k = 0; k < Where::K; ++k) store_one(a, t, at, index, k, whole, v[k]);
  }
};
// B and C of a tile's positions as fp32 in shared memory: [position][B, C][wide], wide = 4 LN per
// pass; zero past dstate and where a position is not valid, so that whatever stands there is not
// used.  The threads go along the states or, where that is B's unit stride, along the sequence; a
// thread's elements for a single pass are loaded a tile ahead.
template <typename T, int NT, int LN, bool MULTI>
struct Coefficients {
  static constexpr int TT = sel_tile(LN), WIDE = 8 * LN, ALL = TT * WIDE, HELD = MULTI || ALL < NT ? 1 : ALL / NT;
  // positions, or states, between two elements of a thread; half the elements are B's
  static constexpr int DT = WIDE <= NT ? NT / WIDE : 1, DN = NT / TT, HALF = HELD > 1 ? HELD / 2 : 1;
  static_assert(WIDE <= 2 * NT, "a thread has one place of B and C, or one of each");
  T v[HELD];
  const T *p, *pc;  // along the states: the thread's tensor, or B; else B and C
  int n, t;
  bool along, is_c;
  __device__ __forceinline__ Coefficients(const SelArgs& a, const SelPlace& at) {
    along = a.B.s1 == 1 || a.B.s2 != 1;
    const int e = threadIdx.x;
    int s;
    if (along) t = e / WIDE, s = e % WIDE;
    else t = e % TT, s = e / TT;
    is_c = s >= 4 * LN;
    n = is_c ? s - 4 * LN : s;
    const T* b = static_cast<const T*>(a.B.data) + at.b * a.B.s0 + at.group * a.B_group;
    const T* c = static_cast<const T*>(a.C.data) + at.b * a.C.s0 + at.group * a.C_group;
    p = is_c ? c + n * a.C.s1 + t * a.C.s2 : b + n * a.B.s1 + t * a.B.s2;
    pc = c + n * a.C.s1 + t * a.C.s2;
  }
  // Element k's position in the tile, and whether it is C's.
  __device__ __forceinline__ int position(int k) const { return !along ? t : WIDE <= NT ? t + k * DT : k / 2; }
  __device__ __forceinline__ bool of_c(int k) const { return along ? (WIDE <= NT ? is_c : k % 2 != 0) : k >= HALF || is_c; }
  __device__ __forceinline__ void load(const SelArgs& a, int64_t t0, bool whole) {
    if constexpr (MULTI) return;
    if (ALL < NT && threadIdx.x >= ALL) return;
    if (along) {
      if (n >= a.dstate) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) v[k] = from_f32<T>(0.f);
        return;
      }
      const int64_t step = is_c ? a.C.s2 : a.B.s2;
      const T* q = p + t0 * step;
      const T* qc = pc + t0 * a.C.s2;
      auto each = [&](auto in) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
          if (WIDE > NT && k % 2) {
            v[k] = in(k) ? *qc : from_f32<T>(0.f);
            qc += a.C.s2;
          } else {
            v[k] = in(k) ? *q : from_f32<T>(0.f);
            q += DT * step;
          }
        }
      };
      if (whole) each([](int) { return true; });
      else each([&](int k) { return t0 + (WIDE <= NT ? t + k * DT : k / 2) < a.seqlen; });
    } else {
      const bool in = t0 + t < a.seqlen;
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        const bool c = of_c(k);
        const T* q = (k >= HALF ? pc : p) + t0 * (c ? a.C.s2 : a.B.s2) + k % HALF * DN * (c ? a.C.s1 : a.B.s1);
        v[k] = in && n + k % HALF * DN < a.dstate ? *q : from_f32<T>(0.f);
      }
    }
  }
  // checked: a position may not be valid
  __device__ __forceinline__ void store(const SelArgs& a, const SelPlace& at, int64_t t0, bool checked, const SelFlags& f, float* bc) const {
    if constexpr (MULTI) {
      const int wide = 4 * LN * a.blocks;
      for (int e = threadIdx.x; e < TT * 2 * wide; e += NT) {
        const int tt = along ? e / (2 * wide) : e % TT, s = along ? e - tt * 2 * wide : e / TT;
        const bool c = s >= wide;
        const int nn = c ? s - wide : s;
        const TensorArg& x = c ? a.C : a.B;
        float r = 0.f;
        if (nn < a.dstate && f.valid(tt))
          r = to_f32(static_cast<const T*>(x.data)[at.b * x.s0 + at.group * (c ? a.C_group : a.B_group) + nn * x.s1 + (t0 + tt) * x.s2]);
        bc[(tt * 2 + c) * wide + nn] = r;
      }
    } else {
      if (ALL < NT && threadIdx.x >= ALL) return;
      auto each = [&](auto valid) {
        float* o = bc + (t * 2 + is_c) * 4 * LN + n;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
          // from the thread's first element on
          const int at_k = !along ? (k >= HALF) * 4 * LN + k % HALF * DN : WIDE <= NT ? k * DT * 8 * LN : k * 4 * LN;
          o[at_k] = valid(position(k)) ? to_f32(v[k]) : 0.f;
        }
      };
      if (checked) each([&](int at_t) { return f.valid(at_t); });
      else each([](int) { return true; });
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
__device__ __forceinline__ Four of4(const float4& f) { return Four{make_float2(f.x, f.y), make_float2(f.z, f.w)}; }
__device__ __forceinline__ float4 to4(const Four& f) { return make_float4(f.lo.x, f.lo.y, f.hi.x, f.hi.y); }
__device__ __forceinline__ Four zero4() { return Four{both(0.f), both(0.f)}; }
__device__ __forceinline__ Four load4(const float* p) { return of4(*reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ void store4(float* p, const Four& f) { *reinterpret_cast<float4*>(p) = to4(f); }
__device__ __forceinline__ Four fma4(const Four& a, const Four& b, const Four& c) { return Four{ffma2(a.lo, b.lo, c.lo), ffma2(a.hi, b.hi, c.hi)}; }
__device__ __forceinline__ Four mul4(const Four& a, float2 b) { return Four{fmul2(a.lo, b), fmul2(a.hi, b)}; }
__device__ __forceinline__ float dot4(const Four& a, const Four& b) {
  const float2 s = ffma2(a.hi, b.hi, fmul2(a.lo, b.lo));
  return s.x + s.y;
}
__device__ __forceinline__ Four decays4(float2 s, const Four& rate) { return Four{decays(s, rate.lo), decays(s, rate.hi)}; }

// Four states of two channels: v[i] is state i of both, as one operand of the instructions with
// which sm_100a multiplies and adds two fp32 values at a time.
struct Eight {
  float2 v[4];
};
__device__ __forceinline__ Eight zero8() {
  Eight r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = both(0.f);
  return r;
}
__device__ __forceinline__ Eight of_channels(const float4& a, const float4& b) {
  return Eight{{make_float2(a.x, b.x), make_float2(a.y, b.y), make_float2(a.z, b.z), make_float2(a.w, b.w)}};
}
__device__ __forceinline__ float4 channel0(const Eight& e) { return make_float4(e.v[0].x, e.v[1].x, e.v[2].x, e.v[3].x); }
__device__ __forceinline__ float4 channel1(const Eight& e) { return make_float4(e.v[0].y, e.v[1].y, e.v[2].y, e.v[3].y); }
// To and from a place of 32 bytes of each thread in shared memory, half of them `half` floats behind.
__device__ __forceinline__ Eight take8(const float* p, int half) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + half);
  return Eight{{make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)}};
}
__device__ __forceinline__ void put8(float* p, int half, const Eight& e) {
  *reinterpret_cast<float4*>(p) = make_float4(e.v[0].x, e.v[0].y, e.v[1].x, e.v[1].y);
  *reinterpret_cast<float4*>(p + half) = make_float4(e.v[2].x, e.v[2].y, e.v[3].x, e.v[3].y);
}
// To and from rows of `padded` fp32 for each channel, on 16 bytes.  n: channels that exist.
__device__ __forceinline__ Eight load8(const float* p, int64_t padded, int n) {
  const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
  return of_channels(n > 0 ? *reinterpret_cast<const float4*>(p) : z, n > 1 ? *reinterpret_cast<const float4*>(p + padded) : z);
}
__device__ __forceinline__ void store8(float* p, int64_t padded, int n, const Eight& e) {
  if (n > 0) *reinterpret_cast<float4*>(p) = channel0(e);
  if (n > 1) *reinterpret_cast<float4*>(p + padded) = channel1(e);
}
// A row of the states (rows, dim, dstate) at channel ch, states n0 .. n0 + 3.
__device__ __forceinline__ float4 load_state(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate) {
  const float* p = static_cast<const float*>(t.data) + row * t.s0 + ch * t.s1;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = n0 + i < dstate ? p[(n0 + i) * t.s2] : 0.f;
  return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_state(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate, const float4& f) {
  float* p = static_cast<float*>(t.data) + row * t.s0 + ch * t.s1;
  const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + i < dstate) p[(n0 + i) * t.s2] = v[i];
}
// The same for the channels ch and ch + 1, n of which exist; zero without the tensor or the row.
__device__ __forceinline__ Eight load_states(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate, int n) {
  const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool is = t.data && row >= 0;
  return of_channels(is && n > 0 ? load_state(t, row, ch, n0, dstate) : z, is && n > 1 ? load_state(t, row, ch + 1, n0, dstate) : z);
}
__device__ __forceinline__ void store_states(const TensorArg& t, int64_t row, int64_t ch, int64_t n0, int64_t dstate, int n, const Eight& e) {
  if (!t.data || row < 0) return;
  if (n > 0) store_state(t, row, ch, n0, dstate, channel0(e));
  if (n > 1) store_state(t, row, ch + 1, n0, dstate, channel1(e));
}
// A[ch, n0 .. n0 + 3] log2(e), so that exp(s A) = 2^(s A log2(e)).
__device__ __forceinline__ float4 load_rates(const TensorArg& A, int64_t ch, int64_t n0, int64_t dstate) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = n0 + i < dstate ? kLog2e * load_any(A.data, A.dtype, ch * A.s0 + (n0 + i) * A.s1) : 0.f;
  return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ Eight load_rates(const SelArgs& a, int64_t ch, int64_t n0, int n) {
  const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
  return of_channels(n > 0 ? load_rates(a.A, ch, n0, a.dstate) : z, n > 1 ? load_rates(a.A, ch + 1, n0, a.dstate) : z);
}
__device__ __forceinline__ Eight decays8(float2 s, const Eight& rate) {
  Eight r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = decays(s, rate.v[i]);
  return r;
}
// Four neighbouring values of shared memory (B or C of a position).
struct Quad {
  float v[4];
};
__device__ __forceinline__ Quad quad(const float* p) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  return Quad{{f.x, f.y, f.z, f.w}};
}
// What a segment's neighbour and those beyond it hand on: x exp(A sum) + e, and e alone where the
// sequence is cut between them (sum infinite) or nothing comes.
__device__ __forceinline__ float handed_on(float x, float rate, float sum, float e) {
  return sum < INFINITY && x != 0.f ? fmaf(exp2f(rate * sum), x, e) : e;
}
// Over segments [from, to) upwards, or with step -1 downwards.
__device__ __forceinline__ Eight handed_over(const SelArgs& a, int64_t b, int64_t from, int64_t to, int64_t step, int64_t ch, int64_t n0, int n, const Eight& rate) {
  Eight x = zero8();
  for (int64_t s = from; s != to; s += step) {
    const int64_t at = (b * a.segments + s) * a.dim + ch;
    const Eight e = load8(a.ends + at * a.padded + n0, a.padded, n);
    const float s0 = n > 0 ? a.steps[at] : 0.f, s1 = n > 1 ? a.steps[at + 1] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x.v[i] = make_float2(handed_on(x.v[i].x, rate.v[i].x, s0, e.v[i].x), handed_on(x.v[i].y, rate.v[i].y, s1, e.v[i].y));
  }
  return x;
}

// The sums over the LN threads of a channel of four positions' values; afterwards thread sl has
// those of positions sl * 4 / LN on, in v[0 .. 4 / LN), or with LN >= 4 that of position sl % 4.
template <int LN>
__device__ __forceinline__ void sum_lanes(float (&v)[4], int sl) {
  if constexpr (LN >= 4) {
    const bool hi = sl & 2;
    const float s0 = hi ? v[0] : v[2], s1 = hi ? v[1] : v[3];
    v[0] = (hi ? v[2] : v[0]) + __shfl_xor_sync(~0u, s0, 2);
    v[1] = (hi ? v[3] : v[1]) + __shfl_xor_sync(~0u, s1, 2);
    const bool odd = sl & 1;
    const float s = odd ? v[0] : v[1];
    v[0] = (odd ? v[1] : v[0]) + __shfl_xor_sync(~0u, s, 1);
#pragma unroll
    for (int bit = 4; bit < LN; bit *= 2) v[0] += __shfl_xor_sync(~0u, v[0], bit);
  } else if constexpr (LN == 2) {
    const bool hi = sl & 1;
    const float s0 = hi ? v[0] : v[2], s1 = hi ? v[1] : v[3];
    v[0] = (hi ? v[2] : v[0]) + __shfl_xor_sync(~0u, s0, 1);
    v[1] = (hi ? v[3] : v[1]) + __shfl_xor_sync(~0u, s1, 1);
  }
}
// Of four positions those that a thread has then, and the first of them; whether it stores them.
template <int LN>
constexpr int kSums = LN >= 4 ? 1 : 4 / LN;
template <int LN>
__device__ __forceinline__ int first_sum(int sl) { return LN >= 4 ? sl & 3 : sl * kSums<LN>; }

}  // namespace cc1d
