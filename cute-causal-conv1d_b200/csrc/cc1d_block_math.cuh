// Element-wise mathematics shared by the recurrent-block kernels.
#pragma once

#include "cc1d_common.cuh"

namespace cc1d {

// The largest (smallest) of two or three, or NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Within +-87 neither exp nor 1 / (1 + exp) leaves the normal numbers.  An e of at most 2^30 has
// finite products of four 1 + e.
constexpr float kMostExponent = 87.f, kMostBits = 30.f;

// exp(-u) for |u| <= 88: 2^v by the hardware's approximation (relative error about 2^-22) and what
// the rounding of v loses: -u log2(e) = t + r, with r from two fused multiply-adds (the second for
// the part of log2(e) below fp32), and 2^r = 1 + r ln 2 to 2^-40.
__device__ __forceinline__ float exp_minus(float u) {
  constexpr double kLog2eExact = 1.4426950408889634074;
  constexpr float kLow = static_cast<float>(kLog2eExact - static_cast<double>(kLog2e));
  const float t = -kLog2e * u;
  const float r = fmaf(-kLow, u, fmaf(-kLog2e, u, -t));
  const float e = ex2_approx(t);
  return fmaf(e, r * 0.693147181f, e);
}
// Any u, NaN included, brought within +-88: exp(-88) is flushed to zero, as is 1 / (1 + exp(88)).
__device__ __forceinline__ float clamp_exponent(float u) { return min_nan(max_nan(u, -88.f), 88.f); }

// a = 1 / (1 + e) and c = e / (1 + e), to 2^-22 or, with NEWTON, a step of Newton's iteration on
// the residual 1 - a - e a, which takes no rounding of 1 + e, to 2^-24.
template <bool NEWTON>
__device__ __forceinline__ void pair_of_exp(float e, float& a, float& c) {
  a = rcp_approx(1.f + e);
  if constexpr (NEWTON) a = fmaf(a, fmaf(-a, e, 1.f - a), a);
  c = e * a;
}

// a = sigmoid(u) and c = 1 - a = sigmoid(-u) for any u, NaN included, each to full relative
// precision and down to zero.
template <bool NEWTON>
__device__ __forceinline__ void sigmoid_pair(float u, float& a, float& c) {
  pair_of_exp<NEWTON>(exp_minus(clamp_exponent(u)), a, c);
  if (u < -kMostExponent) a = 0.f, c = 1.f;
}
// The same for 16-bit tensors, from t = -u log2(e), whose rounding is left in exp.
__device__ __forceinline__ void sigmoid_pair_of_bits(float t, float& a, float& c) {
  pair_of_exp<true>(ex2_approx(min_nan(t, 126.f)), a, c);
  if (t > 125.f) a = 0.f, c = 1.f;
}
template <typename T>
__device__ __forceinline__ void sigmoid_pair_of(float u, float& a, float& c) {
  if constexpr (std::is_same<T, float>::value) sigmoid_pair<true>(u, a, c);
  else sigmoid_pair_of_bits(-kLog2e * u, a, c);
}

// z sigmoid(z); where exp(-z) is infinite, or large enough for its reciprocal to be flushed, zero.
template <typename T>
__device__ __forceinline__ float silu_of(float z) {
  if constexpr (std::is_same<T, float>::value) return z * rcp_approx(1.f + exp_minus(clamp_exponent(z)));
  else return z * rcp_approx(1.f + ex2_approx(-kLog2e * z));
}

// ---------------------------------------------------------------------- Philox4x32-10
// Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3" (2011):
// four 32-bit words for a 128-bit counter under a 64-bit key.
// N blocks from `block` on together, so that they share the rounds' keys.
template <int N>
__device__ __forceinline__ void philox(uint64_t key, const uint64_t (&block)[N], uint64_t stream, uint32_t (&words)[N][4]) {
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    words[n][0] = static_cast<uint32_t>(block[n]);
    words[n][1] = static_cast<uint32_t>(block[n] >> 32);
    words[n][2] = static_cast<uint32_t>(stream);
    words[n][3] = static_cast<uint32_t>(stream >> 32);
  }
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t(&c)[4] = words[n];
      const uint64_t p0 = static_cast<uint64_t>(c[0]) * 0xD2511F53u;
      const uint64_t p1 = static_cast<uint64_t>(c[2]) * 0xCD9E8D57u;
      c[0] = static_cast<uint32_t>(p1 >> 32) ^ c[1] ^ k0;
      c[1] = static_cast<uint32_t>(p1);
      c[2] = static_cast<uint32_t>(p0 >> 32) ^ c[3] ^ k1;
      c[3] = static_cast<uint32_t>(p0);
    }
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

}  // namespace cc1d
