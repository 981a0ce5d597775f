// Element-wise mathematics shared by the recurrent-block kernels.
#pragma once

#include "cc1d_common.cuh"

namespace cc1d {

// min(v, most) that keeps a NaN: e / (1 + e) stays finite where exp overflows, and 1 / (1 + e)
// is then zero to working precision.
__device__ __forceinline__ float clamp_exp(float v, float most) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
  return r;
}

// The larger of two, or NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// exp(-u) for 16-bit tensors: 2^v by the hardware's approximation (relative error about 2^-22,
// plus the rounding of v = -u log2(e)), at most 1e30.
//
// fp32 also takes what that rounding loses: -u log2(e) = t + r, with r from two fused
// multiply-adds (the second for the part of log2(e) below fp32), and 2^r = 1 + r ln 2 to
// 2^-40.  u is held within +-85, where sigmoids are 0 and 1 to working precision and neither
// exp nor 1 / (1 + exp) leaves the normal numbers; a NaN passes.
template <typename T>
__device__ __forceinline__ float exp_minus(float u) {
  if constexpr (std::is_same<T, float>::value) {
    constexpr double kLog2eExact = 1.4426950408889634074;
    constexpr float kLow = static_cast<float>(kLog2eExact - static_cast<double>(kLog2e));
    u = clamp_exp(max_nan(u, -85.f), 85.f);
    const float t = -kLog2e * u;
    const float r = fmaf(-kLow, u, fmaf(-kLog2e, u, -t));
    const float e = ex2_approx(t);
    return fmaf(e, r * 0.693147181f, e);
  } else {
    return clamp_exp(ex2_approx(-kLog2e * u), 1e30f);
  }
}

// a = sigmoid(u) and c = 1 - a = sigmoid(-u), each to full relative precision.
template <typename T>
__device__ __forceinline__ void sigmoid_pair(float u, float& a, float& c) {
  const float e = exp_minus<T>(u);
  a = rcp_approx(1.f + e);
  c = e * a;
}

template <typename T>
__device__ __forceinline__ float silu_of(float z) {
  return z * rcp_approx(1.f + exp_minus<T>(z));
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
