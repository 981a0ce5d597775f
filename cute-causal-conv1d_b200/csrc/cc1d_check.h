// What the extern "C" launchers share: argument checks and the statuses they return.
#pragma once

#include <cstdarg>
#include <cstdio>

#include "cc1d_launch.h"

namespace cc1d {

inline cc1d_status fail(cc1d_status code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
inline cc1d_status fail(cc1d_status code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  try {
    set_last_error(buf);
  } catch (...) {  // out of memory for the message: the status alone has to do
  }
  return code;
}

inline cc1d_status launched(cudaError_t e, const char* what, int kernels) {
  if (e != cudaSuccess)
    return fail(CC1D_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
  count_launches(kernels);
  return CC1D_OK;
}

inline bool is_float(int dt) { return dt == CC1D_FLOAT32 || dt == CC1D_FLOAT16 || dt == CC1D_BFLOAT16; }
constexpr int64_t kMax31 = (int64_t{1} << 31) - 1;

// Sizes whose products stay far inside 64 bits, so that the launchers' own arithmetic cannot wrap.
inline bool sizes_ok(int64_t a, int64_t b, int64_t c) {
  return a >= 0 && b >= 0 && c >= 0 && a <= kMax31 && b <= kMax31 && c <= kMax31 &&
         static_cast<double>(a) * static_cast<double>(b) * static_cast<double>(c) < 4e18;
}

inline cc1d_status workspace_ok(const void* ws, int64_t bytes, int64_t need) {
  if (need > 0 && (!ws || bytes < need))
    return fail(CC1D_ERR_VALUE, "workspace too small: %lld bytes needed", (long long)need);
  if (need > 0 && (reinterpret_cast<uintptr_t>(ws) & 15u)) return fail(CC1D_ERR_VALUE, "workspace must be 16-byte aligned");
  return CC1D_OK;
}

inline int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 148;
  }
  return n;
}

}  // namespace cc1d

// For functions whose params are called p.
#define CC1D_REQUIRE(t, name) \
  if (!(t).data) return fail(CC1D_ERR_VALUE, "%s is required", name)
#define CC1D_SAME_TYPE(t, name)                            \
  if ((t).data && (t).dtype != p->x.dtype) return fail(CC1D_ERR_TYPE, "%s must have x's dtype", name)
#define CC1D_FP32(t, name) \
  if ((t).data && (t).dtype != CC1D_FLOAT32) return fail(CC1D_ERR_TYPE, "%s must be float32", name)
#define CC1D_FLOAT(t, name) \
  if ((t).data && !is_float((t).dtype)) return fail(CC1D_ERR_TYPE, "%s must be a float tensor", name)
