// The kernels' limits of dynamic shared memory.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <functional>
#include <mutex>
#include <unordered_map>

namespace cc1d {

// The largest limit that each kernel has been given on each device.  A limit is only ever raised:
// a thread that has asked for one may launch at any time after it, and the clustered kernels ask
// for a size per cluster size.
class SmemLimits {
 public:
  cudaError_t raise(const void* kernel, int device, size_t bytes) {
    std::lock_guard<std::mutex> lock(mutex_);
    try {
      size_t& limit = limits_[Key{kernel, device}];
      if (limit >= bytes) return cudaSuccess;
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
      if (e == cudaSuccess) limit = bytes;
      return e;
    } catch (...) {  // no room for the entry
      return cudaErrorMemoryAllocation;
    }
  }

 private:
  struct Key {
    const void* kernel;
    int device;
    bool operator==(const Key& o) const { return kernel == o.kernel && device == o.device; }
  };
  struct Hash {
    size_t operator()(const Key& k) const {
      return std::hash<const void*>()(k.kernel) * 31u + static_cast<size_t>(k.device);
    }
  };
  std::mutex mutex_;
  std::unordered_map<Key, size_t, Hash> limits_;
};

inline cudaError_t raise_smem_limit(const void* kernel, size_t bytes) {
  constexpr size_t kDefault = 48 * 1024;
  if (bytes <= kDefault) return cudaSuccess;
  static SmemLimits limits;
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  return e != cudaSuccess ? e : limits.raise(kernel, device, bytes);
}

}  // namespace cc1d
