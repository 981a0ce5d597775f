"""The bookkeeping of the kernels' shared-memory limits, against a fake of the CUDA calls."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cute-causal-conv1d_b200", "csrc")

FAKE = r"""
#pragma once
#include <cstddef>
enum cudaError_t { cudaSuccess = 0, cudaErrorInvalidValue = 1, cudaErrorMemoryAllocation = 2 };
enum cudaFuncAttribute { cudaFuncAttributeMaxDynamicSharedMemorySize = 8 };
cudaError_t cudaGetDevice(int*);
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int);
"""

PROGRAM = r"""
#include "cc1d_smem.h"
#include <atomic>
#include <cstdio>
#include <thread>
#include <vector>

static thread_local int device = 0;
static std::atomic<int> limit[2][4096];
static std::atomic<int> calls{0}, lowered{0}, refuse{0};
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* k, cudaFuncAttribute, int bytes) {
  if (refuse) return cudaErrorInvalidValue;
  ++calls;
  if (limit[device][reinterpret_cast<size_t>(k)].exchange(bytes) > bytes) ++lowered;
  return cudaSuccess;
}
static const void* kernel(size_t i) { return reinterpret_cast<const void*>(i); }

// What a launch does: asks for its size, then needs it to be allowed.
static int launch(size_t k, int bytes) {
  if (cc1d::raise_smem_limit(kernel(k), bytes) != cudaSuccess) return 1;
  return limit[device][k] < bytes && bytes > 48 * 1024;
}

int main() {
  int bad = 0;
  bad += launch(1, 48 * 1024) || calls != 0;  // the default needs no call
  for (int d = 0; d < 2; ++d) {
    device = d;
    for (size_t k = 0; k < 600; ++k)           // many kernels, each with a size for each cluster
      for (int c = 1; c <= 9; ++c) bad += launch(k, 100000 + 2048 * c);
  }
  const int before = calls;
  for (size_t k = 0; k < 600; ++k)
    for (int c = 9; c >= 1; --c) bad += launch(k, 100000 + 2048 * c);  // smaller ones call nothing
  bad += calls != before;
  std::atomic<int> failed{0};
  std::vector<std::thread> threads;
  for (int t = 0; t < 4; ++t)
    threads.emplace_back([&, t] {
      device = t & 1;
      for (int i = 0; i < 20000; ++i) failed += launch(700 + i % 7, 60000 + 512 * ((i * 13 + t * 5) % 90));
    });
  for (auto& t : threads) t.join();
  refuse = 1;
  bad += cc1d::raise_smem_limit(kernel(3000), 60000) != cudaErrorInvalidValue;
  refuse = 0;
  bad += launch(3000, 60000);  // a refusal is not remembered as a limit
  std::printf("%d %d %d\n", bad, failed.load(), lowered.load());
  return 0;
}
"""


def test_limits_are_only_raised(tmp_path):
    (tmp_path / "cuda_runtime.h").write_text(FAKE)
    (tmp_path / "main.cpp").write_text(PROGRAM)
    exe = tmp_path / "main"
    try:
        subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", f"-I{tmp_path}", f"-I{CSRC}", str(tmp_path / "main.cpp"),
                        "-o", str(exe)], check=True, capture_output=True, text=True)
    except OSError:
        pytest.skip("g++ unavailable")
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split() == ["0", "0", "0"]
