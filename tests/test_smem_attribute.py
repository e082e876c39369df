"""CPU: the shared-memory limit of a kernel, set by calls of several threads at once, never falls.

ensure_dynamic_smem (csrc/common.cuh) is compiled against a fake of cudaFuncSetAttribute whose first call, for the
smaller size, is slow: the limit that stands at the end has to hold the larger size, as its caller was told."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "adaptive-kv-memory_b200"))

HARNESS = r"""
#include <cuda_runtime.h>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <thread>
static std::atomic<int> limit{0}, small_in{0};
static cudaError_t fake_set(const void*, cudaFuncAttribute, int bytes) {
  if (bytes == 60000) {
    small_in = 1;
    std::this_thread::sleep_for(std::chrono::milliseconds(300));
  }
  limit = bytes;
  return cudaSuccess;
}
static cudaError_t fake_device(int* d) { *d = 0; return cudaSuccess; }
#define cudaFuncSetAttribute(k, a, b) fake_set((const void*)(k), a, b)
#define cudaGetDevice fake_device
#include "common.cuh"
__global__ void kernel() {}
int main() {
  bool a = false, b = false;
  std::thread t([&] { a = akv::ensure_dynamic_smem<kernel>(60000); });
  while (!small_in) std::this_thread::yield();
  b = akv::ensure_dynamic_smem<kernel>(100000);
  t.join();
  const bool again = akv::ensure_dynamic_smem<kernel>(100000);
  std::printf("%d %d %d %d\n", a, b, again, limit.load());
  return a && b && again && limit >= 100000 ? 0 : 1;
}
"""


def test_two_threads_two_sizes(tmp_path):
    import build
    try:
        nvcc = build.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc here")
    src, exe = tmp_path / "harness.cu", tmp_path / "harness"
    src.write_text(HARNESS)
    r = subprocess.run([nvcc, str(src), "-o", str(exe), *build.flags()], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
