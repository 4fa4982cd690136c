"""The limit of a kernel's dynamic shared memory, raised by calls of different sizes from several threads: host code, with a
runtime that this test plays."""
import subprocess

from xrgpu_b200 import build

PROGRAM = r"""
#include <chrono>
#include <cstdio>
#include <thread>

#include <cuda_runtime.h>

// as the runtime's header has it for device code
template <class T>
cudaError_t cudaFuncSetAttribute(T* f, cudaFuncAttribute a, int v) { return cudaFuncSetAttribute(reinterpret_cast<const void*>(f), a, v); }

#include "mmnb_internal.h"

static std::atomic<int> limit{0}, asked{0};
static void wait_for(const std::atomic<int>& v, int want) {
  const auto end = std::chrono::steady_clock::now() + std::chrono::milliseconds(300);
  while (v.load() != want && std::chrono::steady_clock::now() < end) std::this_thread::yield();
}

// The larger request takes effect first and returns last.
extern "C" cudaError_t cudaGetDevice(int* dev) { *dev = 0; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int bytes) {
  ++asked;
  if (bytes == 200000) {
    limit = bytes;
    wait_for(limit, 100000);
    std::this_thread::sleep_for(std::chrono::milliseconds(100));
  } else {
    if (bytes == 100000) wait_for(limit, 200000);
    limit = bytes;
  }
  return cudaSuccess;
}

void kernel() {}

int main() {
  cudaError_t results[2];
  std::thread large([&] { results[0] = xrgpu::allow_smem<kernel>(200000); });
  std::thread small([&] { results[1] = xrgpu::allow_smem<kernel>(100000); });
  large.join();
  small.join();
  if (results[0] != cudaSuccess || results[1] != cudaSuccess) return 1;
  for (int bytes : {1000, 100000, 150000, 200000, 220000, 210000}) {
    if (xrgpu::allow_smem<kernel>(bytes) != cudaSuccess) return 2;
    if (limit < bytes) return std::printf("limit %d below the %d promised\n", limit.load(), bytes), 3;
  }
  const int calls = asked;  // none for sizes already allowed
  return xrgpu::allow_smem<kernel>(200000) == cudaSuccess && asked == calls ? 0 : 4;
}
"""


def test_limit_is_never_below_a_promise(tmp_path):
    source, program = tmp_path / "limit.cpp", tmp_path / "limit"
    source.write_text(PROGRAM)
    subprocess.run([build.nvcc(), "-std=c++17", "-cudart", "none", "-Xcompiler", "-pthread", f"-I{build.CSRC}", f"-I{build.INCLUDE}", str(source), "-o", str(program)], check=True)
    res = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, (res.returncode, res.stdout)
