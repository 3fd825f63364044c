"""Kernel launches on a device that lost the kernels' attributes (a reset, another context), and failed ones, with a
stand-in for the CUDA runtime: a small C++ program over the launch helpers, compiled and run here."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
PROGRAM = r"""
#include <cstdio>
#include "capi_internal.cuh"

// The device: whether the kernel's attributes are set, whether launches can work at all, the error left behind.
static bool prepared, broken;
static int prepares, launches;
static cudaError_t left = cudaSuccess;

extern "C" cudaError_t cudaGetDevice(int* d) { *d = 3; return cudaSuccess; }
extern "C" cudaError_t cudaGetLastError() { const cudaError_t e = left; left = cudaSuccess; return e; }
extern "C" cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) {
  ++launches;
  if (prepared && !broken) return cudaSuccess;
  return left = cudaErrorInvalidValue;
}
static void kernel(int) {}
static b2a::OncePerDevice once;
static int call() {
  return once.run([] { ++prepares; return prepared = true; },
                  [] { return b2a::launch_dependent(kernel, dim3(1), 32, 0, 0, 0, 5); });
}
#define CHECK(x) if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }

int main() {
  CHECK(call() == 0 && prepares == 1 && launches == 1);
  CHECK(call() == 0 && prepares == 1 && launches == 2);  // set once
  prepared = false;                                      // the device was reset
  CHECK(call() == 0 && prepares == 2);
  CHECK(left == cudaSuccess);
  CHECK(call() == 0 && prepares == 2);
  broken = true;
  CHECK(call() != 0 && left == cudaSuccess);  // reported by the call, not by the next one
  broken = false;
  CHECK(call() == 0 && left == cudaSuccess);
  left = cudaErrorInvalidDevice;  // somebody else's error: the call works, once, and leaves it to them
  launches = 0;
  CHECK(call() == 0 && launches == 1 && left == cudaErrorInvalidDevice);
  return 0;
}
"""


def test_a_reset_device_is_prepared_again_and_no_error_is_left(tmp_path):
    nvcc, cxx = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc", shutil.which("g++")
    include = Path(nvcc).resolve().parent.parent / "include"
    if not cxx or not (include / "cuda_runtime.h").exists():
        pytest.skip("needs g++ and CUDA's headers")
    (tmp_path / "launch.cpp").write_text(PROGRAM)
    r = subprocess.run([cxx, "-std=c++17", "-I", str(ROOT / "npu_b200" / "csrc"), "-isystem", str(include),
                        str(tmp_path / "launch.cpp"), "-o", str(tmp_path / "launch")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(tmp_path / "launch")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
