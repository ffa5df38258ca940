"""OncePerDevice of the library's host code, compiled on its own against a device that is always number 0."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sana_b200", "csrc")
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

PROGRAM = r"""
#include <cuda_runtime.h>
static cudaError_t device_zero(int* d) { *d = 0; return cudaSuccess; }
#define cudaGetDevice(d) device_zero(d)
#include "common.cuh"
int main() {
  static sana::OncePerDevice once;
  int wrong = 0;
  {
    auto first = once.first_time();           // this caller sets up ...
    if (!first) wrong |= 1;
    {
      auto second = once.first_time();        // ... and another thread's call comes before it has finished:
      if (!second) wrong |= 2;                // it must not go on to launch what is not set up yet
    }
  }
  auto third = once.first_time();
  if (third) wrong |= 4;
  return wrong;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no nvcc")
def test_set_up_counts_as_done_when_it_is(tmp_path):
    src, exe = tmp_path / "once.cu", tmp_path / "once"
    src.write_text(PROGRAM)
    r = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", CSRC, "-o", str(exe), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(exe)]).returncode == 0
