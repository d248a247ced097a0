"""The wait for what is still on its way to a barrier (mbar_drain), which the
kernels end with after a wait that gave up: a small program built here, whose
one arrival comes two milliseconds late, in a phase of either parity. Nothing
is copied, and every wait has a limit."""
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "prefree-public_b200", "csrc")
SOURCE = r"""
#include <cstdio>
#include "pf_ptx.cuh"
using namespace pf::ptx;
// phases 0 .. done - 1 of a barrier of one arrival are complete; warp 1 completes
// the next one late, or never
__global__ void late(int done, int arrive, unsigned *out) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    for (int i = 0; i < done; ++i) mbar_arrive(&bar);
  }
  __syncthreads();
  if (threadIdx.x == 32 && arrive) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
    mbar_arrive(&bar);
  }
  if (threadIdx.x == 0) {
    const uint64_t t0 = globaltimer_ns();
    mbar_drain(&bar, 50000000ull);
    out[0] = mbar_test_wait(&bar, done & 1);  // whether that phase is complete
    out[1] = (unsigned)((globaltimer_ns() - t0) / 1000);
  }
}
int main() {
  unsigned *d, h[2];
  if (cudaMalloc(&d, sizeof h) != cudaSuccess) return 1;
  for (int arrive = 1; arrive >= 0; --arrive)
    for (int done = 0; done < 4; ++done) {
      late<<<1, 64>>>(done, arrive, d);
      if (cudaMemcpy(h, d, sizeof h, cudaMemcpyDeviceToHost) != cudaSuccess) return 1;
      std::printf("%d %d %u %u\n", arrive, done, h[0], h[1]);
    }
  return 0;
}
"""


def test_drain_waits_for_either_phase(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    src, exe = tmp_path / "late.cu", tmp_path / "late"
    src.write_text(SOURCE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-std=c++17",
                    f"-I{CSRC}", str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout
    lines = [tuple(map(int, line.split())) for line in out.splitlines()]
    assert len(lines) == 8
    for arrive, done, complete, us in lines:
        if arrive:
            assert complete == 1, f"returned before the arrival in phase {done}"
        else:
            assert complete == 0 and us < 1000000  # gave up within its limit
