"""Waits of the tensor-core operators that run out (GPU): the wait gives up after
about a second, the CTA reports it and the host reads the status; the context
stays usable."""

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from conftest import PKG_NAME, ROOT, load_pkg

pytestmark = pytest.mark.gpu

# one warp waits for an arrival that nothing makes, then (flag 0) for one that has been made
SOURCE = r'''
#include "tcgen05.cuh"
using namespace carekv;
__global__ void wait_kernel(int never, int* out) {
  __shared__ uint64_t bar;
  __shared__ int dead;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    dead = 0;
    fence_mbar_init();
    if (!never) mbar_arrive(&bar);
  }
  __syncthreads();
  const bool ok = wait_or(&bar, 0, &dead);
  out[threadIdx.x] = ok;
  __syncthreads();
  report_wait(&dead);
}
extern "C" int run(int never, int* out, int* status) {
  wait_kernel<<<1, 32>>>(never, out);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = take_wait_errors(status, nullptr);
  return static_cast<int>(e);
}
'''


def test_a_wait_that_runs_out_is_reported(tmp_path):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("needs nvcc")
    src, so = tmp_path / "wait.cu", tmp_path / "wait.so"
    src.write_text(SOURCE)
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
                    "-I", os.path.join(ROOT, PKG_NAME, "csrc"), "-o", str(so), str(src), "-lcudart"], check=True)
    lib = ctypes.CDLL(str(so))
    lib.run.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    out = torch.full((32,), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    status = ctypes.c_int(5)
    for never in (0, 1, 0):      # the flag is cleared when it is read
        assert lib.run(never, out.data_ptr(), ctypes.addressof(status)) == 0
        assert out.tolist() == [1 - never] * 32
        assert (status.value != 0) == bool(never)


def test_nothing_to_report():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    ck = load_pkg()
    packed = torch.randint(0, 256, (3001, 1456), device="cuda", dtype=torch.uint8)
    w = ck.PackedWeight(packed, torch.ones(3001, 91, device="cuda").bfloat16(), 32)
    w.matvec(torch.randn(40, 2912, device="cuda").bfloat16())
    q, k = (torch.randn(4, n, 64, device="cuda").half() for n in (8, 300))
    ck.prefix_attention(q.transpose(0, 1), k, k)
    ck.check_operator_errors()
    flags = ck._lib.i32(9)
    assert ck._lib.lib().carekv_check_operator_errors(ctypes.byref(flags),
                                                      torch.cuda.current_stream().cuda_stream) == 0
    assert flags.value == 0
