"""Calls of the dense e4m3 products that stand in an unusual place: behind a kernel that runs on for long, into their own addend, with
weights that are written just ahead.  Tolerances as in test_gpu_linear.py."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from tests.test_gpu_linear import check, fg, kernel, quant, rows, status, values, weight, weight_values  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def early_trigger(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    so = tmp_path_factory.mktemp("early") / "early_trigger.so"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC", "--cudart", "shared",
                    os.path.join(os.path.dirname(__file__), "early_trigger.cu"), "-o", str(so)], check=True)
    run = ctypes.CDLL(str(so)).early_trigger
    run.argtypes = [ctypes.c_longlong, ctypes.c_void_p]

    def go(clocks):
        assert run(clocks, torch.cuda.current_stream().cuda_stream) == 0

    go(1000)  # loads the module
    torch.cuda.synchronize()
    return go


def test_limit_of_the_waits_does_not_count_the_kernel_before(early_trigger, kernel):
    """A call that starts beside a kernel which runs for longer than the waits' limit (2e9 clocks) gives what it gives alone."""
    T, K, N = 100, 512, 264
    xq, xs = quant(rows(T, K, 1))
    w, ws = weight(N, K, 2)
    want = fg().fp8_block_linear(xq, w, ws, x_scale=xs)
    status()
    early_trigger(2_600_000_000)
    got = fg().fp8_block_linear(xq, w, ws, x_scale=xs)
    status()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
