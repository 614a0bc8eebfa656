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


def test_other_python_threads_run_while_a_call_waits_for_its_launch(tmp_path):
    """A launch waits where the stream's queue is full, perhaps for what another thread has yet to launch: the interpreter is free meanwhile."""
    import threading
    import time

    from flaggems_sglang_b200 import _C

    host, cc = _C.host(), shutil.which("gcc")
    if not cc:
        pytest.skip("no gcc")
    assert host, "the compiled module is not built"
    src, so = tmp_path / "slow.c", tmp_path / "slow.so"
    src.write_text("#include <time.h>\nint slow(void) { struct timespec t = {0, 500000000}; nanosleep(&t, 0); return 0; }\n"
                   "long long none(void) { return 0; }\n")
    subprocess.run([cc, "-shared", "-fPIC", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    slow, none = (ctypes.cast(f, ctypes.c_void_p).value for f in (lib.slow, lib.none))
    w, ws = weight(256, 512, 3)
    w13, s13 = weight(256, 512, 4)
    w2, s2 = weight(512, 128, 5)
    x = rows(4, 512, 6).bfloat16()
    calls = [lambda: fg().fp8_block_linear(x, w, ws), lambda: fg().fp8_gated_mlp(x, w13, s13, w2, s2),
             lambda: fg().rms_norm_quant_fp8(x, torch.ones(512, device="cuda"))]
    for call in calls:
        call()
    ticks, done = [], threading.Event()

    def tick():
        while not done.wait(0.005):
            ticks.append(time.perf_counter())

    thread = threading.Thread(target=tick)
    thread.start()
    try:
        host.bind(slow, slow, none, slow, none)
        for call in calls:
            t0 = time.perf_counter()
            call()
            t1 = time.perf_counter()
            assert t1 - t0 > 0.45, "the call did not go through the module"
            assert sum(t0 + 0.05 < t < t1 - 0.05 for t in ticks) > 5
    finally:
        done.set()
        thread.join()
        _C._host = None
        _C.host()  # the library's entry points again
    assert torch.isfinite(calls[0]()).all()
