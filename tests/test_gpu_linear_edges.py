"""Calls of the dense e4m3 products that stand in an unusual place: behind a kernel that runs on for long, into their own addend, with
weights that are written just ahead.  Tolerances as in test_gpu_linear.py."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from tests.test_gpu_linear import fg, kernel, quant, rows, status, sum_error, values, weight, weight_values  # noqa: F401

pytestmark = pytest.mark.gpu


def check(out, xv, wv, *parts):
    """out against xv wv^T + parts, all in 64 bits.  The terms of the error's bound are those of the product and every part by itself: bias
    and addend join one after the other, and the sum in between is rounded, off by up to 2^-24 (|product| + |bias|), however much of
    the bias the addend then takes away.  (With |bias + addend| in their place one of 16.8 M outputs, the two of which nearly cancel, is
    1.03e-8 further off than allowed, where 2^-24 |bias| is some 6e-8.)"""
    y, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    for part in parts:
        y, size = y + part.double(), size + part.double().abs()
    off = (out.double() - y).abs()
    allowed = y.abs() * 2.0 ** -8 + size * sum_error(xv.shape[1]) * (1 + 2.0 ** -8)
    assert torch.isfinite(out).all()
    assert (off <= allowed).all(), f"off by {float((off - allowed).max())} more than allowed at {(off > allowed).nonzero()[:4].tolist()}"


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


@pytest.mark.parametrize("T,K,N", [(4100, 256, 4104), (2049, 1280, 4616)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("addend", [False, True])
def test_many_tiles_with_what_joins_the_sums(T, K, N, bias, addend):
    """A worker of the pair kernel has four tiles or so: the boxes of addend and output go round, to ragged ends of both sides."""
    from flaggems_sglang_b200 import _C

    xq, xs = quant(rows(T, K, T))
    w, ws = weight(N, K, N)
    g = torch.Generator(device="cuda").manual_seed(7)
    b = torch.randn(N, generator=g, device="cuda") if bias else None
    a = torch.randn(T, N, generator=g, device="cuda").bfloat16() if addend else None
    try:
        for which in (1, 0):
            _C.check(_C.lib().fmoe_debug_linear_kernel(which, 1))
            out = fg().fp8_block_linear(xq, w, ws, x_scale=xs, bias=b, addend=a)
            check(out, values(xq, xs), weight_values(w, ws), *(part for part in (b, a) if part is not None))
    finally:
        _C.check(_C.lib().fmoe_debug_linear_kernel(0, 0))
    status()


def args_of(_C, x, x_scale, w, w_scale, out, **more):
    T, K = x.shape
    return _C.Fp8Args(x_dtype=_C.BF16 if x.dtype == torch.bfloat16 else _C.E4M3, T=T, K=K, N=out.shape[1], x=x.data_ptr(),
                      x_scale=None if x_scale is None else x_scale.data_ptr(), w=w.data_ptr(), w_scale=w_scale.data_ptr(), out=out.data_ptr(), **more)


@pytest.mark.parametrize("T", [1, 16, 50, 100, 300, 4100])
def test_into_its_own_addend(T, kernel):
    """Through the C entry points, which allow it: product and MLP, the MLP with the bias that it has there alone."""
    from flaggems_sglang_b200 import _C

    K, I, N = 512, 256, 1032
    xq, xs = quant(rows(T, K, T, wide=False))
    w, ws = weight(N, K, 11)
    w13, s13 = weight(2 * I, K, 12)
    w2, s2 = weight(N, I, 13)
    g = torch.Generator(device="cuda").manual_seed(T)
    addend = torch.randn(T, N, generator=g, device="cuda").bfloat16()
    bias = torch.randn(N, generator=g, device="cuda")
    out = addend.clone()
    _C.check(_C.lib().fmoe_fp8_linear(args_of(_C, xq, xs, w, ws, out, addend=out.data_ptr(), bias=bias.data_ptr()), _C.stream_ptr()))
    check(out, values(xq, xs), weight_values(w, ws), bias, addend)
    assert torch.equal(out, fg().fp8_block_linear(xq, w, ws, x_scale=xs, addend=addend, bias=bias))

    h, hs = torch.empty(T, I, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(T, I // 128, device="cuda")
    gate_up = args_of(_C, xq, xs, w13, s13, h, I=I, out_scale=hs.data_ptr())
    _C.check(_C.lib().fmoe_fp8_gate_up(gate_up, _C.stream_ptr()))
    out = addend.clone()
    mlp = args_of(_C, xq, xs, w13, s13, out, I=I, w2=w2.data_ptr(), w2_scale=s2.data_ptr(), addend=out.data_ptr(), bias=bias.data_ptr())
    ws_bytes = _C.lib().fmoe_fp8_mlp_workspace_bytes(mlp)
    ws_mem = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
    mlp.workspace, mlp.workspace_bytes = ws_mem.data_ptr(), ws_bytes
    _C.check(_C.lib().fmoe_fp8_mlp(mlp, _C.stream_ptr()))
    check(out, values(h, hs), weight_values(w2, s2), bias, addend)
    status()


@pytest.mark.parametrize("T", [1, 30, 48, 100, 700])
def test_weights_written_just_ahead(T, kernel):
    """A call loads weights before the kernel ahead of it has ended, but none that this kernel, or one before, has yet to write: weights,
    scales and rows change in stream order just ahead of each call, eager and captured, and are overwritten just behind it."""
    K, I, N = 2048, 1024, 2048
    sets = []
    for seed in range(3):
        (w, ws), (w13, s13), (w2, s2) = weight(N, K, 20 + seed), weight(2 * I, K, 30 + seed), weight(N, I, 40 + seed)
        sets.append([rows(T, K, 50 + seed, wide=False).bfloat16(), w, ws, w13, s13, w2, s2])
    now = [torch.empty_like(t) for t in sets[0]]
    lost = [torch.full_like(t, float("nan")) for t in sets[0]]

    def write(new):
        for a, b in zip(now, new):
            a.view(torch.uint8).copy_(b.view(torch.uint8))

    def calls(x, w, ws, w13, s13, w2, s2):
        xq, xs = fg().per_token_group_quant_fp8(x)
        return [fg().fp8_block_linear(x, w, ws), fg().fp8_gated_mlp(x, w13, s13, w2, s2), fg().fp8_gated_mlp(xq, w13, s13, w2, s2, x_scale=xs)]

    torch.cuda.synchronize()
    want = []
    for s in sets:
        want.append(calls(*s))
        torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    source = [t.clone() for t in sets[0]]
    with torch.cuda.graph(graph):
        write(source)
        replayed = calls(*now)
        write(lost)
    got = []
    for _ in range(5):
        for s in sets:
            write(s)
            got.append(calls(*now))
            write(lost)
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, b in zip(outs, want[i % 3]):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    for i in (1, 2, 0):
        for a, b in zip(source, sets[i]):
            a.view(torch.uint8).copy_(b.view(torch.uint8))
        graph.replay()
        for a, b in zip(replayed, want[i]):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    status()


@pytest.mark.parametrize("T", [1, 48, 300])
def test_weights_written_by_the_kernel_ahead(T, kernel):
    """Likewise by a kernel of this library, which lets its successor start before it has ended."""
    K, I, N = 2048, 1024, 2048
    ws, s13, s2 = (torch.rand(r // 128, c // 128, device="cuda") for r, c in ((N, K), (2 * I, K), (N, I)))
    sets = [[rows(r, c, 60 + 10 * seed + r, wide=False).bfloat16() for r, c in ((T, K), (N, K), (2 * I, K), (N, I))] for seed in range(3)]

    def calls(x, *weights, settle=lambda: None):
        xq, xs = fg().per_token_group_quant_fp8(x)
        out = []
        for run in (lambda w, w13, w2: fg().fp8_block_linear(x, w, ws), lambda w, w13, w2: fg().fp8_gated_mlp(x, w13, s13, w2, s2),
                    lambda w, w13, w2: fg().fp8_gated_mlp(xq, w13, s13, w2, s2, x_scale=xs)):
            q = [fg().per_token_group_quant_fp8(t)[0] for t in weights]
            settle()
            out.append(run(*q))
            for t in q:
                t.view(torch.uint8).fill_(0x7F)  # NaN: the next weights are put where these were
        return out

    want = [calls(*s, settle=torch.cuda.synchronize) for s in sets]
    torch.cuda.synchronize()
    got = [calls(*s) for _ in range(4) for s in sets]
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, b in zip(outs, want[i % 3]):
            assert torch.isfinite(b).all() and torch.equal(a.view(torch.int16), b.view(torch.int16))
    status()


def test_calls_from_several_threads():
    """Each thread with a stream of its own, all kinds of calls at once: what a call gives alone."""
    import threading

    K, I, N = 1024, 512, 1032
    w, ws = weight(N, K, 81)
    w13, s13 = weight(2 * I, K, 82)
    w2, s2 = weight(N, I, 83)
    norm_weight = torch.ones(K, device="cuda")
    inputs = [rows(T, K, 84 + T, wide=False).bfloat16() for T in (1, 20, 48, 100, 400, 2000)]

    def calls(x):
        q, s, _ = fg().rms_norm_quant_fp8(x, norm_weight, return_norm=True)
        y = fg().fp8_block_linear(q, w, ws, x_scale=s)
        return fg().fp8_gated_mlp(x, w13, s13, w2, s2, addend=y)

    want = [calls(x) for x in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(60):
                    j = (i + k) % len(inputs)
                    got = calls(inputs[j])
                    if k % 10 == 9 and not torch.equal(got.view(torch.int16), want[j].view(torch.int16)):
                        wrong.append((i, k))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    status()
