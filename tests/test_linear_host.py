"""Refusals and workspaces of the dense e4m3 products and the norm, on the host: nothing is launched."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def C():
    import __graft_entry__ as ge

    ge.build()
    from flaggems_sglang_b200 import _C

    return _C


def test_struct_layout(C):
    assert ctypes.sizeof(C.Fp8Args) == 4 * 4 + 4 * 8 + 11 * 8 + 8
    assert C.Fp8Args.T.offset == 16 and C.Fp8Args.x.offset == 48 and C.Fp8Args.workspace_bytes.offset == 136
    assert C.Fp8Args().struct_size == ctypes.sizeof(C.Fp8Args)


def bad_args(C, entry, **kw):
    a = C.Fp8Args(**{**dict(x_dtype=C.E4M3, T=3, K=256, N=128, I=128), **kw})
    rc = getattr(C.lib(), entry)(a, None)
    return rc, C.lib().fmoe_last_error().decode()


@pytest.mark.parametrize("entry", ["fmoe_fp8_linear", "fmoe_fp8_gate_up", "fmoe_fp8_mlp"])
@pytest.mark.parametrize("kw,says", [
    (dict(x_dtype=0), "bf16 or e4m3"), (dict(T=-1), "bad sizes"), (dict(K=0), "bad sizes"), (dict(K=200), "multiple of 128"),
    (dict(T=1 << 31), "too large"), (dict(T=1 << 29, N=1 << 28, I=1 << 28), "too large"), (dict(), "null")])
def test_products_refuse(C, entry, kw, says):
    rc, msg = bad_args(C, entry, **kw)
    assert rc == C.ERR_INVALID_ARG and says in msg, msg
    assert entry.split("fmoe_")[1] in msg


def test_products_refuse_widths_and_activations(C):
    assert "multiple of 8" in bad_args(C, "fmoe_fp8_linear", N=12)[1]
    assert "multiple of 128" in bad_args(C, "fmoe_fp8_gate_up", I=64)[1]
    assert "multiple of 128" in bad_args(C, "fmoe_fp8_mlp", I=64)[1]
    assert "multiple of 8" in bad_args(C, "fmoe_fp8_mlp", N=12)[1]
    assert "activation" in bad_args(C, "fmoe_fp8_mlp", activation=2)[1]
    a = C.Fp8Args(x_dtype=C.E4M3, T=3, K=256, N=128)
    a.struct_size -= 8
    assert C.lib().fmoe_fp8_linear(a, None) == C.ERR_INVALID_ARG and b"struct_size" in C.lib().fmoe_last_error()
    assert C.lib().fmoe_fp8_linear(None, None) == C.ERR_INVALID_ARG


def test_misaligned_pointers_and_small_workspaces(C):
    ok = dict(x=4096, x_scale=4096, w=4096, w_scale=4096, out=4096)
    for name in ("x", "w", "out", "bias", "addend"):
        rc, msg = bad_args(C, "fmoe_fp8_linear", **{**ok, name: 4104})
        assert rc == C.ERR_INVALID_ARG and "misaligned" in msg, (name, msg)
    assert "x_scale" in bad_args(C, "fmoe_fp8_linear", **{**ok, "x_scale": None})[1]
    a = C.Fp8Args(x_dtype=C.BF16, T=3, K=256, N=128, I=384, w2=4096, w2_scale=4096, **ok)
    lib = C.lib()
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    assert lib.fmoe_fp8_linear_workspace_bytes(a) == up(3 * 256) + up(3 * 2 * 4) == lib.fmoe_fp8_gate_up_workspace_bytes(a)
    need = lib.fmoe_fp8_mlp_workspace_bytes(a)
    assert need == up(3 * 256) + up(3 * 2 * 4) + up(3 * 384) + up(3 * 3 * 4)
    for ws, size in ((None, need), (4096, need - 1), (4096 + 128, need)):
        a.workspace, a.workspace_bytes = ws, size
        assert lib.fmoe_fp8_mlp(a, None) == C.ERR_INVALID_ARG and b"workspace" in lib.fmoe_last_error()
    a.x_dtype = C.E4M3
    assert lib.fmoe_fp8_linear_workspace_bytes(a) == 0
    a.K = 100
    assert lib.fmoe_fp8_linear_workspace_bytes(a) < 0


def test_no_tokens_is_no_work(C):
    for entry in ("fmoe_fp8_linear", "fmoe_fp8_gate_up", "fmoe_fp8_mlp"):
        assert bad_args(C, entry, T=0)[0] == C.OK


def test_norm_refuses(C):
    def call(x=4096, xs=256, r=None, rs=256, dtype=1, w=4096, wd=1, rows=2, K=256, eps=1e-6, tok=0, q=4096, s=4096, n=None):
        rc = C.lib().fmoe_rms_norm_quant(x, xs, r, rs, dtype, w, wd, rows, K, eps, tok, q, s, n, None)
        return rc, C.lib().fmoe_last_error().decode()

    for kw, says in ((dict(dtype=2), "x must be"), (dict(wd=2), "weight"), (dict(K=200), "multiple of 128"), (dict(K=204, tok=1), "multiple of 8"),
                     (dict(K=16512, xs=16512), "16384"), (dict(rows=-1), "rows"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(xs=255), "strides"),
                     (dict(xs=260), "strides"), (dict(r=4096, rs=128), "strides"), (dict(x=None), "null"), (dict(q=None), "null"),
                     (dict(x=4100), "misaligned"), (dict(r=4104), "misaligned"), (dict(n=4104), "misaligned"), (dict(q=4100), "misaligned")):
        rc, msg = call(**kw)
        assert rc == C.ERR_INVALID_ARG and says in msg, (kw, msg)
    assert call(rows=0, x=None)[0] == C.OK


def test_norm_refuses_a_residual_among_the_rows_of_x(C):
    def call(r, rs=256, xs=256, rows=4, dtype=1, x=1 << 20):
        rc = C.lib().fmoe_rms_norm_quant(x, xs, r, rs, dtype, 4096, 1, rows, 256, 1e-6, 0, 4096, 4096, None, None)
        return rc, C.lib().fmoe_last_error().decode()

    x = 1 << 20
    # one row on, half a row on, before x, another stride, interleaved rows that overlap by 16 bytes, fp32
    for kw in (dict(r=x + 512), dict(r=x + 256), dict(r=x - 512), dict(r=x - 16), dict(r=x, rs=512), dict(r=x + 496, rs=512, xs=512),
               dict(r=x + 528, rs=512, xs=512), dict(r=x + 1024, dtype=0), dict(r=x + 16, rows=1)):
        rc, msg = call(**kw)
        assert rc == C.ERR_INVALID_ARG and "shares memory" in msg, (kw, msg)


def test_gate_up_refuses_what_joins_a_last_product(C):
    for name in ("bias", "addend"):
        assert "join the last product" in bad_args(C, "fmoe_fp8_gate_up", x=4096, **{name: 4096})[1]


def test_ops_refuse_cpu_tensors():
    import flaggems_sglang_b200 as fg

    x, w = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(128, 256).to(torch.float8_e4m3fn)
    for call in (lambda: fg.rms_norm_quant_fp8(x, torch.ones(256)), lambda: fg.fp8_block_linear(x, w, torch.ones(1, 2)),
                 lambda: fg.fp8_gated_mlp(x, w, torch.ones(1, 2), w, torch.ones(1, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_norm_kernels_have_the_registers_that_their_plan_counts_on(C):
    """CTAs an SM that the rows' ring is cut into: three of up to 512 threads, two of up to 576 and of up to 768, without a spill where rows
    have a scale per 128 channels.  An SM has 65536 registers; a thread's are a multiple of eight."""
    import re

    from flaggems_sglang_b200.build import ptxas_report

    found = {}
    for name, spills, regs in re.findall(r"Compiling entry function '(\S+)'.*?(\d+) bytes spill stores.*?Used (\d+) registers",
                                         open(ptxas_report("norm.cu")).read(), flags=re.S):
        kernel = re.search(r"stream_kernelILb([01])ELi(\d+)E", name)
        if kernel:
            found[kernel[1] == "1", int(kernel[2])] = int(spills), -(-int(regs) // 8) * 8
    assert set(found) == {(False, 512), (False, 768), (False, 1024), (True, 512), (True, 1024)}
    for (per_token, most), (spills, regs) in found.items():
        for threads, ctas in {512: ((512, 3),), 768: ((768, 2),), 1024: ((1024, 1), (576, 2))}[most]:
            assert regs * threads * ctas <= 65536, (per_token, most, regs)
        assert per_token or spills == 0
