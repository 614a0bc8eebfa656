"""Dense e4m3 products with block scales: a linear layer, and the gated MLP that a shared expert is (csrc/linear.cu)."""
from __future__ import annotations

import torch

from .. import _C

_ACTIVATIONS = {name: _C.ACTIVATIONS[name] for name in ("silu", "gelu")}


def _input(x: torch.Tensor, x_scale: torch.Tensor | None):
    """-> (rows, their scales or None, T, K, type code): bf16 rows that the call quantises, or e4m3 rows with a scale per 128 channels."""
    if x.dim() != 2:
        raise ValueError("x must be a 2-D tensor")
    T, K = x.shape
    if K == 0 or K % 128:
        raise ValueError(f"rows of {K} channels: a multiple of 128 is needed")
    if not x.is_contiguous() or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    dtype = x.dtype
    if dtype is torch.float8_e4m3fn:
        _check_scale(x_scale, T, K, "e4m3 x needs x_scale, fp32 [rows, K/128]")
        return x, x_scale if x_scale.is_contiguous() else x_scale.contiguous(), T, K, _C.E4M3
    if dtype is not torch.bfloat16:
        raise ValueError("x must be bf16 or e4m3")
    if x_scale is not None:
        raise ValueError("x_scale belongs to e4m3 x")
    return x, None, T, K, _C.BF16


def _check_scale(scale, rows: int, K: int, what: str) -> None:
    if scale is not None and scale.dtype is torch.float32 and scale.dim() == 2:
        r, k = scale.shape
        if r == rows and k * 128 == K:
            return
    raise ValueError(what)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _weight(w: torch.Tensor, scale: torch.Tensor, K: int, name: str):
    """-> (weights, scales, N)"""
    if w.dtype is not torch.float8_e4m3fn or w.dim() != 2:
        raise ValueError(f"{name} must be e4m3 [N, {K}]")
    N, k = w.shape
    if k != K or N == 0:
        raise ValueError(f"{name} must be e4m3 [N, {K}]")
    _check_scale(scale, (N + 127) // 128, K, f"the scales of {name} must be fp32 [ceil(N/128), K/128]")
    if not w.is_contiguous() or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    return w, scale if scale.is_contiguous() else scale.contiguous(), N


def _bias(bias: torch.Tensor, N: int) -> torch.Tensor:
    if bias.shape != (N,) or bias.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("bias must be fp32 or bf16 [N]")
    return _aligned(bias.float())


def _addend(addend: torch.Tensor, T: int, N: int) -> torch.Tensor:
    if addend.shape != (T, N) or addend.dtype is not torch.bfloat16:
        raise ValueError("addend must be bf16 [rows, N]")
    return _aligned(addend)


def _call(run, workspace_bytes, args: _C.Fp8Args, dev: torch.device) -> None:
    """`workspace_bytes`: None where the call needs none."""
    if dev.index != _C.current_device():
        with _C.on_device(dev):
            return _call(run, workspace_bytes, args, dev)
    if workspace_bytes is not None:
        need = workspace_bytes(args)
        if need < 0:
            _C.check(_C.ERR_INVALID_ARG)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
    _C.check(run(args, _C.stream_ptr(dev)))


def fp8_block_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, x_scale: torch.Tensor | None = None,
                     bias: torch.Tensor | None = None, addend: torch.Tensor | None = None) -> torch.Tensor:
    """``x w^T`` for e4m3 ``w [N, K]`` with fp32 ``w_scale [ceil(N/128), K/128]``, one scale per 128 x 128 block -> bf16 [T, N].

    ``x [T, K]`` is bf16, quantised in the call with one scale per token and 128 channels (`per_token_group_quant_fp8`), or e4m3 with
    ``x_scale [T, K/128]`` as `rms_norm_quant_fp8` returns them.  Sums are fp32; ``bias [N]`` and ``addend [T, N]`` (bf16: a
    residual, another branch's output) join them before the one rounding.  K is a multiple of 128, N of 8.
    """
    host = _C._host or _C.host()
    if host:
        out = host.linear(x, w, w_scale, x_scale, bias, addend)
        if out is not None:
            return out if type(out) is not int else _C.check(out)
    # what is not dense, on another device, or refused
    dev = _C.require_cuda(x, w, w_scale, x_scale, bias, addend)
    x, x_scale, T, K, code = _input(x, x_scale)
    w, w_scale, N = _weight(w, w_scale, K, "w")
    if N % 8:
        raise ValueError(f"w has {N} rows: a multiple of 8 is needed")
    if bias is not None:
        bias = _bias(bias, N)
    if addend is not None:
        addend = _addend(addend, T, N)
    out = torch.empty(T, N, dtype=torch.bfloat16, device=dev)
    if T:
        lib = _C.lib()
        _call(lib.fmoe_fp8_linear, None if x_scale is not None else lib.fmoe_fp8_linear_workspace_bytes, _C.Fp8Args.of(
            code, 0, 0, T, K, N, 0, x.data_ptr(), None if x_scale is None else x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), None, None,
            None if bias is None else bias.data_ptr(), None if addend is None else addend.data_ptr(), out.data_ptr()), dev)
    return out


def fp8_gated_mlp(x: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
                  x_scale: torch.Tensor | None = None, activation: str = "silu", addend: torch.Tensor | None = None) -> torch.Tensor:
    """``(act(x Wg^T) * (x Wu^T)) W2^T`` -> bf16 [T, N]: the shared expert beside `fused_moe`, or a dense layer's block.

    ``w13 [2I, K]`` e4m3 (gate rows, then up rows) and ``w2 [N, I]`` e4m3 with fp32 scales per 128 x 128 block; ``x`` and ``x_scale`` as
    in `fp8_block_linear`.  The activation (``silu`` or ``gelu``) is taken in fp32 and quantised with one scale per token and 128
    channels.  ``addend [T, N]`` (bf16) joins the sums: ``fp8_gated_mlp(..., addend=fused_moe(...))`` is the layer's output.
    K and I are multiples of 128, N of 8.
    """
    code = _ACTIVATIONS.get(activation)
    host = _C._host or _C.host()
    if host and code is not None:
        out = host.mlp(x, w13, w13_scale, w2, w2_scale, x_scale, code, addend)
        if out is not None:
            return out if type(out) is not int else _C.check(out)
    dev = _C.require_cuda(x, w13, w13_scale, w2, w2_scale, x_scale, addend)
    if code is None:
        raise ValueError(f"Unsupported activation: {activation}")
    x, x_scale, T, K, x_code = _input(x, x_scale)
    w13, w13_scale, rows = _weight(w13, w13_scale, K, "w13")
    if rows % 256:
        raise ValueError(f"w13 has {rows} rows: 2I with I a multiple of 128 is needed")
    I = rows // 2
    w2, w2_scale, N = _weight(w2, w2_scale, I, "w2")
    if N % 8:
        raise ValueError(f"w2 has {N} rows: a multiple of 8 is needed")
    if addend is not None:
        addend = _addend(addend, T, N)
    out = torch.empty(T, N, dtype=torch.bfloat16, device=dev)
    if T:
        lib = _C.lib()
        _call(lib.fmoe_fp8_mlp, lib.fmoe_fp8_mlp_workspace_bytes, _C.Fp8Args.of(
            x_code, code, 0, T, K, N, I, x.data_ptr(), None if x_scale is None else x_scale.data_ptr(), w13.data_ptr(),
            w13_scale.data_ptr(), w2.data_ptr(), w2_scale.data_ptr(), None, None if addend is None else addend.data_ptr(), out.data_ptr()), dev)
    return out


__all__ = ["fp8_block_linear", "fp8_gated_mlp"]
