"""Residual addition, root-mean-square norm and e4m3 quantisation in one kernel (csrc/norm.cu)."""
from __future__ import annotations

import torch

from .. import _C


_CODES = {torch.bfloat16: _C.BF16, torch.float32: _C.F32}


def _rows(t: torch.Tensor) -> bool:
    """Rows that the kernel reads in place: contiguous channels, rows at multiples of 16 bytes that do not overlap."""
    per16 = 16 // t.element_size()
    return (t.stride(1) == 1 and (t.shape[0] == 1 or (t.stride(0) >= t.shape[1] and t.stride(0) % per16 == 0))
            and t.data_ptr() % 16 == 0)


def rms_norm_quant_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                       per_token: bool = False, return_norm: bool = False):
    """x [rows, K] (bf16 or fp32) -> (q e4m3 [rows, K], scale f32 [rows, K/128]); the input of the e4m3 layers.

    With ``residual [rows, K]`` (x's type) the norm is of ``x + residual``, and ``residual`` holds that sum, rounded to its type,
    afterwards (in place).  ``y = h / sqrt(mean(h^2) + eps) * weight`` is computed in fp32 and rounded once, by the rule of
    `per_token_group_quant_fp8`; with ``per_token`` by that of `per_token_quant_fp8` (scale [rows]).  ``return_norm`` appends
    y in x's type, for what reads the layer's input unquantised (a router, bf16 experts).
    K is a multiple of 128 (``per_token``: of 8), at most 16384.  Rows of x and residual may be strided; weight is bf16 or fp32 [K].
    """
    host = _C._host or _C.host()
    if host:
        got = host.norm(x, weight, eps, residual, per_token, return_norm)
        if got is not None:
            return got if type(got) is tuple else _C.check(got)
    # what is not dense, on another device, or refused
    dev = _C.require_cuda(x, weight, residual)
    code, w_code = _CODES.get(x.dtype), _CODES.get(weight.dtype)
    if x.dim() != 2 or code is None:
        raise ValueError("x must be a 2-D bf16 or fp32 tensor")
    rows, K = x.shape
    if weight.dim() != 1 or weight.numel() != K or w_code is None:
        raise ValueError("weight must be a bf16 or fp32 tensor of x's row length")
    if K == 0 or K > 16384 or K % (8 if per_token else 128):
        raise ValueError(f"rows of {K} channels: a multiple of {8 if per_token else 128} up to 16384 is needed")
    x_ptr, x_stride = x.data_ptr(), K
    dense = x.is_contiguous() and x_ptr % 16 == 0
    if not dense:
        if not _rows(x):
            x = x.contiguous() if not x.is_contiguous() else x.clone()
        x_ptr, x_stride = x.data_ptr(), x.stride(0) if rows > 1 else K
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    r_ptr, r_stride = None, K
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError("residual must have x's shape and type")
        r_ptr = residual.data_ptr()
        if not (residual.is_contiguous() and r_ptr % 16 == 0):
            if not _rows(residual):
                raise ValueError("residual is updated in place: its channels must be contiguous and its rows start at multiples of 16 bytes")
            r_stride = residual.stride(0) if rows > 1 else K
    if dense:
        q = torch.empty_like(x, dtype=torch.float8_e4m3fn)
        norm = torch.empty_like(x) if return_norm else None
    else:
        q = torch.empty(rows, K, dtype=torch.float8_e4m3fn, device=dev)
        norm = torch.empty(rows, K, dtype=x.dtype, device=dev) if return_norm else None
    s = torch.empty(rows, dtype=torch.float32, device=dev) if per_token else torch.empty(rows, K // 128, dtype=torch.float32, device=dev)
    args = (x_ptr, x_stride, r_ptr, r_stride, code, weight.data_ptr(), w_code, rows, K, eps, int(per_token), q.data_ptr(), s.data_ptr(),
            None if norm is None else norm.data_ptr(), _C.stream_ptr(dev))
    if dev.index == _C.current_device():
        _C.check(_C.lib().fmoe_rms_norm_quant(*args))
    else:
        with _C.on_device(dev):
            _C.check(_C.lib().fmoe_rms_norm_quant(*args))
    return (q, s, norm) if return_norm else (q, s)


__all__ = ["rms_norm_quant_fp8"]
