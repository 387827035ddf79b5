"""Root-mean-square norm of a decoder layer, with the residual's addition, its
output in the input's type or in 8-bit floating point (csrc/tp_norm.hip).

The reference leaves these to the HF decoder between its packed projections
(scripts/graph_decode_bench.py:86-115), which runs them as five to eight
elementwise launches each.  Inference only: no gradient flows through.
"""

from __future__ import annotations

import torch
from torch import Tensor

from turbopress_amd import _lib
from turbopress_amd import hip_kernel as hk

__all__ = ["rms_norm", "rms_norm_fp8", "FP8_BLOCK"]

FP8_BLOCK = 128  # columns that share a scale

DTYPE_CODES = {torch.float16: _lib.TP_F16, torch.bfloat16: _lib.TP_BF16, torch.float32: _lib.TP_F32}


def _rows(x: Tensor) -> tuple:
    """(tensor, rows, inner, outer stride, inner stride) of x's rows: row r
    starts at (r // inner) * outer + (r % inner) * inner_stride.  Slices of
    wider tensors are read in place; what two strides cannot say is copied."""
    d = x.shape[-1]
    if x.is_contiguous():
        return x, x.numel() // d if d else 0, 1, d, 0
    if x.dim() <= 3 and (x.stride(-1) == 1 or d == 1):
        if x.dim() == 1:
            return x, 1, 1, d, 0
        if x.dim() == 2:
            return x, x.shape[0], 1, x.stride(0), 0
        return x, x.shape[0] * x.shape[1], max(1, x.shape[1]), x.stride(0), x.stride(1)
    x = x.contiguous()
    return x, x.numel() // d if d else 0, 1, d, 0


def _check(x: Tensor, weight: Tensor, residual: Tensor | None) -> int:
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    code = DTYPE_CODES.get(x.dtype)
    if code is None:
        raise ValueError(f"x must be fp16, bf16 or fp32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs a last dimension of at least 1")
    if weight.dtype != x.dtype or weight.device != x.device or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must be {x.dtype} [{x.shape[-1]}] on {x.device}, "
                         f"got {weight.dtype} {list(weight.shape)} on {weight.device}")
    if residual is not None and (residual.dtype != x.dtype or residual.device != x.device or residual.shape != x.shape):
        raise ValueError(f"residual must be {x.dtype} {list(x.shape)} on {x.device}, "
                         f"got {residual.dtype} {list(residual.shape)} on {residual.device}")
    return code


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, residual: Tensor | None = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, in one
    launch: h = x, or x + residual.  Returns y of x's type and shape, and with
    a residual ``(y, h)``.  h enters the norm in fp32; y and h round once."""
    code = _check(x, weight, residual)
    xr, rows, inner, outer, step = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h, rp, ro, rs = None, 0, 0, 0
    if residual is not None:
        r, _, r_inner, ro, rs = _rows(residual)
        if r_inner != inner:  # (one of the two is contiguous: say its rows as the other's)
            xr, r = xr.contiguous(), r.contiguous()
            inner, outer, step, ro, rs = 1, x.shape[-1], 0, x.shape[-1], 0
        rp = r.data_ptr()
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    st = _lib.lib().tp_rms_norm(code, rows, inner, x.shape[-1], xr.data_ptr(), outer, step, rp, ro, rs,
                                weight.contiguous().data_ptr(), eps, y.data_ptr(), 0 if h is None else h.data_ptr(),
                                hk.current_stream_ptr(x.device))
    _lib.check(st, "rms_norm")
    return y if h is None else (y, h)


def rms_norm_fp8(x: Tensor, weight: Tensor, eps: float = 1e-6, residual: Tensor | None = None,
                 block: int | None = FP8_BLOCK):
    """``rms_norm`` with its output in 8-bit floating point: ``(codes, scales)``,
    with a residual ``(codes, scales, h)``.  codes: float8_e4m3fn of x's shape
    (its rows 16-byte aligned, so not contiguous for odd lengths); scales: fp32
    [..., ceil(d / 128)], or [..., 1] with block=None; y = code * scale."""
    if block not in (None, FP8_BLOCK):
        raise ValueError(f"block must be {FP8_BLOCK} or None (a scale per row), got {block}")
    code = _check(x, weight, residual)
    d = x.shape[-1]
    xr, rows, inner, outer, step = _rows(x)
    ldc = -(-d // 16) * 16
    lead = x.shape[:-1]
    codes = torch.empty(*lead, ldc, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(*lead, -(-d // FP8_BLOCK) if block else 1, dtype=torch.float32, device=x.device)
    h, rp, ro, rs = None, 0, 0, 0
    if residual is not None:
        r, _, r_inner, ro, rs = _rows(residual)
        if r_inner != inner:
            xr, r = xr.contiguous(), r.contiguous()
            inner, outer, step, ro, rs = 1, d, 0, d, 0
        rp = r.data_ptr()
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    st = _lib.lib().tp_rms_norm_fp8(code, rows, inner, d, xr.data_ptr(), outer, step, rp, ro, rs,
                                    weight.contiguous().data_ptr(), eps, block or 0, codes.data_ptr(), ldc,
                                    scales.data_ptr(), 0 if h is None else h.data_ptr(),
                                    hk.current_stream_ptr(x.device))
    _lib.check(st, "rms_norm_fp8")
    if ldc != d:
        codes = codes[..., :d]
    return (codes, scales) if h is None else (codes, scales, h)
