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
from turbopress_amd.hip_kernel import raw_stream as _raw_stream

__all__ = ["rms_norm", "rms_norm_fp8", "FP8_BLOCK"]

FP8_BLOCK = 128  # columns that share a scale

DTYPE_CODES = {torch.float16: _lib.TP_F16, torch.bfloat16: _lib.TP_BF16, torch.float32: _lib.TP_F32}


def _rows(x: Tensor, d: int) -> tuple:
    """(tensor, rows, inner, outer stride, inner stride) of x's rows: row r
    starts at (r // inner) * outer + (r % inner) * inner_stride.  Slices of
    wider tensors are read in place; what two strides cannot say is copied."""
    if not x.is_contiguous():
        if x.dim() <= 3 and (x.stride(-1) == 1 or d == 1):
            if x.dim() == 1:
                return x, 1, 1, d, 0
            if x.dim() == 2:
                return x, x.shape[0], 1, x.stride(0), 0
            return x, x.shape[0] * x.shape[1], max(1, x.shape[1]), x.stride(0), x.stride(1)
        x = x.contiguous()
    return x, x.numel() // d, 1, d, 0


def _refuse(x: Tensor, weight: Tensor, residual: Tensor | None) -> None:
    """Raise for arguments that the norms do not take (x, weight, residual in order)."""
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    if x.dtype not in DTYPE_CODES:
        raise ValueError(f"x must be fp16, bf16 or fp32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs a last dimension of at least 1")
    if weight.dtype != x.dtype or weight.device != x.device or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must be {x.dtype} [{x.shape[-1]}] on {x.device}, "
                         f"got {weight.dtype} {list(weight.shape)} on {weight.device}")
    raise ValueError(f"residual must be {x.dtype} {list(x.shape)} on {x.device}, "
                     f"got {residual.dtype} {list(residual.shape)} on {residual.device}")


def _inputs(x: Tensor, weight: Tensor, residual: Tensor | None) -> tuple:
    """What both entry points take of their checked inputs: (type code, device
    index, d, rows, inner, x, its strides, residual, its strides).  (Small calls
    are bound by the host: the checks compare as little as they can, and the
    words for a refusal are found only once there is one.)"""
    code, index, shape = DTYPE_CODES.get(x.dtype), x.get_device(), x.shape
    if code is None or index < 0 or not shape or weight.dtype is not x.dtype or weight.get_device() != index \
            or weight.shape != shape[-1:] or shape[-1] < 1 or (residual is not None and (
                residual.dtype is not x.dtype or residual.get_device() != index or residual.shape != shape)):
        _refuse(x, weight, residual)
    d = shape[-1]
    x, rows, inner, outer, step = _rows(x, d)
    if residual is None:
        return code, index, d, rows, inner, x, outer, step, None, 0, 0
    residual, _, r_inner, r_outer, r_step = _rows(residual, d)
    if r_inner != inner:  # (one of the two is contiguous: its rows do not say the other's)
        x, residual = x.contiguous(), residual.contiguous()
        inner, outer, step, r_outer, r_step = 1, d, 0, d, 0
    return code, index, d, rows, inner, x, outer, step, residual, r_outer, r_step


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6, residual: Tensor | None = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, in one
    launch: h = x, or x + residual.  Returns y of x's type and shape, and with
    a residual ``(y, h)``.  h enters the norm in fp32; y and h round once."""
    code, index, d, rows, inner, xr, outer, step, res, r_outer, r_step = _inputs(x, weight, residual)
    # (xr holds x's rows; its shape is x's, but for copies' strides)
    y = torch.empty_like(xr, memory_format=torch.contiguous_format)
    h = None if res is None else torch.empty_like(y)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    st = _lib.lib().tp_rms_norm(code, rows, inner, d, xr.data_ptr(), outer, step, 0 if res is None else res.data_ptr(),
                                r_outer, r_step, weight.data_ptr(), eps, y.data_ptr(), 0 if h is None else h.data_ptr(),
                                _raw_stream(index))
    if st:
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
    code, index, d, rows, inner, xr, outer, step, res, r_outer, r_step = _inputs(x, weight, residual)
    ldc = -(-d // 16) * 16
    lead = x.shape[:-1]
    codes = xr.new_empty((*lead, ldc), dtype=torch.float8_e4m3fn)
    scales = xr.new_empty((*lead, -(-d // FP8_BLOCK) if block else 1), dtype=torch.float32)
    h = None if res is None else torch.empty_like(xr, memory_format=torch.contiguous_format)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    st = _lib.lib().tp_rms_norm_fp8(code, rows, inner, d, xr.data_ptr(), outer, step,
                                    0 if res is None else res.data_ptr(), r_outer, r_step, weight.data_ptr(), eps,
                                    block or 0, codes.data_ptr(), ldc, scales.data_ptr(),
                                    0 if h is None else h.data_ptr(), _raw_stream(index))
    if st:
        _lib.check(st, "rms_norm_fp8")
    if ldc != d:
        codes = codes[..., :d]
    return (codes, scales) if h is None else (codes, scales, h)
