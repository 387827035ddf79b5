"""Product of 8-bit floating point activations and weights with a scale for
every 128 columns (csrc/tp_fp8.hip): what stays dense in a packed model, above
all its head, at half of fp16's bytes.

Activations come from ``turbopress_amd.norm.rms_norm_fp8``.  Inference only.
"""

from __future__ import annotations

import torch
from torch import Tensor

from turbopress_amd import _lib
from turbopress_amd.hip_kernel import raw_stream as _raw_stream
from turbopress_amd.norm import DTYPE_CODES, FP8_BLOCK

__all__ = ["fp8_linear", "quantize_fp8_weight"]

F8 = torch.float8_e4m3fn
_F8_MAX = 448.0
_LEAST_SCALE = 2.0 ** -126


@torch.no_grad()
def quantize_fp8_weight(w: Tensor) -> tuple:
    """(codes, scales) of a dense weight [n, k], once at load time: e4m3 codes
    whose rows are padded to whole 128-column blocks in memory (so that they
    are aligned), and fp32 scales [ceil(n / 128), ceil(k / 128)], the largest
    magnitude of each 128 x 128 block / 448 (at least 2^-126)."""
    if w.dim() != 2 or not w.is_floating_point():
        raise ValueError(f"expected a floating-point weight [n, k], got {w.dtype} {list(w.shape)}")
    n, k = w.shape
    kb = -(-k // FP8_BLOCK)
    codes = torch.zeros(n, kb * FP8_BLOCK, dtype=F8, device=w.device)
    scales = torch.empty(-(-n // FP8_BLOCK), kb, dtype=torch.float32, device=w.device)
    step = 128 * FP8_BLOCK  # rows at a time: a head in fp32 would be 1.5 GB
    for r in range(0, n, step):
        part = w[r:r + step].float()
        rows = part.shape[0]
        nb = -(-rows // FP8_BLOCK)
        part = torch.nn.functional.pad(part, (0, kb * FP8_BLOCK - k, 0, nb * FP8_BLOCK - rows))
        part = part.view(nb, FP8_BLOCK, kb, FP8_BLOCK)
        s = (part.abs().amax((1, 3)) / _F8_MAX).clamp(min=_LEAST_SCALE)
        q = (part / s[:, None, :, None]).clamp(-_F8_MAX, _F8_MAX).to(F8)
        codes[r:r + rows] = q.view(nb * FP8_BLOCK, -1)[:rows]
        scales[r // FP8_BLOCK:r // FP8_BLOCK + nb] = s
    return codes[:, :k], scales


def fp8_linear(a: Tensor, a_scales: Tensor, w: Tensor, w_scales: Tensor, bias: Tensor | None = None,
               out_dtype: torch.dtype = torch.float16) -> Tensor:
    """``(a * a_scales) @ (w * w_scales)^T + bias``: a float8_e4m3fn [..., k] with
    scales fp32 [..., ceil(k / 128)], w float8_e4m3fn [n, k] with scales fp32
    [ceil(n / 128), ceil(k / 128)], bias of out_dtype: [..., n] of out_dtype
    (fp16, bf16 or fp32).  The scaled sums of blocks of 128 columns are added in
    fp32 in a fixed order and rounded once.  A block's own sum is in fp32 for fp32
    outputs; for the others it is the 8-bit matrix instructions', good to about
    2^-16 of the result (1.3e-5 rms), well below their rounding.  Rows may lie
    anywhere (any alignment, any distance)."""
    code, index, shape = DTYPE_CODES.get(out_dtype), a.get_device(), a.shape
    n, k = w.shape if w.dim() == 2 else (0, 0)
    kb = -(-k // FP8_BLOCK)
    if code is None or index < 0 or a.dtype is not F8 or w.dtype is not F8 or k < 1 or not shape or shape[-1] != k \
            or a_scales.dtype is not torch.float32 or a_scales.shape != (*shape[:-1], kb) \
            or w_scales.dtype is not torch.float32 or w_scales.shape != (-(-n // FP8_BLOCK), kb) \
            or a_scales.get_device() != index or w.get_device() != index or w_scales.get_device() != index \
            or (bias is not None and (bias.dtype is not out_dtype or bias.shape != (n,) or bias.get_device() != index)):
        _refuse(a, a_scales, w, w_scales, bias, out_dtype)
    flat = a if len(shape) == 2 else a.reshape(-1, k)
    lda, step = flat.stride()
    if step != 1 or lda < k:
        flat = flat.contiguous()
        lda = k
    ldw, step = w.stride()
    if step != 1 or ldw < k:
        w = w.contiguous()
        ldw = k
    m = flat.shape[0]
    y = a.new_empty((*shape[:-1], n), dtype=out_dtype)
    lib = _lib.lib()
    ap, wp = flat.data_ptr(), w.data_ptr()
    need = lib.tp_fp8_workspace_bytes(m, n, k, ap, lda, wp, ldw)
    ws = a.new_empty(need, dtype=torch.uint8) if need > 0 else None
    if not a_scales.is_contiguous():
        a_scales = a_scales.contiguous()
    if not w_scales.is_contiguous():
        w_scales = w_scales.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    st = lib.tp_fp8_linear(code, m, n, k, ap, lda, a_scales.data_ptr(), wp, ldw, w_scales.data_ptr(),
                           0 if bias is None else bias.data_ptr(), y.data_ptr(), n,
                           0 if ws is None else ws.data_ptr(), need, _raw_stream(index))
    if st:
        _lib.check(st, "fp8_linear")
    return y


def _refuse(a, a_scales, w, w_scales, bias, out_dtype) -> None:
    """Raise for arguments that fp8_linear does not take."""
    if not a.is_cuda:
        raise RuntimeError("a must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    if out_dtype not in DTYPE_CODES:
        raise ValueError(f"out_dtype must be fp16, bf16 or fp32, got {out_dtype}")
    if a.dtype != F8 or w.dtype != F8 or w.dim() != 2 or a.dim() < 1 or a.shape[-1] != w.shape[1] or w.shape[1] < 1:
        raise ValueError(f"expected float8_e4m3fn a [..., k] and w [n, k], got {a.dtype} {list(a.shape)} "
                         f"and {w.dtype} {list(w.shape)}")
    n, k = w.shape
    kb, dev = -(-k // FP8_BLOCK), a.device
    if a_scales.dtype != torch.float32 or a_scales.shape != (*a.shape[:-1], kb) or a_scales.device != dev:
        raise ValueError(f"a_scales must be fp32 {[*a.shape[:-1], kb]} on {dev}, "
                         f"got {a_scales.dtype} {list(a_scales.shape)} on {a_scales.device}")
    if w_scales.dtype != torch.float32 or w_scales.shape != (-(-n // FP8_BLOCK), kb) or w_scales.device != dev \
            or w.device != dev:
        raise ValueError(f"w_scales must be fp32 {[-(-n // FP8_BLOCK), kb]} beside w on {dev}, "
                         f"got {w_scales.dtype} {list(w_scales.shape)} on {w_scales.device}")
    raise ValueError(f"bias must be {out_dtype} [{n}] on {dev}, got {bias.dtype} {list(bias.shape)} on {bias.device}")
