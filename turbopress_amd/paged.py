"""Rotary positions, the paged cache's writes, and attention of one new token
over it (csrc/tp_rotary.hip, csrc/tp_paged.hip).

A paged cache is two tensors ``k_cache`` and ``v_cache`` [n_pages, page_size,
kv heads, head_dim] (any strides with contiguous head columns, so a [n_pages, kv
heads, page_size, head_dim] store is passed as its transposed view) and a
``block_table`` int32 [sequences, width]: token t of sequence s is slot
``t % page_size`` of page ``block_table[s, t // page_size]``.

The reference decodes over transformers' StaticCache, one sequence of fixed
length (scripts/graph_decode_bench.py:39-60); pages serve many sequences of any
lengths from one store.  Inference only: no gradient flows through.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from turbopress_amd import _lib
from turbopress_amd import hip_kernel as hk
from turbopress_amd.norm import DTYPE_CODES

__all__ = ["rotary_frequencies", "rotary_table", "rotary", "rotary_append", "paged_attention"]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple:
    """(frequencies float64 [rotary_dim / 2], factor of cosines and sines).

    scaling (keys as in transformers' ``rope_scaling``): None; ``linear`` (every
    frequency / factor); ``llama3`` (frequencies of wavelengths above
    original / low_freq_factor / factor, below original / high_freq_factor
    kept, between them blended); ``yarn`` (frequencies that turn fewer than
    beta_slow times over the original length / factor, more than beta_fast
    times kept, a ramp between; cosines and sines times attention_factor or
    0.1 ln(factor) + 1)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    half = rotary_dim // 2
    freq = float(base) ** (-torch.arange(half, dtype=torch.float64) / half)
    kind = None if scaling is None else scaling.get("rope_type", scaling.get("type"))
    if kind in (None, "default"):
        return freq, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r}: linear, llama3 or yarn")
    factor = float(scaling["factor"])
    if not factor > 0:
        raise ValueError(f"a scaling factor above 0 is needed, got {factor}")
    if kind == "linear":
        return freq / factor, 1.0
    original = float(scaling["original_max_position_embeddings"])
    turns = original * freq / (2 * math.pi)  # over the original length
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return freq * keep + freq / factor * (1 - keep), 1.0
    # yarn: the ramp is linear in the index between those of beta_fast and beta_slow turns
    fast, slow = float(scaling.get("beta_fast") or 32), float(scaling.get("beta_slow") or 1)

    def index(t):
        return half * math.log(original / (t * 2 * math.pi)) / math.log(base)

    lo, hi = index(fast), index(slow)
    if scaling.get("truncate", True):
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
    ramp = ((torch.arange(half, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    attention = scaling.get("attention_factor")
    if attention is None:
        attention = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freq * (1 - ramp) + freq / factor * ramp, float(attention)


def rotary_table(n_positions: int, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                 device="cuda") -> Tensor:
    """fp32 [n_positions, rotary_dim]: the cosines, then the sines, of every
    position's angles, formed in 64 bits (an angle formed in fp32 is off by
    2^-24 of the position).  Made once per model."""
    freq, factor = rotary_frequencies(rotary_dim, base, scaling)
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
    return torch.cat((angle.cos(), angle.sin()), 1).mul_(factor).float()


_STRIDES: dict = {}


def _strides(t: Tensor):
    """A tensor's first three strides as the C array the library takes (one
    array per distinct set of strides)."""
    key = t.stride()[:3]
    got = _STRIDES.get(key)
    if got is None:
        got = _STRIDES[key] = (ctypes.c_int64 * 3)(*key)
    return got


def _heads(t: Tensor, name: str, like: Tensor | None = None) -> Tensor:
    """t [tokens, heads, d] with contiguous columns, checked against `like`."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {list(t.shape)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[0] != like.shape[0]
                             or t.shape[2] != like.shape[2]):
        raise ValueError(f"{name} must be {like.dtype} [{like.shape[0]}, heads, {like.shape[2]}] on {like.device}, "
                         f"got {t.dtype} {list(t.shape)} on {t.device}")
    return t if t.stride(2) == 1 else t.contiguous()


def _check_cache(k_cache: Tensor, v_cache: Tensor, block_table: Tensor, like: Tensor) -> None:
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.dtype != like.dtype or c.device != like.device or c.stride(3) != 1 \
                or c.shape[3] != like.shape[2]:
            raise ValueError(f"{name} must be {like.dtype} [pages, page_size, kv heads, {like.shape[2]}] on "
                             f"{like.device} with contiguous columns, got {c.dtype} {list(c.shape)} on {c.device}")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache differ in shape: {list(k_cache.shape)} and {list(v_cache.shape)}")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != like.device \
            or not block_table.is_contiguous():
        raise ValueError(f"block_table must be contiguous int32 [sequences, width] on {like.device}, "
                         f"got {block_table.dtype} {list(block_table.shape)} on {block_table.device}")


def _rotary(q, k, v, table, positions, k_cache, v_cache, block_table, sequences, interleaved, what):
    q = _heads(q, "q")
    code = DTYPE_CODES.get(q.dtype)
    if code is None:
        raise ValueError(f"q must be fp16, bf16 or fp32, got {q.dtype}")
    tokens, hq, d = q.shape
    dev = q.device
    if table.dtype != torch.float32 or table.dim() != 2 or table.device != dev or not table.is_contiguous():
        raise ValueError(f"table must be contiguous fp32 [positions, rotary_dim] on {dev}, "
                         f"got {table.dtype} {list(table.shape)} on {table.device}")
    rd = table.shape[1]
    if d % 2 or rd < 2 or rd % 2 or rd > d:
        raise ValueError(f"head_dim {d} and rotary_dim {rd} must be even, with 2 <= rotary_dim <= head_dim")
    if positions.shape != (tokens,) or positions.dtype != torch.int64 or positions.device != dev:
        raise ValueError(f"positions must be int64 [{tokens}] on {dev}, "
                         f"got {positions.dtype} {list(positions.shape)} on {positions.device}")
    positions = positions.contiguous()
    hk_ = 0
    k_out = None
    kp = ks0 = ks1 = vp = vs0 = vs1 = kc = vc = 0
    kcp = vcp = btp = sp = n_pages = width = n_seq = 0
    page_size = 1
    if k is not None:
        k = _heads(k, "k", q)
        hk_ = k.shape[1]
        kp, (ks0, ks1, _) = k.data_ptr(), k.stride()
    if k_cache is not None:
        v = _heads(v, "v", k)
        if v.shape != k.shape:
            raise ValueError(f"k and v differ in shape: {list(k.shape)} and {list(v.shape)}")
        _check_cache(k_cache, v_cache, block_table, q)
        if k_cache.shape[2] != hk_:
            raise ValueError(f"the caches hold {k_cache.shape[2]} heads, k has {hk_}")
        if sequences is not None:
            if sequences.shape != (tokens,) or sequences.dtype != torch.int32 or sequences.device != dev:
                raise ValueError(f"sequences must be int32 [{tokens}] on {dev}, "
                                 f"got {sequences.dtype} {list(sequences.shape)} on {sequences.device}")
            sequences = sequences.contiguous()
            sp = sequences.data_ptr()
        elif tokens > block_table.shape[0]:
            raise ValueError(f"{tokens} tokens without sequences need as many rows of block_table, "
                             f"got {block_table.shape[0]}")
        vp, (vs0, vs1, _) = v.data_ptr(), v.stride()
        kcp, vcp, btp = k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr()
        kc, vc = _strides(k_cache), _strides(v_cache)
        n_pages, page_size = k_cache.shape[0], k_cache.shape[1]
        n_seq, width = block_table.shape
    elif k is not None:
        k_out = torch.empty(tokens, hk_, d, dtype=q.dtype, device=dev)
    q_out = torch.empty(tokens, hq, d, dtype=q.dtype, device=dev)
    st = _lib.lib().tp_rotary(
        code, tokens, hq, hk_, d, rd, int(interleaved), q.data_ptr(), q.stride(0), q.stride(1), kp, ks0, ks1,
        table.data_ptr(), table.shape[0], positions.data_ptr(), q_out.data_ptr(),
        0 if k_out is None else k_out.data_ptr(), vp, vs0, vs1, kcp, kc or None, vcp, vc or None, n_pages, page_size, btp,
        width, n_seq, sp, hk.current_stream_ptr(dev))
    _lib.check(st, what)
    return q_out, k_out


def rotary(q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor, interleaved: bool = False) -> tuple:
    """Rotary positions of q [tokens, heads, d] and k [tokens, kv heads, d] (or
    None) in one launch: ``(q_out, k_out)``, contiguous.

    table: fp32 [n_positions, rotary_dim] (``rotary_table``); the first
    rotary_dim columns of a head turn, the rest are copied.  positions: int64
    [tokens].  Pairs are columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where
    interleaved.  A negative position is padding and gives zeros; one past the
    table gives NaN."""
    return _rotary(q, k, None, table, positions, None, None, None, None, interleaved, "rotary")


def rotary_append(q: Tensor, k: Tensor, v: Tensor, table: Tensor, positions: Tensor, k_cache: Tensor, v_cache: Tensor,
                  block_table: Tensor, sequences: Tensor | None = None, interleaved: bool = False) -> Tensor:
    """``rotary`` with the rotated k and v written into a paged cache in the same
    launch; returns the rotated q.

    Token t goes to position positions[t] of sequence sequences[t] (int32
    [tokens]; None: token t is sequence t's).  Padding (a negative position), a
    position past the table or past block_table's width, and a page or a
    sequence that does not exist write nothing."""
    if k is None or v is None or k_cache is None or v_cache is None or block_table is None:
        raise ValueError("rotary_append needs k, v, k_cache, v_cache and block_table")
    return _rotary(q, k, v, table, positions, k_cache, v_cache, block_table, sequences, interleaved, "rotary_append")[0]


def paged_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor,
                    scale: float | None = None, window: int = 0) -> Tensor:
    """Attention of one new token per sequence, q [sequences, heads, d] (fp16 or
    bf16), over its cached tokens [0, lengths[s]), or the last `window` of them:
    [sequences, heads, d], contiguous.  Query head h reads cache head
    h // (heads / kv heads); d is a multiple of 8 up to 256; lengths: int32
    [sequences], on the device (the host never waits for them), a length of 0
    gives zeros; scale: 1 / sqrt(d) by default.

    The new token's own key and value are read from the cache like the others
    (``rotary_append`` first).  Several new tokens of one sequence are several
    rows of q with that sequence's row of block_table and growing lengths."""
    q = _heads(q, "q")
    b, hq, d = q.shape
    dev = q.device
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q must be fp16 or bf16, got {q.dtype}")
    _check_cache(k_cache, v_cache, block_table, q)
    hkv = k_cache.shape[2]
    if d % 8 or not 8 <= d <= 256 or hq < 1 or hkv < 1 or hq % hkv:
        raise ValueError(f"head_dim {d} must be a multiple of 8 up to 256 and {hq} query heads a multiple of {hkv}")
    if block_table.shape[0] != b:
        raise ValueError(f"block_table has {block_table.shape[0]} rows, expected {b}")
    if lengths.shape != (b,) or lengths.dtype != torch.int32 or lengths.device != dev:
        raise ValueError(f"lengths must be int32 [{b}] on {dev}, "
                         f"got {lengths.dtype} {list(lengths.shape)} on {lengths.device}")
    if window < 0:
        raise ValueError(f"window must be 0 (none) or positive, got {window}")
    if (q.data_ptr() | 2 * q.stride(0) | 2 * q.stride(1)) & 15:
        q = q.contiguous()
        if q.data_ptr() & 15:
            q = q.clone()
    lengths = lengths.contiguous()
    out = torch.empty(b, hq, d, dtype=q.dtype, device=dev)
    lib = _lib.lib()
    if b == 0:
        return out
    need = lib.tp_paged_attention_workspace_bytes(b, hq, hkv, d)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    count = lib.tp_paged_attention_counter_bytes(b, hq, hkv, d)
    counters = hk.shared_workspace(dev, count)  # zero between launches, as the split-K sums' counters
    st = lib.tp_paged_attention(
        DTYPE_CODES[q.dtype], b, hq, hkv, d, q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(),
        _strides(k_cache), v_cache.data_ptr(), _strides(v_cache), k_cache.shape[0], k_cache.shape[1],
        block_table.data_ptr(), block_table.shape[1], lengths.data_ptr(),
        1.0 / math.sqrt(d) if scale is None else scale, window, out.data_ptr(),
        ws.data_ptr(), need, counters.data_ptr(), count, hk.current_stream_ptr(dev))
    _lib.check(st, "paged_attention")
    return out
