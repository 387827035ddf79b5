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
import functools
import math

import torch
from torch import Tensor

from turbopress_amd import _lib
from turbopress_amd import hip_kernel as hk
from turbopress_amd.hip_kernel import raw_stream as _raw_stream
from turbopress_amd.norm import DTYPE_CODES

__all__ = ["rotary_frequencies", "rotary_table", "rotary", "rotary_append", "paged_attention"]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None) -> tuple:
    """(frequencies float64 [rotary_dim / 2], factor of cosines and sines).

    scaling (keys as in transformers' ``rope_scaling``): None; ``linear`` (every
    frequency / factor); ``llama3`` (frequencies of wavelengths above
    original / low_freq_factor / factor, below original / high_freq_factor
    kept, between them blended); ``yarn`` (frequencies that turn fewer than
    beta_slow times over the original length / factor, more than beta_fast
    times kept, a ramp between; cosines and sines times attention_factor or, with
    t(m) = 0.1 m ln(factor) + 1, t(mscale) / t(mscale_all_dim) where both are
    given and t(1) where not)."""
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
        def temperature(m):
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        attention = temperature(m) / temperature(m_all) if m and m_all else temperature(1.0)
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


def _expect(ok: bool, name: str, t, what: str) -> None:
    if not ok:
        got = "None" if t is None else f"{t.dtype} {list(t.shape)} on {t.device}"
        raise ValueError(f"{name} must be {what}, got {got}")


def _refuse(q, k, v, table, positions, k_cache, v_cache, block_table, sequences, lengths=None) -> None:
    """Raise for the first argument that is not as the entry points take it."""
    if not q.is_cuda:
        raise RuntimeError("q must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    _expect(q.dim() == 3, "q", q, "[tokens, heads, head_dim]")
    dt, dev, (tokens, heads, d) = q.dtype, q.device, q.shape
    _expect(dt in DTYPE_CODES and (lengths is None or dt != torch.float32), "q", q,
            "fp16 or bf16" if lengths is not None else "fp16, bf16 or fp32")
    for name, t in (("k", k), ("v", v)):
        if t is not None:
            _expect(t.dtype == dt and t.device == dev and t.dim() == 3 and t.shape[0] == tokens and t.shape[2] == d and
                    (k is None or t.shape == k.shape), name, t, f"{dt} [{tokens}, kv heads, {d}] on {dev}, k like v")
    if lengths is None:
        _expect(table.dtype == torch.float32 and table.device == dev and table.dim() == 2 and table.is_contiguous(), "table",
                table, f"contiguous fp32 [positions, rotary_dim] on {dev}")
        rd = table.shape[1]
        if d % 2 or rd < 2 or rd % 2 or rd > d:
            raise ValueError(f"head_dim {d} and rotary_dim {rd} must be even, with 2 <= rotary_dim <= head_dim")
        _expect(positions.dtype == torch.int64 and positions.device == dev and positions.shape == (tokens,), "positions",
                positions, f"int64 [{tokens}] on {dev}")
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c is not None:
            _expect(c.dtype == dt and c.device == dev and c.dim() == 4 and c.stride(3) == 1 and c.shape[3] == d and
                    c.shape == k_cache.shape and (k is None or c.shape[2] == k.shape[1]), name, c,
                    f"{dt} [pages, page_size, kv heads, {d}] on {dev} with contiguous columns, both caches alike")
    if block_table is not None:
        _expect(block_table.dtype == torch.int32 and block_table.device == dev and block_table.dim() == 2 and
                block_table.is_contiguous(), "block_table", block_table, f"contiguous int32 [sequences, width] on {dev}")
        if sequences is not None:
            _expect(sequences.dtype == torch.int32 and sequences.device == dev and sequences.shape == (tokens,), "sequences",
                    sequences, f"int32 [{tokens}] on {dev}")
        elif block_table.shape[0] < tokens or (lengths is not None and block_table.shape[0] != tokens):
            raise ValueError(f"block_table has {block_table.shape[0]} rows for {tokens} tokens of as many sequences")
    if lengths is not None:
        _expect(lengths.dtype == torch.int32 and lengths.device == dev and lengths.shape == (tokens,), "lengths", lengths,
                f"int32 [{tokens}] on {dev}")
        if d % 8 or not 8 <= d <= 256 or heads < 1 or k_cache.shape[2] < 1 or heads % k_cache.shape[2]:
            raise ValueError(f"head_dim {d} must be a multiple of 8 up to 256 and {heads} query heads a multiple of "
                             f"the caches' {k_cache.shape[2]}")
    raise ValueError("arguments do not belong together")


def _columns(t: Tensor) -> Tensor:
    return t if t.stride(2) == 1 else t.contiguous()


def _turn(q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor) -> tuple:
    """(type code, device index, tokens, heads, d, rotary_dim) of arguments that
    rotary positions take.  (Small calls are bound by the host: the checks
    compare as little as they can; the words are found where one fails.)"""
    code, index = DTYPE_CODES.get(q.dtype), q.get_device()
    if q.dim() == 3 and table.dim() == 2:
        tokens, hq, d = q.shape
        rd = table.shape[1]
        if code is not None and index >= 0 and table.dtype is torch.float32 and table.get_device() == index \
                and table.is_contiguous() and 2 <= rd <= d and not (d | rd) & 1 and positions.dtype is torch.int64 \
                and positions.get_device() == index and positions.shape == (tokens,) and (
                    k is None or (k.dtype is q.dtype and k.get_device() == index and k.dim() == 3 and k.shape[0] == tokens
                                  and k.shape[2] == d)):
            return code, index, tokens, hq, d, rd
    _refuse(q, k, None, table, positions, None, None, None, None)


def _cached(k_cache: Tensor, v_cache: Tensor, block_table: Tensor, q: Tensor, index: int, d: int) -> bool:
    shape = k_cache.shape
    return (k_cache.dtype is q.dtype and v_cache.dtype is q.dtype and len(shape) == 4 and shape[3] == d
            and v_cache.shape == shape and k_cache.stride(3) == 1 and v_cache.stride(3) == 1
            and k_cache.get_device() == index and v_cache.get_device() == index and block_table.dtype is torch.int32
            and block_table.get_device() == index and block_table.dim() == 2 and block_table.is_contiguous())


def rotary(q: Tensor, k: Tensor | None, table: Tensor, positions: Tensor, interleaved: bool = False) -> tuple:
    """Rotary positions of q [tokens, heads, d] and k [tokens, kv heads, d] (or
    None) in one launch: ``(q_out, k_out)``, contiguous.

    table: fp32 [n_positions, rotary_dim] (``rotary_table``); the first
    rotary_dim columns of a head turn, the rest are copied.  positions: int64
    [tokens].  Pairs are columns (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where
    interleaved.  A negative position is padding and gives zeros; one past the
    table gives NaN."""
    code, index, tokens, hq, d, rd = _turn(q, k, table, positions)
    q = _columns(q)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    heads, kp, k_token, k_head, k_out = 0, 0, 0, 0, None
    if k is not None:
        k = _columns(k)
        heads, kp = k.shape[1], k.data_ptr()
        k_token, k_head, _ = k.stride()
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    q_token, q_head, _ = q.stride()
    st = _lib.lib().tp_rotary(code, tokens, hq, heads, d, rd, interleaved, q.data_ptr(), q_token, q_head, kp, k_token, k_head,
                              table.data_ptr(), table.shape[0], positions.data_ptr(), q_out.data_ptr(),
                              0 if k_out is None else k_out.data_ptr(), 0, 0, 0, 0, None, 0, None, 0, 1, 0, 0, 0, 0,
                              _raw_stream(index))
    if st:
        _lib.check(st, "rotary")
    return q_out, k_out


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
    code, index, tokens, hq, d, rd = _turn(q, k, table, positions)
    if v.dtype is not q.dtype or v.get_device() != index or v.shape != k.shape \
            or not _cached(k_cache, v_cache, block_table, q, index, d) or k_cache.shape[2] != k.shape[1] \
            or (sequences is None and tokens > block_table.shape[0]) or (sequences is not None and (
                sequences.dtype is not torch.int32 or sequences.shape != (tokens,) or sequences.get_device() != index)):
        _refuse(q, k, v, table, positions, k_cache, v_cache, block_table, sequences)
    q, k, v = _columns(q), _columns(k), _columns(v)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if sequences is not None and not sequences.is_contiguous():
        sequences = sequences.contiguous()
    pages, page_size, heads, _ = k_cache.shape
    rows, width = block_table.shape
    q_token, q_head, _ = q.stride()
    k_token, k_head, _ = k.stride()
    v_token, v_head, _ = v.stride()
    st = _lib.lib().tp_rotary(code, tokens, hq, heads, d, rd, interleaved, q.data_ptr(), q_token, q_head, k.data_ptr(),
                              k_token, k_head, table.data_ptr(), table.shape[0], positions.data_ptr(), q_out.data_ptr(), 0,
                              v.data_ptr(), v_token, v_head, k_cache.data_ptr(), _strides(k_cache), v_cache.data_ptr(),
                              _strides(v_cache), pages, page_size, block_table.data_ptr(), width, rows,
                              0 if sequences is None else sequences.data_ptr(), _raw_stream(index))
    if st:
        _lib.check(st, "rotary_append")
    return q_out


# Workspaces of paged_attention by (device index, stream): a buffer whose first
# bytes are the counters, zero between calls, and how many those are.  Calls in
# stream order share one; a graph's capture makes its own, whatever its stream
# has here (a graph may be replayed beside eager calls and other graphs).
_WORKSPACES: dict = {}
_COUNTERS = 1 << 16  # bytes of counters at least


@functools.lru_cache(maxsize=1024)
def _needs(index: int, batch: int, hq: int, hkv: int, d: int) -> tuple:
    """(workspace bytes, counter bytes) of a call on a device."""
    lib = _lib.lib()
    return (lib.tp_paged_attention_workspace_bytes(batch, hq, hkv, d), lib.tp_paged_attention_counter_bytes(batch, hq, hkv, d))


def _workspace(index: int, stream: int, need: int, count: int) -> tuple:
    """(workspace pointer, counters pointer, buffers to hold until the launch)."""
    if torch.cuda.is_current_stream_capturing():
        dev = torch.device("cuda", index)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        counters = hk.shared_workspace(dev, count)  # the capture's own; zero between launches, as split-K sums leave it
        return ws.data_ptr(), counters.data_ptr(), (ws, counters)
    got = _WORKSPACES.get((index, stream))
    if got is None or got[1] < count or got[0].numel() - got[1] < need:
        counts = max(_COUNTERS, -(-count // 256) * 256, 0 if got is None else got[1])
        size = max(need, 0 if got is None else got[0].numel() - got[1])
        got = _WORKSPACES[(index, stream)] = (torch.zeros(counts + size, dtype=torch.uint8, device=torch.device("cuda", index)), counts)
    p = got[0].data_ptr()
    return p + got[1], p, got


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
    index = q.get_device()
    code = DTYPE_CODES.get(q.dtype, _lib.TP_F32)
    if window < 0:
        raise ValueError(f"window must be 0 (none) or positive, got {window}")
    if q.dim() != 3 or index < 0 or code == _lib.TP_F32 or not _cached(k_cache, v_cache, block_table, q, index, q.shape[2]) \
            or block_table.shape[0] != q.shape[0] or lengths.dtype is not torch.int32 or lengths.shape != q.shape[:1] \
            or lengths.get_device() != index:
        _refuse(q, None, None, None, None, k_cache, v_cache, block_table, None, lengths)
    b, hq, d = q.shape
    pages, page_size, hkv, _ = k_cache.shape
    if d % 8 or not 8 <= d <= 256 or hq < 1 or hkv < 1 or hq % hkv:
        _refuse(q, None, None, None, None, k_cache, v_cache, block_table, None, lengths)
    q = _columns(q)
    q_row, q_head, _ = q.stride()
    qp = q.data_ptr()
    if (qp | q_row << 1 | q_head << 1) & 15:  # (a row of 16-byte pieces)
        q = q.clone(memory_format=torch.contiguous_format)
        q_row, q_head, qp = hq * d, d, q.data_ptr()
    if not lengths.is_contiguous():
        lengths = lengths.contiguous()
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if b == 0:
        return out
    stream = _raw_stream(index)
    need, count = _needs(index, b, hq, hkv, d)
    ws, counters, _held = _workspace(index, stream, need, count)
    st = _lib.lib().tp_paged_attention(
        code, b, hq, hkv, d, qp, q_row, q_head, k_cache.data_ptr(), _strides(k_cache), v_cache.data_ptr(), _strides(v_cache),
        pages, page_size, block_table.data_ptr(), block_table.shape[1], lengths.data_ptr(),
        d ** -0.5 if scale is None else scale, window, out.data_ptr(), ws, need, counters, count, stream)
    if st:
        _lib.check(st, "paged_attention")
    return out
