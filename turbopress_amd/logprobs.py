"""Log probabilities of tokens, entropies and the most likely tokens of rows of
logits (csrc/tp_logprobs.hip): what a server answers beside its tokens, and what
checks drafted ones.  Inference only: no gradient flows through.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch import Tensor

from turbopress_amd import _lib
from turbopress_amd.hip_kernel import raw_stream as _raw_stream
from turbopress_amd.norm import DTYPE_CODES
from turbopress_amd.paged import _elsewhere, _workspace

__all__ = ["token_logprobs", "TokenLogprobs", "MAX_TOP"]

MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    """Of each row: the given token's log probability, the entropy (fp32), the
    `top` largest log probabilities (fp32 [rows, top]) and their tokens (int64),
    in falling order, the lower token first of equal ones."""
    logprobs: Tensor | None
    entropy: Tensor
    top_logprobs: Tensor | None
    top_tokens: Tensor | None


@functools.lru_cache(maxsize=1024)
def _needs(rows: int, vocab: int, top: int) -> tuple:
    """(workspace bytes, counter bytes) of a call."""
    lib = _lib.lib()
    return lib.tp_token_logprobs_workspace_bytes(rows, vocab, top), lib.tp_token_logprobs_counter_bytes(rows, vocab, top)


def _refuse(logits: Tensor, tokens: Tensor | None, top: int) -> None:
    """Raise for arguments that token_logprobs does not take."""
    if not logits.is_cuda:
        raise RuntimeError("logits must be a CUDA (ROCm) tensor; turbopress_amd has no CPU path")
    if logits.dtype not in DTYPE_CODES or logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be fp16, bf16 or fp32 [rows, vocabulary], got {logits.dtype} {list(logits.shape)}")
    if not 0 <= top <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"top must lie between 0 and {min(MAX_TOP, logits.shape[1])}, got {top}")
    raise ValueError(f"tokens must be int64 [{logits.shape[0]}] on {logits.device}, "
                     f"got {tokens.dtype} {list(tokens.shape)} on {tokens.device}")


def token_logprobs(logits: Tensor, tokens: Tensor | None = None, top: int = 0) -> TokenLogprobs:
    """Log probabilities (softmax over the vocabulary) of rows of logits [rows,
    vocabulary] (fp16, bf16 or fp32; rows may lie apart): of tokens (int64
    [rows]; a negative one is padding and gives 0, one past the vocabulary NaN),
    of the `top` most likely tokens (up to 64), and the entropy, in nats.

    Sums are fp32; log probabilities near 0 and entropies near 0 keep their
    relative accuracy.  A logit of -infinity has log probability -infinity; where
    every logit of a row is, all have, and the entropy is 0.  A row that holds a
    NaN or +infinity gives NaN; its largest are its NaNs, then +infinity."""
    code, index, shape = DTYPE_CODES.get(logits.dtype), logits.get_device(), logits.shape
    if code is None or index < 0 or len(shape) != 2 or shape[1] < 1 or not 0 <= top <= min(MAX_TOP, shape[1]) \
            or (tokens is not None and (tokens.dtype is not torch.int64 or tokens.shape != shape[:1]
                                        or tokens.get_device() != index)):
        _refuse(logits, tokens, top)
    if _elsewhere(index):
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top)
    rows, vocab = shape
    ld, step = logits.stride()
    if step != 1 and vocab > 1 or ld < 0:
        logits = logits.contiguous()
        ld = vocab
    if tokens is not None and not tokens.is_contiguous():
        tokens = tokens.contiguous()
    lib = _lib.lib()
    out = torch.empty(rows * (2 + top), dtype=torch.float32, device=logits.device)
    ids = torch.empty(rows, top, dtype=torch.int64, device=logits.device) if top else None
    p = out.data_ptr()
    stream = _raw_stream(index)
    need, count = _needs(rows, vocab, top)
    ws, counters, _held = _workspace(index, stream, max(need, 16), count)
    st = lib.tp_token_logprobs(code, rows, vocab, logits.data_ptr(), ld, 0 if tokens is None else tokens.data_ptr(), p,
                               p + 4 * rows, top, p + 8 * rows, 0 if ids is None else ids.data_ptr(), ws, need, counters,
                               count, stream)
    if st:
        _lib.check(st, "token_logprobs")
    return TokenLogprobs(None if tokens is None else out[:rows], out[rows:2 * rows], out[2 * rows:].view(rows, top) if top else None,
                         ids)
