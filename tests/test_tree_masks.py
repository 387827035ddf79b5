"""Attention of drafted trees under masks of any bits: rows that see new tokens
whose own entry is 0 (they are at the position of the last token before them),
with windows about as long as a row is deep."""

import random

import pytest
import torch

from oracle import serving_oracle as O
from test_serving_ops import BF16, F16, _attention_tol, _bits, _gen, _paged, _randn, _within


def _check(masks, lengths, hq, hkv, d, dtype, window, sinks):
    from turbopress_amd import paged_tree_attention
    count = len(masks[0])
    g = _gen(count + window)
    k, v, bt = _paged(g, [n + count for n in lengths], hkv, d, 16, dtype)
    q = _randn(g, len(lengths), count, hq, d, dtype=dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ancestors = torch.tensor([_bits(m) for m in masks], dtype=torch.int64, device="cuda")
    want, size, dots = O.paged_tree_attention(q, k, v, bt, n, ancestors, None, window, sinks)
    got = paged_tree_attention(q, k, v, bt, n, ancestors=ancestors, window=window, sinks=sinks)
    _within(got, want, _attention_tol(want, size, dots, d, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 3])
@pytest.mark.parametrize("sinks", [0, 11])
def test_a_row_as_deep_as_the_window(cuda, window, sinks):
    """Token 1 sees token 0, whose entry is 0: hidden from it by windows of up to 2."""
    for length in (10, 0, 40):
        _check([[0, 3]], [length], 1, 1, 64, F16, window, sinks)


def _masks(r, count, most):
    """Entries of up to `most` bits, every third one 0."""
    return [0 if r.random() < 0.34 else sum(1 << j for j in r.sample(range(count), r.randint(1, min(most, count)))) for _ in range(count)]


# rows of a cache head up to 16, 32, 64 and 128, and past those in each form
@pytest.mark.gpu
@pytest.mark.parametrize("count,group", [(3, 2), (12, 1), (14, 2), (24, 1), (20, 3), (64, 1), (64, 2), (36, 4), (64, 5)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (256, F16)])
@pytest.mark.parametrize("deeper", [False, True])
def test_masks_of_any_bits(cuda, count, group, d, dtype, deeper):
    """No row deeper than the window, or one beside the others."""
    r = random.Random(count * group)
    lengths = [0, 5, 40, 130, 300]
    for window in (1, 2, 4, 7):
        masks = [_masks(r, count, window) for _ in lengths]
        if deeper:
            for m in masks:
                m[r.randrange(count)] = (1 << count) - 1
        for sinks in (0, 3, 41):
            _check(masks, lengths, group, 1, d, dtype, window, sinks)
