"""Attention of drafted trees where scores are so large that fp32 holds them to
whole units and more only: what one token, equal keys, or one far largest score
decide does not depend on that."""

import pytest
import torch

from test_serving_ops import BF16, F16, LEAST, U, _gen, _paged, _randn, _within


def _case(count, group, d, dtype, size, keys):
    """Queries of `size` in every column, keys of `size` times keys[t % len] at token t."""
    g = _gen(count + d)
    lengths = [0, 40, 300]
    k, v, bt = _paged(g, [n + count for n in lengths], 1, d, 16, dtype)
    q = torch.full((3, count, group, d), size, dtype=dtype, device="cuda")
    for s, n in enumerate(lengths):
        for t in range(n + count):
            k[bt[s, t // 16].long(), t % 16] = size * keys[t % len(keys)]
    values = [torch.stack([v[bt[s, t // 16].long(), t % 16, 0] for t in range(n + count)]).double() for s, n in enumerate(lengths)]
    return q, k, v, bt, torch.tensor(lengths, dtype=torch.int32, device="cuda"), lengths, values


SIZES = [(F16, x) for x in (100.0, 1000.0, 3000.0, 10000.0, 60000.0)] + [(BF16, x) for x in (1e3, 1e4, 1e5, 1e7, 1e10, 1e15)]


@pytest.mark.gpu
@pytest.mark.parametrize("count,group", [(5, 2), (24, 1), (20, 3), (40, 4)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype,size", SIZES)
@pytest.mark.parametrize("scale", [None, -0.3])
def test_large_scores(cuda, count, group, d, dtype, size, scale):
    from turbopress_amd import paged_tree_attention
    # a token that sees itself alone answers with its value; of equal keys the mean: sums
    # of up to 2^9 products, each probability in two pieces (2^-16), one rounding
    q, k, v, bt, n, lengths, values = _case(count, group, d, dtype, size, [1.0])
    got = paged_tree_attention(q, k, v, bt, n, window=1, scale=scale)
    for s, m in enumerate(lengths):
        want = values[s][m:, None].expand(-1, group, -1)
        _within(got[s], want, (U[dtype] + 2.0 ** -14) * want.abs() + LEAST[dtype])
    got = paged_tree_attention(q, k, v, bt, n, scale=scale)
    for s, m in enumerate(lengths):
        want = torch.stack([values[s][:m + i + 1].mean(0) for i in range(count)])[:, None].expand(-1, group, -1)
        size_ = torch.stack([values[s][:m + i + 1].abs().mean(0) for i in range(count)])[:, None]
        _within(got[s], want, U[dtype] * want.abs() + 2.0 ** -14 * size_ + LEAST[dtype])
    # one of 32 scores lies above (of a negative scale below) the others by an eighth and more
    ladder = [0.5 + (t * 5 % 32 == 7) * 0.5 - (t % 3) / 8 for t in range(32)]
    q, k, v, bt, n, lengths, values = _case(count, group, d, dtype, size, ladder)
    got = paged_tree_attention(q, k, v, bt, n, scale=scale)
    for s, m in enumerate(lengths):
        for i in range(count):
            at = [ladder[t % 32] for t in range(m + i + 1)]
            best = (max if scale is None else min)(at)
            if size ** 2 * d * (d ** -0.5 if scale is None else 0.3) / 16 < 100:
                continue  # (others still count)
            few = values[s][[t for t, x in enumerate(at) if x == best]]
            want = few.mean(0)[None].expand(group, -1)
            _within(got[s, i], want, U[dtype] * want.abs() + 2.0 ** -14 * few.abs().mean(0) + LEAST[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("count,group", [(5, 2), (24, 1), (20, 3), (40, 4)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (256, F16)])
@pytest.mark.parametrize("window", [0, 20])
def test_rows_of_ordinary_scores_beside_them(cuda, count, group, d, dtype, window):
    """Every third row's queries are 2^15 times the others', of powers of two: its scores are exact."""
    from oracle import serving_oracle as O
    from test_serving_ops import _attention_tol, _trees
    from turbopress_amd import paged_tree_attention
    g = _gen(count + d)
    lengths = [0, 40, 300]
    k, v, bt = _paged(g, [n + count for n in lengths], 1, d, 16, dtype)
    k.copy_(torch.where(k.isnan(), k, (k * 4).round() / 4))  # (quarters up to 2^2: sums of products are exact)
    q = _randn(g, 3, count, group, d, dtype=dtype)
    far = (torch.arange(count * group, device="cuda") % 3 == 1).view(count, group)
    q[:, far] = torch.where(torch.rand(3, int(far.sum()), d, generator=g, device="cuda") < 0.5, -2.0 ** 15, 2.0 ** 15).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ancestors = _trees(g, 3, count)
    args = dict(scale=2.0 ** -3, window=window, sinks=2)
    got = paged_tree_attention(q, k, v, bt, n, ancestors=ancestors, **args)
    want, size, dots = O.paged_tree_attention(q, k, v, bt, n, ancestors, **args)
    tol = _attention_tol(want, size, torch.where(far, 0, dots), d, dtype)
    # (exact scores times log2 e, off by 2^-24 of them: two that differ do by 2^10 at least)
    assert dots[:, far].max() < 2.0 ** 23
    _within(got, want, tol)
