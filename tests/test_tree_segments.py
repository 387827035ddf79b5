"""Attention of drafted trees where a workgroup takes many short sequences, every
second of which holds values that are not finite: one sequence's leave no trace in
the next."""

import math

import pytest
import torch

from test_serving_ops import BF16, F16, _gen, _paged, _randn, _trees


@pytest.mark.gpu
@pytest.mark.parametrize("count,group,batch", [(2, 1, 1500), (5, 3, 900), (16, 1, 900), (9, 2, 900), (16, 4, 900), (24, 6, 600)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (256, F16)])
def test_values_that_are_not_finite_in_every_second_sequence(cuda, count, group, batch, d, dtype):
    from turbopress_amd import paged_tree_attention
    g = _gen(count + group)
    lengths = [(7 * s) % 40 for s in range(batch)]
    k, v, bt = _paged(g, [n + count for n in lengths], 2, d, 16, dtype)
    q = _randn(g, batch, count, 2 * group, d, dtype=dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ancestors = _trees(g, batch, count)
    clean = paged_tree_attention(q, k, v, bt, n, ancestors=ancestors)
    assert torch.isfinite(clean).all()
    # one value of a new token in every second sequence, of its first cache head
    s = torch.arange(0, batch, 2, device="cuda")
    token = s // 2 % count
    at = n[s].long() + token
    value = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype, device="cuda")[s // 2 % 3]
    column = s % d
    v[bt[s, at // 16].long(), at % 16, 0, column] = value
    want = clean.clone()
    sees = (ancestors[s] >> token[:, None] & 1).bool()  # [sequence, row]
    for h in range(group):
        was = want[s[:, None], torch.arange(count, device="cuda"), h, column[:, None]]
        want[s[:, None], torch.arange(count, device="cuda"), h, column[:, None]] = torch.where(sees, value[:, None], was)
    for _ in range(3):
        got = paged_tree_attention(q, k, v, bt, n, ancestors=ancestors)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
