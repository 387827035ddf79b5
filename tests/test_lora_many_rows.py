"""Adapters of prompts' rows (more than a tile's rows, several ranks' tiles, parts
of long sums, 64 rows of several adapters together) against the plain
implementation in 64 bits."""

import math

import pytest
import torch

from test_serving_ops import BF16, F16, _check_lora, _gen, _lora_case, _lora_tol, _within


def _ids(g, rows, count, order):
    ids = torch.randint(-1, count + 1, (rows,), generator=g, device="cuda").int()
    return ids if order == "none" else ids.sort().values


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16, 17, 32, 40, 64, 65, 130, 200, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("order", ["runs", "none"])
def test_ranks(cuda, rank, dtype, order):
    g = _gen(rank)
    _check_lora(g, 1087, 1001, 77, rank, 5, dtype, ids=_ids(g, 1087, 5, order))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1023, 1024, 1025, 1087, 1088, 1089, 2047])
@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("order", ["runs", "none"])
def test_rows(cuda, rows, count, order):
    g = _gen(rows + count)
    _check_lora(g, rows, 300, 130, 24, count, F16, ids=_ids(g, rows, count, order))
    _check_lora(g, rows, 300, 130, 24, count, BF16, ids=_ids(g, rows, count, order), scaled=False)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 7, 64, 100, 1001, 2560, 9728, 10001])
@pytest.mark.parametrize("n", [1, 33, 64, 77, 1000])
@pytest.mark.parametrize("rank", [20, 64])
def test_sizes(cuda, k, n, rank):
    g = _gen(k + n)
    _check_lora(g, 1090, k, n, rank, 6, BF16 if n % 2 else F16, ids=_ids(g, 1090, 6, "runs" if k % 2 else "none"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank,k", [(16, 200), (40, 2600), (100, 9728)])
def test_rows_do_not_mix(cuda, dtype, rank, k):
    """NaN and infinity in a row, in an adapter or in the weights of others stay there."""
    from turbopress_amd import lora_add
    rows = 1100
    g = _gen(rank)
    y, x, a, b, _, scales = _lora_case(g, rows, k, 100, rank, 4, dtype)
    row = torch.arange(rows, device="cuda")
    ids = (row % 4).int()
    ids[7::60] = -1
    clean = lora_add(y, x, a, b, ids, scales=scales)
    x[3::64, 5], x[8::64, k - 1], a[1, rank - 1, 4], b[2, 9] = math.nan, math.inf, math.nan, math.inf
    x[ids == -1] = math.nan
    got = lora_add(y, x, a, b, ids, scales=scales)
    bad = ((row % 64 == 3) | (row % 64 == 8)) & (ids >= 0)
    touched = bad | (ids == 1) | (ids == 2)
    assert torch.equal(got[~touched], clean[~touched]) and torch.equal(got[ids == -1], y[ids == -1])
    assert not got[bad].isfinite().any() and got[ids == 1].isnan().all()
    others = torch.arange(100, device="cuda") != 9
    mine = (ids == 2) & ~bad
    assert torch.equal(got[mine][:, others], clean[mine][:, others]) and not got[mine][:, 9].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_leading_dimensions_and_rows_apart(cuda, dtype):
    from oracle import serving_oracle as O
    from turbopress_amd import lora_add
    g = _gen(4)
    y, x, a, b, ids, scales = _lora_case(g, 1200, 700, 130, 33, 5, dtype)
    want, size = O.lora_add(y, x, a, b, ids, scales)
    tol = _lora_tol(want, size, 700, 33, dtype)
    wide = torch.full((1200, 1000), math.nan, dtype=dtype, device="cuda")
    wide[:, 3:703], wide[:, 801:931] = x, y
    for yy, xx, ii in ((y, x, ids), (y.view(12, 100, 130), x.view(12, 100, 700), ids.view(12, 100)), (wide[:, 801:931], wide[:, 3:703], ids)):
        _within(lora_add(yy, xx, a, b, ii, scales=scales).view(1200, 130), want, tol)
