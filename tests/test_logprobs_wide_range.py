"""Log probabilities of rows whose logits are of any size that their type holds:
masks by ordinary large negative numbers, rows that hold nothing else, and large
positive logits, against the plain implementation in 64 bits."""

import math

import pytest
import torch

from oracle import serving_oracle as O
from test_serving_ops import BF16, E, F16, F32, LEAST, _gen, _randn, _within


def _equal_or_within(got, want, tol):
    """A logit of -infinity (fp16 has no less than -65504) has log probability -infinity."""
    none = want == -math.inf
    assert (got[none] == -math.inf).all()
    _within(torch.where(none, 0, got), torch.where(none, 0, want), torch.where(none, 0, tol))


def _check(logits, tokens, top):
    from turbopress_amd import token_logprobs
    given, log_sum, off, lp, order, y_top, y_given = O.token_logprobs(logits, tokens, top)
    got = token_logprobs(logits, tokens, top=top)
    # each exponential e^y off by (2 |y| + 4) E; their sum by up to 2^8 additions
    # more, or those of a lane that adds every 64th of the row; the log of 1 + s by
    # what s is, of itself
    near = (4 * off + 300 + logits.shape[1] / 64) * E
    # the hardware's exponential of a result below 2^-126, the least normal number, is
    # 0: each logit may lose so much of the sum, and of the entropy's terms -p log p,
    # which grow with p there, 2^-126 * 126 log 2 < 2^-119
    lse = near * log_sum + logits.shape[1] * 2.0 ** -126
    assert torch.equal(got.top_tokens, order)
    _equal_or_within(got.top_logprobs, lp, lse[:, None] + 4 * E * (y_top.abs() + log_sum[:, None]) + LEAST[F32])
    _equal_or_within(got.logprobs, given, lse + 4 * E * (y_given.abs() + log_sum) + LEAST[F32])
    _within(got.entropy, log_sum + off, near * (log_sum + off) + logits.shape[1] * 2.0 ** -119 + LEAST[F32])
    alone = token_logprobs(logits, tokens)
    assert torch.equal(alone.logprobs, got.logprobs) and torch.equal(alone.entropy, got.entropy)


# (few rows: a wave takes one piece of a row; many: a whole row)
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("mask", [-6e4, -1e9, -1e10, -1e12, -1e20, -1e30, -1e36, -1e37, -5e37, -1e38, -3e38])
@pytest.mark.parametrize("rows,vocab", [(6, 300), (6, 9000), (6, 151936), (300, 20000), (2100, 6000)])
def test_masks_of_large_negative_numbers(cuda, dtype, mask, rows, vocab):
    if dtype == F16 and mask < -7e4:
        mask = mask * 6e4 / 3e38 - 1  # (of its range)
    g = _gen(rows + vocab)
    row, at = torch.arange(rows, device="cuda"), torch.arange(vocab, device="cuda")
    live = 3 * _randn(g, rows, vocab)
    form = (row % 6)[:, None]
    lone = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
    dropped = torch.where(form == 0, torch.rand(rows, vocab, generator=g, device="cuda") > 0.1,  # a grammar's
                          torch.where(form == 1, at < vocab - vocab // 8,                        # a whole beginning
                                      torch.where(form == 2, at != lone,                         # all but one
                                                  torch.where(form == 5, at < vocab - 1, True))))
    # (form 3: one value alone; form 4: a few values, sums of a mask and something)
    several = mask * (1 + torch.randint(0, 4, (rows, vocab), generator=g, device="cuda") * 2.0 ** -5)
    logits = torch.where(dropped, torch.where(form == 4, several, mask), live).to(dtype)
    tokens = torch.where(row % 4 == 0, lone[:, 0], torch.randint(0, vocab, (rows,), generator=g, device="cuda"))
    _check(logits, tokens, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [300, 9000, 40001])
@pytest.mark.parametrize("largest", [4.1e6, 4194303.0, 4194304.0, 5.9e6, 8.5e6, 1e7, 1e12, 1e20, 1e37, 2.3e38, 2.4e38, 3.3e38])
def test_large_logits(cuda, dtype, vocab, largest):
    """The largest is far from 0, on either side, alone or with others beside it."""
    g = _gen(vocab)
    logits = 3 * _randn(g, 300, vocab)
    at = torch.randint(0, vocab, (300, 3), generator=g, device="cuda")
    form = torch.arange(300, device="cuda") % 6
    logits.scatter_(1, at[:, :1], largest)
    logits[form == 1] = logits[form == 1].scatter(1, at[form == 1], largest)
    near = largest * (1 - torch.rand(300, vocab, generator=g, device="cuda") / 64)
    logits[form == 2] = near[form == 2]
    logits[form == 3] = -largest
    logits[form == 4] = -near[form == 4]
    few = largest - 20 * torch.rand(300, vocab, generator=g, device="cuda")
    logits[form == 5] = few[form == 5]
    logits = logits.to(dtype)
    _check(logits, at[:, 0], 5)
    _check(logits[:7], at[:7, 1], 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_log_probabilities_below_the_least(cuda, dtype):
    """3e38 beside -3e38: a log probability below what 32 bits hold is -infinity."""
    from turbopress_amd import token_logprobs
    for rows, vocab in ((3, 9000), (300, 9000)):
        logits = torch.full((rows, vocab), -3e38, dtype=dtype, device="cuda")
        logits[:, 4321] = 3e38
        got = token_logprobs(logits, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=2)
        assert (got.entropy == 0).all() and (got.logprobs == -math.inf).all()
        assert (got.top_logprobs[:, 0] == 0).all() and (got.top_logprobs[:, 1] == -math.inf).all()
        assert (got.top_tokens == torch.tensor([4321, 0], device="cuda")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [300, 9000, 40001])
def test_rows_without_a_distribution_among_large_logits(cuda, vocab):
    """NaN and +infinity are told from large logits in the same row."""
    from turbopress_amd import token_logprobs
    logits = 3 * _randn(_gen(vocab), 300, vocab)
    logits[:, 5:200:3], logits[:, 6:200:5] = -1e30, 3e38
    logits[::4, 250], logits[1::4, 251], logits[2::4] = math.nan, math.inf, -math.inf
    got = token_logprobs(logits, torch.full((300,), 7, device="cuda"), top=2)
    for r in (0, 1):
        assert got.entropy[r::4].isnan().all() and got.logprobs[r::4].isnan().all() and got.top_logprobs[r::4].isnan().all()
    assert (got.entropy[2::4] == 0).all() and (got.logprobs[2::4] == -math.inf).all()
    assert torch.isfinite(got.entropy[3::4]).all() and torch.isfinite(got.top_logprobs[3::4]).all()
