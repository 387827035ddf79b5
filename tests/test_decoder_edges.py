"""Decoder operators at values, strides and sizes where a shorter way would show
(the tolerances are those of the operators' other tests)."""

import ctypes
import math

import pytest
import torch

from oracle import decoder_oracle as O
from test_decoder_ops import _attention_tol, _fp8_case, _fp8_tol, _gen, _randn, _within

F16, BF16, F32, F8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
E = 2.0 ** -24


def _ties(d, block, seed):
    """(weights fp32 [d], scales): in every block its largest magnitude, then
    values at ties between two e4m3 codes times the scale, and beside them."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.arange(0, 0x7f, dtype=torch.uint8).view(F8).float()
    mid = (codes[1:] + codes[:-1]) / 2
    w, scales = [], []
    for c in range(0, d, block):
        n = min(block, d - c)
        top = torch.exp(4 * torch.randn(1, generator=g))
        s = top / 448
        v = mid[torch.randint(0, len(mid), (n,), generator=g)] * s
        for away in (math.inf, 0.0):
            v = torch.where(torch.rand(n, generator=g) < 0.3, torch.nextafter(v, torch.tensor(away)), v)
        v[torch.randint(0, n, (1,), generator=g)] = top
        w.append(v * (1 - 2 * torch.randint(0, 2, (n,), generator=g)))
        scales.append(s)
    return torch.cat(w), torch.cat(scales)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [100, 128, 1000, 2560, 9728, 30001])
@pytest.mark.parametrize("block", [128, None])
def test_norm_codes_are_those_of_the_quotient(cuda, d, block):
    """Rows of 1 and -1 without an epsilon have the norm 1, so y is the weight:
    codes are e4m3 of y / scale as a division gives it, at ties too (a product
    with the scale's reciprocal takes one in eight of those to the other side)."""
    from turbopress_amd import rms_norm_fp8
    for seed in range(20):
        w, scales = _ties(d, block or d, seed)
        x = (1 - 2 * torch.randint(0, 2, (2, d), generator=torch.Generator().manual_seed(seed))).float()
        codes, got = rms_norm_fp8(x.to(cuda), w.to(cuda), 0.0, block=block)
        assert torch.equal(got.cpu(), scales.expand(2, -1))
        want = (x * w / scales.repeat_interleave(block or d)[:d]).to(F8)
        assert torch.equal(codes.cpu().contiguous().view(torch.uint8), want.view(torch.uint8)), seed


@pytest.mark.gpu
@pytest.mark.parametrize("block", [128, None])
def test_norm_codes_of_zeros_and_infinities(cuda, block):
    """Signs of zeros stay; a block whose scale is infinite has zeros where y is
    finite and NaN where it is not, as the division has."""
    from turbopress_amd import rms_norm_fp8
    w = torch.ones(256)
    w[3], w[7], w[9], w[200] = 0, -0.0, math.inf, 0
    x = torch.ones(2, 256)
    x[1, 200] = -1
    codes, scales = rms_norm_fp8(x.to(cuda), w.to(cuda), 0.0, block=block)
    s = scales.cpu().repeat_interleave(block or 256, 1)
    want = (x * w / s).to(F8)
    assert torch.isinf(s[:, 0]).all() and torch.isnan(want[:, 9].float()).all()
    assert torch.equal(codes.cpu().float().nan_to_num(7), want.float().nan_to_num(7))
    finite = ~torch.isnan(want.float())
    assert torch.equal(codes.cpu().view(torch.uint8)[finite], want.view(torch.uint8)[finite])
