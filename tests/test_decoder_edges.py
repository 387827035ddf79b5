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


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 4, 20, 40, 100])
def test_fp8_linear_rows_far_apart(cuda, m):
    """The last token of each of m prompts of 2048: rows 5 242 880 codes apart,
    through operand registers and through tiles, with weights as far apart."""
    from turbopress_amd import fp8_linear
    k = 2560
    a, sa, w, sw = _fp8_case(_gen(m), m, 7000, k)
    far = torch.full((m, 2048, k), 0x7f, dtype=torch.uint8, device="cuda").view(F8)
    far[:, -1] = a
    scales = sa[:, None].expand(m, 3, sa.shape[1])[:, -1]
    assert far[:, -1].stride(0) == 2048 * k
    for n in (300, 7000):
        got = fp8_linear(far[:, -1], scales, w[:n], sw[:-(-n // 128)], out_dtype=F32)
        if not 16 < m <= 32:  # (of those, wide weights' rows as they lie and copied ones take different paths)
            assert torch.equal(got, fp8_linear(a, sa, w[:n], sw[:-(-n // 128)], out_dtype=F32))
        want, size = O.fp8_linear(a, sa, w[:n], sw[:-(-n // 128)])
        _within(got, want, _fp8_tol(want, size, k, F32))
    wide = torch.full((70, 2048, k), 0x7f, dtype=torch.uint8, device="cuda").view(F8)
    wide[:, -1] = w[:70]
    assert torch.equal(fp8_linear(a, sa, wide[:, -1], sw[:1], out_dtype=F32), fp8_linear(a, sa, w[:70], sw[:1], out_dtype=F32))


def test_fp8_entry_points_take_rows_far_apart(built_lib):
    """A row stride above 2^22 is copied for the tiles and read in place by few
    rows; only offsets past 64 bits are refused."""
    from turbopress_amd import _lib as L
    lib, p, far = built_lib, ctypes.c_void_p(256), 5242880
    assert lib.tp_fp8_workspace_bytes(1, 300, 2560, p, far, p, 2560) == 0
    assert lib.tp_fp8_workspace_bytes(100, 300, 2560, p, far, p, 2560) == 100 * 2560
    assert lib.tp_fp8_workspace_bytes(100, 300, 2560, p, 2560, p, far) == 300 * 2560

    def fp8(lda, ldw, m=100):
        return lib.tp_fp8_linear(0, m, 300, 2560, p, lda, p, p, ldw, p, None, p, 300, None, 0, None)

    assert fp8(far, 2560) == fp8(2560, far) == L.TP_ERR_WORKSPACE
    assert fp8(1 << 40, 2560) == fp8(2560, 1 << 40) == fp8(1 << 40, 2560, 1) == L.TP_ERR_BAD_DIMS


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_paged_attention_keeps_small_weights(cuda, d, dtype):
    """Tokens of value zero whose scores are the largest, then 8000 whose
    weights are 2^-26 of theirs and which alone make up the output."""
    from turbopress_amd import paged_attention
    g = _gen(d)
    n, first, batch = 8192, 256, 512  # (more heads than workgroups: a wave meets both kinds)
    k = torch.zeros(n // 64, 64, 1, d, dtype=dtype, device="cuda")
    v = (3e4 + 1e4 * torch.rand(n // 64, 64, 1, d, generator=g, device="cuda")).to(dtype)
    k.view(n, d)[:first, 0], v.view(n, d)[:first] = 18, 0
    bt = torch.arange(n // 64, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    q = torch.zeros(batch, 1, d, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    want, size, dots = O.paged_attention(q[:1], k, v, bt[:1], lengths[:1], 1.0)
    assert 0.005 < want.min() and want.max() < 0.05
    got = paged_attention(q, k, v, bt, lengths, scale=1.0)
    _within(got, want.expand(batch, -1, -1), _attention_tol(want, size, dots, d, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_paged_attention_of_values_that_cancel(cuda, d, dtype):
    """Values of either sign whose weighted mean nearly vanishes: the error is of
    the fp32 scores and exponentials and of the output's rounding, not of the
    probabilities' (held in two pieces of the cache's type, 2^-16 of each at
    least)."""
    from turbopress_amd import paged_attention
    g = _gen(d)
    lengths = [2, 5, 33, 400, 3000]
    page, width = 16, -(-3000 // 16)
    bt = torch.randperm(5 * width, generator=g, device="cuda").view(5, width).int()
    k = (_randn(g, 5 * width, page, 2, d) * d ** -0.25).to(dtype)
    v = (1 - 2 * torch.randint(0, 2, (5 * width, page, 2, d), generator=g, device="cuda")).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = _randn(g, 5, 6, d, dtype=dtype)
    want, size, dots = O.paged_attention(q, k, v, bt, n)
    u, least = (2.0 ** -11, 2.0 ** -24) if dtype == F16 else (2.0 ** -8, 2.0 ** -130)
    near = 2 * (d + 8) * E * dots[..., None] + 2.0 ** -18 + 2.0 ** -16
    _within(paged_attention(q, k, v, bt, n), want, u * want.abs() + near * size + least)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_paged_attention_infinite_values(cuda, dtype):
    """A value that is infinite makes its column so where its token has weight,
    whatever that weight is; the other columns and sequences are as without it."""
    from turbopress_amd import paged_attention
    g = _gen(2)
    k, v = (_randn(g, 40, 16, 1, 64, dtype=dtype) for _ in "kv")
    bt = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
    n = torch.tensor([300, 1], dtype=torch.int32, device="cuda")
    q = _randn(g, 2, 4, 64, dtype=dtype)
    clean = paged_attention(q, k, v, bt, n)
    v[20, 0, 0, 9] = -math.inf  # (the second sequence's only token: its weight is 1)
    v[3, 5, 0, 7] = math.inf
    got = paged_attention(q, k, v, bt, n)
    assert (got[0, :, 7] == math.inf).all() and (got[1, :, 9] == -math.inf).all()
    got[0, :, 7], got[1, :, 9] = clean[0, :, 7], clean[1, :, 9]
    assert torch.equal(got, clean)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_paged_attention_keys_without_weight(cuda, dtype):
    """Tokens whose keys are at -infinity have no weight at all, whatever their values."""
    from turbopress_amd import paged_attention
    g = _gen(3)
    k, v = (_randn(g, 700, 16, 1, 64, dtype=dtype) for _ in "kv")
    bt = torch.arange(700, dtype=torch.int32, device="cuda").view(2, 350)
    n = torch.tensor([5600, 4001], dtype=torch.int32, device="cuda")
    q = _randn(g, 2, 4, 64, dtype=dtype).abs()
    none = torch.rand(700, 16, generator=g, device="cuda") < 0.9
    k[none] = -math.inf
    v[none] = 0
    want = paged_attention(q, k, v, bt, n)
    v[none] = 65504
    assert torch.equal(paged_attention(q, k, v, bt, n), want)


def test_rotary_refuses_tokens_of_more_than_31_bits_of_pairs(built_lib):
    """One token of 65536 + 40 heads of 65536 columns, of which two turn."""
    from turbopress_amd import _lib as L
    p, d = ctypes.c_void_p(4096), 65536
    st = built_lib.tp_rotary(0, 1, 65536, 40, d, 2, 0, p, 65536 * d, d, p, 40 * d, d, p, 8, p, p, p, None, 0, 0, None, None,
                             None, None, 0, 1, None, 0, 0, None, None)
    assert st == L.TP_ERR_BAD_DIMS


# (weight rows, activation rows, teams) of a tile -> a call that takes it, of several
# tiles either way and ragged ends, and a K past three of its groups of staged scales
# (8 blocks of 128 columns each, 4 of the largest tile's, per team)
TILES = {(320, 256, 1): (1537, 10000, 1801), (256, 256, 1): (2045, 6000, 3301), (256, 192, 1): (1537, 5000, 3301),
         (128, 128, 1): (400, 10000, 3301), (128, 64, 1): (200, 4100, 3301), (64, 64, 1): (1277, 1597, 3301),
         (64, 64, 2): (70, 150, 6401)}
CODE = {F16: 0, BF16: 1, F32: 2}


def _fp8_plan(dtype, m, n, k, cus):
    from turbopress_amd import _lib
    out = (ctypes.c_int64 * 5)()
    _lib.check(_lib.lib().tp_fp8_plan(CODE[dtype], m, n, k, 1, cus, out), "fp8_plan")
    return tuple(out)


@pytest.mark.gpu
@pytest.mark.parametrize("tile,dtype", [(t, dt) for t in TILES for dt in (F16, BF16, F32) if dt != F32 or t[0] <= 128])
@pytest.mark.parametrize("tail", [True, False])
def test_fp8_linear_every_tile(cuda, tile, tail, dtype):
    """Each tile by the plan's word, at K of no multiple of 16 (NaN behind it) and
    of 16, over all of its rings of stages and scales; scales differ from block to
    block by up to 2^12."""
    from turbopress_amd import fp8_linear
    m, n, k = TILES[tile]
    if not tail:
        k += -k % 16
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert _fp8_plan(dtype, m, n, k, cus)[:4] == (0, *tile)
    g = _gen(m + n + k)
    a, sa, w, sw = _fp8_case(g, m, n, k, -k % 16, -k % 16)
    sa, sw = (s * torch.exp2(torch.randint(-6, 7, s.shape, generator=g, device="cuda").float()) for s in (sa, sw))
    bias = _randn(g, n, dtype=dtype)
    if dtype == F16:  # (inside its range)
        top = O.fp8_linear(a, sa, w, sw)[0].abs().max()
        sa = sa * torch.exp2(-torch.ceil(torch.log2(top / 30000))).float()
    want, size = O.fp8_linear(a, sa, w, sw, bias)
    got = fp8_linear(a, sa, w, sw, bias=bias, out_dtype=dtype)
    _within(got, want, _fp8_tol(want, size, k, dtype))
    assert torch.equal(got, fp8_linear(a, sa, w, sw, bias=bias, out_dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 20])
@pytest.mark.parametrize("n", [150, 17000])
def test_fp8_linear_few_rows_of_long_columns(cuda, m, n):
    """The rows kernel past several rounds of its waves over the columns."""
    from turbopress_amd import fp8_linear
    k = 8165 if n == 150 else 1701
    plan = _fp8_plan(F32, m, n, k, torch.cuda.get_device_properties(0).multi_processor_count)
    g = _gen(m + n)
    a, sa, w, sw = _fp8_case(g, m, n, k, -k % 16, -k % 16)
    sa, sw = (s * torch.exp2(torch.randint(-6, 7, s.shape, generator=g, device="cuda").float()) for s in (sa, sw))
    want, size = O.fp8_linear(a, sa, w, sw)
    _within(fp8_linear(a, sa, w, sw, out_dtype=F32), want, _fp8_tol(want, size, k, F32))
    assert plan[0] == (m <= 16 or n <= 6144) and (not plan[0] or plan[3] == 8)


def test_fp8_plan(built_lib):
    """The plan on 256 compute units, and its refusals."""
    from turbopress_amd import _lib as L
    assert _fp8_plan(F32, 1, 151936, 2560, 256) == (1, 32, 16, 8, 4748)
    assert _fp8_plan(F16, 20, 4096, 300, 256) == (1, 16, 32, 2, 256)
    assert _fp8_plan(F16, 199, 4096, 2560, 256) == (0, 64, 64, 2, 256)
    assert _fp8_plan(BF16, 2048, 9728, 2560, 256) == (0, 320, 256, 1, 248)
    assert _fp8_plan(F32, 2048, 9728, 2560, 256)[1] <= 128
    for tile, (m, n, k) in TILES.items():
        assert _fp8_plan(F32, m, n, k, 256)[1] <= 128  # (fp32 outputs do not take the largest)
        assert _fp8_plan(BF16, m, n, k, 256)[:4] == _fp8_plan(F16, m, n, k + -k % 16, 256)[:4] == (0, *tile)
    out = (ctypes.c_int64 * 5)(7, 7, 7, 7, 7)
    assert built_lib.tp_fp8_plan(3, 1, 1, 1, 1, 256, out) == L.TP_ERR_BAD_TYPE and list(out) == [0] * 5
    assert built_lib.tp_fp8_plan(0, 0, 1, 1, 1, 256, out) == built_lib.tp_fp8_plan(0, 1, 1, 1, 1, 0, out) == L.TP_ERR_BAD_DIMS
    assert built_lib.tp_fp8_plan(0, 1, 1, 0, 1, 256, out) == L.TP_ERR_BAD_DIMS
    assert built_lib.tp_fp8_plan(0, 1, 1, 1, 1, 256, None) == L.TP_ERR_NULL_POINTER
