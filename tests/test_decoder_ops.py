"""The decoder operators between the packed projections (norm, e4m3 product,
rotary positions, paged attention) against plain 64-bit implementations, and
their refusals.

Tolerances come from the formats.  U[t] is the unit roundoff of type t: an
output that rounds once is off by at most U |y|, beside what the fp32 arithmetic
before it leaves.  E = 2^-24 is fp32's own."""

import math

import pytest
import torch

from oracle import decoder_oracle as O

F16, BF16, F32, F8 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
LEAST = {F16: 2.0 ** -24, BF16: 2.0 ** -130, F32: 2.0 ** -140}  # below the normal numbers
E = 2.0 ** -24
EPS = 1e-6


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _within(got, want, tol):
    """Every element of got within tol of want (both finite)."""
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got.float()).all()
    assert off.max().item() <= 0, f"{off.max().item():.3g} over at {off.argmax().item()} of {off.numel()}"


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
# (a row in 16, 32 or 64 lanes, in 2..8 waves, in several passes; whole vectors
# of 8 and rests of them)
NORM = [(1, 1), (3, 7), (5, 8), (4, 64), (9, 128), (2, 129), (33, 200), (6, 257), (3, 512), (1025, 576), (2, 1000),
        (1, 2560), (3, 2561), (2, 9727), (1500, 2560), (1, 24576), (2, 24577), (1, 60001)]


def _norm_tol(y, dtype):
    # the sum of squares: at most 64 sequential and 10 pairwise additions; its
    # square root halves that; then three products
    return (U[dtype] + 64 * E) * y.abs() + LEAST[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", NORM)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(cuda, rows, d, dtype, residual):
    from turbopress_amd import rms_norm
    g = _gen(rows + d)
    x, w = _randn(g, rows, d, dtype=dtype), (1 + 0.3 * _randn(g, d)).to(dtype)
    r = (5 * _randn(g, rows, d)).to(dtype) if residual else None
    want, h = O.rms_norm(x, w, EPS, r)
    got = rms_norm(x, w, EPS, residual=r)
    if residual:
        assert torch.equal(got[1], (x.float() + r.float()).to(dtype))
        got = got[0]
    assert got.dtype == dtype and got.shape == x.shape
    _within(got, want, _norm_tol(want, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,pad", [(5, 128, 1), (70, 100, 3), (9, 7, 0), (3, 256, 1), (33, 200, 5), (4, 2560, 1), (2000, 2560, 3),
                                        (6, 9727, 0), (3, 9728, 1), (2, 30001, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rms_norm_rows_off_their_words(cuda, rows, d, pad, dtype):
    """Rows of 2-byte elements that begin in the middle of a word, NaN between them."""
    from turbopress_amd import rms_norm, rms_norm_fp8
    g = _gen(rows + d + pad)

    def moved(t, off):
        raw = torch.full((off + rows * (d + pad) + 1,), float("nan"), dtype=dtype, device="cuda")
        out = raw[off:off + rows * (d + pad)].view(rows, d + pad)[:, :d]
        return out.copy_(t)

    x, r, w = _randn(g, rows, d, dtype=dtype), _randn(g, rows, d, dtype=dtype), _randn(g, d, dtype=dtype)
    for off in (0, 1):
        assert torch.equal(rms_norm(moved(x, off), w), rms_norm(x, w))
        for got, want in zip(rms_norm(moved(x, off), w, residual=moved(r, 1 - off)), rms_norm(x, w, residual=r)):
            assert torch.equal(got, want)
        for got, want in zip(rms_norm_fp8(moved(x, off), w, residual=moved(r, 0)), rms_norm_fp8(x, w, residual=r)):
            assert torch.equal(got.float(), want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", NORM)
@pytest.mark.parametrize("dtype,residual", [(F16, True), (BF16, False), (F32, True)])
@pytest.mark.parametrize("block", [128, None])
def test_rms_norm_fp8(cuda, rows, d, dtype, residual, block):
    from turbopress_amd import rms_norm_fp8
    g = _gen(rows + d)
    x, w = _randn(g, rows, d, dtype=dtype), (1 + 0.3 * _randn(g, d)).to(dtype)
    r = (5 * _randn(g, rows, d)).to(dtype) if residual else None
    want, h = O.rms_norm(x, w, EPS, r)
    values, scales = O.block_scales(want, block)
    got = rms_norm_fp8(x, w, EPS, residual=r, block=block)
    assert len(got) == (3 if residual else 2) and got[0].dtype == F8 and got[0].shape == x.shape
    assert got[1].dtype == F32 and got[1].shape == scales.shape
    if residual:
        assert torch.equal(got[2], (x.float() + r.float()).to(dtype))
    near = 70 * E  # of y, as above, and of the scale's division
    _within(got[1], scales, near * scales)
    # e4m3: half a unit in the last of 4 places, 2^-10 below the normal numbers
    _within(got[0].float(), values, torch.clamp(values.abs() * 2.0 ** -4, min=2.0 ** -10) + 3 * near * values.abs())


@pytest.mark.gpu
def test_norm_rows_of_slices(cuda):
    """Rows of slices of wider tensors, of three dimensions, of transposes."""
    from turbopress_amd import rms_norm, rms_norm_fp8
    g = _gen(5)
    qkv = _randn(g, 7, 5 * 128 + 64, dtype=F16)
    w = _randn(g, 128, dtype=F16)
    heads = qkv[:, 64:64 + 3 * 128].view(7, 3, 128)
    other = _randn(g, 3, 7, 128, dtype=F16).transpose(0, 1)
    for x, r in ((heads, None), (heads, other), (heads, heads.contiguous()), (other, heads), (qkv[::2, 1:129], None),
                 (_randn(g, 128, 7, dtype=F16).t(), None), (_randn(g, 2, 3, 4, 128, dtype=F16).transpose(0, 2), None)):
        want, _ = O.rms_norm(x, w, EPS, r)
        got = rms_norm(x, w, EPS, residual=r)
        _within(got if r is None else got[0], want, _norm_tol(want, F16))
        assert torch.equal(rms_norm_fp8(x, w, EPS, residual=r)[0].float(),
                           rms_norm_fp8(x.contiguous(), w, EPS, residual=None if r is None else r.contiguous())[0].float())
    assert rms_norm(qkv[:0, :128], w).shape == (0, 128)
    one = rms_norm(qkv[0, :128], w)
    assert one.shape == (128,) and torch.equal(one, rms_norm(qkv[:1, :128], w)[0])


@pytest.mark.gpu
def test_norm_rows_do_not_mix(cuda):
    """NaN, infinity, zeros and the type's largest values stay in their rows, in
    8 bits a NaN's too (its whole row: the mean is NaN)."""
    from turbopress_amd import rms_norm, rms_norm_fp8
    g = _gen(6)
    for d in (100, 300, 1000):
        x, w = _randn(g, 6, d, dtype=F16), _randn(g, d, dtype=F16)
        x[1, 3], x[2, 5], x[3], x[4] = float("nan"), float("inf"), 0, 65504
        y = rms_norm(x, w)
        clean = rms_norm(x[[0, 5]], w)
        assert torch.equal(y[[0, 5]], clean) and y[1].isnan().all()
        assert y[2, 5].isnan() and (y[2, :5] == 0).all() and (y[3] == 0).all()
        want, _ = O.rms_norm(x[4], w, EPS)
        _within(y[4], want, _norm_tol(want, F16))
        codes, scales = rms_norm_fp8(x, w)
        assert codes[1].float().isnan().all() and scales[1].isnan().all()
        assert scales[2, 0].isnan() and (codes[3].float() == 0).all() and (scales[3] == 2.0 ** -126).all()
        clean8 = rms_norm_fp8(x[[0, 5]], w)
        assert torch.equal(codes[[0, 5]].float(), clean8[0].float()) and torch.equal(scales[[0, 5]], clean8[1])


@pytest.mark.gpu
def test_norm_past_32_bit_offsets(cuda):
    from turbopress_amd import rms_norm
    rows, d = 270000, 8192  # 2.2e9 elements
    x = torch.zeros(rows, d, dtype=F16, device="cuda")
    w = torch.ones(d, dtype=F16, device="cuda")
    g = _gen(7)
    x[-2:] = _randn(g, 2, d, dtype=F16)
    y = rms_norm(x, w)
    want, _ = O.rms_norm(x[-2:], w, EPS)
    _within(y[-2:], want, _norm_tol(want, F16))
    assert (y[-4:-2] == 0).all()


# ---------------------------------------------------------------------------
# e4m3 product
# ---------------------------------------------------------------------------
def _codes(g, rows, k, ld=None):
    """e4m3 rows, ld bytes apart, NaN between them."""
    ld = ld or k
    c = torch.full((rows, ld), 0x7f, dtype=torch.uint8, device="cuda").view(F8)
    c[:, :k] = (_randn(g, rows, k) * torch.exp(_randn(g, rows, 1))).clamp(-448, 448).to(F8)
    return c[:, :k]


def _fp8_case(g, m, n, k, pad_a=0, pad_w=0):
    kb = -(-k // 128)
    return (_codes(g, m, k, k + pad_a), 0.01 + torch.rand(m, kb, generator=g, device="cuda"),
            _codes(g, n, k, k + pad_w), 0.01 + torch.rand(-(-n // 128), kb, generator=g, device="cuda"))


def _fp8_tol(want, size, k, dtype):
    # fp32 outputs: at most 128 additions in a block and one per block.  Others:
    # the 8-bit instructions keep about 2^-16 of a block's largest sums
    inner = (128 + k / 128 + 8) * E if dtype == F32 else 2.0 ** -13
    return U[dtype] * want.abs() + inner * size + LEAST[dtype]


# (few rows; tiles of 64 x 64 to 256 x 256; blocks, rows and columns that end
# inside a tile)
FP8 = [(1, 1, 1), (1, 16, 128), (2, 40, 129), (3, 17, 300), (16, 100, 256), (17, 300, 300), (32, 128, 1000), (1, 20000, 300),
       (33, 65, 127), (64, 64, 128), (65, 130, 384), (200, 257, 777), (130, 1000, 3001), (300, 400, 2576), (33, 20000, 256),
       (512, 4096, 256), (2048, 4096, 256), (2048, 9728, 384), (4000, 8100, 272),
       (2000, 5000, 300), (20000, 64, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", FP8)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_fp8_linear(cuda, m, n, k, dtype):
    from turbopress_amd import fp8_linear
    g = _gen(m + n + k)
    case = _fp8_case(g, m, n, k)
    bias = _randn(g, n, dtype=dtype) if (m + n) % 2 else None
    if dtype == F16:
        case = (case[0], case[1] / 64, case[2], case[3])  # inside fp16's range
    want, size = O.fp8_linear(*case, bias)
    got = fp8_linear(*case, bias=bias, out_dtype=dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    _within(got, want, _fp8_tol(want, size, k, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 100, 700])
@pytest.mark.parametrize("k", [128, 200, 333])
@pytest.mark.parametrize("pads", [(16, 48), (3, 0), (0, 5), (7, 9)])
def test_fp8_linear_rows_apart(cuda, m, k, pads):
    """Rows of any distance, aligned or not, with NaN between them."""
    from turbopress_amd import fp8_linear
    g = _gen(m + k)
    to16 = -k % 16
    case = _fp8_case(g, m, 150, k, *(p + to16 if p % 16 == 0 and p else p for p in pads))
    want, size = O.fp8_linear(*case)
    _within(fp8_linear(*case, out_dtype=F32), want, _fp8_tol(want, size, k, F32))
    _within(fp8_linear(*case, out_dtype=BF16), want, _fp8_tol(want, size, k, BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("m,n,k", [(1, 70, 33), (5, 6200, 257), (20, 6200, 130), (24, 33600, 1001), (40, 70, 1027)])
def test_fp8_linear_rows_off_their_words(cuda, m, n, k, offset):
    """Operands that begin anywhere in a word of memory, and rows that begin
    elsewhere in theirs; the bytes around them are NaN."""
    from turbopress_amd import fp8_linear
    g = _gen(m + k + offset)
    a, sa, w, sw = _fp8_case(g, m, n, k)

    def moved(t, off):
        ld = t.shape[1] + 3
        raw = torch.full((off + t.shape[0] * ld + 8,), 0x7f, dtype=torch.uint8, device="cuda")
        rows = raw[off:off + t.shape[0] * ld].view(-1, ld)[:, :t.shape[1]]
        rows.copy_(t.view(torch.uint8))
        return rows.view(torch.float8_e4m3fn)

    want, size = O.fp8_linear(a, sa, w, sw)
    got = fp8_linear(moved(a, offset), sa, moved(w, 5 * offset), sw, out_dtype=F32)
    _within(got, want, _fp8_tol(want, size, k, F32))


@pytest.mark.gpu
def test_fp8_linear_rows_do_not_mix(cuda):
    from turbopress_amd import fp8_linear
    g = _gen(9)
    for m in (5, 90):
        a, sa, w, sw = _fp8_case(g, m, 70, 200)
        clean = fp8_linear(a, sa, w, sw)
        a2, w2 = a.clone(), w.clone()
        a2.view(torch.uint8)[3, 199] = 0x7f
        w2.view(torch.uint8)[60, 0] = 0x7f
        y = fp8_linear(a2, sa, w2, sw)
        assert y[3].isnan().all() and y[:, 60].isnan().all()
        keep = [i for i in range(m) if i != 3]
        cols = [j for j in range(70) if j != 60]
        assert torch.equal(y[keep][:, cols], clean[keep][:, cols])


@pytest.mark.gpu
def test_fp8_linear_of_norm_and_weights(cuda):
    """Norm, quantised weights and product together, over leading dimensions."""
    from turbopress_amd import fp8_linear, quantize_fp8_weight, rms_norm_fp8
    g = _gen(10)
    dense = 0.02 * _randn(g, 333, 576, dtype=F16)
    w, sw = quantize_fp8_weight(dense)
    # half a unit of e4m3 at the block's scale, of the value itself above it
    back = w.double() * sw.double().repeat_interleave(128, 0)[:333].repeat_interleave(128, 1)[:, :576]
    least = sw.double().repeat_interleave(128, 0)[:333].repeat_interleave(128, 1)[:, :576] * 2.0 ** -10
    _within(back, dense.double(), torch.maximum(dense.double().abs() * 2.0 ** -4, least) * (1 + 2.0 ** -20))
    x, nw = _randn(g, 2, 3, 576, dtype=F16), _randn(g, 576, dtype=F16)
    codes, scales = rms_norm_fp8(x, nw)
    y = fp8_linear(codes, scales, w, sw, out_dtype=F32)
    want, size = O.fp8_linear(codes.reshape(-1, 576), scales.reshape(-1, 5), w, sw)
    assert y.shape == (2, 3, 333)
    _within(y.view(-1, 333), want, _fp8_tol(want, size, 576, F32))
    assert fp8_linear(codes[:0], scales[:0], w, sw).shape == (0, 3, 333)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------
def _table(positions, rd):
    from turbopress_amd import rotary_table
    return rotary_table(positions, rd, device="cuda")


def _turn_tol(want, size, dtype):
    return U[dtype] * want.abs() + 3 * E * size + LEAST[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("d,rd", [(2, 2), (6, 4), (64, 64), (80, 40), (96, 36), (128, 128), (128, 32), (128, 2), (192, 64), (256, 256)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(cuda, d, rd, dtype, interleaved):
    from turbopress_amd import rotary
    g = _gen(d + rd)
    for tokens, hq, hk in ((1, 1, 1), (5, 6, 2), (67, 3, 3)):
        table = _table(100, rd)
        qkv = _randn(g, tokens, hq + 2 * hk, d, dtype=dtype)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
        pos = torch.randint(0, 100, (tokens,), generator=g, device="cuda")
        for x, y in zip((q, k), rotary(q, k, table, pos, interleaved=interleaved)):
            want, size = O.rotary(x, table, pos, interleaved)
            assert y.shape == x.shape and y.is_contiguous() and torch.equal(y[..., rd:], x[..., rd:])
            _within(y, want, _turn_tol(want, size, dtype))
    alone, none = rotary(q, None, table, pos, interleaved=interleaved)
    assert none is None and torch.equal(alone, rotary(q, k, table, pos, interleaved=interleaved)[0])


@pytest.mark.gpu
def test_rotary_padding_and_positions_past_the_table(cuda):
    from turbopress_amd import rotary
    g = _gen(12)
    q, k, table = _randn(g, 4, 2, 64, dtype=F16), _randn(g, 4, 1, 64, dtype=F16), _table(10, 32)
    pos = torch.tensor([9, -1, 10, 2 ** 40], device="cuda")
    for y in rotary(q, k, table, pos):
        assert torch.isfinite(y[0]).all() and (y[1] == 0).all() and y[2].isnan().all() and y[3].isnan().all()
    assert rotary(q[:0], k[:0], table, pos[:0])[0].shape == (0, 2, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("d,rd,interleaved", [(64, 64, False), (96, 36, True), (128, 32, False)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_rotary_append(cuda, page, d, rd, interleaved, heads_first):
    """Tokens of several sequences at once: their keys and values arrive, and
    nothing else of the caches changes, whatever the tokens that have no place."""
    from turbopress_amd import rotary, rotary_append
    g = _gen(page + d)
    seqs, hq, hk, width, pages = 3, 4, 2, -(-40 // page), 3 * -(-40 // page) + 2
    shape = (pages, hk, page, d) if heads_first else (pages, page, hk, d)
    stores = [_randn(g, *shape, dtype=F16) for _ in "kv"]
    caches = [c.transpose(1, 2) if heads_first else c for c in stores]
    before = [c.clone() for c in caches]
    bt = torch.randperm(pages, generator=g, device="cuda")[:seqs * width].view(seqs, width).int()
    table = _table(45, rd)
    seq = torch.tensor([0, 0, 2, 1, 2, 1, 0, 9, 1, -1], device="cuda", dtype=torch.int32)
    pos = torch.tensor([0, 1, 39, 17, 38, -1, 44 if width * page < 44 else 60, 3, 16, 3], device="cuda")
    bad = int(bt[2, 38 // page]) if page == 1 else None
    if bad is not None:
        bt[2, 38 // page] = pages + 5  # a page that does not exist
    t = len(seq)
    q, k, v = _randn(g, t, hq, d, dtype=F16), _randn(g, t, hk, d, dtype=F16), _randn(g, t, hk, d, dtype=F16)
    got = rotary_append(q, k, v, table, pos, *caches, bt, sequences=seq, interleaved=interleaved)
    q_want, k_want = rotary(q, k, table, pos, interleaved=interleaved)
    assert torch.equal(got.nan_to_num(7), q_want.nan_to_num(7))
    for i in range(t):
        s, p = int(seq[i]), int(pos[i])
        if not 0 <= s < seqs or not 0 <= p < 45 or p // page >= width or not 0 <= int(bt[s, p // page]) < pages:
            continue
        at = int(bt[s, p // page]), p % page
        before[0][at], before[1][at] = k_want[i], v[i]
    assert all(torch.equal(a, b) for a, b in zip(caches, before))
    # without `sequences` token t is sequence t's
    pos3 = torch.tensor([5, 6, 7], device="cuda")
    rotary_append(q[:3], k[:3], v[:3], table, pos3, *caches, bt, interleaved=interleaved)
    _, k3 = rotary(q[:3], k[:3], table, pos3, interleaved=interleaved)
    for s in range(3):
        at = int(bt[s, int(pos3[s]) // page]), int(pos3[s]) % page
        assert torch.equal(caches[0][at], k3[s]) and torch.equal(caches[1][at], v[s])


def test_rotary_frequencies_match_transformers():
    """Against transformers' own frequencies of the same configurations (its
    fp32 ones: 2^-21 apart at most)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    from turbopress_amd.paged import rotary_frequencies
    for kind, scaling in (("linear", {"rope_type": "linear", "factor": 4.0}),
                          ("llama3", {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                      "original_max_position_embeddings": 8192}),
                          ("yarn", {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}),
                          ("yarn", {"rope_type": "yarn", "factor": 16.0, "beta_fast": 24, "beta_slow": 2,
                                    "attention_factor": 1.3, "original_max_position_embeddings": 4096})):
        for dim, base in ((64, 10000.0), (128, 1e6)):
            cfg = LlamaConfig(hidden_size=4 * dim, num_attention_heads=4, head_dim=dim, rope_theta=base,
                              max_position_embeddings=int(scaling.get("original_max_position_embeddings", 2048) * scaling["factor"]),
                              rope_scaling=dict(scaling, rope_theta=base))
            want, factor = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu")
            got, mine = rotary_frequencies(dim, base, scaling)
            assert got.dtype == torch.float64 and abs(mine - factor) < 1e-6
            assert ((got - want.double()).abs() <= 2.0 ** -21 * want.double()).all(), (kind, dim, base)
    assert torch.equal(rotary_frequencies(8)[0], 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4))


def test_rotary_table_on_the_cpu():
    from turbopress_amd import rotary_table
    t = rotary_table(50, 16, base=500.0, device="cpu")
    assert t.shape == (50, 16) and t.dtype == F32
    i, p = 3, 37
    angle = p * 500.0 ** (-i / 8)
    assert abs(t[p, i].item() - math.cos(angle)) <= E and abs(t[p, 8 + i].item() - math.sin(angle)) <= E


# ---------------------------------------------------------------------------
# paged attention
# ---------------------------------------------------------------------------
def _paged(g, lengths, hkv, d, page, dtype, junk=float("nan"), spare=3, heads_first=False, extra=1):
    """Caches whose every unused place holds `junk`, pages in random order, and
    table columns past a sequence's own that name no page."""
    width = max([-(-n // page) for n in lengths] + [0]) + extra
    count = sum(-(-n // page) for n in lengths) + spare
    shape = (count, hkv, page, d) if heads_first else (count, page, hkv, d)
    caches = [torch.full(shape, junk, dtype=dtype, device="cuda") for _ in "kv"]
    if heads_first:
        caches = [c.transpose(1, 2) for c in caches]
    order = torch.randperm(count, generator=g, device="cuda").tolist()
    bt = torch.full((len(lengths), width), -7, dtype=torch.int32)
    bt[:, ::2] = 2 ** 31 - 1
    for i, n in enumerate(lengths):
        for c in range(-(-n // page)):
            bt[i, c] = p = order.pop()
            m = min(page, n - c * page)
            caches[0][p, :m] = _randn(g, m, hkv, d, dtype=dtype)
            caches[1][p, :m] = _randn(g, m, hkv, d, dtype=dtype)
    return *caches, bt.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _attention_tol(want, size, dots, d, dtype):
    # scores in fp32 (d products of magnitudes that sum to `dots`) and their
    # exponentials, above and below the fraction; the probabilities round once
    # to the values' type for their products
    near = 2 * (d + 8) * E * dots[..., None] + 2.0 ** -18
    return U[dtype] * want.abs() + (U[dtype] + near) * size + LEAST[dtype]


def _check_attention(g, lengths, hq, hkv, d, page, dtype, window=0, scale=None, **kw):
    from turbopress_amd import paged_attention
    k, v, bt, n = _paged(g, lengths, hkv, d, page, dtype, **kw)
    q = _randn(g, len(lengths), hq, d, dtype=dtype)
    want, size, dots = O.paged_attention(q, k, v, bt, n, scale, window)
    got = paged_attention(q, k, v, bt, n, scale=scale, window=window)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    _within(got, want, _attention_tol(want, size, dots, d, dtype))
    for i, m in enumerate(lengths):
        if m == 0:
            assert (got[i] == 0).all()
    assert torch.equal(got, paged_attention(q, k, v, bt, n, scale=scale, window=window))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 24, 64, 80, 96, 120, 128, 136, 192, 248, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_paged_attention_head_sizes(cuda, d, dtype):
    _check_attention(_gen(d), [0, 1, 31, 33, 200, 700], 6, 2, d, 16, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (9, 3), (7, 1), (16, 1), (17, 1), (40, 2), (8, 8)])
def test_paged_attention_head_groups(cuda, hq, hkv):
    _check_attention(_gen(hq), [5, 0, 130, 999], hq, hkv, 64, 16, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 3, 16, 31, 32, 48, 100, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_paged_attention_pages(cuda, page, heads_first):
    _check_attention(_gen(page), [1, 2, 3, 15, 16, 17, 32, 127, 128, 129, 500], 4, 2, 64, page, BF16, heads_first=heads_first)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0], [1], [128], [129], [5000], [40000], [0] * 70, [1] * 200, [0, 3000] * 40,
                                     list(range(0, 260, 2)), [20000] + [1] * 65])
def test_paged_attention_lengths(cuda, lengths):
    """One sequence and many, empty ones among them, so that a sequence is one
    workgroup's, several's, or shares one."""
    _check_attention(_gen(len(lengths)), lengths, 4, 2, 64, 16, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 31, 32, 33, 128, 100, 1000, 10 ** 6])
def test_paged_attention_window(cuda, window):
    _check_attention(_gen(window), [0, 1, 32, 33, 100, 500, 1500], 4, 1, 64, 16, F16, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5, 4.0])
def test_paged_attention_scales(cuda, scale):
    """Down to no scores at all, and up to ones that single tokens decide."""
    _check_attention(_gen(3), [1, 64, 300, 2000], 4, 2, 64, 16, BF16, scale=scale)


@pytest.mark.gpu
def test_paged_attention_infinities(cuda):
    """A key at -infinity (and a query that meets it with a positive sign) has
    no weight; where every key is, the output is zero; at +infinity, NaN."""
    from turbopress_amd import paged_attention
    g = _gen(4)
    k, v, bt, n = _paged(g, [100, 40, 300], 1, 64, 16, F16)
    q = _randn(g, 3, 2, 64, dtype=F16).abs()
    flat = [bt[i].long()[torch.arange(m, device="cuda") // 16] for i, m in enumerate((100, 40, 300))]
    at = [torch.arange(m, device="cuda") % 16 for m in (100, 40, 300)]
    k[flat[0][70:], at[0][70:], 0, 0] = -math.inf
    k[flat[1], at[1], 0, 3] = -math.inf
    k[flat[2][200], at[2][200], 0, 3] = math.inf
    y = paged_attention(q, k, v, bt, n)
    short = n.clone()
    short[0] = 70
    want = paged_attention(q, k, v, bt, short)
    assert (y[0].float() - want[0].float()).abs().max() <= 2 ** -9 and (y[1] == 0).all() and y[2].isnan().all()


@pytest.mark.gpu
def test_paged_attention_odd_inputs(cuda):
    """Pages that do not exist are left out, lengths stop at the table's width,
    negative ones are empty; queries may be slices of a wider tensor."""
    from turbopress_amd import paged_attention
    g = _gen(8)
    k, v, bt, n = _paged(g, [100, 64, 33, 20], 2, 64, 16, F16, extra=0, junk=0.5)
    bt[0, 3], bt[1, :4] = -1, torch.tensor([k.shape[0], -5, 2 ** 31 - 1, k.shape[0] + 1])
    bt = bt.clamp(min=-5)
    n[3] = -4
    wide = _randn(g, 4, 10, 72, dtype=F16)
    for q in (wide[:, 3:7, :64], wide[:, 3:7, 4:68], _randn(g, 4, 4, 64, dtype=F16)):
        want, size, dots = O.paged_attention(q, k, v, bt, n)
        got = paged_attention(q, k, v, bt, n)
        _within(got, want, _attention_tol(want, size, dots, 64, F16))
        assert (got[1] == 0).all() and (got[3] == 0).all()
    far = n.clone()
    far[0] = 2 ** 31 - 1
    bt[0] = torch.arange(bt.shape[1], device="cuda")
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    want, size, dots = O.paged_attention(q, k, v, bt, far)
    _within(paged_attention(q, k, v, bt, far), want, _attention_tol(want, size, dots, 64, F16))
    none = torch.empty(4, 0, dtype=torch.int32, device="cuda")
    assert (paged_attention(q, k, v, none, n) == 0).all()
    assert paged_attention(q[:0], k, v, bt[:0], n[:0]).shape == (0, 4, 64)


@pytest.mark.gpu
def test_paged_cache_past_32_bit_offsets(cuda):
    """A cache of more than 2^31 elements: written and read at both its ends."""
    from turbopress_amd import paged_attention, rotary_append
    g = _gen(11)
    pages, page, hk, d = 17000, 64, 16, 128  # 2.2e9 elements each
    caches = [torch.zeros(pages, page, hk, d, dtype=F16, device="cuda") for _ in "kv"]
    bt = torch.tensor([[0, pages - 1], [pages - 2, 1]], dtype=torch.int32, device="cuda")
    table = _table(128, d)
    t = 2 * 128
    q, k, v = (_randn(g, t, h, d, dtype=F16) for h in (32, hk, hk))
    pos = torch.arange(128, device="cuda").repeat(2)
    seq = torch.arange(2, device="cuda", dtype=torch.int32).repeat_interleave(128)
    turned = rotary_append(q, k, v, table, pos, *caches, bt, sequences=seq)
    n = torch.tensor([128, 128], dtype=torch.int32, device="cuda")
    last = turned[127::128]
    small = [torch.cat([c[[0, pages - 1]], c[[pages - 2, 1]]]) for c in caches]
    assert torch.equal(small[1].view(t, hk, d), v)
    want, size, dots = O.paged_attention(last, *small, torch.tensor([[0, 1], [2, 3]], device="cuda"), n)
    _within(paged_attention(last, *caches, bt, n), want, _attention_tol(want, size, dots, d, F16))


# ---------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------
def _step(g):
    """One token of three sequences through all operators, into fresh outputs."""
    from turbopress_amd import fp8_linear, paged_attention, rms_norm, rms_norm_fp8, rotary_append
    k_cache, v_cache, bt, n = _paged(g, [1000, 31, 2000], 2, 64, 16, F16, junk=0.0)
    x, r, nw = _randn(g, 3, 512, dtype=F16), _randn(g, 3, 512, dtype=F16), _randn(g, 512, dtype=F16)
    w, sw = _codes(g, 700, 512), torch.rand(6, 4, generator=g, device="cuda")
    table = _table(2100, 64)
    pos = (n - 1).long()

    def run():
        y, h = rms_norm(x, nw, residual=r)
        qkv = y.view(3, 8, 64)
        q = rotary_append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], table, pos, k_cache, v_cache, bt)
        o = paged_attention(q, k_cache, v_cache, bt, n)
        codes, scales = rms_norm_fp8(torch.cat((o.view(3, 256), h[:, :256]), 1), nw)
        return h, o, fp8_linear(codes, scales, w, sw)

    return x, run


@pytest.mark.gpu
def test_operators_in_a_graph(cuda):
    x, run = _step(_gen(20))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(5):
        x.copy_(_randn(_gen(100 + i), 3, 512, dtype=F16))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


@pytest.mark.gpu
def test_a_graph_stands_without_the_one_captured_before(cuda):
    """Two graphs captured in a row, the second replayed alone: its counters'
    zeros are its own, not the first one's."""
    _, run = _step(_gen(21))
    want = [t.clone() for t in run()]
    graphs = []
    for _ in range(2):
        junk = torch.full((1 << 24,), 255, dtype=torch.uint8, device="cuda")  # (what memory may hold)
        del junk
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graphs.append((graph, outs))
    for i in (1, 1, 0, 1):
        graphs[i][0].replay()
        assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want))


@pytest.mark.gpu
def test_operators_on_two_streams(cuda):
    """The same calls on two streams at once, each with workspaces of its own."""
    steps = [_step(_gen(30 + i)) for i in range(2)]
    want = [[t.clone() for t in run()] for _, run in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(steps[i][1]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for o in outs[i] for a, b in zip(o, want[i]))


def test_cpu_tensors_are_refused():
    import turbopress_amd as T
    x, w = torch.zeros(2, 8, dtype=F16), torch.ones(8, dtype=F16)
    q, pos, table = torch.zeros(2, 1, 8, dtype=F16), torch.zeros(2, dtype=torch.int64), torch.zeros(4, 8)
    cache, bt, n = torch.zeros(1, 4, 1, 8, dtype=F16), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    f8, s = torch.zeros(2, 8, dtype=F8), torch.ones(2, 1)
    for call in (lambda: T.rms_norm(x, w), lambda: T.rms_norm_fp8(x, w), lambda: T.fp8_linear(f8, s, f8, s[:1]),
                 lambda: T.rotary(q, q, table, pos), lambda: T.rotary_append(q, q, q, table, pos, cache, cache, bt),
                 lambda: T.paged_attention(q, cache, cache, bt, n)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.gpu
def test_bad_arguments_are_refused(cuda):
    import turbopress_amd as T
    dev = cuda

    def z(*shape, dtype=F16):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    x, w = z(2, 8), z(8)
    a, sa, wt, sw = z(2, 200, dtype=F8), z(2, 2, dtype=F32), z(3, 200, dtype=F8), z(1, 2, dtype=F32)
    q, k, pos, table = z(2, 4, 8), z(2, 2, 8), z(2, dtype=torch.int64), z(4, 8, dtype=F32)
    c, bt, n = z(3, 4, 2, 8), z(2, 1, dtype=torch.int32), z(2, dtype=torch.int32)
    bad = [
        lambda: T.rms_norm(z(2, 8, dtype=torch.float64), z(8, dtype=torch.float64)), lambda: T.rms_norm(x, z(7)),
        lambda: T.rms_norm(x, z(8, dtype=F32)), lambda: T.rms_norm(x, w.cpu()), lambda: T.rms_norm(x, w, residual=z(1, 8)),
        lambda: T.rms_norm(x, w, residual=z(2, 8, dtype=F32)), lambda: T.rms_norm(z(2, 0), z(0)),
        lambda: T.rms_norm_fp8(x, w, block=64), lambda: T.rms_norm_fp8(x, z(9)),
        lambda: T.fp8_linear(a, sa, wt, sw, out_dtype=F8), lambda: T.fp8_linear(x, sa, wt, sw),
        lambda: T.fp8_linear(a, sa, z(3, 199, dtype=F8), sw), lambda: T.fp8_linear(a, z(2, 1, dtype=F32), wt, sw),
        lambda: T.fp8_linear(a, sa, wt, z(2, 2, dtype=F32)), lambda: T.fp8_linear(a, sa.half(), wt, sw),
        lambda: T.fp8_linear(a, sa, wt, sw, bias=z(4)), lambda: T.fp8_linear(a, sa, wt, sw, bias=z(3, dtype=F32)),
        lambda: T.quantize_fp8_weight(z(4)), lambda: T.quantize_fp8_weight(z(4, 4, dtype=torch.int32)),
        lambda: T.rotary(q[0], k, table, pos), lambda: T.rotary(q, k, table.half(), pos), lambda: T.rotary(q, k, table[:, :7], pos),
        lambda: T.rotary(q, k, z(4, 10, dtype=F32), pos), lambda: T.rotary(q, k, table, pos.int()),
        lambda: T.rotary(q, k, table, pos[:1]), lambda: T.rotary(q, k[:1], table, pos), lambda: T.rotary(q, k.float(), table, pos),
        lambda: T.rotary_append(q, k, None, table, pos, c, c, bt), lambda: T.rotary_append(q, k, k[:, :1], table, pos, c, c, bt),
        lambda: T.rotary_append(q, k, k, table, pos, c, c[:2], bt), lambda: T.rotary_append(q, k, k, table, pos, c[:, :, :1], c[:, :, :1], bt),
        lambda: T.rotary_append(q, k, k, table, pos, c, c, bt.long()), lambda: T.rotary_append(q, k, k, table, pos, c, c, bt[:1]),
        lambda: T.rotary_append(q, k, k, table, pos, c, c, bt, sequences=pos),
        lambda: T.paged_attention(q.float(), c.float(), c.float(), bt, n), lambda: T.paged_attention(q, c, c, bt[:1], n),
        lambda: T.paged_attention(q, c, c, bt, n.long()), lambda: T.paged_attention(q, c, c, bt, n[:1]),
        lambda: T.paged_attention(q[:, :3], c, c, bt, n), lambda: T.paged_attention(q, c, c, bt, n, window=-1),
        lambda: T.paged_attention(q, c.bfloat16(), c.bfloat16(), bt, n), lambda: T.paged_attention(q[..., :4], c[..., :4], c[..., :4], bt, n),
        lambda: T.paged_attention(z(2, 4, 264), z(3, 4, 2, 264), z(3, 4, 2, 264), bt, n),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_c_entry_points_refuse_on_the_host(built_lib):
    import ctypes

    from turbopress_amd import _lib as L
    lib, p, odd = built_lib, ctypes.c_void_p(256), ctypes.c_void_p(257)
    i3 = (ctypes.c_int64 * 3)(1024, 64, 8)

    def norm(dtype=0, rows=2, inner=1, d=8, x=p, w=p, y=p):
        return lib.tp_rms_norm(dtype, rows, inner, d, x, d, 0, None, 0, 0, w, 1e-6, y, None, None)

    assert norm(rows=0) == L.TP_OK
    assert norm(dtype=3) == L.TP_ERR_BAD_TYPE
    assert norm(d=0) == norm(inner=0) == norm(rows=-1) == norm(rows=2 ** 31) == L.TP_ERR_BAD_DIMS
    assert norm(x=None) == norm(w=None) == norm(y=None) == L.TP_ERR_NULL_POINTER
    assert norm(x=odd) == norm(y=odd) == L.TP_ERR_MISALIGNED

    def norm8(block=128, ldc=16, codes=p, scales=p):
        return lib.tp_rms_norm_fp8(0, 2, 1, 8, p, 8, 0, None, 0, 0, p, 1e-6, block, codes, ldc, scales, None, None)

    assert norm8(block=64) == L.TP_ERR_BAD_BLOCK and norm8(ldc=7) == L.TP_ERR_BAD_DIMS
    assert norm8(ldc=24) == norm8(codes=ctypes.c_void_p(264)) == L.TP_ERR_MISALIGNED
    assert norm8(codes=None) == norm8(scales=None) == L.TP_ERR_NULL_POINTER

    def fp8(dtype=0, m=2, n=4, k=64, a=p, lda=64, sa=p, w=p, ldw=64, y=p, ldy=4, ws=None, size=0):
        return lib.tp_fp8_linear(dtype, m, n, k, a, lda, sa, w, ldw, p, None, y, ldy, ws, size, None)

    assert fp8(m=0) == fp8(n=0) == L.TP_OK and fp8(dtype=7) == L.TP_ERR_BAD_TYPE
    assert fp8(k=0) == fp8(m=-1) == fp8(lda=63) == fp8(ldw=63) == fp8(ldy=3) == L.TP_ERR_BAD_DIMS
    assert fp8(a=None) == fp8(sa=None) == fp8(w=None) == fp8(y=None) == L.TP_ERR_NULL_POINTER
    assert fp8(sa=odd) == fp8(y=odd) == L.TP_ERR_MISALIGNED
    need = lib.tp_fp8_workspace_bytes(100, 10, 65, p, 65, p, 80)
    assert need == 100 * 80 and lib.tp_fp8_workspace_bytes(100, 10, 65, odd, 80, p, 65) == 110 * 80
    assert lib.tp_fp8_workspace_bytes(1, 10, 65, p, 65, p, 65) == 0 and lib.tp_fp8_workspace_bytes(1, 1, 0, p, 1, p, 1) == -1
    assert fp8(m=100, n=10, k=65, lda=65, ldw=80, ldy=10, ws=p, size=need - 1) == L.TP_ERR_WORKSPACE
    assert fp8(m=100, n=10, k=65, lda=65, ldw=80, ldy=10, ws=ctypes.c_void_p(264), size=need) == L.TP_ERR_MISALIGNED

    def rot(dtype=0, tokens=2, hq=2, hk=1, d=8, rd=8, q=p, k=p, table=p, pos=p, k_out=p, kc=None, v=p, strides=i3, page=4):
        return lib.tp_rotary(dtype, tokens, hq, hk, d, rd, 0, q, 16, 8, k, 8, 8, table, 4, pos, p, k_out, v, 8, 8, kc, strides,
                             kc, strides, 3, page, p, 1, 2, None, None)

    assert rot(tokens=0) == L.TP_OK and rot(dtype=9) == L.TP_ERR_BAD_TYPE
    assert rot(d=7) == rot(rd=10) == rot(rd=3) == rot(rd=0) == rot(hq=-1) == rot(kc=p, page=0) == L.TP_ERR_BAD_DIMS
    assert rot(q=None) == rot(k=None) == rot(table=None) == rot(pos=None) == rot(k_out=None) == L.TP_ERR_NULL_POINTER
    assert rot(kc=p, v=None) == rot(kc=p, strides=None) == L.TP_ERR_NULL_POINTER
    assert rot(q=odd) == rot(pos=ctypes.c_void_p(260)) == L.TP_ERR_MISALIGNED

    need = lib.tp_paged_attention_workspace_bytes(2, 4, 2, 64)
    count = lib.tp_paged_attention_counter_bytes(2, 4, 2, 64)
    assert need > 0 and count == 16 and lib.tp_paged_attention_counter_bytes(3, 40, 2, 64) == 3 * 2 * 2 * 4

    def att(dtype=0, batch=2, hq=4, hkv=2, d=64, q=p, kc=p, strides=i3, page=16, window=0, ws=p, size=need, cnt=p, csize=count):
        return lib.tp_paged_attention(dtype, batch, hq, hkv, d, q, 256, 64, kc, strides, p, i3, 5, page, p, 1, p, 1.0, window, p,
                                      ws, size, cnt, csize, None)

    assert att(batch=0) == L.TP_OK and att(dtype=2) == L.TP_ERR_BAD_TYPE
    assert att(d=60) == att(d=264) == att(hq=5) == att(page=0) == att(window=-1) == att(batch=-1) == L.TP_ERR_BAD_DIMS
    assert lib.tp_paged_attention_workspace_bytes(1, 3, 2, 64) == lib.tp_paged_attention_counter_bytes(1, 1, 1, 4) == -1
    assert att(q=None) == att(kc=None) == att(strides=None) == L.TP_ERR_NULL_POINTER
    assert att(q=ctypes.c_void_p(264)) == att(strides=(ctypes.c_int64 * 3)(1024, 64, 4)) == L.TP_ERR_MISALIGNED
    assert att(ws=None) == att(size=need - 1) == att(cnt=None) == att(csize=count - 1) == L.TP_ERR_WORKSPACE


def test_c_entry_points_refuse_more_threads_than_a_launch_holds(built_lib):
    import ctypes

    from turbopress_amd import _lib as L
    lib, p = L.lib(), ctypes.c_void_p(4096)

    def rot(tokens, hq, d):
        return lib.tp_rotary(0, tokens, hq, 0, d, d, 0, p, d * hq, d, None, 0, 0, p, 16, p, p, None, None, 0, 0, None, None,
                             None, None, 0, 1, None, 0, 0, None, None)

    assert rot(1 << 40, 65536, 65536) == rot(1 << 33, 1, 2) == rot(1 << 28, 8, 64) == L.TP_ERR_BAD_DIMS
    for rows, d in ((1 << 28, 128), (1 << 23, 30000)):
        assert lib.tp_rms_norm(0, rows, 1, d, p, d, 0, None, 0, 0, p, 1e-6, p, None, None) == L.TP_ERR_BAD_DIMS
    assert lib.tp_fp8_linear(0, 1, 1 << 27, 16, p, 16, p, p, 16, p, None, p, 1 << 27, None, 0, None) == L.TP_ERR_BAD_DIMS
