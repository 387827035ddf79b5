"""The operators of serving many requests (attention of drafted trees, windows
with first tokens that stay visible, log probabilities, adapters) against plain
64-bit implementations, and their refusals.

Tolerances come from the formats.  U[t] is the unit roundoff of type t: an
output that rounds once is off by at most U |y|, beside what the fp32 arithmetic
before it leaves.  E = 2^-24 is fp32's own."""

import math

import pytest
import torch

from oracle import serving_oracle as O

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
LEAST = {F16: 2.0 ** -24, BF16: 2.0 ** -130, F32: 2.0 ** -140}  # below the normal numbers
E = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _within(got, want, tol):
    """Every element of got within tol of want (both finite)."""
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got.float()).all()
    assert off.max().item() <= 0, f"{off.max().item():.3g} over at {off.argmax().item()} of {off.numel()}"


def _bits(masks):
    return [m - (1 << 64) if m >> 63 else m for m in masks]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _paged(g, lengths, hkv, d, page, dtype, junk=float("nan"), heads_first=False, extra=1):
    """Caches that hold `lengths` tokens of each sequence, `junk` in every unused
    place, pages in random order, table columns past a sequence's own that name no page."""
    width = max([-(-n // page) for n in lengths] + [0]) + extra
    count = sum(-(-n // page) for n in lengths) + 3
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
    return *caches, bt.cuda()


def _attention_tol(want, size, dots, d, dtype):
    # scores in fp32 (d products of magnitudes that sum to `dots`) above and below
    # the fraction; exponentials and the two pieces of a probability 2^-16; sums of
    # up to 2^8 steps of a wave, two roundings each, 2^-15
    near = 2 * (d + 8) * E * dots[..., None] + 2.0 ** -16 + 2.0 ** -15
    return U[dtype] * want.abs() + near * size + LEAST[dtype]


def _trees(g, batch, count):
    """Ancestors of random trees, some of fewer tokens."""
    parents = torch.full((batch, count), -1)
    rand = torch.rand(batch, count + 1, generator=g, device="cuda").tolist()
    for s in range(batch):
        n = count if s % 2 == 0 else 1 + int(rand[s][-1] * count)
        for i in range(1, count):
            parents[s, i] = int(rand[s][i] * (i + 1)) - 1 if i < n else -2
    from turbopress_amd import tree_ancestors
    return tree_ancestors(parents).cuda()


def _check_tree(g, lengths, count, hq, hkv, d, page, dtype, tree=True, window=0, sinks=0, scale=None, **kw):
    from turbopress_amd import paged_tree_attention
    k, v, bt = _paged(g, [n + count for n in lengths], hkv, d, page, dtype, **kw)
    q = _randn(g, len(lengths), count, hq, d, dtype=dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ancestors = _trees(g, len(lengths), count) if tree else None
    want, size, dots = O.paged_tree_attention(q, k, v, bt, n, ancestors, scale, window, sinks)
    args = dict(ancestors=ancestors, scale=scale, window=window, sinks=sinks)
    got = paged_tree_attention(q, k, v, bt, n, **args)
    assert got.shape == q.shape and got.dtype == dtype and got.is_contiguous()
    _within(got, want, _attention_tol(want, size, dots, d, dtype))
    assert torch.equal(got, paged_tree_attention(q, k, v, bt, n, **args))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 24, 64, 80, 96, 120, 128, 136, 192, 248, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("count,group", [(3, 2), (11, 2), (13, 3), (31, 3)])
def test_tree_head_sizes(cuda, d, dtype, count, group):
    _check_tree(_gen(d + count), [0, 1, 31, 130], count, group, 1, d, 16, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 64, 72, 96, 104, 128, 136, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("count,group", [(43, 3), (64, 5)])
def test_tree_rows_of_many_heads(cuda, d, dtype, count, group):
    """129 rows of a cache head, and 320: more than one group of them."""
    _check_tree(_gen(d + group), [0, 1, 31, 130, 700], count, 2 * group, 2, d, 16, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0] * 40, [1] * 90, [0, 1500] * 4, list(range(0, 260, 16)), [6000] + [1] * 20])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 3), (300, 40)])
def test_tree_rows_of_many_heads_of_uneven_sequences(cuda, lengths, window, sinks):
    _check_tree(_gen(len(lengths) + window), lengths, 36, 4, 1, 128, 16, F16, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv", [(1, 1), (9, 3), (7, 1), (16, 1), (17, 1), (40, 2)])
@pytest.mark.parametrize("count", [1, 2, 7, 16])
def test_tree_head_groups(cuda, hq, hkv, count):
    _check_tree(_gen(hq), [5, 0, 130], count, hq, hkv, 64, 16, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 5, 8, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64])
@pytest.mark.parametrize("tree", [False, True])
def test_tree_sizes(cuda, count, tree):
    _check_tree(_gen(count), [0, 33, 200], count, 4, 2, 64, 16, BF16, tree=tree)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 2, 3, 16, 31, 48, 100, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_tree_pages(cuda, page, heads_first):
    _check_tree(_gen(page), [0, 1, 15, 16, 31, 32, 127, 128, 300], 9, 2, 1, 64, page, F16, heads_first=heads_first)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[0], [1], [5000], [0] * 70, [1] * 100, [0, 1500] * 4, list(range(0, 260, 8)), [6000] + [1] * 65])
@pytest.mark.parametrize("count", [2, 20])
def test_tree_lengths(cuda, lengths, count):
    """One sequence and many, empty ones among them, so that a sequence is one
    workgroup's, several's, or shares one."""
    _check_tree(_gen(len(lengths)), lengths, count, 2, 1, 64, 16, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 5, 31, 32, 33, 100, 128, 1000, 10 ** 6])
@pytest.mark.parametrize("sinks", [0, 1, 4, 40, 10 ** 6])
def test_tree_window_and_sinks(cuda, window, sinks):
    _check_tree(_gen(window + sinks), [0, 1, 3, 33, 100, 150, 500], 12, 2, 1, 64, 16, F16, window=window, sinks=sinks)
    _check_tree(_gen(window + sinks), [0, 2, 40, 300], 64, 1, 1, 64, 16, BF16, tree=False, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1.0, -0.5, 4.0])
def test_tree_scales(cuda, scale):
    _check_tree(_gen(3), [1, 64, 300, 700], 6, 4, 2, 64, 16, BF16, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("count,group", [(6, 1), (20, 1), (20, 4), (36, 4)])
@pytest.mark.parametrize("window", [0, 9])
def test_tree_hidden_tokens_do_not_matter(cuda, dtype, count, group, window):
    """NaN and infinity in keys and values of new tokens, and of cached ones that a
    window hides from some, reach the tokens that see them and no others."""
    from turbopress_amd import paged_tree_attention
    g = _gen(9)
    lengths = [3, 40, 100]
    k, v, bt = _paged(g, [n + count for n in lengths], 1, 64, 16, dtype)
    q = _randn(g, 3, count, group, 64, dtype=dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ancestors = _trees(g, 3, count)
    args = dict(ancestors=ancestors, window=window, sinks=1)
    clean = paged_tree_attention(q, k, v, bt, n, **args)
    bad = [(0, 1, math.nan), (0, 2, math.inf), (1, 3, -math.inf), (1, 0, math.nan), (2, 4, math.inf), (2, 5, -math.inf),
           (1, -5, math.inf), (2, -7, math.nan)]  # (sequence, new token or, below 0, one of the cache's last, value)
    for what in "kv":
        kk, vv = k.clone(), v.clone()
        for s, j, x in bad:
            t = lengths[s] + j
            place = (bt[s, t // 16].long(), t % 16, 0)
            (kk if what == "k" else vv)[place][7:9] = x
        got = paged_tree_attention(q, kk, vv, bt, n, **args)
        want, size, dots = O.paged_tree_attention(q, kk, vv, bt, n, ancestors, None, window, 1)
        for s in range(3):
            masks = [int(m) & ((1 << count) - 1) for m in ancestors[s]]
            for i in range(count):
                seen = O.seen_by_new_token(lengths[s], masks, i, window, 1)
                if any(r == s and lengths[s] + j in seen for r, j, _ in bad):
                    if what == "v":
                        finite = torch.isfinite(want[s, i])
                        assert torch.equal(torch.isfinite(got[s, i]), finite) and torch.equal(got[s, i].isnan(), want[s, i].isnan())
                        assert torch.equal(got[s, i][~finite & ~want[s, i].isnan()].double(), want[s, i][~finite & ~want[s, i].isnan()])
                    else:
                        assert torch.equal(got[s, i].isnan(), want[s, i].isnan())
                else:
                    _within(got[s, i], want[s, i], _attention_tol(want[s, i], size[s, i], dots[s, i], 64, dtype))
                    _within(got[s, i], clean[s, i].double(), 2 * _attention_tol(want[s, i], size[s, i], dots[s, i], 64, dtype))


@pytest.mark.gpu
def test_tree_odd_inputs(cuda):
    """Pages that do not exist are left out, negative lengths are 0, bits past the
    tokens are not looked at, queries may be slices of a wider tensor."""
    from turbopress_amd import paged_tree_attention
    g = _gen(8)
    k, v, bt = _paged(g, [100, 64, 33, 20], 2, 64, 16, F16, extra=0, junk=0.5)
    bt[0, 3], bt[1, :4] = -1, torch.tensor([k.shape[0], -5, 2 ** 31 - 1, k.shape[0] + 1])
    n = torch.tensor([93, 60, 26, -9], dtype=torch.int32, device="cuda")
    ancestors = _trees(g, 4, 7)
    high = ancestors | torch.tensor(-1 << 7, device="cuda")
    wide = _randn(g, 7, 4, 10, 72, dtype=F16).transpose(0, 1)
    for q in (wide[:, :, 3:7, :64], wide[:, :, 3:7, 4:68], wide[:, :, 3:7, :64].contiguous(),
              _randn(g, 4, 7, 64, 4, dtype=F16).transpose(2, 3)):
        for masks in (ancestors, high, ancestors.t().contiguous().t()):
            want, size, dots = O.paged_tree_attention(q, k, v, bt, n, ancestors)
            got = paged_tree_attention(q, k, v, bt, n, ancestors=masks)
            _within(got, want, _attention_tol(want, size, dots, 64, F16))
            assert (got[1] == 0).all()
    far = torch.tensor([2 ** 31 - 1, 2 ** 31 - 65, 500, 0], dtype=torch.int32, device="cuda")
    bt[0] = torch.arange(bt.shape[1], device="cuda")
    got = paged_tree_attention(q, k, v, bt, far, ancestors=torch.zeros_like(ancestors))
    want, size, dots = O.paged_tree_attention(q[:1], k, v, bt[:1], torch.tensor([bt.shape[1] * 16]), ancestors[:1] * 0)
    _within(got[:1], want, _attention_tol(want, size, dots, 64, F16))
    assert (got[3] == 0).all()
    none = torch.empty(4, 0, dtype=torch.int32, device="cuda")
    assert (paged_tree_attention(q, k, v, none, n) == 0).all()
    assert paged_tree_attention(q[:0], k, v, bt[:0], n[:0]).shape == (0, 7, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 0), (50, 6)])
def test_tree_of_one_token_is_paged_attention(cuda, window, sinks):
    from turbopress_amd import paged_attention, paged_tree_attention
    g = _gen(4)
    lengths = [0, 1, 60, 700]
    k, v, bt = _paged(g, [n + 1 for n in lengths], 2, 64, 16, F16)
    q = _randn(g, 4, 8, 64, dtype=F16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    one = paged_attention(q, k, v, bt, n + 1, window=window, sinks=sinks)
    tree = paged_tree_attention(q[:, None], k, v, bt, n, window=window, sinks=sinks)[:, 0]
    want, size, dots = O.paged_attention(q, k, v, bt, n + 1, None, window, sinks)
    for got in (one, tree):
        _within(got, want, _attention_tol(want, size, dots, 64, F16))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 31, 32, 33, 128, 100, 1000, 10 ** 6])
@pytest.mark.parametrize("sinks", [0, 1, 4, 32, 33, 130, 10 ** 9])
def test_paged_attention_sinks(cuda, window, sinks):
    from turbopress_amd import paged_attention
    g = _gen(window + sinks)
    lengths = [0, 1, 32, 33, 100, 500, 1500]
    for dtype, hq, hkv, d, page in ((F16, 4, 1, 64, 16), (BF16, 2, 2, 128, 48)):
        k, v, bt = _paged(g, lengths, hkv, d, page, dtype)
        q = _randn(g, len(lengths), hq, d, dtype=dtype)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        want, size, dots = O.paged_attention(q, k, v, bt, n, None, window, sinks)
        got = paged_attention(q, k, v, bt, n, window=window, sinks=sinks)
        _within(got, want, _attention_tol(want, size, dots, d, dtype))
        assert torch.equal(got, paged_attention(q, k, v, bt, n, window=window, sinks=sinks))


@pytest.mark.gpu
def test_sinks_read_nothing_between(cuda):
    """Pages between the first tokens and the window may be given back: what they
    name and hold does not matter."""
    from turbopress_amd import paged_attention, paged_tree_attention
    g = _gen(5)
    k, v, bt = _paged(g, [1000], 2, 64, 16, F16)
    n = torch.tensor([1000], dtype=torch.int32, device="cuda")
    q = _randn(g, 1, 4, 64, dtype=F16)
    want = paged_attention(q, k, v, bt, n, window=100, sinks=5)
    tree = paged_tree_attention(q[:, None], k, v, bt, n - 1, window=100, sinks=5)
    gone = bt.clone()
    k[bt[0, 1:56].long()] = math.nan
    v[bt[0, 1:56].long()] = math.nan
    gone[0, 1:56:2] = -1
    assert torch.equal(paged_attention(q, k, v, gone, n, window=100, sinks=5), want)
    assert torch.equal(paged_tree_attention(q[:, None], k, v, gone, n - 1, window=100, sinks=5), tree)


@pytest.mark.gpu
def test_tree_cache_past_32_bit_offsets(cuda):
    """A cache of more than 2^31 elements, read at both its ends."""
    from turbopress_amd import paged_tree_attention
    g = _gen(11)
    pages, page, hk, d = 17000, 64, 16, 128  # 2.2e9 elements each
    k, v = (torch.zeros(pages, page, hk, d, dtype=F16, device="cuda") for _ in "kv")
    bt = torch.tensor([[0, pages - 1], [pages - 2, 1]], dtype=torch.int32, device="cuda")
    small = [torch.cat([_randn(g, 2, page, hk, d, dtype=F16) for _ in range(2)]) for _ in "kv"]
    for c, s in zip((k, v), small):
        c[bt.long().flatten()] = s
    n = torch.tensor([120, 100], dtype=torch.int32, device="cuda")
    q = _randn(g, 2, 5, 16, d, dtype=F16)
    ancestors = _trees(g, 2, 5)
    want, size, dots = O.paged_tree_attention(q, *small, torch.tensor([[0, 1], [2, 3]], device="cuda"), n, ancestors)
    _within(paged_tree_attention(q, k, v, bt, n, ancestors=ancestors), want, _attention_tol(want, size, dots, d, F16))


def test_tree_ancestors_on_the_host():
    from turbopress_amd import tree_ancestors
    parents = torch.tensor([[-1, 0, 0, 1, -1, 3, -2], [-1, 0, 1, 2, 3, 4, 5]])
    want = [[1, 3, 5, 11, 16, 43, 0], [1, 3, 7, 15, 31, 63, 127]]
    assert tree_ancestors(parents).tolist() == want and tree_ancestors(parents[0]).tolist() == want[0]
    chain = tree_ancestors(torch.arange(64) - 1)
    assert chain.tolist() == _bits([(1 << i + 1) - 1 for i in range(64)])
    with pytest.raises(ValueError):
        tree_ancestors(torch.zeros(2, 65, dtype=torch.int64))
    with pytest.raises(ValueError):
        tree_ancestors(torch.zeros(2, 5, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 16, 48])
def test_rotary_append_slots(cuda, page):
    """Keys and values go to their slots, queries and keys turn by their positions."""
    from turbopress_amd import rotary, rotary_append, rotary_table
    g = _gen(page)
    table = rotary_table(64, 64)
    tokens, hk = 40, 2
    q, k, v = (_randn(g, tokens, h, 64, dtype=F16) for h in (4, hk, hk))
    seq = torch.arange(tokens, device="cuda", dtype=torch.int32) % 2
    positions = torch.randint(0, 64, (tokens,), generator=g, device="cuda")
    slots = torch.arange(tokens, device="cuda") // 2 + 5
    positions[3], slots[4], slots[5], positions[6] = -1, -1, 10 ** 12, 64
    width = -(-30 // page)
    bt = torch.randperm(2 * width, generator=g, device="cuda").view(2, width).int()
    k_cache, v_cache = (torch.full((2 * width, page, hk, 64), 7.0, dtype=F16, device="cuda") for _ in "kv")
    want_k, want_v = k_cache.clone(), v_cache.clone()
    tq, tk = rotary(q, k, table, positions)
    for t in range(tokens):
        if t not in (3, 4, 5, 6):
            at = bt[seq[t].item(), slots[t].item() // page].item(), slots[t].item() % page
            want_k[at], want_v[at] = tk[t], v[t]
    got = rotary_append(q, k, v, table, positions, k_cache, v_cache, bt, sequences=seq, slots=slots)
    assert torch.equal(got[:6], tq[:6]) and torch.equal(got[7:], tq[7:]) and got[6].isnan().all()
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)
    other = [torch.full_like(c, 7.0) for c in (k_cache, v_cache)]
    rotary_append(q, k, v, table, positions, *other, bt, sequences=seq, slots=torch.stack((slots, slots), 1)[:, 0])
    assert torch.equal(other[0], want_k)


# ---------------------------------------------------------------------------
# log probabilities
# ---------------------------------------------------------------------------
def _check_logprobs(logits, tokens, top):
    from turbopress_amd import token_logprobs
    given, log_sum, off, lp, order, y_top, y_given = O.token_logprobs(logits, tokens, top)
    got = token_logprobs(logits, tokens, top=top)
    # each exponential e^y off by (2 |y| + 4) E, the sum of them by 2^8 additions
    # more; a log of 1 + s is off by what s is, of itself
    near = (4 * off + 300) * E
    lse = near * log_sum
    if top:
        assert got.top_tokens.dtype == torch.int64 and torch.equal(got.top_tokens, order)
        _within(got.top_logprobs, lp, lse[:, None] + 4 * E * (y_top.abs() + log_sum[:, None]) + LEAST[F32])
    else:
        assert got.top_tokens is None and got.top_logprobs is None
    if tokens is not None:
        real = tokens >= 0
        _within(got.logprobs[real], given[real], (lse + 4 * E * (y_given.abs() + log_sum))[real] + LEAST[F32])
        assert (got.logprobs[~real] == 0).all()
    else:
        assert got.logprobs is None
    _within(got.entropy, log_sum + off, near * (log_sum + off) + LEAST[F32])
    again = token_logprobs(logits, tokens, top=top)
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, again))


LOGPROBS = [(1, 1), (3, 2), (2, 7), (5, 64), (4, 255), (3, 1000), (2, 2048), (2, 2049), (3, 8191), (2, 8192), (5, 8193), (9, 16385),
            (2, 40001), (600, 1000), (70, 49152), (3, 151936), (1, 262147), (1, 1000003)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", LOGPROBS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
def test_token_logprobs(cuda, rows, vocab, dtype, top):
    g = _gen(rows + vocab)
    logits = (3 * _randn(g, rows, vocab) * torch.exp(_randn(g, rows, 1))).to(dtype)
    tokens = torch.randint(-1 if rows > 1 else 0, vocab, (rows,), generator=g, device="cuda")
    _check_logprobs(logits, tokens if top != 5 else None, min(top, vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_token_logprobs_ties(cuda, dtype, vocab):
    """Equal logits in the order of their tokens, zeros of either sign among them."""
    g = _gen(vocab)
    logits = torch.randint(-3, 3, (6, vocab), generator=g, device="cuda").to(dtype)
    logits[1] = 0
    logits[2] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, -0.0, 0.0).to(dtype)
    logits[3], logits[3, 1::7] = -5, 2
    logits[4, :] = torch.arange(vocab, device="cuda").to(dtype) / vocab
    logits[5] = -logits[4]
    _check_logprobs(logits, torch.arange(6, device="cuda"), 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_token_logprobs_near_certain(cuda, dtype):
    """Rows whose largest probability is 1 but for 1e-3 to 1e-20, and rows under a
    mask of the type's lowest value or of -infinity."""
    g = _gen(7)
    logits = _randn(g, 8, 30000, dtype=dtype)
    for r, x in enumerate((17, 24, 30, 40, 57)):
        logits[r, 12345] = x
    logits[5], logits[6] = torch.finfo(dtype).min, -math.inf
    logits[5:7, 77], logits[5:7, 29000] = 1.5, 1.0
    logits[7] = 0.25
    tokens = torch.full((8,), 12345, device="cuda")
    tokens[5], tokens[6] = 77, 29000
    _check_logprobs(logits, tokens, 2)
    from turbopress_amd import token_logprobs
    got = token_logprobs(logits, torch.zeros_like(tokens), top=4)
    assert got.logprobs[6] == -math.inf and (got.top_logprobs[6, 2:] == -math.inf).all()
    assert got.top_tokens[6].tolist() == [77, 29000, 0, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50, 9000, 40000])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_token_logprobs_without_a_distribution(cuda, vocab, dtype):
    """Nothing possible: -infinity and entropy 0.  NaN or +infinity: NaN.  The rows
    beside them are as without."""
    from turbopress_amd import token_logprobs
    g = _gen(vocab)
    logits = _randn(g, 5, vocab, dtype=dtype)
    clean = token_logprobs(logits, torch.arange(5, device="cuda"), top=3)
    logits[1], logits[2, 7], logits[2, 40] = -math.inf, math.nan, math.inf
    logits[3, 44], logits[3, 2] = math.inf, math.inf
    tokens = torch.arange(5, device="cuda")
    tokens[4] = vocab
    got = token_logprobs(logits, tokens, top=3)
    assert all(torch.equal(a[0], b[0]) for a, b in zip(got, clean))
    assert got.logprobs[1] == -math.inf and got.entropy[1] == 0 and (got.top_logprobs[1] == -math.inf).all()
    assert got.top_tokens[1].tolist() == [0, 1, 2]
    for r in (2, 3):
        assert got.logprobs[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all()
    assert got.top_tokens[2, :2].tolist() == [7, 40] and got.top_tokens[3, :2].tolist() == [2, 44]
    assert got.logprobs[4].isnan() and torch.equal(got.entropy[4], clean.entropy[4])
    # (a logit of +infinity among -infinity is no distribution either)
    logits[1, 3] = math.inf
    assert token_logprobs(logits, tokens).logprobs[1].isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (0, 1), (5, 3), (64, 8)])
def test_token_logprobs_rows_apart(cuda, dtype, pad, offset):
    """Rows of slices of wider tensors at any alignment, NaN between them."""
    from turbopress_amd import token_logprobs
    g = _gen(pad + offset)
    for rows, vocab in ((4, 1001), (3, 20003)):
        raw = torch.full((rows * (vocab + pad) + offset,), math.nan, dtype=dtype, device="cuda")
        logits = raw[offset:].view(rows, vocab + pad)[:, :vocab]
        logits.copy_(_randn(g, rows, vocab))
        tokens = torch.arange(rows, device="cuda") * 7
        want = token_logprobs(logits.contiguous(), tokens, top=9)
        got = token_logprobs(logits, torch.stack((tokens, tokens), 1)[:, 0], top=9)
        for a, b in zip(got, want):
            if a.dtype == torch.int64:
                assert torch.equal(a, b)
            else:  # (an alignment may cut a row elsewhere: sums in another order)
                assert (a - b).abs().max() <= 2.0 ** -20 * (1 + b.abs().max())
        _check_logprobs(logits, tokens, 9)
    wide = _randn(g, 50, 6, dtype=dtype)
    _check_logprobs(wide.t(), None, 3)
    _check_logprobs(wide[:1].expand(4, 6), None, 3)
    assert token_logprobs(wide[:0], top=2).top_tokens.shape == (0, 2)


@pytest.mark.gpu
def test_token_logprobs_past_32_bit_offsets(cuda):
    from turbopress_amd import token_logprobs
    rows, vocab = 15000, 151936  # 2.3e9 elements
    x = torch.zeros(rows, vocab, dtype=F16, device="cuda")
    x[-2:] = _randn(_gen(3), 2, vocab, dtype=F16)
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    got = token_logprobs(x, tokens, top=3)
    want = token_logprobs(x[-2:].clone(), tokens[-2:], top=3)
    assert torch.equal(got.top_tokens[-2:], want.top_tokens)
    assert (got.entropy[-2:] - want.entropy).abs().max() <= 2.0 ** -18 and (got.top_tokens[:-2] == torch.arange(3, device="cuda")).all()
    assert (got.logprobs[:-2] + math.log(vocab)).abs().max() <= 2.0 ** -18


# ---------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------
def _lora_case(g, rows, k, n, rank, count, dtype):
    y, x = _randn(g, rows, n, dtype=dtype), _randn(g, rows, k, dtype=dtype)
    a, b = (_randn(g, count, rank, k) / math.sqrt(k)).to(dtype), _randn(g, count, n, rank, dtype=dtype)
    ids = torch.randint(-1, count + 1, (rows,), generator=g, device="cuda").int()
    return y, x, a, b, ids, torch.exp2(torch.randint(-2, 3, (count,), generator=g, device="cuda").float())


def _lora_tol(want, size, k, rank, dtype):
    # sums of 8 products and more at a time in fp32 (k + rank at most), the first
    # product's result in two pieces (2^-16 of it lost)
    return U[dtype] * want.abs() + ((k + rank) * E + 2.0 ** -16) * size + LEAST[dtype]


def _check_lora(g, rows, k, n, rank, count, dtype, ids=None, scaled=True):
    from turbopress_amd import lora_add
    y, x, a, b, drawn, scales = _lora_case(g, rows, k, n, rank, count, dtype)
    ids = drawn if ids is None else ids
    scales = scales if scaled else None
    want, size = O.lora_add(y, x, a, b, ids, scales)
    before = y.clone()
    got = lora_add(y, x, a, b, ids, scales=scales)
    assert got.shape == y.shape and got.dtype == dtype and got.is_contiguous() and torch.equal(y, before)
    _within(got, want, _lora_tol(want, size, k, rank, dtype))
    none = (ids < 0) | (ids >= count)
    assert torch.equal(got[none], y[none])
    assert torch.equal(got, lora_add(y, x, a, b, ids, scales=scales))


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 2, 7, 8, 16, 17, 31, 32, 33, 64, 65, 100, 128, 200, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_lora_ranks(cuda, rank, dtype):
    _check_lora(_gen(rank), 20, 256, 192, rank, 3, dtype)
    _check_lora(_gen(rank), 3, 100, 77, rank, 2, dtype, scaled=False)


@pytest.mark.gpu
@pytest.mark.parametrize("k,n", [(1, 1), (7, 3), (8, 16), (33, 65), (100, 1000), (256, 255), (576, 1536), (1001, 999), (2560, 4096),
                                 (9728, 2560), (10001, 130)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rank", [16, 40])
def test_lora_sizes(cuda, k, n, dtype, rank):
    _check_lora(_gen(k + n), 5, k, n, rank, 2, dtype)
    _check_lora(_gen(k + n), 70, k, n, rank, 2, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 129, 300, 1000])
@pytest.mark.parametrize("count", [1, 4, 100])
def test_lora_rows_and_adapters(cuda, rows, count):
    """One adapter for all, as many as rows, none at all; in any order and in runs."""
    g = _gen(rows + count)
    _check_lora(g, rows, 320, 200, 16, count, F16)
    runs = torch.randint(-1, count, (rows,), generator=g, device="cuda").int().sort().values
    _check_lora(g, rows, 320, 200, 16, count, BF16, ids=runs)
    _check_lora(g, rows, 320, 200, 16, count, F16, ids=torch.full((rows,), -1, dtype=torch.int32, device="cuda"))
    _check_lora(g, rows, 320, 200, 16, count, F16, ids=torch.full((rows,), count - 1, dtype=torch.int32, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_lora_rows_do_not_mix(cuda, dtype):
    """NaN and infinity in a row, in an adapter or in the weights of others stay there."""
    from turbopress_amd import lora_add
    g = _gen(2)
    y, x, a, b, _, scales = _lora_case(g, 40, 200, 100, 16, 4, dtype)
    ids = (torch.arange(40, device="cuda") % 4).int()
    ids[7] = -1
    clean = lora_add(y, x, a, b, ids, scales=scales)
    x[3, 5], x[8, 7], a[1, 3, 4], b[2, 9] = math.nan, math.inf, math.nan, math.inf
    x[7], y[10, 3] = math.nan, math.inf
    got = lora_add(y, x, a, b, ids, scales=scales)
    row = torch.arange(40, device="cuda")
    touched = (row == 3) | (row == 8) | (ids == 1) | (ids == 2)
    assert torch.equal(got[~touched], clean[~touched])
    assert got[3].isnan().all() and got[ids == 1].isnan().all() and not got[8].isfinite().any()
    others = torch.arange(100, device="cuda") != 9
    mine = (ids == 2) & (row != 10)
    assert torch.equal(got[mine][:, others], clean[mine][:, others]) and not got[mine][:, 9].isfinite().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_lora_wide_range(cuda, dtype):
    """Inner products beyond fp16's largest and below its least."""
    from turbopress_amd import lora_add
    g = _gen(6)
    y, x, a, b, ids, _ = _lora_case(g, 24, 256, 64, 16, 2, dtype)
    ids = (ids % 2).abs().int()
    for xs, bs in ((2.0 ** 12, 2.0 ** -12), (2.0 ** -10, 2.0 ** 8)):
        x2, a2, b2 = (x * xs), (a * 16 * (xs if xs < 1 else 16)).to(dtype), (b * bs).to(dtype)
        y2 = y if xs > 1 else (y * 2.0 ** -9).to(dtype)
        want, size = O.lora_add(y2, x2, a2, b2, ids)
        got = lora_add(y2, x2, a2, b2, ids)
        _within(got, want, _lora_tol(want, size, 256, 16, dtype))


@pytest.mark.gpu
def test_lora_shapes_and_strides(cuda):
    """Leading dimensions, slices of wider tensors, transposed and unaligned weights."""
    from turbopress_amd import lora_add
    g = _gen(12)
    y, x, a, b, ids, scales = _lora_case(g, 24, 200, 120, 24, 3, F16)
    want = lora_add(y, x, a, b, ids, scales=scales)
    tol = 2 * _lora_tol(want.double(), O.lora_add(y, x, a, b, ids, scales)[1], 200, 24, F16)
    wide = torch.full((24, 1000), math.nan, dtype=F16, device="cuda")
    wide[:, 3:203], wide[:, 301:421] = x, y
    views = [(y.view(2, 3, 4, 120), x.view(2, 3, 4, 200), a, b, ids.view(2, 3, 4)),
             (wide[:, 301:421], wide[:, 3:203], a, b, ids),
             (y, x, a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(1, 2).contiguous().transpose(1, 2), ids),
             (y.t().contiguous().t(), x.t().contiguous().t(), a, b, torch.stack((ids, ids), 1)[:, 0]),
             (y, x, torch.cat((a, a), 1)[:, :24], torch.cat((b, b), 2)[:, :, :24], ids),
             (y, x, torch.cat((a.flatten(), a.flatten()))[1:1 + a.numel()].copy_(a.flatten()).view(a.shape), b, ids)]
    for yy, xx, aa, bb, ii in views:
        _within(lora_add(yy, xx, aa, bb, ii, scales=scales).view(24, 120), want.double(), tol)
    one = lora_add(y[0], x[0], a, b, ids[0], scales=scales)
    assert one.shape == (120,)
    _within(one, want[0].double(), tol[0])
    assert lora_add(y[:0], x[:0], a, b, ids[:0]).shape == (0, 120)
    assert torch.equal(lora_add(y, x, a[:0], b[:0], ids), y)
    same = lora_add(y, x[:1].expand(24, 200), a, b, ids, scales=scales)
    _within(same, lora_add(y, x[:1].repeat(24, 1), a, b, ids, scales=scales).double(), tol + 1e-2)


@pytest.mark.gpu
def test_lora_past_32_bit_offsets(cuda):
    from turbopress_amd import lora_add
    g = _gen(13)
    rows, k, n = 230000, 64, 9728  # 2.2e9 elements
    y = torch.zeros(rows, n, dtype=F16, device="cuda")
    x = torch.zeros(rows, k, dtype=F16, device="cuda")
    x[-3:] = _randn(g, 3, k, dtype=F16)
    _, _, a, b, _, _ = _lora_case(g, 1, k, n, 8, 2, F16)
    ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids[-2] = 1
    got = lora_add(y, x, a, b, ids)
    want, size = O.lora_add(y[-3:], x[-3:], a, b, ids[-3:])
    _within(got[-3:], want, _lora_tol(want, size, k, 8, F16))
    assert (got[-100:-3] == 0).all() and (got[:100] == 0).all()


# ---------------------------------------------------------------------------
# together, in graphs, on streams; refusals
# ---------------------------------------------------------------------------
def _serve(g):
    """A checked step of drafted tokens of three sequences: an adapter beside the
    projection, keys and values appended, attention of the trees, another adapter,
    log probabilities."""
    from turbopress_amd import lora_add, paged_attention, paged_tree_attention, rotary_append, rotary_table, token_logprobs
    lengths, count = [700, 31, 0], 5
    k_cache, v_cache, bt = _paged(g, [n + count for n in lengths], 2, 64, 16, F16, junk=0.0)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    x = _randn(g, 3 * count, 256, dtype=F16)
    base = _randn(g, 3 * count, 512, dtype=F16)
    a, b = (0.1 * _randn(g, 2, 16, 256)).to(F16), (0.1 * _randn(g, 2, 512, 16)).to(F16)
    head = _randn(g, 256, 3001, dtype=F16) * 0.1
    seq = torch.arange(3, device="cuda", dtype=torch.int32).repeat_interleave(count)
    ids = torch.tensor([0, -1, 1], dtype=torch.int32, device="cuda").repeat_interleave(count)
    ancestors = _trees(g, 3, count)
    table = rotary_table(1000, 64)
    depth = torch.tensor([[bin(int(m) & 31).count("1") for m in row] for row in ancestors], device="cuda")
    positions = (n[:, None] + depth - 1).flatten().clamp(min=0)
    slots = (n[:, None] + torch.arange(count, device="cuda")).flatten()

    def run():
        qkv = lora_add(base, x, a, b, ids).view(-1, 8, 64)
        q = rotary_append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], table, positions, k_cache, v_cache, bt, sequences=seq, slots=slots)
        o = paged_tree_attention(q.view(3, count, 4, 64), k_cache, v_cache, bt, n, ancestors=ancestors)
        one = paged_attention(q.view(3, count, 4, 64)[:, 0], k_cache, v_cache, bt, n + 1, window=100, sinks=4)
        got = token_logprobs(o.view(-1, 256) @ head, seq.long(), top=7)
        return o, one, *got

    return x, run


@pytest.mark.gpu
def test_serving_operators_in_a_graph(cuda):
    x, run = _serve(_gen(20))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(5):
        x.copy_(_randn(_gen(100 + i), *x.shape, dtype=F16))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


@pytest.mark.gpu
def test_serving_operators_on_two_streams_and_in_two_graphs(cuda):
    """The same calls on two streams at once beside two graphs, each with
    workspaces of its own."""
    steps = [_serve(_gen(30 + i)) for i in range(4)]
    want = [[t.clone() for t in run()] for _, run in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    graphs = []
    for i in (2, 3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = steps[i][1]()
        graphs.append((i, graph, outs))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(steps[i][1]())
        for i, graph, _ in graphs:
            with torch.cuda.stream(streams[i]):
                graph.replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for o in outs[i] for a, b in zip(o, want[i]))
    for i, _, o in graphs:
        assert all(torch.equal(a, b) for a, b in zip(o, want[i]))


def _c(shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def test_cpu_tensors_are_refused():
    import turbopress_amd as T
    cache, bt, n = _c((1, 4, 1, 8)), _c((2, 1), torch.int32), _c((2,), torch.int32)
    for call in (lambda: T.paged_tree_attention(_c((2, 3, 1, 8)), cache, cache, bt, n),
                 lambda: T.paged_attention(_c((2, 1, 8)), cache, cache, bt, n, window=2, sinks=1),
                 lambda: T.token_logprobs(_c((2, 8))),
                 lambda: T.lora_add(_c((2, 8)), _c((2, 8)), _c((1, 2, 8)), _c((1, 8, 2)), n)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.gpu
def test_bad_arguments_are_refused(cuda):
    import turbopress_amd as T

    def z(*shape, dtype=F16):
        return torch.zeros(*shape, dtype=dtype, device=cuda)

    i32, i64 = torch.int32, torch.int64
    q, c, bt, n, m = z(2, 3, 4, 8), z(3, 4, 2, 8), z(2, 1, dtype=i32), z(2, dtype=i32), z(2, 3, dtype=i64)
    rq, rk, pos, table = z(2, 4, 8), z(2, 2, 8), z(2, dtype=i64), z(4, 8, dtype=F32)
    x, t = z(2, 9), z(2, dtype=i64)
    y, lx, a, b, ids, s = z(2, 6), z(2, 5), z(3, 2, 5), z(3, 6, 2), z(2, dtype=i32), z(3, dtype=F32)
    bad = [
        lambda: T.paged_tree_attention(q[:, 0], c, c, bt, n), lambda: T.paged_tree_attention(q.float(), c.float(), c.float(), bt, n),
        lambda: T.paged_tree_attention(z(2, 65, 4, 8), c, c, bt, n), lambda: T.paged_tree_attention(z(2, 0, 4, 8), c, c, bt, n),
        lambda: T.paged_tree_attention(q, c.bfloat16(), c, bt, n), lambda: T.paged_tree_attention(q, c, c[:, :3], bt, n),
        lambda: T.paged_tree_attention(q, c, c, bt.long(), n), lambda: T.paged_tree_attention(q, c, c, bt[:1], n),
        lambda: T.paged_tree_attention(q, c, c, bt, n[:1]), lambda: T.paged_tree_attention(q, c, c, bt, n.long()),
        lambda: T.paged_tree_attention(q, c, c, bt, n, ancestors=m[:1]), lambda: T.paged_tree_attention(q, c, c, bt, n, ancestors=m.int()),
        lambda: T.paged_tree_attention(q, c, c, bt, n, ancestors=m.cpu()), lambda: T.paged_tree_attention(q, c, c, bt, n, window=-1),
        lambda: T.paged_tree_attention(q, c, c, bt, n, window=4, sinks=-1), lambda: T.paged_tree_attention(q[:, :, :3], c, c, bt, n),
        lambda: T.paged_tree_attention(q[..., :4], c[..., :4], c[..., :4], bt, n),
        lambda: T.paged_tree_attention(z(2, 3, 4, 264), z(3, 4, 2, 264), z(3, 4, 2, 264), bt, n),
        lambda: T.paged_attention(rq, c, c, bt, n, window=3, sinks=-1),
        lambda: T.rotary_append(rq, rk, rk, table, pos, c, c, bt, slots=pos.int()),
        lambda: T.rotary_append(rq, rk, rk, table, pos, c, c, bt, slots=pos[:1]),
        lambda: T.rotary_append(rq, rk, rk, table, pos, c, c, bt, slots=pos.cpu()),
        lambda: T.token_logprobs(x[0]), lambda: T.token_logprobs(x.double()), lambda: T.token_logprobs(z(2, 0)),
        lambda: T.token_logprobs(x, t.int()), lambda: T.token_logprobs(x, t[:1]), lambda: T.token_logprobs(x, t.cpu()),
        lambda: T.token_logprobs(x, t, top=10), lambda: T.token_logprobs(x, t, top=-1), lambda: T.token_logprobs(z(2, 100), t, top=65),
        lambda: T.lora_add(y.float(), lx, a, b, ids), lambda: T.lora_add(y, lx.bfloat16(), a, b, ids), lambda: T.lora_add(y, lx[:1], a, b, ids),
        lambda: T.lora_add(y, lx, a[0], b, ids), lambda: T.lora_add(y, lx, a, b[:2], ids), lambda: T.lora_add(y, lx, a, b[:, :5], ids),
        lambda: T.lora_add(y, lx, a[:, :1], b, ids), lambda: T.lora_add(y, lx, a[..., :4], b, ids),
        lambda: T.lora_add(y, lx, a, b, ids.long()), lambda: T.lora_add(y, lx, a, b, ids[:1]), lambda: T.lora_add(y, lx, a, b, ids.cpu()),
        lambda: T.lora_add(y, lx, a, b, ids, scales=s[:2]), lambda: T.lora_add(y, lx, a, b, ids, scales=s.half()),
        lambda: T.lora_add(y, lx, z(3, 257, 5), z(3, 6, 257), ids), lambda: T.lora_add(y, lx, z(3, 0, 5), z(3, 6, 0), ids),
        lambda: T.lora_add(y, z(2, 0), z(3, 2, 0), b, ids), lambda: T.lora_add(y[:, :0], lx, a, b[:, :0], ids),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
