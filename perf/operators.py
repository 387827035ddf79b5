"""Cases of the decoder operators that run between the packed projections.

  norm       -- root-mean-square norm, with the residual's addition or without,
                its output in the input's type or in 8-bit floating point
                (e4m3) with a scale per row or per 128 columns
  fp8        -- product of 8-bit floating point activations and weights, a scale
                per row and 128 columns of the one and per 128 x 128 block of
                the other (the dense head of a packed model)
  rotary     -- rotary positions of queries and keys, alone or with keys and
                values written into a paged cache
  attention  -- attention of one new token per sequence over a paged cache

``run`` computes them by elementary torch operations in 32 bits, or, where
``own`` is set, through ``turbopress_amd``'s entry points.  Sizes are those of
the decoders that the package configures (SmolLM2-135M, Qwen3-0.6B, Qwen3-4B)
and, for ``draw``, sizes between and around them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
BLOCK = 128
LEAST_SCALE = 2.0 ** -126  # the scale of a block of zeros
EPS = 1e-6
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _norm(name, rows, d, dtype, residual, scales, pad=0):
    """scales: "none" (output in the input's type), "row" or "block" (e4m3);
    pad: columns by which the input's rows lie further apart than d."""
    return {"name": name, "op": "norm", "rows": rows, "d": d, "type": dtype, "residual": residual, "scales": scales,
            "pad": pad}


def _fp8(name, m, n, k, dtype):
    return {"name": name, "op": "fp8", "m": m, "n": n, "k": k, "type": dtype}


def _rotary(name, tokens, hq, hkv, d, rotary, interleaved, append, dtype, page=16, sequences=1, fused=False):
    """sequences: how many the tokens are of (each of tokens / sequences new
    ones); fused: q, k and v are slices of one projection's output."""
    return {"name": name, "op": "rotary", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rotary": rotary,
            "interleaved": interleaved, "append": append, "type": dtype, "page": page, "sequences": sequences,
            "fused": fused}


def _attention(name, batch, length, ragged, hq, hkv, d, page, dtype, window=0):
    """ragged: the sequences' lengths lie between 0 and `length`, else all have it."""
    return {"name": name, "op": "attention", "batch": batch, "length": length, "ragged": ragged, "hq": hq, "hkv": hkv,
            "d": d, "page": page, "type": dtype, "window": window}


def listed() -> list:
    return [
        # before a projection of one decode step of one sequence (Qwen3-4B)
        _norm("norm_step", 1, 2560, "fp16", True, "none"),
        # a prompt's rows for products in 8 bits
        _norm("norm_prompt_8bit", 2048, 2560, "bf16", True, "block"),
        # rows as long as the MLP's, of odd length, a large batch of prompts
        _norm("norm_long_rows", 8191, 9727, "fp16", False, "none"),
        # the head of a decode step: every weight read for one row (Qwen3-4B)
        _fp8("fp8_head_step", 1, 151936, 2560, "fp32"),
        # a short prompt of an odd length through q_proj's shape
        _fp8("fp8_prompt_199", 199, 4096, 2560, "fp16"),
        # a long prompt through the widest projection's shape
        _fp8("fp8_prompt_2048", 2048, 9728, 2560, "bf16"),
        # one decode step of four sequences (Qwen3-4B heads), into the cache
        _rotary("rotary_step", 4, 32, 8, 128, 128, False, True, "fp16", sequences=4),
        # a prompt into the cache, a quarter of the head rotated in pairs
        _rotary("rotary_prompt", 2047, 16, 8, 128, 32, True, True, "bf16", page=64, fused=True),
        # a batch of prompts, small heads (SmolLM2-135M), no cache
        _rotary("rotary_long", 32768, 9, 3, 64, 64, False, False, "fp16", sequences=16),
        # one sequence with a short context (Qwen3-0.6B heads)
        _attention("attention_short", 1, 577, False, 16, 8, 128, 16, "fp16"),
        # one sequence with a long context (Qwen3-4B heads): few rows, a long axis
        _attention("attention_long", 1, 131072, False, 32, 8, 128, 64, "fp16"),
        # many sequences of uneven lengths, some of them empty
        _attention("attention_batch", 64, 8192, True, 32, 8, 128, 16, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(("norm", "fp8", "rotary", "attention"))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "norm":
        d = rng.choice((_log(rng, 64, 16384), rng.choice((64, 128, 576, 1024, 2560, 9728))))
        rows = _log(rng, 1, max(1, min(65536, 8191 * 9727 // (2 * d))))
        c = _norm("", rows, d, rng.choice((dtype, dtype, "fp32")), rng.random() < 0.5, rng.choice(("none", "none", "row", "block")),
                  rng.choice((0, 0, d, 3)))
    elif op == "fp8":
        n, k = _log(rng, 100, 16384), _log(rng, 100, 10000)
        m = min(_log(rng, 1, 2048), max(1, 2048 * 9728 * 2560 // (n * k)))
        c = _fp8("", m, n, k, rng.choice((dtype, dtype, "fp32")))
    elif op == "rotary":
        hkv, d = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 80, 96, 128, 256))
        hq = hkv * rng.choice((1, 2, 3, 4, 8))
        sequences = _log(rng, 1, 64)
        each = _log(rng, 1, max(1, min(8192, 32768 * 12 * 64 // (sequences * (hq + 2 * hkv) * d))))
        c = _rotary("", sequences * each, hq, hkv, d, rng.choice((d, d, d // 2, d // 4)), rng.random() < 0.5,
                    rng.random() < 0.5, dtype, rng.choice((1, 16, 48, 64, 256)), sequences, rng.random() < 0.5)
    else:
        hkv, d = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 80, 96, 128, 256))
        batch = _log(rng, 1, 256)
        length = _log(rng, 1, max(1, min(131072, 64 * 4096 * 8 * 128 // (batch * hkv * d))))
        c = _attention("", batch, length, rng.random() < 0.5, hkv * rng.choice((1, 2, 3, 4, 7, 8, 16)), hkv, d,
                       rng.choice((1, 16, 48, 64, 256)), dtype, rng.choice((0, 0, 0, _log(rng, 1, 4096))))
    del c["name"]
    return c


def _lengths(case) -> list:
    """The sequences' lengths: the case's own, whatever the seed."""
    if not case["ragged"]:
        return [case["length"]] * case["batch"]
    rng = random.Random(case["batch"] * 1000003 + case["length"])
    return [0 if rng.random() < 0.05 else rng.randint(1, case["length"]) for _ in range(case["batch"])]


def _seen(case) -> int:
    """Cached tokens that the attention of the case reads."""
    w = case["window"]
    return sum(min(n, w) if w else n for n in _lengths(case))


def work(case) -> dict:
    s = BYTES[case["type"]]
    if case["op"] == "norm":
        el = case["rows"] * case["d"]
        out = el * s if case["scales"] == "none" else el + 4 * case["rows"] * (
            1 if case["scales"] == "row" else -(-case["d"] // BLOCK))
        return {"bytes": el * s * (3 if case["residual"] else 1) + out + case["d"] * s, "flops": 4 * el}
    if case["op"] == "fp8":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": m * k + n * k + 4 * kb * (m + -(-n // BLOCK)) + m * n * s, "flops": 2 * m * n * k}
    if case["op"] == "rotary":
        heads = case["hq"] + case["hkv"] * (2 if case["append"] else 1)
        return {"bytes": case["tokens"] * (2 * heads * case["d"] * s + 4 * case["rotary"] + 8),
                "flops": 3 * case["tokens"] * (case["hq"] + case["hkv"]) * case["rotary"]}
    seen = _seen(case)
    return {"bytes": 2 * seen * case["hkv"] * case["d"] * s + 2 * case["batch"] * case["hq"] * case["d"] * s
            + 4 * -(-seen // case["page"]) + 4 * case["batch"],
            "flops": 4 * seen * case["hq"] * case["d"]}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _outliers(x, g):
    """Activations as a decoder has them: one column in a hundred 20 times larger."""
    big = torch.rand(x.shape[-1], generator=g, device=DEV) < 0.01
    return x * (1 + 19 * big.to(x.dtype))


def _in_blocks(w):
    """(codes, scales) of a weight matrix, a scale per 128 x 128 block."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    p = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    s = (p.abs().amax((1, 3)) / F8_MAX).clamp(min=LEAST_SCALE)
    codes = (p / s[:, None, :, None]).to(F8).view(nb * BLOCK, kb * BLOCK)
    return codes[:n, :k].contiguous(), s


def _in_rows(x):
    """(codes, scales) of activations, a scale per row and 128 columns."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    p = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).view(m, kb, BLOCK)
    s = (p.abs().amax(2) / F8_MAX).clamp(min=LEAST_SCALE)
    return (p / s[:, :, None]).to(F8).view(m, kb * BLOCK)[:, :k].contiguous(), s


def _pages(count, pages, width, g):
    """A block table [count, width]: the cache's pages in the order in which a
    server has handed them out."""
    return torch.randperm(pages, generator=g, device=DEV)[:count * width].view(count, width).to(torch.int32)


def prepare(case, seed) -> dict:
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    dtype = TYPES[case["type"]]
    st = {"case": case}
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        st["x"] = _outliers(normal(rows, d + case["pad"]), g).to(dtype)[:, :d]
        st["residual"] = (4 * normal(rows, d)).to(dtype) if case["residual"] else None
        st["weight"] = (1 + 0.2 * normal(d)).to(dtype)
    elif case["op"] == "fp8":
        st["w"], st["w_scales"] = _in_blocks(0.02 * normal(case["n"], case["k"]))
        st["a"], st["a_scales"] = _in_rows(_outliers(normal(case["m"], case["k"]), g))
    elif case["op"] == "rotary":
        t, hq, hkv, d, n = case["tokens"], case["hq"], case["hkv"], case["d"], case["sequences"]
        each = t // n
        if case["fused"]:
            qkv = normal(t, (hq + 2 * hkv) * d).to(dtype).view(t, hq + 2 * hkv, d)
            st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            st["q"], st["k"], st["v"] = (normal(t, h, d).to(dtype) for h in (hq, hkv, hkv))
        past = torch.randint(0, 512, (n, 1), generator=g, device=DEV)
        st["positions"] = (past + torch.arange(each, device=DEV)).reshape(-1)
        # frequencies at base 10000, their cosines and sines from 64 bits
        half = case["rotary"] // 2
        angle = torch.arange(512 + each, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device=DEV, dtype=torch.float64) / half)
        st["table"] = torch.cat((angle.cos(), angle.sin()), 1).float()
        if case["append"]:
            width = -(-(512 + each) // case["page"])
            pages = n * width + 3
            st["sequences"] = torch.arange(n, device=DEV, dtype=torch.int32).repeat_interleave(each)
            st["block_table"] = _pages(n, pages, width, g)
            st["k_cache"], st["v_cache"] = (torch.zeros(pages, case["page"], hkv, d, dtype=dtype, device=DEV) for _ in "kv")
    else:
        lengths = _lengths(case)
        width = max(1, -(-max(lengths) // case["page"]))
        b, pages = case["batch"], case["batch"] * width + 3
        st["q"] = (1.5 * normal(b, case["hq"], case["d"])).to(dtype)
        st["k_cache"], st["v_cache"] = (
            torch.empty(pages, case["page"], case["hkv"], case["d"], dtype=dtype, device=DEV).normal_(generator=g) for _ in "kv")
        st["block_table"] = _pages(b, pages, width, g)
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st, st["case"])


def _run_own(st, case):
    if case["op"] == "norm":
        from turbopress_amd import rms_norm, rms_norm_fp8
        if case["scales"] == "none":
            got = rms_norm(st["x"], st["weight"], EPS, residual=st["residual"])
        else:
            got = rms_norm_fp8(st["x"], st["weight"], EPS, residual=st["residual"],
                               block=BLOCK if case["scales"] == "block" else None)
        return got if isinstance(got, tuple) else (got,)
    if case["op"] == "fp8":
        from turbopress_amd import fp8_linear
        return fp8_linear(st["a"], st["a_scales"], st["w"], st["w_scales"], out_dtype=TYPES[case["type"]])
    if case["op"] == "rotary":
        from turbopress_amd import rotary, rotary_append
        if not case["append"]:
            return rotary(st["q"], st["k"], st["table"], st["positions"], interleaved=case["interleaved"])
        q = rotary_append(st["q"], st["k"], st["v"], st["table"], st["positions"], st["k_cache"], st["v_cache"],
                          st["block_table"], sequences=st["sequences"], interleaved=case["interleaved"])
        return q, st["k_cache"], st["v_cache"]
    from turbopress_amd import paged_attention
    return paged_attention(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["lengths"], window=case["window"])


def _run_plain(st, case):
    if case["op"] == "norm":
        return _plain_norm(st, case)
    if case["op"] == "fp8":
        a = st["a"].float() * _columns(st["a_scales"], case["k"])
        w = st["w"].float() * _columns(st["w_scales"], case["k"]).repeat_interleave(BLOCK, 0)[:case["n"]]
        return torch.matmul(a, w.t()).to(TYPES[case["type"]])
    if case["op"] == "rotary":
        return _plain_rotary(st, case)
    return _plain_attention(st, case)


def _columns(scales, k):
    return scales.repeat_interleave(BLOCK, 1)[:, :k]


def _plain_norm(st, case):
    x, dtype, d = st["x"], st["x"].dtype, case["d"]
    h = x.float() if st["residual"] is None else x.float() + st["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * st["weight"].float()
    if case["scales"] == "none":
        got = (y.to(dtype),)
    else:
        width = d if case["scales"] == "row" else BLOCK
        count = -(-d // width)
        p = torch.nn.functional.pad(y, (0, count * width - d)).view(-1, count, width)
        s = (p.abs().amax(2) / F8_MAX).clamp(min=LEAST_SCALE)
        got = ((p / s[:, :, None]).clamp(-F8_MAX, F8_MAX).to(F8).view(-1, count * width)[:, :d], s)
    return got if st["residual"] is None else (*got, h.to(dtype))


def _plain_turn(x, table, positions, interleaved):
    rd = table.shape[1]
    cos, sin = (t[:, None] for t in table[positions].split(rd // 2, 1))
    f = x.float()
    a, b = (f[..., 0:rd:2], f[..., 1:rd:2]) if interleaved else (f[..., :rd // 2], f[..., rd // 2:rd])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, f[..., rd:]), -1).to(x.dtype)


def _plain_rotary(st, case):
    q, k = (_plain_turn(st[n], st["table"], st["positions"], case["interleaved"]) for n in "qk")
    if not case["append"]:
        return q, k
    page = st["block_table"][st["sequences"].long(), st["positions"] // case["page"]].long()
    at = st["positions"] % case["page"]
    st["k_cache"][page, at] = k
    st["v_cache"][page, at] = st["v"]
    return q, st["k_cache"], st["v_cache"]


def _plain_attention(st, case):
    b, hkv, d = case["batch"], case["hkv"], case["d"]
    pages = st["block_table"].long()
    at = torch.arange(pages.shape[1] * case["page"], device=DEV)
    seen = at < st["lengths"][:, None]
    if case["window"]:
        seen &= at >= st["lengths"][:, None] - case["window"]
    # [sequence, token, head, column] of the pages that each sequence has
    k, v = (c[pages].flatten(1, 2).float() for c in (st["k_cache"], st["v_cache"]))
    q = st["q"].float().view(b, hkv, -1, d) / math.sqrt(d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous())
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill(~seen[:, :, None, None], 0).transpose(1, 2).contiguous()
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1)
    return out.view(b, -1, d).to(st["q"].dtype)


# ---------------------------------------------------------------------------
# in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"norm": _exact_norm, "fp8": _exact_fp8, "rotary": _exact_rotary, "attention": _exact_attention}[case["op"]](st, case)


def _exact_norm(st, case):
    h = st["x"].double()
    if st["residual"] is not None:
        h = h + st["residual"].double()
    y = st["weight"].double() * h / (h.square().sum(1, keepdim=True) / case["d"] + EPS).sqrt()
    if case["scales"] == "none":
        got = [y]
    else:
        parts = list(y.split(case["d"] if case["scales"] == "row" else BLOCK, 1))
        scales = [p.abs().max(1, keepdim=True).values.div(F8_MAX).clamp(min=LEAST_SCALE) for p in parts]
        # (the values before they are rounded to 8 bits)
        got = [torch.cat([p / s for p, s in zip(parts, scales)], 1), torch.cat(scales, 1)]
    return (*got, h) if st["residual"] is not None else tuple(got)


def _exact_fp8(st, case):
    k, n = case["k"], case["n"]
    y = torch.zeros(case["m"], n, dtype=torch.float64, device=DEV)
    for j in range(st["a_scales"].shape[1]):
        cols = slice(BLOCK * j, min(k, BLOCK * (j + 1)))
        a = st["a"][:, cols].double() * st["a_scales"][:, j:j + 1].double()
        w = st["w"][:, cols].double()
        for i in range(0, n, 16384):
            r = torch.arange(i, min(n, i + 16384), device=DEV)
            y[:, i:i + 16384] += a @ (w[r] * st["w_scales"][r // BLOCK, j, None].double()).t().contiguous()
    return y


def _exact_rotary(st, case):
    rd, d = case["rotary"], case["d"]
    table = st["table"].double()[st["positions"]]
    turn = torch.complex(table[:, :rd // 2], table[:, rd // 2:])[:, None]
    i = torch.arange(rd // 2, device=DEV)
    one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rd // 2)
    got = []
    for x in (st["q"].double(), st["k"].double()):
        z = torch.complex(x[..., one], x[..., two]) * turn
        x = x.clone()
        x[..., one], x[..., two] = z.real, z.imag
        got.append(x)
    if not case["append"]:
        return tuple(got)
    slots = (st["block_table"].long().gather(
        1, (st["positions"] // case["page"]).view(case["sequences"], -1)).reshape(-1) * case["page"] + st["positions"] % case["page"])
    caches = [torch.zeros(st["k_cache"].shape, dtype=torch.float64, device=DEV) for _ in "kv"]
    for c, x in zip(caches, (got[1], st["v"].double())):
        c.view(-1, case["hkv"], d)[slots] = x
    return (got[0], *caches)


def _exact_attention(st, case):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    groups = case["hq"] // case["hkv"]
    for b, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        t = torch.arange(first, n, device=DEV)
        page, at = st["block_table"][b].long()[t // case["page"]], t % case["page"]
        k, v = (c[page, at].double().transpose(0, 1).contiguous() for c in (st["k_cache"], st["v_cache"]))
        q = st["q"][b].double().view(case["hkv"], groups, case["d"])
        p = torch.softmax(torch.matmul(k, q.transpose(1, 2).contiguous()) * case["d"] ** -0.5, 1)
        out[b] = torch.matmul(p.transpose(1, 2).contiguous(), v).view(-1, case["d"])
    return out
