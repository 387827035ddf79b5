"""Cases of the operators of serving many requests over one model: drafted
tokens checked together, long contexts cut to a window, adapters, and the log
probabilities of what came out.

  tree      -- attention of a tree (or a chain) of drafted tokens of each
               sequence over its paged cache
  sinks     -- attention of one new token per sequence over the last tokens of
               its paged cache and a few first ones that stay visible
  logprobs  -- log probabilities of given tokens, entropies and the most likely
               tokens of rows of logits
  adapters  -- low-rank adapters, one per row, added to a shared projection's
               output

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
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _tree(name, batch, length, ragged, tokens, tree, hq, hkv, d, page, dtype, window=0, sinks=0):
    """tokens: drafted ones per sequence, whose keys and values are in the cache
    behind the `length` others; tree: each follows some earlier one, else the
    one before; ragged: lengths between 0 and `length`, fewer drafted tokens."""
    return {"name": name, "op": "tree", "batch": batch, "length": length, "ragged": ragged, "tokens": tokens, "tree": tree,
            "hq": hq, "hkv": hkv, "d": d, "page": page, "type": dtype, "window": window, "sinks": sinks}


def _sinks(name, batch, length, ragged, hq, hkv, d, page, dtype, window, sinks):
    return {"name": name, "op": "sinks", "batch": batch, "length": length, "ragged": ragged, "hq": hq, "hkv": hkv, "d": d,
            "page": page, "type": dtype, "window": window, "sinks": sinks}


def _logprobs(name, rows, vocab, dtype, top, given=True, masked=False, pad=0):
    """top: how many of the most likely tokens; masked: some rows allow a tenth
    of the vocabulary; pad: columns by which the rows lie further apart."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "type": dtype, "top": top, "given": given,
            "masked": masked, "pad": pad}


def _adapters(name, rows, k, n, rank, adapters, segments, dtype):
    """segments: each adapter's rows follow each other (prompts), else any row
    has any adapter, or none (decode steps)."""
    return {"name": name, "op": "adapters", "rows": rows, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "segments": segments, "type": dtype}


def listed() -> list:
    return [
        # one sequence, a short context, eight drafted tokens (Qwen3-0.6B heads)
        _tree("tree_short", 1, 577, False, 8, True, 16, 8, 128, 16, "fp16"),
        # one sequence with a long context (Qwen3-4B heads)
        _tree("tree_long", 1, 131072, False, 16, True, 32, 8, 128, 64, "bf16"),
        # a server's batch: uneven contexts, trees of uneven sizes, some empty
        _tree("tree_batch", 32, 8191, True, 13, True, 32, 8, 128, 16, "fp16"),
        # pieces of prompts, 64 tokens of each sequence over what came before
        _tree("tree_chunk", 16, 4096, False, 64, False, 32, 8, 128, 64, "bf16"),
        # long streams cut to their last 4096 tokens and the first four
        _sinks("sinks_step", 16, 32768, False, 32, 8, 128, 64, "bf16", 4096, 4),
        # uneven streams, small heads (SmolLM2-135M), sizes off every tile
        _sinks("sinks_ragged", 61, 5000, True, 9, 3, 64, 48, "fp16", 1001, 7),
        # a decode step of four sequences: the sampled tokens and five others
        _logprobs("logprobs_step", 4, 151936, "fp16", 5),
        # scoring a long text: every position's token, twenty alternatives
        _logprobs("logprobs_score", 2047, 151936, "bf16", 20),
        # logits of the 8-bit head, some rows under a grammar's mask
        _logprobs("logprobs_masked", 64, 49152, "fp32", 1, masked=True),
        # one decode step of four requests, q_proj (Qwen3-4B), an adapter each
        _adapters("adapters_step", 4, 2560, 4096, 16, 4, False, "fp16"),
        # a decode step of many requests, gate_proj, adapters in any order
        _adapters("adapters_batch", 64, 2560, 9728, 64, 32, False, "bf16"),
        # prompts of seven requests through down_proj
        _adapters("adapters_prompt", 2047, 9728, 2560, 64, 7, True, "fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(("tree", "sinks", "logprobs", "adapters"))
    dtype = rng.choice(("fp16", "bf16"))
    if op in ("tree", "sinks"):
        hkv, d = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 80, 96, 128, 256))
        hq = hkv * rng.choice((1, 2, 3, 4, 7, 8))
        batch = _log(rng, 1, 64)
        page = rng.choice((1, 16, 48, 64, 256))
        window, sinks = rng.choice(((0, 0), (0, 0), (_log(rng, 1, 4096), rng.choice((0, 1, 4, 50)))))
        if op == "tree":
            tokens = _log(rng, 1, 64)
            most = min(16 * 4096 * 8 * 128 // (batch * hkv * d), 16 * 4096 * 64 * 32 * 128 // (batch * tokens * hq * d))
            c = _tree("", batch, _log(rng, 1, max(1, min(131072, most))), rng.random() < 0.5, tokens, rng.random() < 0.6,
                      hq, hkv, d, page, dtype, window, sinks)
        else:
            most = 16 * 32768 * 8 * 128 // (batch * hkv * d)
            c = _sinks("", batch, _log(rng, 1, max(1, min(131072, most))), rng.random() < 0.5, hq, hkv, d, page, dtype,
                       window or _log(rng, 1, 4096), rng.choice((1, 4, 5, 50, 300)))
    elif op == "logprobs":
        vocab = _log(rng, 100, 262144)
        rows = _log(rng, 1, max(1, min(8192, 2047 * 151936 // (2 * vocab))))
        c = _logprobs("", rows, vocab, rng.choice((dtype, dtype, "fp32")), rng.choice((0, 1, 5, 20, _log(rng, 1, 64))),
                      rng.random() < 0.8, vocab >= 1000 and rng.random() < 0.4, rng.choice((0, 0, 3, 64)))
    else:
        k, n, rank = _log(rng, 100, 10000), _log(rng, 100, 10000), rng.choice((8, 16, 32, 64, _log(rng, 1, 128)))
        segments = rng.random() < 0.5
        rows = _log(rng, 1, min(2047 if segments else 256, max(1, 2047 * (9728 + 2 * 2560) // (k + 2 * n))))
        c = _adapters("", rows, k, n, rank, _log(rng, 1, 64), segments, dtype)
    del c["name"]
    return c


def _own_random(case) -> random.Random:
    """Of a case's lengths and trees, which are its own whatever the seed."""
    return random.Random(case["batch"] * 1000003 + case["length"] * 101 + case.get("tokens", 0))


def _lengths(case) -> list:
    """Tokens in the cache (of a tree: before the drafted ones)."""
    if not case["ragged"]:
        return [case["length"]] * case["batch"]
    rng = _own_random(case)
    return [0 if rng.random() < 0.05 else rng.randint(1, case["length"]) for _ in range(case["batch"])]


def _ancestors(case) -> list:
    """Per sequence and drafted token the drafted tokens that it sees, itself
    among them, as bits; 0: no token is drafted there."""
    rng = _own_random(case)
    got = []
    for _ in range(case["batch"]):
        count = rng.randint(1, case["tokens"]) if case["ragged"] and case["tree"] else case["tokens"]
        masks = []
        for i in range(case["tokens"]):
            if i >= count:
                masks.append(0)
                continue
            parent = i - 1 if not case["tree"] or rng.random() < 0.5 else rng.randint(0, max(0, i - 1))
            masks.append((masks[parent] if i else 0) | 1 << i)
        got.append(masks)
    return got


def _seen(case) -> tuple:
    """(cached tokens that any query of a sequence reads, those that each query
    reads), summed."""
    w, sinks, any_query, each = case["window"], case["sinks"], 0, 0
    if case["op"] == "sinks":
        for n in _lengths(case):
            s = min(n, w + sinks) if w else n
            any_query, each = any_query + s, each + s
        return any_query, each
    for n, masks in zip(_lengths(case), _ancestors(case)):
        drafted = 0
        least = n
        for m in masks:
            depth = bin(m).count("1")
            first = max(0, n + depth - w) if w else 0
            least = min(least, first)
            each += n - min(first, n) + min(sinks, first, n) + (min(depth, w) if w else depth)
            drafted += m != 0
        any_query += n - least + min(sinks, least) + drafted
    return any_query, each


def work(case) -> dict:
    s = BYTES[case["type"]]
    if case["op"] in ("tree", "sinks"):
        any_query, each = _seen(case)
        queries = case["batch"] * case.get("tokens", 1)
        bytes_ = (2 * any_query * case["hkv"] * case["d"] * s + 2 * queries * case["hq"] * case["d"] * s
                  + 4 * -(-any_query // case["page"]) + 4 * case["batch"])
        if case.get("tree"):
            bytes_ += 8 * queries
        return {"bytes": bytes_, "flops": 4 * each * case["hq"] * case["d"]}
    if case["op"] == "logprobs":
        el = case["rows"] * case["vocab"]
        return {"bytes": el * s + case["rows"] * ((12 if case["given"] else 0) + 4 + 12 * case["top"]), "flops": 6 * el}
    rows, k, n, rank = case["rows"], case["k"], case["n"], case["rank"]
    used = len({i for i in _rows_adapters(case) if i >= 0})
    return {"bytes": rows * (k + 2 * n) * s + used * rank * (k + n) * s + 4 * rows + 4 * case["adapters"],
            "flops": 2 * rows * rank * (k + n)}


def _rows_adapters(case) -> list:
    """The adapter of each row, the case's own; -1: none."""
    rng = random.Random(case["rows"] * 1009 + case["adapters"])
    rows, count = case["rows"], case["adapters"]
    if not case["segments"]:
        return [-1 if rng.random() < 0.1 else rng.randrange(count) for _ in range(rows)]
    cuts = sorted(rng.randint(0, rows) for _ in range(count - 1))
    order = rng.sample(range(-1, count), count)  # (one of them, or none at all, is left out)
    return [i for i, lo, hi in zip(order, [0, *cuts], [*cuts, rows]) for _ in range(hi - lo)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _outliers(x, g):
    """Activations as a decoder has them: one column in a hundred 20 times larger."""
    big = torch.rand(x.shape[-1], generator=g, device=DEV) < 0.01
    return x * (1 + 19 * big.to(x.dtype))


def prepare(case, seed) -> dict:
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    dtype = TYPES[case["type"]]
    st = {"case": case}
    if case["op"] in ("tree", "sinks"):
        lengths, b = _lengths(case), case["batch"]
        tokens = case.get("tokens", 0)
        width = max(1, -(-(max(lengths) + tokens) // case["page"]))
        pages = b * width + 3
        lead = (b, tokens) if tokens else (b,)
        st["q"] = (1.5 * normal(*lead, case["hq"], case["d"])).to(dtype)
        st["k_cache"], st["v_cache"] = (
            torch.empty(pages, case["page"], case["hkv"], case["d"], dtype=dtype, device=DEV).normal_(generator=g) for _ in "kv")
        # the cache's pages in the order in which a server has handed them out
        st["block_table"] = torch.randperm(pages, generator=g, device=DEV)[:b * width].view(b, width).to(torch.int32)
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        if tokens:
            signed = [[m - (1 << 64) if m >> 63 else m for m in masks] for masks in _ancestors(case)]
            st["ancestors"] = torch.tensor(signed, dtype=torch.int64, device=DEV) if case["tree"] else None
    elif case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # rows from nearly even to nearly certain
        x = normal(rows, vocab + case["pad"]) * torch.exp(0.5 * normal(rows, 1)) * 2.0
        likely = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        at = torch.arange(rows, device=DEV)
        x[at, likely] += 12.0 * torch.rand(rows, generator=g, device=DEV)
        if case["masked"]:
            refused = torch.rand(rows, vocab + case["pad"], generator=g, device=DEV) >= 0.1
            refused[at, likely] = False
            for row in range(0, rows, 3):  # by -infinity, or by the type's lowest value
                x[row].masked_fill_(refused[row], -math.inf if row % 2 else torch.finfo(dtype).min)
        st["logits"] = x.to(dtype)[:, :vocab]
        # a text's padding has no token
        padding = torch.rand(rows, generator=g, device=DEV) < (0.05 if rows > 1 else 0.0)
        st["tokens"] = torch.where(padding, -1, likely) if case["given"] else None
    else:
        rows, k, n, rank, count = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
        ids = _rows_adapters(case)
        st["x"] = _outliers(normal(rows, k), g).to(dtype)
        st["y"] = (2 * normal(rows, n)).to(dtype)
        st["a"] = (normal(count, rank, k) / math.sqrt(k)).to(dtype)
        st["b"] = (0.1 * normal(count, n, rank)).to(dtype)
        st["scales"] = torch.exp2(torch.randint(-1, 3, (count,), generator=g, device=DEV).float())
        st["ids"] = torch.tensor(ids, dtype=torch.int32, device=DEV)
        # (a server knows each adapter's rows)
        st["groups"] = [(i, torch.tensor([r for r, j in enumerate(ids) if j == i], device=DEV)) for i in sorted(set(ids)) if i >= 0]
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    return (_run_own if own else _run_plain)(st, st["case"])


def _run_own(st, case):
    if case["op"] == "tree":
        from turbopress_amd import paged_tree_attention
        return paged_tree_attention(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["lengths"],
                                    ancestors=st["ancestors"], window=case["window"], sinks=case["sinks"])
    if case["op"] == "sinks":
        from turbopress_amd import paged_attention
        return paged_attention(st["q"], st["k_cache"], st["v_cache"], st["block_table"], st["lengths"], window=case["window"],
                               sinks=case["sinks"])
    if case["op"] == "logprobs":
        from turbopress_amd import token_logprobs
        got = token_logprobs(st["logits"], st["tokens"], top=case["top"])
        return tuple(t for t in (got.logprobs, got.entropy, got.top_logprobs, got.top_tokens) if t is not None)
    from turbopress_amd import lora_add
    return lora_add(st["y"], st["x"], st["a"], st["b"], st["ids"], scales=st["scales"])


def _run_plain(st, case):
    if case["op"] == "logprobs":
        return _plain_logprobs(st, case)
    if case["op"] == "adapters":
        return _plain_adapters(st, case)
    return _plain_attention(st, case)


def _visible(st, case, at):
    """[sequence, query, token]: which tokens `at` of the cache a query sees.  The
    last of a sequence's tokens that a query sees is at the query's position."""
    n = st["lengths"][:, None, None]
    window, sinks = case["window"], case["sinks"]
    if case["op"] == "sinks":
        return (at < n) & ((at >= n - window) | (at < sinks) if window else True)
    t = case["tokens"]
    i = torch.arange(t, device=DEV)
    if st["ancestors"] is None:
        bits = (i[None] <= i[:, None])[None].expand(case["batch"], t, t)
    else:
        bits = (st["ancestors"][:, :, None] >> i & 1).bool()
    position = n[:, :, 0] + bits.sum(2) - 1  # of the drafted tokens
    drafted = at - n  # (of no use below 0 and from t on)
    is_drafted = (drafted >= 0) & (drafted < t)
    index = drafted.clamp(0, t - 1).expand(case["batch"], t, at.shape[0])
    seen = torch.where(is_drafted, bits.gather(2, index), drafted < 0)
    if window:
        place = torch.where(is_drafted, position[:, None].expand(-1, t, -1).gather(2, index), at)
        seen = seen & ((place > position[:, :, None] - window) | (place < sinks))
    return seen


def _plain_attention(st, case):
    b, hkv, d = case["batch"], case["hkv"], case["d"]
    pages = st["block_table"].long()
    at = torch.arange(pages.shape[1] * case["page"], device=DEV)
    seen = _visible(st, case, at)
    t, group = seen.shape[1], case["hq"] // hkv
    # [sequence, token, head, column] of the pages that each sequence has
    k, v = (c[pages].flatten(1, 2).float() for c in (st["k_cache"], st["v_cache"]))
    q = st["q"].float().view(b, t, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * t, d) / math.sqrt(d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(b, hkv, group, t, -1)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    v = v.transpose(1, 2).contiguous()
    out = torch.matmul(p.view(b, hkv, group * t, -1), v).view(b, hkv, group, t, d) / torch.where(total > 0, total, 1)
    return out.permute(0, 3, 1, 2, 4).reshape(st["q"].shape).to(st["q"].dtype)


def _plain_logprobs(st, case):
    x = st["logits"].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    # sum of p (log_total - (x - top)): tokens without probability add nothing
    off = torch.where(e > 0, e * (x - top), 0).sum(1, keepdim=True)
    got = [(log_total - off / total)[:, 0]]
    if case["given"]:
        tokens = st["tokens"]
        value = x.gather(1, tokens.clamp(min=0)[:, None]) - top - log_total
        got.insert(0, torch.where(tokens >= 0, value[:, 0], 0))
    if case["top"]:
        index = torch.empty(case["rows"], case["top"], dtype=torch.int64, device=DEV)
        value = torch.empty(case["rows"], case["top"], device=DEV)
        left = x.clone()
        for j in range(case["top"]):
            best = left.argmax(1, keepdim=True)  # (the first of equals)
            index[:, j:j + 1], value[:, j:j + 1] = best, left.gather(1, best)
            left.scatter_(1, best, -math.inf)
        got += [value - top - log_total, index]
    return tuple(got)


def _plain_adapters(st, case):
    y = st["y"].float()
    for i, rows in st["groups"]:
        h = torch.matmul(st["x"][rows].float(), st["a"][i].float().t())
        y[rows] += st["scales"][i] * torch.matmul(h, st["b"][i].float().t())
    return y.to(st["y"].dtype)


# ---------------------------------------------------------------------------
# in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_tree, "sinks": _exact_sinks, "logprobs": _exact_logprobs, "adapters": _exact_adapters}[case["op"]](
        st, case)


def _cached(st, case, b, t):
    """Keys and values [head, token, column] of tokens t of sequence b."""
    page, at = st["block_table"][b].long()[t // case["page"]], t % case["page"]
    return (c[page, at].double().transpose(0, 1).contiguous() for c in (st["k_cache"], st["v_cache"]))


def _exact_sinks(st, case):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    w, sinks = case["window"], case["sinks"]
    for b, n in enumerate(_lengths(case)):
        t = torch.tensor([*range(min(sinks, max(0, n - w))), *range(max(0, n - w), n)] if w else range(n), device=DEV)
        if n == 0:
            continue
        k, v = _cached(st, case, b, t.long())
        q = st["q"][b].double().view(case["hkv"], -1, case["d"])
        p = torch.softmax(torch.matmul(k, q.transpose(1, 2).contiguous()) * case["d"] ** -0.5, 1)
        out[b] = torch.matmul(p.transpose(1, 2).contiguous(), v).view(-1, case["d"])
    return out


def _exact_tree(st, case):
    """A query at a time decides what it sees; a sequence's queries together meet
    its keys."""
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    count, w, sinks = case["tokens"], case["window"], case["sinks"]
    for b, (n, masks) in enumerate(zip(_lengths(case), _ancestors(case))):
        t = torch.arange(n + count, device=DEV)
        hidden = torch.ones(count, n + count, dtype=torch.bool)
        place = [*range(n), *(n + bin(m).count("1") - 1 for m in masks)]
        for i, m in enumerate(masks):
            here = place[n + i]
            low = max(0, min(n, here + 1 - w)) if w else 0
            hidden[i, low:n] = False
            hidden[i, :min(sinks, n)] = False
            for j in range(count):
                if m >> j & 1 and (not w or place[n + j] > here - w or place[n + j] < sinks):
                    hidden[i, n + j] = False
        hidden = hidden.to(DEV)
        k, v = _cached(st, case, b, t)
        q = st["q"][b].double().view(count, case["hkv"], -1, case["d"]).permute(1, 2, 0, 3).contiguous()
        s = torch.matmul(q.flatten(1, 2), k.transpose(1, 2).contiguous()).view(*q.shape[:3], -1) * case["d"] ** -0.5
        p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        p = p.masked_fill(hidden.all(1)[:, None], 0)  # (a query that sees nothing)
        out[b] = torch.matmul(p.flatten(1, 2), v).view(q.shape).permute(2, 0, 1, 3).reshape(count, -1, case["d"])
    return out


def _exact_logprobs(st, case):
    parts = []
    ids = torch.arange(case["vocab"], device=DEV)
    for lo in range(0, case["rows"], 256):
        x = st["logits"][lo:lo + 256].double()
        total = torch.logsumexp(x, 1, keepdim=True)
        log_p = x - total
        p = log_p.exp()
        got = [-torch.where(p > 0, p * log_p, 0).sum(1)]
        if case["given"]:
            t = st["tokens"][lo:lo + 256]
            got.insert(0, torch.where(t < 0, 0, log_p[torch.arange(len(t), device=DEV), t.clamp(min=0)]))
        if case["top"]:
            # the value's order, then the lower token, as one whole number (+ 0: no negative zeros)
            bits = (st["logits"][lo:lo + 256].float() + 0.0).contiguous().view(torch.int32).long()
            order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
            index = ((order << 20) + (2 ** 20 - 1 - ids)).topk(case["top"], 1).indices
            got += [log_p.gather(1, index), index]
        parts.append(got)
    return tuple(torch.cat(p) for p in zip(*parts))


def _exact_adapters(st, case):
    y = st["y"].double()
    for r0 in range(0, case["rows"], 64):
        for i in sorted(set(_rows_adapters(case)[r0:r0 + 64])):
            if i >= 0:
                mine = (st["ids"][r0:r0 + 64] == i).double()[:, None] * st["scales"][i].double()
                x = st["x"][r0:r0 + 64].double()
                y[r0:r0 + 64] += mine * ((x @ st["a"][i].double().t().contiguous()) @ st["b"][i].double().t().contiguous())
    return y
