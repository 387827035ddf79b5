"""Plain 64-bit implementations of the operators of serving many requests (test
infrastructure only): attention of drafted trees and of windows with first
tokens, log probabilities, adapters.  Tensors of any device in, float64 tensors
out; each follows its formula, a query or a row at a time."""

from __future__ import annotations

import math

import torch


def seen_by_new_token(length, masks, i, window, sinks):
    """Tokens of the cache that new token i sees, in order: `length` tokens are
    there before the new ones, masks[j] holds new token j's ancestors as bits."""
    count = len(masks)

    def position(t):
        return t if t < length else length - 1 + sum(masks[t - length] >> j & 1 for j in range(count))

    here = position(length + i)
    got = [t for t in range(length) if not window or t > here - window or t < sinks]
    for j in range(count):
        if masks[i] >> j & 1:
            p = position(length + j)
            if not window or p > here - window or p < sinks:
                got.append(length + j)
    return got


def _attend(q, k_cache, v_cache, pages, seen, scale):
    """Queries q [count, heads, d] of one sequence, of which query i sees the
    tokens seen[i]: (out, weighted mean magnitude of v, largest sum of |q k|
    terms [count, heads]).  Tokens of pages that do not exist are left out."""
    n_pages, page, hkv = k_cache.shape[:3]
    count, hq, d = q.shape
    out = torch.zeros(count, hq, d, dtype=torch.float64, device=q.device)
    size, dots = torch.zeros_like(out), torch.zeros(count, hq, dtype=torch.float64, device=q.device)
    t = torch.tensor(sorted(set().union(*seen)), dtype=torch.int64)
    mask = torch.zeros(count, len(t), dtype=torch.bool)
    for i, tokens in enumerate(seen):
        mask[i, torch.searchsorted(t, torch.tensor(tokens, dtype=torch.int64))] = True
    t, mask = t.to(q.device), mask.to(q.device)
    held = t < pages.shape[0] * page
    t, mask = t[held], mask[:, held]
    p = pages.long()[t // page]
    held = (p >= 0) & (p < n_pages)
    t, mask, p = t[held], mask[:, held], p[held]
    k, v = k_cache[p, t % page].double(), v_cache[p, t % page].double()  # [token, kv head, column]
    qd = q.double()
    together = bool(torch.isfinite(k).all() and torch.isfinite(v).all())
    for rows in [slice(0, count)] if together else [slice(i, i + 1) for i in range(count)]:
        # (a value that is not finite may meet only the queries that see it)
        some = mask[rows].any(0)
        m, ks, vs = mask[rows][:, some], k[some], v[some]
        if not m.any():
            continue
        for h in range(hq):
            kh, vh = ks[:, h // (hq // hkv)], vs[:, h // (hq // hkv)]
            s = (qd[rows, h][:, None] * kh[None]).sum(2) * scale
            w = torch.softmax(s.masked_fill(~m, -math.inf), 1)
            w = torch.where(m, w, 0) if together else w
            w = w.masked_fill(~m.any(1)[:, None], 0)
            out[rows, h] = (w[:, :, None] * vh[None]).sum(1)
            size[rows, h] = (w[:, :, None] * vh.abs()[None]).sum(1)
            dots[rows, h] = (kh.abs()[None] * qd[rows, h].abs()[:, None]).sum(2).amax(1) * abs(scale)
    return out, size, dots


def paged_tree_attention(q, k_cache, v_cache, block_table, lengths, ancestors=None, scale=None, window=0, sinks=0):
    """As ``_attend``, of all sequences, new tokens and heads."""
    b, count, hq, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    got = []
    for s in range(b):
        length = max(int(lengths[s]), 0)
        masks = [(1 << i + 1) - 1 for i in range(count)] if ancestors is None else [
            m & ((1 << count) - 1) for m in ancestors[s].tolist()]
        seen = [seen_by_new_token(min(length, 1 << 20), masks, i, window, sinks) for i in range(count)]
        got.append(_attend(q[s], k_cache, v_cache, block_table[s], seen, scale))
    return tuple(torch.stack(c) for c in zip(*got))


def paged_attention(q, k_cache, v_cache, block_table, lengths, scale=None, window=0, sinks=0):
    """As ``_attend``, of one new token per sequence, itself in the cache."""
    d = q.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    got = []
    for s in range(q.shape[0]):
        n = max(int(lengths[s]), 0)
        seen = [t for t in range(n) if not window or t >= n - window or t < sinks]
        got.append(_attend(q[s:s + 1], k_cache, v_cache, block_table[s], [seen], scale))
    return tuple(torch.cat(c) for c in zip(*got))


def token_logprobs(logits, tokens=None, top=0):
    """(log probabilities, their entropy's two parts, tokens in falling order):
    per row of finite or -infinite logits, of which one is finite at least.

    log p = (x - m) - L with m the largest and L = log sum e^(x - m), entropy = L
    + A with A = sum p (m - x)."""
    rows = []
    for r, x in enumerate(logits.double()):
        y = x - x.max()
        others = y.clone()
        others[x.argmax()] = -math.inf
        log_sum = torch.log1p(others.exp().sum())
        p = (y - log_sum).exp()
        off = torch.where(p > 0, -p * y, 0).sum()
        lp = y - log_sum
        order = torch.sort(x + 0.0, descending=True, stable=True).indices[:top]
        given = None if tokens is None else lp[tokens[r]] if tokens[r] >= 0 else torch.zeros_like(log_sum)
        rows.append((given, log_sum, off, lp[order], order, y[order], None if tokens is None else y[tokens[r]]))
    return [None if c[0] is None else torch.stack(c) for c in zip(*rows)]


def lora_add(y, x, a, b, adapters, scales=None):
    """(y + scale (x a^T) b^T, magnitudes of the second product's terms), a row at a time."""
    out, size = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    for r, i in enumerate(adapters.tolist()):
        if 0 <= i < a.shape[0]:
            s = 1.0 if scales is None else scales[i].double()
            ad, bd, xd = a[i].double(), b[i].double(), x[r].double()
            out[r] += s * (bd @ (ad @ xd))
            size[r] = abs(s) * (bd.abs() @ (ad.abs() @ xd.abs()))
    return out, size
