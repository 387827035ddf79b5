"""Plain 64-bit implementations of the decoder operators (test infrastructure
only): norm, e4m3 product, rotary positions, paged attention.  Tensors of any
device in, float64 tensors out; each follows its formula, a sequence or a token
at a time where that is the formula's own order."""

from __future__ import annotations

import math

import torch

F8_MAX = 448.0
LEAST_SCALE = 2.0 ** -126


def rms_norm(x, weight, eps, residual=None):
    """(y, h): h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight."""
    h = x.double() if residual is None else x.double() + residual.double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double(), h


def block_scales(y, block):
    """Scales of y's rows: largest magnitude of each `block` columns (None: of
    the row) / 448, at least 2^-126; and y / scale, unrounded."""
    d = y.shape[-1]
    width = d if block is None else block
    scales, values = [], []
    for c in range(0, d, width):
        part = y[..., c:c + width]
        s = (part.abs().amax(-1, keepdim=True) / F8_MAX).clamp(min=LEAST_SCALE)
        scales.append(s)
        values.append(part / s)
    return torch.cat(values, -1), torch.cat(scales, -1)


def fp8_linear(a, a_scales, w, w_scales, bias=None):
    """(y, sum of the terms' magnitudes)."""
    k, n = w.shape[1], w.shape[0]
    ad = a.double() * a_scales.double().repeat_interleave(128, -1)[..., :k]
    wd = w.double() * w_scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    wt = wd.t().contiguous()
    y, size = ad @ wt, ad.abs() @ wt.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def rotary(x, table, positions, interleaved):
    """(turned x, magnitudes of the two terms of each element)."""
    x = x.double()
    out, size = x.clone(), torch.zeros_like(x)
    half = table.shape[1] // 2
    c, s = table.double()[positions].split(half, 1)
    for i in range(half):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[:, :, p], x[:, :, q]
        ci, si = c[:, i, None], s[:, i, None]
        out[:, :, p], out[:, :, q] = a * ci - b * si, b * ci + a * si
        size[:, :, p], size[:, :, q] = (a * ci).abs() + (b * si).abs(), (b * ci).abs() + (a * si).abs()
    return out, size


def paged_attention(q, k_cache, v_cache, block_table, lengths, scale=None, window=0):
    """(out, weighted mean magnitude of v, largest sum of |q k| terms): a sequence
    at a time; tokens of pages that do not exist are left out."""
    b, hq, d = q.shape
    n_pages, page, hkv = k_cache.shape[:3]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size, dots = torch.zeros_like(out), torch.zeros(b, hq, dtype=torch.float64, device=q.device)
    for i in range(b):
        n = min(max(int(lengths[i]), 0), block_table.shape[1] * page)
        t = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        p = block_table[i].long()[t // page]
        t, p = t[(p >= 0) & (p < n_pages)], p[(p >= 0) & (p < n_pages)]
        if not len(t):
            continue
        k, v = k_cache[p, t % page].double(), v_cache[p, t % page].double()
        for h in range(hq):
            kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
            w = torch.softmax((kh * q[i, h].double()).sum(1) * scale, 0)
            out[i, h] = (w[:, None] * vh).sum(0)
            size[i, h] = (w[:, None] * vh.abs()).sum(0)
            dots[i, h] = (kh * q[i, h].double()).abs().sum(1).max() * abs(scale)
    return out, size, dots
