"""Rotary positions, the cache store and paged attention from their
definitions, in binary64 on the CPU (test infrastructure only).

Besides each result the attention oracle returns what a bound of a binary32
kernel's error needs: per output element sum_j p_j |v_j|, and per row the
largest sum_i |q_i k_i| over its keys (times the scale)."""
from __future__ import annotations

import math

import torch


def rotary(x, positions, inv_freq, layout="half", factor=1.0):
    """(turned rows, |a c| + |b s| of each element) in binary64."""
    out = x.double().cpu().clone()
    size = out.abs()
    n = inv_freq.numel()
    angle = positions.double().cpu()[:, None] * inv_freq.double().cpu()
    c, s = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
    i = torch.arange(n)
    first, second = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = out[..., first].clone(), out[..., second].clone()
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = (a * c).abs() + (b * s).abs()
    size[..., second] = (b * c).abs() + (a * s).abs()
    return out, size


def keys_of(cache, table, b, head, n):
    """The first n rows of sequence b's pages, and which of them lie in a page
    of the cache."""
    pages, _, page, dim = cache.shape
    if n == 0 or pages == 0:
        return torch.zeros(n, dim, dtype=torch.float64), torch.zeros(n, dtype=torch.bool)
    own = table[b, :-(-n // page)].long()
    known = ((own >= 0) & (own < pages)).repeat_interleave(page)[:n]
    rows = cache[own.clamp(0, pages - 1), head].flatten(0, 1)[:n].double()
    return rows.masked_fill(~known[:, None], 0.0), known


def attention(q, k_cache, v_cache, table, lengths, q_starts=None, scale=None):
    """(out, sum p |v|, max scale sum |q k|); rows of no sequence are NaN."""
    q, k_cache, v_cache = q.cpu(), k_cache.cpu(), v_cache.cpu()
    table, lengths = table.cpu(), lengths.cpu().tolist()
    t, h, d = q.shape
    group = h // k_cache.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((t, h, d), math.nan, dtype=torch.float64)
    size, dots = out.clone(), torch.full((t, h), math.nan, dtype=torch.float64)
    starts = list(range(len(lengths) + 1)) if q_starts is None else q_starts.cpu().tolist()
    most = table.shape[1] * k_cache.shape[2]
    for b, total in enumerate(lengths):
        total = max(0, min(total, most))
        rows = slice(starts[b], starts[b + 1])
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        last = total - n + torch.arange(n)
        for g in range(k_cache.shape[1]):
            k, known = keys_of(k_cache, table, b, g, total)
            v, _ = keys_of(v_cache, table, b, g, total)
            seen = (torch.arange(total) <= last[:, None]) & known
            for i in range(g * group, (g + 1) * group):
                x = q[rows, i].double()
                s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
                peak = s.amax(-1, keepdim=True) if total else torch.full((n, 1), -math.inf)
                p = torch.exp(s - peak.masked_fill(peak == -math.inf, 0.0))
                p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
                out[rows, i], size[rows, i] = p @ v, p @ v.abs()
                a = (x.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0)
                dots[rows, i] = a.amax(-1) if total else 0.0
    return out, size, dots
