"""Attention under a mask of its own (windows with sinks, trees of drafted
tokens), accepted paths and log probabilities from their definitions, in binary64
on the CPU (test infrastructure only)."""
from __future__ import annotations

import math

import torch

from .attention_oracle import keys_of


def window_sight(n, total, window, sinks):
    """[n, total]: what the newest n rows of a sequence see of its keys."""
    place = torch.arange(total - n, total)[:, None]
    key = torch.arange(total)
    seen = key <= place
    return seen if window is None else seen & ((key < sinks) | (key > place - window))


def tree_sight(masks, total):
    """[n, total]: what drafted rows see; masks [n, words] as Python reads them."""
    n = masks.shape[0]
    seen = torch.ones(n, total, dtype=torch.bool)
    for i, words in enumerate(masks.tolist()):
        bits = sum((w & (2 ** 64 - 1)) << (64 * at) for at, w in enumerate(words))
        for j in range(max(0, total - n), total):
            seen[i, j] = bool(bits >> (j - (total - n)) & 1)
    return seen


def attention(q, k_cache, v_cache, table, lengths, starts, sight, scale=None):
    """(out, sum p |v|, max scale sum |q k|); rows of no sequence are NaN.
    ``sight(b, n, total)``: the [n, total] mask of sequence b."""
    q, k_cache, v_cache, table = q.cpu(), k_cache.cpu(), v_cache.cpu(), table.cpu()
    t, h, d = q.shape
    group = h // k_cache.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.full((t, h, d), math.nan, dtype=torch.float64)
    size, dots = out.clone(), torch.full((t, h), math.nan, dtype=torch.float64)
    lengths, starts = lengths.cpu().tolist(), starts.cpu().tolist()
    most = table.shape[1] * k_cache.shape[2]
    for b, total in enumerate(lengths):
        total = max(0, min(total, most))
        rows, n = slice(starts[b], starts[b + 1]), starts[b + 1] - starts[b]
        if n <= 0:
            continue
        allowed = sight(b, n, total)
        for g in range(k_cache.shape[1]):
            k, known = keys_of(k_cache, table, b, g, total)
            v, _ = keys_of(v_cache, table, b, g, total)
            seen = allowed & known
            # What no row sees may hold anything.
            k = k.masked_fill(~seen.any(0)[:, None], 0.0)
            for i in range(g * group, (g + 1) * group):
                x = q[rows, i].double()
                s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
                peak = s.amax(-1, keepdim=True) if total else torch.full((n, 1), -math.inf)
                p = torch.exp(s - peak.masked_fill(peak == -math.inf, 0.0))
                p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
                # A weight of a masked key is 0 whatever its value.
                out[rows, i] = torch.stack([(p[r, seen[r]] @ v[seen[r]]) for r in range(n)])
                size[rows, i] = torch.stack([(p[r, seen[r]] @ v[seen[r]].abs()) for r in range(n)])
                a = (x.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0)
                dots[rows, i] = a.amax(-1) if total else 0.0
    return out, size, dots


def accept(cache, table, lengths, path):
    """The cache [..., pages, heads, page, dim] with the accepted rows moved."""
    before, after = cache.cpu(), cache.cpu().clone()
    pages, _, page, _ = cache.shape[-4:]
    table = table.cpu().tolist()
    for b, (n, nodes) in enumerate(zip(lengths.tolist(), path.tolist())):
        n = max(n, 0)
        for i, node in enumerate(nodes):
            if node < i or max(n + node, n + i) >= len(table[b]) * page:
                continue
            source, target = table[b][(n + node) // page], table[b][(n + i) // page]
            if 0 <= source < pages and 0 <= target < pages:
                after[..., target, :, (n + i) % page, :] = \
                    before[..., source, :, (n + node) % page, :]
    return after


def logprobs(x, tokens, top):
    """(log probabilities, entropy, top log probabilities, top tokens) of rows x
    [rows, vocab], tokens [rows, n]; and per row (R, D, Q): the sums over the
    logits but one largest of e, |d| e and d^2 e, d = x - max, e = exp(d)."""
    x = x.double().cpu()
    v = x.shape[1]
    p = torch.log_softmax(x, -1)
    t = tokens.cpu()
    inside = (t >= 0) & (t < v)
    given = p.gather(1, t.clamp(0, v - 1)).masked_fill(~inside, math.nan)
    given = given.masked_fill(t == -1, 0.0)
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    first = torch.zeros_like(e, dtype=torch.bool).scatter_(1, x.argmax(-1, keepdim=True), True)
    rest = e.masked_fill(first, 0.0).sum(-1)
    flat = torch.where(e == 0.0, torch.zeros_like(d), d.abs())
    spread, square = (flat * e).sum(-1), (flat * flat * e).sum(-1)
    entropy = torch.log1p(rest) + spread / (1.0 + rest)
    order = torch.sort(x.nan_to_num(nan=math.inf, posinf=1.7e308, neginf=-math.inf), stable=True,
                       dim=-1, descending=True).indices[:, :top]
    return given, entropy, p.gather(1, order), order, (rest, spread, square)
