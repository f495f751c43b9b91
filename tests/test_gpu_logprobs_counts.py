"""Log probabilities of rows in which every token counts, and of as many rows as
change how a row is cut.

Rows hold one value at the tokens of a residue class and -inf elsewhere, for all
classes: between them every token of the vocabulary, the ends of slices and vectors
among them, is in exactly one row, and a token that is lost or taken twice changes
that row's sum by one part in its count.

Tolerances (u = 2^-24).  Equal tokens are counted: whole numbers below 2^24, added
without an error, terms of -inf are 0; their log is within 4 u log n, its
difference to the logit rounded once more: 5 u log n.  Sums of a row: a thread adds
at most 17 vectors of 8 logits, a wavefront's 64 lanes in 6 steps, up to 16
wavefronts and 32 slices one by one; a thread's sum changes its reference up to 17
times, then for the row and for the join, each a factor within 2 u and a rounding:
N = 136 + 6 + 16 + 32 + 19 * 3 = 247 roundings in a row, all terms of one sign.  An
exponential is off by (2 |d| + 4) u.  So log S is off by ((N + 4) R + 2 D) u / S + 4 u
log S, with R, D, Q the sums of e, |d| e and d^2 e over all but one largest logit, S
= 1 + R; a log probability by 2 u |d| + u |y| more, the entropy log S + D / S by ((2 N
+ 12) D + 2 Q) u / S + u of itself.
"""
from __future__ import annotations

import math

import pytest
import torch

import test_gpu_attention as G
from nanopointllm_amd import lm_head as L
from oracle import drafts_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
N = 247
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def rows_in(wide, rows, vocab):
    """Rows of ``vocab`` logits at every alignment, NaN around them."""
    wide.fill_(math.nan)
    return wide.as_strided((rows, vocab), (vocab + 13, 1), 3)


def room(rows, vocab, dtype, device):
    return torch.empty(rows * (vocab + 13) + 16, dtype=dtype, device=device)


def count_of(vocab, period, r):
    """How many tokens of the vocabulary are r behind a multiple of the period."""
    return (vocab - r + period - 1) // period


def check_classes(cuda, vocab, period, classes, dtype, top=4):
    rows = len(classes)
    r = torch.tensor(classes, device=cuda)
    n = torch.tensor([count_of(vocab, period, c) for c in classes], dtype=torch.float64)
    assert int(n.min()) >= top + 1
    own = torch.arange(vocab, device=cuda)[None] % period == r[:, None]
    x = rows_in(room(rows, vocab, dtype, cuda), rows, vocab)
    first, last = r, r + period * (n.long().to(cuda) - 1)
    other = torch.where(r > 0, r - 1, r + 1)
    tokens = torch.stack((first, last, other, torch.full_like(r, -1)), 1)

    # Equal ones.
    x.copy_(torch.where(own, 1.5, -math.inf))
    out = L.token_logprobs(x, tokens, top=top)
    want, tol = -n.log(), 5 * U * n.log()
    assert (tol < 0.25 / n).all()
    y = out.logprobs.double().cpu()
    for got in (y[:, 0], y[:, 1], -out.entropy.double().cpu(), out.top_logprobs[:, top - 1].double().cpu()):
        bad = (got - want).abs() > tol
        assert not bad.any(), (bad.nonzero()[:3].tolist(), got[bad][:3], want[bad][:3])
    assert (y[:, 2] == -math.inf).all() and (y[:, 3] == 0).all()
    assert torch.equal(out.top_tokens, r[:, None] + period * torch.arange(top, device=cuda))

    # One of another class far above them: they are summed, not counted.
    x.copy_(torch.where(own, -1.0, -math.inf))
    at = (other + period * (torch.arange(rows, device=cuda) * 7919 % (n.long().to(cuda) - 1)))
    x.scatter_(1, at[:, None], 1.0)
    out = L.token_logprobs(x, tokens, top=top)
    e = math.exp(-2.0)
    rest = n * e
    norm = torch.log1p(rest)
    off = U * (((N + 4) * rest + 4 * rest) / (1 + rest) + 4 * norm)
    assert (off < 0.4 * e / (1 + rest)).all()
    y = out.logprobs.double().cpu()
    tol = off + U * (4 + 2 + norm)
    for got in (y[:, 0], y[:, 1], out.top_logprobs[:, 1].double().cpu()):
        bad = (got + 2.0 + norm).abs() > tol
        assert not bad.any(), (bad.nonzero()[:3].tolist(), got[bad][:3], -2.0 - norm[bad][:3])
    entropy = norm + 2 * rest / (1 + rest)
    tol = off + U * (((2 * N + 12) * 2 * rest + 8 * rest) / (1 + rest) + entropy)
    assert ((out.entropy.double().cpu() - entropy).abs() <= tol).all()
    assert torch.equal(out.top_tokens, torch.cat(
        (at[:, None], r[:, None] + period * torch.arange(top - 1, device=cuda)), 1))


# one to 32 slices of a row, workgroups of every size
VOCABS = [331, 1023, 4097, 9001, 32003, 65521, 65537, 131072, 131085, 140003, 262147, 500009,
          1 << 20]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_every_token_counts_once(cuda, vocab, dtype):
    G.note(f"logprobs counts {vocab} {dtype}")
    check_classes(cuda, vocab, 61, range(61), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [32003, 65537, 140003, 262147])
def test_every_token_counts_once_among_few(cuda, vocab, dtype):
    """Classes so sparse that a wavefront has the maximum in a few threads."""
    G.note(f"logprobs sparse counts {vocab} {dtype}")
    period = 4099
    for c in range(0, period, 512):
        check_classes(cuda, vocab, period, range(c, min(c + 512, period)), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [32769, 32787, 65541, 65552, 131073])
def test_every_token_counts_once_in_many_rows(cuda, vocab, dtype):
    """More rows than fill the card: long ones are cut earlier."""
    G.note(f"logprobs counts of many rows {vocab} {dtype}")
    check_classes(cuda, vocab, 61, [i % 61 for i in range(549)], dtype)


def check(out, x, tokens, top):
    x = x.cpu()
    given, entropy, best, ids, (rest, spread, square) = O.logprobs(x, tokens[:, None].cpu(), top)
    s, log = 1.0 + rest, torch.log1p(rest)
    norm = U * (((N + 4) * rest + 2 * spread) / s + 4 * log)

    def close(got, want, tol):
        err = (got.double().cpu() - want).abs()
        same = got.double().cpu() == want      # infinities
        assert (same | (err <= tol)).all(), float((err - tol).nan_to_num(0.0).max())

    def tol(want):
        return norm[:, None] + U * (3 * want.abs() + 2 * log[:, None])

    close(out.logprobs[:, None], given, tol(given))
    close(out.entropy, entropy, norm + U * (((2 * N + 12) * spread + 2 * square) / s + entropy))
    if top:
        assert torch.equal(out.top_tokens.cpu(), ids)
        close(out.top_logprobs, best, tol(best))


@pytest.mark.parametrize("top", [0, 64])
@pytest.mark.parametrize("vocab,dtype", [(65552, torch.bfloat16), (65552, torch.float16),
                                         (32776, torch.float32)])
def test_one_row_more_than_keep_a_workgroup_each(cuda, vocab, dtype, top):
    """512 rows, a workgroup each, and 513 and 600, cut in two: each against the
    definition, and the bits of a row do not depend on its place or on how many
    rows of either kind there are."""
    G.note(f"logprobs 513 rows {vocab} {dtype} {top}")
    rows = 600
    g = torch.Generator(device=cuda).manual_seed(vocab + top)
    sharp = torch.logspace(-1, 1, rows, device=cuda)[torch.randperm(rows, generator=g, device=cuda)]
    x = rows_in(room(rows, vocab, dtype, cuda), rows, vocab)
    x.copy_(torch.randn(rows, vocab, generator=g, device=cuda) * sharp[:, None])
    x[::3, vocab // 3:vocab // 2] = -math.inf
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=cuda)

    def pick(out, at):
        return L.TokenLogprobs(*(None if t is None else t[at] for t in out))

    def call(n):
        return L.token_logprobs(x[:n], tokens[:n], top=top)

    outs = {n: call(n) for n in (200, 512, 513, 600)}
    some = torch.tensor([0, 1, 2, 3, 5, 100, 199, 255, 256, 400, 511], device=cuda)
    check(pick(outs[512], some), x[some], tokens[some], top)
    some = torch.cat((some, torch.tensor([512], device=cuda)))
    check(pick(outs[513], some), x[some], tokens[some], top)
    for few, many in ((200, 512), (513, 600)):
        for a, b in zip(outs[few], outs[many]):
            assert a is None or torch.equal(a, b[:few])
    if top:
        assert torch.equal(outs[512].top_tokens, outs[513].top_tokens[:512])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 1000, 1025, 5003, 65537, 140003, 262147])
@pytest.mark.parametrize("top", [1, 33])
def test_rows_of_many_nan(cuda, top, vocab, dtype):
    """More NaN than candidates are ranked, the first token's and the last one's
    among them: they come first, by their number, then infinity."""
    G.note(f"logprobs many nan {vocab} {top} {dtype}")
    x = torch.zeros(8, vocab, dtype=dtype, device=cuda)
    x[0] = math.nan
    x[1, 1:] = math.nan
    x[2, :-1] = math.nan
    x[3, ::2] = math.nan
    x[4, 1::2] = math.nan
    x[4, 0] = math.inf
    x[5] = math.inf
    x[5, :12] = math.nan
    x[6] = -math.inf
    x[6, 0] = math.nan
    x[7] = math.inf
    x[7, vocab - 1] = math.nan
    tokens = torch.zeros(8, dtype=torch.int64, device=cuda)
    out = L.token_logprobs(x, tokens, top=top)
    value = x.double().cpu()
    key = torch.where(value.isnan(), 3.0, torch.where(value == math.inf, 2.0, torch.where(
        value == 0, 1.0, 0.0)))
    want = torch.sort(key, stable=True, dim=-1, descending=True).indices[:, :top]
    assert torch.equal(out.top_tokens.cpu(), want)
    assert out.logprobs.isnan().all() and out.entropy.isnan().all()
    assert out.top_logprobs.isnan().all()
