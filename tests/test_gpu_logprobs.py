"""Log probabilities of given tokens on the GPU against log_softmax in binary64
(oracle/drafts_oracle.py).

Tolerances, from the arithmetic (u = 2^-24).  With d = x - m, e = exp(d), m the
largest logit: R = sum e over all logits but one largest, D = sum |d| e, Q = sum
d^2 e, and S = 1 + R.  d is rounded once; the exponential's argument a second time
and its result within 2 u: e is off by (2 |d| + 4) u relative.  A sum has at
most N = vocab / 256 + 64 additions in a row (256 threads at least, a tree over
them), N u relative, all terms of one sign.  So log S is off by ((N + 8) R + 2 D) u / S
(of a function of slope 1 / S) and its own rounding, 4 u log S; a log probability
by that and 2 u |d| + u |y|.  The entropy log S + D / S adds ((2 N + 16) D + 2 Q) u / S.
"""
from __future__ import annotations

import math

import pytest
import torch

import test_gpu_attention as G
from nanopointllm_amd import lm_head as L
from nanopointllm_amd.runner import DecodeGraphBucket
from oracle import drafts_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def same_or_close(got, want, tol, what):
    got = got.double().cpu()
    special = ~torch.isfinite(want)
    assert torch.equal(got[special].nan_to_num(nan=5.0, posinf=6.0, neginf=7.0),
                       want[special].nan_to_num(nan=5.0, posinf=6.0, neginf=7.0)), what
    err = (got - want).abs()[~special]
    bad = ~(err <= tol[~special])
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {err[bad].max()}"


def check(out, x, tokens, top):
    rows, v = x.shape
    t = tokens.reshape(rows, -1)
    given, entropy, best, ids, (rest, spread, square) = O.logprobs(x, t, top)
    s = 1.0 + rest
    n = v / 256 + 64
    norm = U * (((n + 8) * rest + 2 * spread) / s + 4 * torch.log1p(rest))
    y = out.logprobs.reshape(rows, -1)
    def tol(want):
        return norm[:, None] + U * (3 * want.abs() + 2 * torch.log1p(rest)[:, None]) + 1e-44

    same_or_close(y, given, tol(given), "logprobs")
    same_or_close(out.entropy, entropy.masked_fill(torch.isnan(spread + rest), math.nan),
                  norm + U * ((2 * n + 16) * spread + 2 * square) / s + U * entropy.abs() + 1e-44,
                  "entropy")
    if top:
        assert torch.equal(out.top_tokens.cpu(), ids)
        same_or_close(out.top_logprobs, best, tol(best), "top")
    else:
        assert out.top_logprobs is None and out.top_tokens is None


def rows_of(seed, rows, vocab, dtype, device):
    """From flat to decided rows, some with masked tokens."""
    g = G.gen_of(seed)
    sharp = torch.logspace(-1, 1.2, rows)[torch.randperm(rows, generator=g)]
    x = (torch.randn(rows, vocab, generator=g) * sharp[:, None]).to(dtype)
    for i in range(0, rows, 3):
        hide = torch.rand(vocab, generator=g) < 0.7
        hide[i % vocab] = False
        x[i] = x[i].masked_fill(hide, -math.inf)
    return x.to(device)


SHAPES = [
    # rows, vocab, tokens a row (0: the rows' shape), top
    (1, 1, 0, 1), (3, 2, 0, 2), (5, 7, 3, 7), (2, 64, 0, 64), (9, 65, 2, 64), (4, 511, 0, 5),
    (3, 512, 1, 0), (3, 513, 0, 33), (2, 1000, 5, 20), (8, 32003, 0, 5), (3, 32003, 4, 64),
    (1, 50257, 0, 1), (2, 65536, 0, 20), (2, 65537, 0, 3), (3, 128256, 4, 20),
    (1, 131073, 0, 64), (2, 262144, 0, 10), (1, 1 << 20, 2, 64), (700, 300, 0, 4),
    (2500, 40, 0, 0), (300, 4097, 2, 2),
    # few groups of threads hold a logit: hundreds of candidates
    (67, 1004, 0, 64), (3, 700, 2, 64), (5, 520, 0, 40), (2, 420, 0, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,per,top", SHAPES)
def test_logprobs_against_the_definition(cuda, rows, vocab, per, top, dtype):
    G.note(f"logprobs {rows} {vocab} {per} {top} {dtype}")
    x = rows_of(rows + vocab, rows, vocab, dtype, cuda)
    g = G.gen_of(vocab)
    shape = (rows, per) if per else (rows,)
    tokens = torch.randint(0, vocab, shape, generator=g).to(cuda)
    out = L.token_logprobs(x, tokens, top=top)
    assert out.logprobs.shape == tokens.shape and out.entropy.shape == (rows,)
    check(out, x, tokens, top)
    again = L.token_logprobs(x, tokens, top=top)
    for a, b in zip(out, again):
        assert a is None and b is None or torch.equal(a, b) or torch.equal(
            a.nan_to_num(nan=9.0), b.nan_to_num(nan=9.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 5, 8])
def test_rows_at_any_alignment(cuda, offset, dtype):
    """Rows inside a larger tensor, whose other columns hold what must not count;
    more axes in front."""
    G.note(f"logprobs alignment {offset} {dtype}")
    vocab, rows = 1003, 6
    wide = torch.full((rows, vocab + 19), math.nan, dtype=dtype, device=cuda)
    x = rows_of(offset, rows, vocab, dtype, cuda)
    wide[:, offset:offset + vocab] = x
    tokens = torch.randint(0, vocab, (2, 3), generator=G.gen_of(1)).to(cuda)
    out = L.token_logprobs(wide.view(2, 3, -1)[..., offset:offset + vocab], tokens, top=9)
    assert out.top_tokens.shape == (2, 3, 9) and out.entropy.shape == (2, 3)
    flat = L.TokenLogprobs(out.logprobs.view(-1), out.entropy.view(-1),
                           out.top_logprobs.view(-1, 9), out.top_tokens.view(-1, 9))
    check(flat, x, tokens.view(-1), 9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [40, 600, 1000, 5000, 70000, 300000])
def test_ties_and_special_rows(cuda, vocab, dtype):
    """Equal logits (the lowest token first), zeros of both signs, fewer finite
    logits than asked for, rising and falling rows, NaN, infinities, and rows of
    nothing."""
    G.note(f"logprobs ties {vocab} {dtype}")
    g = G.gen_of(vocab)
    top = 33
    x = torch.randn(12, vocab, generator=g)
    x[0] = 0.75
    x[1] = torch.where(torch.rand(vocab, generator=g) < 0.5, 0.0, -0.0)
    x[2] = -math.inf
    x[2, [3, 17, 21]] = torch.tensor([1.0, 2.0, 1.0])
    x[3] = torch.arange(vocab) / vocab * 20
    x[4] = -torch.arange(vocab) / vocab * 20
    x[5] = torch.randint(0, 3, (vocab,), generator=g).float()
    x[6, vocab // 2] = math.nan
    x[7, 5] = math.inf
    x[8] = -math.inf
    x[9] = -1000.0
    x[9, vocab - 1] = 1000.0
    x[10] = torch.finfo(dtype).min
    x[10, 1] = 0.0
    x[11, :] = x[11].abs().neg() * 1e-3
    x = x.to(dtype).to(cuda)
    tokens = torch.tensor([-1, 0, 17, vocab, vocab - 1, -7, 4, 2 ** 40, -2 ** 63, 0, 1, 39],
                          device=cuda)
    out = L.token_logprobs(x, tokens, top=top)
    check(out, x, tokens, top)
    assert out.logprobs[0] == 0 and out.logprobs[3].isnan() and out.logprobs[5].isnan()
    assert out.top_tokens[0].tolist() == list(range(top))
    assert out.top_tokens[1].tolist() == list(range(top))
    assert out.top_tokens[2, :5].tolist() == [17, 3, 21, 0, 1]
    assert out.entropy[6:9].isnan().all() and out.entropy[9] == 0


def test_nearly_decided_rows_keep_their_digits(cuda):
    """One logit far above the rest: the entropy and the top log probability are
    tiny, and right to a few units of their own last place."""
    G.note("logprobs decided")
    vocab = 32003
    x = torch.zeros(3, vocab)
    for i, top in enumerate((20.0, 40.0, 70.0)):
        x[i, 100 * i] = top
    out = L.token_logprobs(x.to(cuda), torch.tensor([0, 100, 200], device=cuda), top=2)
    rest = (vocab - 1) * torch.exp(-torch.tensor([20.0, 40.0, 70.0], dtype=torch.float64))
    d = torch.tensor([20.0, 40.0, 70.0], dtype=torch.float64)
    tol = U * (vocab / 256 + 64 + 16 + 4 * d)
    assert ((out.logprobs.double().cpu() / -torch.log1p(rest) - 1).abs() <= tol).all()
    want = torch.log1p(rest) + rest * d / (1 + rest)
    assert ((out.entropy.double().cpu() / want - 1).abs() <= 3 * tol).all()


def test_captured_and_on_another_stream(cuda):
    G.note("logprobs graph")
    x = rows_of(1, 6, 140000, torch.bfloat16, cuda)
    tokens = torch.randint(0, 140000, (6,), generator=G.gen_of(1)).to(cuda)
    bucket = DecodeGraphBucket(cuda)
    bucket.capture(lambda: L.token_logprobs(x, tokens, top=7))
    for turn in range(3):
        x.copy_(rows_of(20 + turn, 6, 140000, torch.bfloat16, cuda))
        want = L.token_logprobs(x, tokens, top=7)
        torch.cuda.synchronize()
        got = bucket.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = L.token_logprobs(x, tokens, top=7)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_calls(cuda):
    G.note("logprobs empty")
    x = torch.zeros(0, 50, device=cuda)
    out = L.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device=cuda), top=2)
    assert out.logprobs.shape == out.entropy.shape == (0,) and out.top_tokens.shape == (0, 2)
    x = rows_of(1, 3, 50, torch.float16, cuda)
    out = L.token_logprobs(x, torch.zeros(3, 0, dtype=torch.int64, device=cuda), top=2)
    assert out.logprobs.shape == (3, 0)
    want = L.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=cuda), top=2)
    assert all(torch.equal(a, b) for a, b in zip(out[1:], want[1:]))


@pytest.mark.parametrize("vocab", [5000, 200000])
def test_offsets_past_32_bits(cuda, vocab):
    """Rows 2^31 logits apart, the last more than 2^32 behind the first."""
    G.note(f"logprobs far rows {vocab}")
    apart = (1 << 31) + 24
    store = torch.empty(2 * apart + vocab, dtype=torch.bfloat16, device=cuda)
    x = store.as_strided((3, vocab), (apart, 1))
    near = rows_of(4, 3, vocab, torch.bfloat16, cuda)
    x.copy_(near)
    tokens = torch.randint(0, vocab, (3, 4), generator=G.gen_of(1)).to(cuda)
    got, want = (L.token_logprobs(y, tokens, top=9) for y in (x, near))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,top,skew", [(1300, 20, 0), (32003, 5, 1), (32003, 64, 3),
                                            (140003, 33, 5), (262144, 64, 0), (50001, 1, 7)])
def test_thousands_of_equal_or_close_tokens(cuda, vocab, top, skew, dtype):
    """More candidates than are ranked: rows of one value, masks of the type's
    lowest value that leave fewer tokens than are asked for, tokens allowed in one
    short range only, runs of equal ones at either end, and values of which
    thousands are equal."""
    G.note(f"logprobs ties {vocab} {top} {skew} {dtype}")
    g = G.gen_of(vocab + top)
    low = torch.finfo(dtype).min
    x = torch.full((12, vocab), low, dtype=dtype)
    x[0] = 0.0
    x[1] = -3.5
    few = torch.randperm(vocab, generator=g)[:3]
    x[2, few] = torch.tensor([1.0, 3.0, 2.0], dtype=dtype)
    x[3, [0, vocab - 1]] = 1.0
    x[5, vocab // 3:vocab // 3 + 1200] = torch.randn(1200, generator=g).to(dtype)[:vocab - vocab // 3]
    x[6:9] = -math.inf
    x[6, vocab // 3:vocab // 3 + 1200] = x[5, vocab // 3:vocab // 3 + 1200]
    x[7, -1200:] = 1.0
    x[7, vocab // 2] = 4.0
    x[8, :1200] = -1.0
    x[8, -3:] = 0.0
    x[9] = torch.randint(0, 3, (vocab,), generator=g).to(dtype)
    x[10] = torch.randint(0, 3, (vocab,), generator=g).to(dtype)
    x[10, few] = 7.0
    x[11] = torch.arange(vocab).div(2000, rounding_mode="floor").to(dtype)
    wide = torch.full((12, vocab + 8), math.nan, dtype=dtype, device=cuda)
    y = wide[:, skew:skew + vocab]
    y.copy_(x)
    tokens = torch.randint(0, vocab, (12,), generator=g)
    check(L.token_logprobs(y, tokens.to(cuda), top=top), x, tokens, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(3, 40, 3), (4, 1300, 20), (5, 32003, 5), (3, 140003, 64),
                                            (2, 300000, 0)])
def test_rows_far_from_zero(cuda, rows, vocab, top, dtype):
    """All of a row's logits far below or above zero, with and without masked
    tokens, where some threads have none."""
    G.note(f"logprobs far {rows} {vocab} {top} {dtype}")
    g = G.gen_of(vocab)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    for shift in (-90.0, -700.0, -60000.0, 700.0, 60000.0):
        x = (torch.randn(rows, vocab, generator=g) + shift).to(dtype)
        x[0, 3:] = -math.inf
        x[1] = x[1, 0]
        check(L.token_logprobs(x.to(cuda), tokens.to(cuda), top=top), x, tokens, top)
