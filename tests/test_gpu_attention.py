"""The attention core on the GPU against its definitions in binary64
(oracle/attention_oracle.py).

Tolerances, from the arithmetic (u = 2^-24, e = finfo(dtype).eps / 2: half a
step of a rounding to the 16-bit type):

* rotary: cos and sin within 4 u of their values (amplitude a), two products
  and one sum in binary32 (3 u), one rounding:
  e |y| + 8 u (|a c x| + |a s y|).
* attention: a score is off by at most (D + 4) u sum |q k| (binary32 products
  and sums, the scale, the change of base); exp2 and its argument's rounding
  give 8 u more per probability, relative, and scores s of size S another 4 u S
  from the rounding of s - max.  Numerator and denominator both carry this:
  r = 2 ((D + 4 + 8) u S + 16 u).  The probabilities of prompts are rounded to
  the 16-bit type, in numerator and denominator: 2 e more; below that type's
  smallest normal value the step is 2^-24 for binary16 at a probability scale
  of at least 1, so n 2^-25 max|v| for n keys.  Sums over n keys: 2 n u.  In
  all (r + 2 e + 2 n u) sum p |v| + n 2^-25 max|v| + e |out| (+ the smallest
  step of the type).  A wrong key, row, head or mask misses this by orders of
  magnitude: values are of order 1.
"""
from __future__ import annotations

import sys

import pytest
import torch

from nanopointllm_amd import attention as A
from oracle import attention_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float16, torch.bfloat16]


def note(msg: str) -> None:
    sys.__stderr__.write(f"[gpu-case] {msg}\n")
    sys.__stderr__.flush()


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def smallest(dtype) -> float:
    return 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133


def randn(gen, *shape, dtype, device, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype).to(device)


def gen_of(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------- rotary
def check_rotary(got, x, positions, freq, layout, factor, what=""):
    want, size = O.rotary(x, positions, freq, layout, factor)
    err = (got.double().cpu() - want).abs()
    tol = half_step(x.dtype) * want.abs() + 8 * U * size + smallest(x.dtype)
    assert not (err > tol).any(), f"{what} worst {(err - tol).max()}"


ROTARY = [
    # tokens, heads, dim, rotary dim
    (1, 32, 128, 128), (3, 5, 128, 64), (7, 2, 80, 80), (7, 3, 80, 40), (2, 1, 64, 24),
    (5, 4, 96, 48), (4, 2, 256, 256), (3, 2, 8, 2), (3, 2, 8, 0), (9, 40, 64, 6), (130, 3, 24, 22),
]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("t,h,d,rot", ROTARY)
def test_rotary_against_the_definition(cuda, t, h, d, rot, layout):
    for dtype in DTYPES:
        note(f"rotary {t} {h} {d} {rot} {layout} {dtype}")
        g = gen_of(t * 1000 + d + rot)
        x = randn(g, t, h, d, dtype=dtype, device=cuda)
        # Positions of every size, negative ones among them.
        positions = (torch.randint(-10 ** 6, 10 ** 7, (t,), generator=g)).to(cuda)
        positions[0] = 0 if t > 1 else 10 ** 9 + 7
        freq = A.rotary_frequencies(rot, device=cuda).inv_freq
        y = A.rotary(x, positions, freq, layout=layout, attention_factor=1.25)
        check_rotary(y, x, positions, freq, layout, 1.25)
        assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_rotary_strides_and_in_place(cuda, layout, offset):
    """Rows at any 2-byte alignment, token and head strides of their own, and
    the same tensor as input and output: the neighbours keep their values."""
    note(f"rotary strides {layout} offset {offset}")
    t, h, d, rot = 6, 3, 64, 48
    g = gen_of(3 + offset)
    base = randn(g, t, h, 2 * d + 8, dtype=torch.float16, device=cuda)
    x = base[:, :, offset:offset + d]
    positions = torch.arange(t, device=cuda) * 1000
    freq = A.rotary_frequencies(rot, device=cuda).inv_freq
    want = A.rotary(x.contiguous(), positions, freq, layout=layout)
    assert torch.equal(A.rotary(x, positions, freq, layout=layout), want)
    before = base.clone()
    assert A.rotary(x, positions, freq, layout=layout, out=x) is x
    assert torch.equal(x, want)
    before[:, :, offset:offset + d] = want
    assert torch.equal(base, before)
    by_head = base.transpose(0, 1)[:, :, :d]     # head stride past the token stride
    assert torch.equal(A.rotary(by_head, torch.arange(h, device=cuda), freq, layout=layout),
                       A.rotary(by_head.contiguous(), torch.arange(h, device=cuda), freq,
                                layout=layout))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h,g,d,rot,page", [
    (1, 32, 32, 128, 128, 16), (37, 32, 8, 128, 64, 16), (19, 28, 4, 80, 80, 8),
    (5, 8, 1, 64, 24, 1), (3, 3, 3, 96, 40, 128), (70, 2, 2, 8, 8, 4)])
def test_rotary_store_against_the_definition(cuda, t, h, g, d, rot, page, dtype):
    """Views of a packed matrix into scattered slots, some rows padded; the
    cache's other rows keep their bits, and the [page, head] order of a cache
    changes nothing."""
    note(f"rotary_store {t} {h} {g} {d} {rot} {page} {dtype}")
    r = gen_of(t + h)
    rows = randn(r, t, (h + 2 * g) * d, dtype=dtype, device=cuda)
    q, k, v = rows.split((h * d, g * d, g * d), 1)
    q, k, v = q.view(t, h, d), k.view(t, g, d), v.view(t, g, d)
    pages = -(-t // page) + 3
    slots = torch.randperm(pages * page, generator=r)[:t]
    if t > 4:
        slots[1], slots[3], slots[4] = -1, pages * page, 2 ** 62
    positions = torch.randint(0, 200000, (t,), generator=r)
    freq = A.rotary_frequencies(rot, device=cuda).inv_freq
    caches = [randn(r, pages, g, page, d, dtype=dtype, device=cuda) for _ in range(2)]
    before = [c.clone() for c in caches]
    other = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    for layout in ("half", "interleaved"):
        for c, b in zip(caches, before):
            c.copy_(b)
        out = A.rotary_store(q, k, v, positions.to(cuda), slots.to(cuda), freq, *caches,
                             layout=layout, attention_factor=0.75)
        check_rotary(out, q, positions, freq, layout, 0.75, "q")
        turned = A.rotary(k, positions.to(cuda), freq, layout=layout, attention_factor=0.75)
        check_rotary(turned, k, positions, freq, layout, 0.75, "k")
        want = [b.clone() for b in before]
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                want[0][s // page, :, s % page] = turned[i]
                want[1][s // page, :, s % page] = v[i]
        assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])
        A.rotary_store(q, k, v, positions.to(cuda), slots.to(cuda), freq, *other, layout=layout,
                       attention_factor=0.75)
        assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    # q in place inside the packed rows: k and v keep their bits.
    kv = rows[:, h * d:].clone()
    A.rotary_store(q, k, v, positions.to(cuda), slots.to(cuda), freq, *caches,
                   layout="interleaved", attention_factor=0.75, out=q)
    assert torch.equal(q, out) and torch.equal(rows[:, h * d:], kv)


# ---------------------------------------------------------------- attention
def paged(seed, lengths, g, d, page, dtype, device, *, order="head", spare=2, poison=True):
    """(k_cache, v_cache, table): scattered pages; rows past each length, and
    pages of no sequence, hold NaN and infinities."""
    r = gen_of(seed)
    needs = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(needs) + spare
    at = torch.randperm(pages, generator=r).tolist()
    shape = (pages, g, page, d) if order == "head" else (pages, page, g, d)
    caches = []
    for i in range(2):
        c = randn(r, *shape, dtype=dtype, device=device)
        caches.append(c if order == "head" else c.transpose(1, 2))
    table = torch.full((len(lengths), max(needs + [1]) + 1), -1, dtype=torch.int32)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for i in range(needs[b]):
            table[b, i] = at.pop()
            used[table[b, i], :max(0, min(page, n - i * page))] = True
    if poison:
        bad = ~used.to(device)[:, None, :, None]
        caches[0].masked_fill_(bad, float("nan"))
        caches[1].masked_fill_(bad, float("nan"))
        caches[1][..., ::2].masked_fill_(bad, float("inf"))
    return caches[0], caches[1], table.to(device)


def check_attention(out, q, k, v, table, lengths, starts=None, scale=None, what=""):
    want, size, dots = O.attention(q, k, v, table, lengths, starts, scale)
    owned = ~torch.isnan(want)
    assert owned.all() or starts is not None
    d, e, n = q.shape[2], half_step(q.dtype), int(lengths.max()) if lengths.numel() else 0
    finite = v.float().cpu()
    most = float(finite[torch.isfinite(finite)].abs().max()) if finite.numel() else 0.0
    rel = 2 * ((d + 12) * U * dots + 16 * U) + 2 * e + 2 * n * U
    tol = rel[..., None] * size + n * 2.0 ** -25 * most * (size > 0) + e * want.abs() \
        + smallest(q.dtype)
    err = (out.double().cpu() - want).abs()
    bad = owned & ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} off, worst {err[bad].max()} "
                           f"at {bad.nonzero()[0].tolist()}")


DECODE = [
    # heads, kv heads, dim, page, lengths
    (32, 32, 128, 16, [601]), (32, 8, 128, 16, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0]),
    (4, 4, 64, 32, [129, 0, 700, 1]), (28, 4, 80, 8, [77, 255, 256, 257]), (6, 2, 96, 1, [5, 40]),
    (16, 1, 128, 64, [1000, 3]), (71, 1, 64, 16, [300, 90]), (40, 2, 8, 16, [50]),
    (8, 2, 256, 16, [333, 64]), (8, 8, 24, 4, [9, 0, 0, 130]), (34, 2, 192, 128, [500]),
    (2, 2, 128, 16, [5000]), (4, 1, 128, 64, [9000, 17, 0, 4097]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,lengths", DECODE)
def test_decode_against_the_definition(cuda, h, g, d, page, lengths, dtype):
    note(f"decode {h} {g} {d} {page} {lengths} {dtype}")
    k, v, table = paged(h + d, lengths, g, d, page, dtype, cuda)
    q = randn(gen_of(d), len(lengths), h, d, dtype=dtype, device=cuda, std=1.7)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    out = A.paged_decode(q, k, v, table, n)
    check_attention(out, q, k, v, table, n)
    assert (out[n <= 0] == 0).all()
    assert torch.equal(out, A.paged_decode(q, k, v, table, n))      # the same bits again
    # The same cache with heads inside tokens, a wider table, strided rows.
    k2, v2 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    wide = torch.full((len(lengths), table.shape[1] + 5), 2 ** 31 - 1, dtype=torch.int32,
                      device=cuda)
    wide[:, :table.shape[1]] = table
    rows = torch.zeros(len(lengths), h + 2, d, dtype=dtype, device=cuda)
    rows[:, 1:-1] = q
    into = torch.full((len(lengths), h + 1, d), 7.0, dtype=dtype, device=cuda)
    A.paged_decode(rows[:, 1:-1], k2, v2, wide[:, :table.shape[1]], n, out=into[:, :h])
    assert torch.equal(into[:, :h], out) and (into[:, h] == 7.0).all()


@pytest.mark.parametrize("batch,h,g,d,page,longest", [
    (130, 2, 2, 128, 16, 400),     # a workgroup of 8 wavefronts per sequence and head
    (260, 2, 2, 64, 64, 300),      # ... of 4
    (70, 34, 2, 96, 8, 500),       # blocks of 16 queries of one key head
    (129, 4, 2, 80, 2, 333),       # pages smaller than a lane's four keys
    (65, 4, 4, 256, 32, 400),      # wide heads
    (37, 8, 8, 128, 16, 2500),     # cut, each sequence by its length
])
def test_decode_of_large_batches(cuda, batch, h, g, d, page, longest):
    """Batches with a workgroup for every CU, lengths of zero and one among
    them."""
    note(f"decode batch {batch} {h} {g} {d} {page} {longest}")
    r = gen_of(batch)
    lengths = torch.randint(0, longest, (batch,), generator=r).tolist()
    lengths[0], lengths[1], lengths[2] = longest, 0, 1
    for dtype in DTYPES:
        k, v, table = paged(batch + d, lengths, g, d, page, dtype, cuda)
        q = randn(r, batch, h, d, dtype=dtype, device=cuda, std=1.7)
        n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        out = A.paged_decode(q, k, v, table, n)
        check_attention(out, q, k, v, table, n)
        # The last ten by themselves, cut otherwise.
        few = A.paged_decode(q[-10:], k, v, table[-10:], n[-10:])
        check_attention(few, q[-10:], k, v, table[-10:], n[-10:])


PREFILL = [
    # heads, kv heads, dim, page, new tokens, lengths
    (4, 4, 128, 16, [560], [560]),
    (8, 2, 128, 16, [1, 2, 31, 32, 33, 64, 0, 65, 127, 128, 129], None),
    (4, 1, 64, 32, [5, 100, 0, 3], [300, 100, 50, 9]), (7, 1, 80, 8, [40, 130], [41, 400]),
    (2, 2, 96, 1, [17, 33], [17, 80]), (4, 2, 256, 16, [70, 9], [70, 150]),
    (3, 3, 8, 4, [21], [30]), (2, 1, 192, 64, [140], [200]),
    # fewer keys than new rows: the first rows see none
    (4, 2, 128, 16, [10, 50, 4], [3, 0, 4]), (2, 2, 64, 16, [200], [70]),
    # few rows far into a long context
    (8, 2, 128, 64, [3], [5000]), (4, 4, 64, 16, [40, 1], [3333, 2000]),
    (2, 1, 128, 16, [300], [4400]),
    # many sequences; row tiles of uneven prompts by their keys; more than 2048
    # workgroups
    (8, 1, 64, 16, [1 + 7 * i % 41 for i in range(70)], [1 + 11 * i % 60 for i in range(70)]),
    (16, 2, 96, 32, [200, 0, 77, 31, 130], [200, 40, 500, 31, 300]),
    (128, 128, 8, 16, [900, 350, 600], [900, 700, 590]),
    # a token's queries over more than one row tile
    (200, 1, 64, 16, [3, 0, 70], [40, 9, 70]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,new,lengths", PREFILL)
def test_prefill_against_the_definition(cuda, h, g, d, page, new, lengths, dtype):
    note(f"prefill {h} {g} {d} {page} {new} {lengths} {dtype}")
    lengths = new if lengths is None else lengths
    k, v, table = paged(h + d + len(new), lengths, g, d, page, dtype, cuda)
    before, behind = 3, 5                     # rows of no sequence
    starts = torch.tensor([before] + new).cumsum(0).to(torch.int32).to(cuda)
    rows = before + sum(new) + behind
    q = randn(gen_of(d + h), rows, h, d, dtype=dtype, device=cuda, std=1.7)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    into = torch.full((rows, h, d), 7.0, dtype=dtype, device=cuda)
    out = A.paged_prefill(q, k, v, table, n, starts, out=into)
    assert out is into
    check_attention(out, q, k, v, table, n, starts)
    assert (out[:before] == 7.0).all() and (out[rows - behind:] == 7.0).all()
    again = torch.full_like(into, 7.0)
    k2, v2 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    A.paged_prefill(q, k2, v2, table, n, starts, out=again)
    assert torch.equal(out, again)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_given_scales(cuda, scale):
    note(f"scale {scale}")
    k, v, table = paged(5, [70, 33], 2, 64, 16, torch.float16, cuda)
    n = torch.tensor([70, 33], dtype=torch.int32, device=cuda)
    q = randn(gen_of(1), 2, 4, 64, dtype=torch.float16, device=cuda)
    check_attention(A.paged_decode(q, k, v, table, n, scale=scale), q, k, v, table, n, None, scale)
    q = randn(gen_of(2), 25, 4, 64, dtype=torch.float16, device=cuda)
    starts = torch.tensor([0, 20, 25], dtype=torch.int32, device=cuda)
    check_attention(A.paged_prefill(q, k, v, table, n, starts, scale=scale), q, k, v, table, n,
                    starts, scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sharp_and_flat_rows(cuda, dtype):
    """Scores hundreds apart (one key takes all), all equal, and a first key
    far above or far below the rest: the running maximum has to follow."""
    note(f"sharp rows {dtype}")
    lengths = [300, 300, 300, 300]
    k, v, table = paged(9, lengths, 1, 64, 16, dtype, cuda, poison=False)
    q = randn(gen_of(3), 4, 4, 64, dtype=dtype, device=cuda)
    q[0] *= 60.0
    q[1] = 0.0
    first = k[table[2, 0].long(), 0, 0]
    first *= 8.0
    q[2] = first * 0.5
    low = k[table[3, 0].long(), 0, 0]
    low *= 8.0
    q[3] = -low * 0.5
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    check_attention(A.paged_decode(q, k, v, table, n), q, k, v, table, n, what="decode")
    # The rows as the newest of one sequence each.
    for b in range(4):
        starts = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
        out = A.paged_prefill(q[b:b + 1], k, v, table[b:b + 1], n[b:b + 1], starts)
        check_attention(out, q[b:b + 1], k, v, table[b:b + 1], n[b:b + 1], starts, what="prefill")
    rows = q[2].expand(40, 4, 64).contiguous()
    starts = torch.tensor([0, 40], dtype=torch.int32, device=cuda)
    out = A.paged_prefill(rows, k, v, table[2:3], n[2:3], starts)
    check_attention(out, rows, k, v, table[2:3], n[2:3], starts, what="chunk")


@pytest.mark.parametrize("below", [14, 20, 23, 26])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_small_probabilities_count(cuda, dtype, below):
    """One key ahead of 90 thousand others by 2^below each: together they weigh
    up to 5 times as much, or 0.1%.  With values of one the result is the sum
    of the weights over itself, 1, whatever a weight's rounding, as long as
    numerator and denominator hold the same weights; with the first value 0
    and the others 1 it is their share."""
    note(f"small probabilities {dtype} 2^-{below}")
    n, d, page = 90001, 64, 64
    k, v, table = paged(31, [n], 1, d, page, dtype, cuda, poison=False)
    k.zero_()
    v.fill_(1.0)
    k[table[0, 0].long(), 0, 0, 0] = 1.0
    q = torch.zeros(1, 1, d, dtype=dtype, device=cuda)
    q[..., 0] = 16.0
    scale = below * 0.6931471805599453 / 16.0
    lengths = torch.tensor([n], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    share = (n - 1) / (n - 1 + 2.0 ** below)
    # Weights: r of the module's bound with D sum |q k| = 16 once, the 16-bit
    # rounding of a weight 2 e (binary16 below 2^-14 of a scale of at least 1:
    # 2^-25 absolute, of a weight of 2^(7 - below)), sums of n terms 2 n u.
    step = half_step(dtype)
    if dtype == torch.float16:
        step = max(step, 2.0 ** -25 / 2.0 ** (7 - below))
    rel = 2 * ((d + 12) * U * 16 * scale + 16 * U) + 2 * step + 2 * n * U
    for name, out in (("decode", A.paged_decode(q, k, v, table, lengths, scale=scale)),
                      ("prefill", A.paged_prefill(q, k, v, table, lengths, starts, scale=scale))):
        assert (out.float() - 1.0).abs().max() <= half_step(dtype) + 2 * n * U, name
    v[table[0, 0].long(), 0, 0] = 0.0
    for name, out in (("decode", A.paged_decode(q, k, v, table, lengths, scale=scale)),
                      ("prefill", A.paged_prefill(q, k, v, table, lengths, starts, scale=scale))):
        err = (out.double() - share).abs().max()
        assert err <= (rel + half_step(dtype)) * share, f"{name} {float(err)} of {share}"


def test_infinities_and_nans_stay_where_they_are_seen(cuda):
    """A NaN or infinite value is seen by the rows at and after its token, and
    by no row before it; a NaN key likewise.  The other elements stay within
    the bound of the definition without it (rows that met such a value may be
    summed in another order, and with unrounded probabilities)."""
    note("causal NaN")
    n = 200
    k, v, table = paged(4, [n], 2, 128, 16, torch.float16, cuda, poison=False)
    q = randn(gen_of(8), n, 4, 128, dtype=torch.float16, device=cuda)
    lengths = torch.tensor([n], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    clean = A.paged_prefill(q, k, v, table, lengths, starts)
    check_attention(clean, q, k, v, table, lengths, starts, what="clean")
    for at, value in ((0, float("nan")), (77, float("inf")), (150, float("nan")),
                      (199, float("-inf"))):
        page, row = int(table[0, at // 16]), at % 16
        bad = v.clone()
        bad[page, 0, row, 5] = value
        out = A.paged_prefill(q, k, bad, table, lengths, starts)
        assert torch.equal(out[:, 2:], clean[:, 2:])                 # the other head's queries
        assert (~torch.isfinite(out[at:, :2, 5])).all()
        out[at:, :2, 5] = clean[at:, :2, 5]
        check_attention(out, q, k, v, table, lengths, starts, what=f"value {value} at {at}")
        bad = k.clone()
        bad[page, 1, row, 9] = float("nan")
        out = A.paged_prefill(q, bad, v, table, lengths, starts)
        assert torch.equal(out[:, :2], clean[:, :2])
        assert torch.isnan(out[at:, 2:]).all()
        out[at:, 2:] = clean[at:, 2:]
        check_attention(out, q, k, v, table, lengths, starts, what=f"key {value} at {at}")


def test_pages_outside_the_cache_are_masked(cuda):
    """A page of -1 or past the cache inside a sequence is never read: its keys
    are masked, and a sequence of such pages alone gives zeros."""
    note("bad pages")
    lengths = [100, 64, 90]
    k, v, table = paged(6, lengths, 2, 64, 16, torch.bfloat16, cuda)
    table[0, 2], table[1, :], table[2, 0] = -1, 2 ** 31 - 1, k.shape[0]
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = randn(gen_of(8), 3, 4, 64, dtype=torch.bfloat16, device=cuda)
    out = A.paged_decode(q, k, v, table, n)
    check_attention(out, q, k, v, table, n)
    assert (out[1] == 0).all()
    new = [40, 20, 90]
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda)
    q = randn(gen_of(9), sum(new), 4, 64, dtype=torch.bfloat16, device=cuda)
    check_attention(A.paged_prefill(q, k, v, table, n, starts), q, k, v, table, n, starts)


@pytest.mark.parametrize("page", [4, 16])
def test_caches_that_share_rows(cuda, page):
    """A cache that repeats one row, one head or one page by a stride of zero is
    read as its copy is."""
    note(f"shared rows {page}")
    g, d, lengths = 2, 64, [3 * page, 2 * page - 3]
    table = torch.tensor([[2, 0, 1], [1, 2, 0]], dtype=torch.int32, device=cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    new = [7, 2]
    starts = torch.tensor([0, 7, 9], dtype=torch.int32, device=cuda)
    r = gen_of(31)
    for shape in ((3, g, 1, d), (3, 1, page, d), (1, g, page, d), (1, 1, 1, d)):
        k, v = (randn(r, *shape, dtype=torch.float16, device=cuda).expand(3, g, page, d)
                for _ in range(2))
        whole = k.contiguous(), v.contiguous()
        q = randn(r, 2, 4, d, dtype=torch.float16, device=cuda)
        assert torch.equal(A.paged_decode(q, k, v, table, n), A.paged_decode(q, *whole, table, n))
        q = randn(r, sum(new), 4, d, dtype=torch.float16, device=cuda)
        out = A.paged_prefill(q, k, v, table, n, starts)
        check_attention(out, q, *whole, table, n, starts, what=f"{shape}")


def test_lengths_past_the_table_are_cut(cuda):
    note("long lengths")
    k, v, table = paged(7, [64, 64], 2, 64, 16, torch.float16, cuda)
    table = table[:, :4]
    n = torch.tensor([10 ** 9, -5], dtype=torch.int32, device=cuda)
    cut = torch.tensor([64, 0], dtype=torch.int32, device=cuda)
    q = randn(gen_of(1), 2, 4, 64, dtype=torch.float16, device=cuda)
    out = A.paged_decode(q, k, v, table, n)
    assert torch.equal(out, A.paged_decode(q, k, v, table, cut)) and (out[1] == 0).all()
    q = randn(gen_of(2), 12, 4, 64, dtype=torch.float16, device=cuda)
    starts = torch.tensor([0, 9, 12], dtype=torch.int32, device=cuda)
    assert torch.equal(A.paged_prefill(q, k, v, table, n, starts),
                       A.paged_prefill(q, k, v, table, cut, starts))


def test_refusals_of_gpu_tensors(cuda):
    """Shapes, dtypes and layouts that no kernel may see."""
    note("refusals")
    q = torch.zeros(3, 4, 64, dtype=torch.float16, device=cuda)
    kv = torch.zeros(3, 2, 64, dtype=torch.float16, device=cuda)
    c = torch.zeros(5, 2, 16, 64, dtype=torch.float16, device=cuda)
    c2 = torch.zeros_like(c)
    i64 = torch.zeros(3, dtype=torch.int64, device=cuda)
    n = torch.ones(3, dtype=torch.int32, device=cuda)
    table = torch.zeros(3, 2, dtype=torch.int32, device=cuda)
    starts = torch.arange(4, dtype=torch.int32, device=cuda)
    freq = A.rotary_frequencies(64, device=cuda).inv_freq

    def store(q=q, k=kv, v=kv, positions=i64, slots=i64, freq=freq, kc=c, vc=c2, **kw):
        return A.rotary_store(q, k, v, positions, slots, freq, kc, vc, **kw)

    def decode(q=q, kc=c, vc=c2, table=table, n=n, **kw):
        return A.paged_decode(q, kc, vc, table, n, **kw)

    def prefill(q=q, kc=c, vc=c2, table=table, n=n, starts=starts, **kw):
        return A.paged_prefill(q, kc, vc, table, n, starts, **kw)

    turned = q.transpose(1, 2).contiguous().transpose(1, 2)    # heads not contiguous
    refused = [
        lambda: store(q=q.float()), lambda: store(q=q[0]), lambda: store(k=kv.bfloat16()),
        lambda: store(k=kv[:2]), lambda: store(v=kv[:, :1]), lambda: store(k=kv[..., :32]),
        lambda: store(positions=i64.int()), lambda: store(slots=i64[:2]),
        lambda: store(freq=freq.float()), lambda: store(freq=torch.cat((freq, freq))),
        lambda: store(layout="spiral"), lambda: store(kc=c.bfloat16()), lambda: store(vc=c2[:4]),
        lambda: store(kc=c[:, :1], vc=c2[:, :1]), lambda: store(vc=c), lambda: store(out=q[:2]),
        lambda: store(vc=c2.transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: store(q=turned, out=turned), lambda: store(out=kv.repeat(1, 2, 1).bfloat16()),
        lambda: store(attention_factor=float("inf")),
        lambda: A.rotary(turned, i64, freq, out=turned), lambda: A.rotary(q, i64[:1], freq),
        lambda: A.rotary(q, i64, freq, out=q.float()),
    ]
    for call in (decode, prefill):
        refused += [
            lambda call=call: call(q=q.float()), lambda call=call: call(q=q[..., :32]),
            lambda call=call: call(q=q[:, :3]), lambda call=call: call(kc=c.float(), vc=c2.float()),
            lambda call=call: call(table=table.long()), lambda call=call: call(table=table[:2]),
            lambda call=call: call(n=n.long()), lambda call=call: call(n=n[:2]),
            lambda call=call: call(out=q), lambda call=call: call(out=q[:2].clone()),
            lambda call=call: call(scale=float("nan")), lambda call=call: call(vc=c2[..., :32]),
            lambda call=call: call(kc=c[:, :, :12], vc=c2[:, :, :12]),
        ]
    refused += [lambda: prefill(starts=starts[:3]), lambda: prefill(starts=starts.long()),
                lambda: prefill(n=n.reshape(3, 1))]
    for at, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {at} was accepted")
    for call in (store, decode, prefill):
        with pytest.raises(RuntimeError, match="only on the GPU"):
            call(q=q.cpu())
        with pytest.raises(RuntimeError, match="only on the GPU"):
            call(vc=c2.cpu())
    assert not c.any() and not c2.any()
    # What the checks make contiguous is taken: rows with scattered elements, a
    # transposed table, lengths of every second place.
    assert torch.equal(store(q=turned), store())
    wide = torch.ones(6, dtype=torch.int32, device=cuda)
    assert torch.equal(decode(n=wide[::2], table=table.T.contiguous().T), decode())


def test_empty_calls(cuda):
    note("empty")
    k, v, table = paged(7, [64], 2, 64, 16, torch.float16, cuda)
    none = torch.empty(0, 4, 64, dtype=torch.float16, device=cuda)
    i32 = torch.zeros(0, dtype=torch.int32, device=cuda)
    assert A.paged_decode(none, k, v, table[:0], i32).shape == (0, 4, 64)
    starts = torch.zeros(2, dtype=torch.int32, device=cuda)
    n = torch.tensor([64], dtype=torch.int32, device=cuda)
    assert A.paged_prefill(none, k, v, table, n, starts).shape == (0, 4, 64)
    i64 = torch.zeros(0, dtype=torch.int64, device=cuda)
    freq = A.rotary_frequencies(64, device=cuda).inv_freq
    assert A.rotary_store(none, none[:, :2], none[:, :2], i64, i64, freq, k, v).shape == (0, 4, 64)
    # No page at all: every row is empty.
    q = torch.ones(1, 4, 64, dtype=torch.float16, device=cuda)
    assert (A.paged_decode(q, k, v, table[:, :0], n) == 0).all()
    assert (A.paged_decode(q, k[:0], v[:0], table, n) == 0).all()


def test_offsets_past_32_bits(cuda):
    """Pages more than 2^32 elements into the cache."""
    note("far pages")
    g, page, d = 2, 64, 128
    pages = (1 << 32) // (g * page * d) + 40
    k = torch.empty(pages, g, page, d, dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    lengths, r = [150, 70], gen_of(5)
    table = torch.tensor([[pages - 1, 3, pages - 30], [pages - 7, pages - 2, -1]],
                         dtype=torch.int32, device=cuda)
    for p in table.flatten().tolist():
        if p >= 0:
            k[p] = randn(r, g, page, d, dtype=k.dtype, device=cuda)
            v[p] = randn(r, g, page, d, dtype=k.dtype, device=cuda)
    small = torch.tensor([[0, 1, 2], [3, 4, -1]], dtype=torch.int32, device=cuda)
    at = table.flatten()[:5].long()
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    new = torch.randn(2, 4, d, generator=r).to(k.dtype).to(cuda)
    freq = A.rotary_frequencies(d, device=cuda).inv_freq
    slots = torch.tensor([(pages - 30) * page + 149 % page, (pages - 2) * page + 69 % page],
                         device=cuda)
    q = A.rotary_store(new, new[:, :2].contiguous(), new[:, 2:].contiguous(),
                       n.long() - 1, slots, freq, k, v)
    assert torch.equal(v[pages - 30, :, 149 % page], new[0, 2:])
    ks, vs = k[at], v[at]
    out = A.paged_decode(q, k, v, table, n)
    assert torch.equal(out, A.paged_decode(q, ks, vs, small, n))
    check_attention(out, q, ks, vs, small, n)
    starts = torch.tensor([0, 20, 29], dtype=torch.int32, device=cuda)
    rows = torch.randn(29, 4, d, generator=r).to(k.dtype).to(cuda)
    assert torch.equal(A.paged_prefill(rows, k, v, table, n, starts),
                       A.paged_prefill(rows, ks, vs, small, n, starts))


# ------------------------------------------------------ streams and graphs
def _step(seed, cuda, lengths, dtype=torch.float16, h=8, g=2, d=128, page=16, room=64):
    """The tensors of a decode step over sequences with pages for `room` more
    tokens."""
    k, v, table = paged(seed, [n + room for n in lengths], g, d, page, dtype, cuda, poison=False)
    q = randn(gen_of(seed), len(lengths), h, d, dtype=dtype, device=cuda)
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=cuda)


def test_calls_on_another_stream(cuda):
    note("streams")
    cases = [_step(s, cuda, [900 + 7 * s, 40, 3000]) for s in range(4)]
    want = [A.paged_decode(*c) for c in cases]
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(3):
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append((A.paged_decode(*c), A.paged_prefill(*c, starts)))
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(got):
        assert torch.equal(a, want[i % 4])
        torch.testing.assert_close(b, a, rtol=4e-3, atol=4e-3)


def test_two_graphs_replayed_in_turn(cuda):
    """Two captured steps with their own workspaces, replayed on growing
    lengths between eager calls: every replay equals the eager result."""
    note("graphs")
    cases = [_step(11, cuda, [700, 64, 2000]), _step(12, cuda, [5, 1500])]
    graphs = []
    for q, k, v, table, n in cases:
        b = len(n)
        starts = torch.arange(b + 1, dtype=torch.int32, device=cuda)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            A.paged_decode(q, k, v, table, n)
            A.paged_prefill(q, k, v, table, n, starts)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = (A.paged_decode(q, k, v, table, n),
                    A.paged_prefill(q, k, v, table, n, starts))
        graphs.append((graph, outs, starts))
    for step in range(4):
        for (q, k, v, table, n), (graph, outs, starts) in zip(cases, graphs):
            n += step
            graph.replay()
        for (q, k, v, table, n), (graph, outs, starts) in zip(cases, graphs):
            assert torch.equal(outs[0], A.paged_decode(q, k, v, table, n))
            assert torch.equal(outs[1], A.paged_prefill(q, k, v, table, n, starts))
        torch.cuda.synchronize()


# -------------------------------------------------------- the core, together
def _dense_causal(q, k, v):
    """Causal attention over whole sequences in binary64: [T, H, D] rows."""
    t, h, _ = q.shape
    k, v = (x.double().repeat_interleave(h // x.shape[1], 1) for x in (k, v))
    s = torch.einsum("qhd,khd->hqk", q.double(), k) * q.shape[2] ** -0.5
    s = s.masked_fill(torch.ones(t, t, dtype=torch.bool).triu(1), float("-inf"))
    return torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_core_over_prompt_chunks_and_steps(cuda, layout):
    """One layer's core over two sequences: prompts in chunks, then a mixed
    step, then decode with a padded row; every row against dense attention
    over the rotated rows in binary64."""
    note(f"core {layout}")
    h, g, d, page, dtype = 4, 2, 64, 8, torch.float16
    total = [57, 30]
    r = gen_of(21)
    rows = [randn(r, n, (h + 2 * g) * d, dtype=dtype, device=cuda) for n in total]
    parts = []
    for x in rows:
        q, k, v = x.split((h * d, g * d, g * d), 1)
        parts.append((q.reshape(-1, h, d), k.reshape(-1, g, d), v.reshape(-1, g, d)))
    freq = A.rotary_frequencies(d, scaling={"type": "yarn", "factor": 4.0,
                                            "original_max_position_embeddings": 32}, device=cuda)
    cache = A.PagedKVCache(3, 12, g, d, page_size=page, dtype=dtype, device=cuda)
    core = A.PagedAttentionCore(cache, freq, layout=layout)
    pages = [[4, 9, 1, 0, 7, 11, 2, 10], [3, 8, 5, 6]]
    got = [torch.empty(n, h * d, dtype=dtype, device=cuda) for n in total]

    def step(new, ends):
        state = A.AttentionState.build(pages, ends, new, page, device=cuda)
        cut = [[p[e - n:e] for p in part] for part, e, n in zip(parts, ends, new)]
        out = core(*[torch.cat([c[i] for c in cut]) for i in range(3)], 1, state)
        at = 0
        for b, (n, e) in enumerate(zip(new, ends)):
            got[b][e - n:e] = out[at:at + n]
            at += n

    step([40, 9], [40, 9])
    step([1, 20], [41, 29])          # one token next to a chunk: a mixed step
    step([15, 0], [56, 29])
    # The last tokens as a padded decode batch of three.
    state = A.AttentionState.build(pages, total, [1, 1], page, device=cuda)
    state = A.AttentionState(
        torch.cat((state.positions, state.positions[:1])),
        torch.cat((state.slots, state.slots.new_tensor([-1]))),
        torch.cat((state.page_table, state.page_table.new_full((1, 8), -1))),
        torch.cat((state.lengths, state.lengths.new_zeros(1))))
    last = [torch.cat([part[i][-1:] for part in parts] + [parts[0][i][:1]]) for i in range(3)]
    out = core(*last, 1, state)
    assert (out[2] == 0).all()
    for b in range(2):
        got[b][-1] = out[b]
        q, k, v = (x.cpu() for x in parts[b])
        at = torch.arange(total[b])
        turned = [O.rotary(x, at, freq.inv_freq, layout, freq.attention_factor)[0]
                  .to(dtype) for x in (q, k)]
        want = _dense_causal(*turned, v).reshape(total[b], h * d)
        # Rotated rows may round the other way (one step of 2^-10 of a value
        # of a few units): scores move by up to D^-0.5 sum |q| 2^-11 |k| ~ 1e-2.
        torch.testing.assert_close(got[b].double().cpu(), want, rtol=0.0, atol=2e-2)
    assert not cache.k[0].any() and not cache.k[2].any()      # the other layers


def test_runner_with_the_paged_core(cuda):
    """Prompt then captured decode steps through W8A8LlamaRunner: logits equal
    those of the whole prefix run as one prompt, within the W8A8 stack's
    sensitivity to the 16-bit rounding of the attention's rows."""
    note("runner")
    from nanopointllm_amd.runner import DecodeGraphBucket, W8A8LlamaRunner
    from workloads import llama_model

    heads, kv, hidden, page = 4, 2, 256, 16
    model = llama_model(cuda, layers=2, hidden=hidden, heads=heads, kv_heads=kv, intermediate=384,
                        vocab=512)
    freq = A.rotary_frequencies(hidden // heads, device=cuda)
    ids = torch.randint(0, 512, (1, 43), generator=gen_of(2)).to(cuda)

    def fresh():
        return A.PagedKVCache(2, 4, kv, hidden // heads, page_size=page, device=cuda)

    runner = W8A8LlamaRunner(model, A.PagedAttentionCore(fresh(), freq))
    embeds = runner.embed_tokens(ids)
    pages = [[2, 0, 3]]
    whole = runner(inputs_embeds=embeds,
                   attention_state=A.AttentionState.build(pages, [43], [43], page, device=cuda))
    for layer in runner.layers:
        layer.attention_core.cache = fresh()
    first = runner(inputs_embeds=embeds[:, :40],
                   attention_state=A.AttentionState.build(pages, [40], [40], page, device=cuda))
    state = A.AttentionState.build(pages, [41], [1], page, device=cuda)
    token = embeds[:, 40:41].clone()
    bucket = DecodeGraphBucket(cuda)
    static = bucket.capture(lambda: runner(inputs_embeds=token, attention_state=state))
    logits = [first]
    for i in range(40, 43):
        now = A.AttentionState.build(pages, [i + 1], [1], page, device=cuda)
        token.copy_(embeds[:, i:i + 1])
        for name in ("positions", "slots", "lengths"):
            getattr(state, name).copy_(getattr(now, name))
        bucket.replay()
        logits.append(static.clone())
        assert torch.equal(static, runner(inputs_embeds=token, attention_state=now))
    got = torch.cat(logits, 1).double()
    off = (got - whole.double()).norm() / whole.double().norm()
    assert off < 0.05, float(off)
