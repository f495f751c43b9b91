"""Calls of the attention core that its documentation allows at the edges:
addresses, tables, padded rows, values that are not finite.

Tolerances as in test_gpu_attention.py where its check is used; others are
derived at the test."""
from __future__ import annotations

import math

import pytest
import torch

from nanopointllm_amd import attention as A
from oracle import attention_oracle as O
from test_gpu_attention import (DTYPES, check_attention, check_rotary, gen_of, note, paged, randn,
                                smallest)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------ addresses and strides
@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_at_any_address_and_stride(cuda, dtype):
    """A contiguous q at an odd element, and one row or one head of a stride
    that is no multiple of 8, give the bits of an aligned copy."""
    note(f"misaligned queries {dtype}")
    h, g, d, lengths = 4, 2, 64, [300, 45]
    k, v, table = paged(3, lengths, g, d, 16, dtype, cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    flat = randn(gen_of(4), 3 * h * d + 8, dtype=dtype, device=cuda)
    wide = randn(gen_of(5), 3, h * d + 3, dtype=dtype, device=cuda)
    cases = [(flat[i:i + 2 * h * d].view(2, h, d), slice(0, 2)) for i in (0, 1, 3, 4)]
    cases += [(wide[:1, :h * d].view(1, h, d), slice(0, 1)),
              (wide[1:2, 1:h * d + 1].view(1, h, d), slice(1, 2)),
              (wide[:2, :h * d].view(2, h, d), slice(0, 2))]
    for q, at in cases:
        copy = torch.empty_like(q, memory_format=torch.contiguous_format)
        copy.copy_(q)
        out = A.paged_decode(q, k, v, table[at], n[at])
        assert torch.equal(out, A.paged_decode(copy, k, v, table[at], n[at]))
        check_attention(out, q, k, v, table[at], n[at], what="decode")
        starts = torch.arange(len(q) + 1, dtype=torch.int32, device=cuda)
        out = A.paged_prefill(q, k, v, table[at], n[at], starts)
        assert torch.equal(out, A.paged_prefill(copy, k, v, table[at], n[at], starts))
        check_attention(out, q, k, v, table[at], n[at], starts, what="prefill")


def test_one_page_one_head_and_one_row_of_unused_strides(cuda):
    """out and caches whose axes of one carry odd strides."""
    note("unused strides")
    d, page = 64, 16
    r = gen_of(6)
    wide = [randn(r, page * d + 8, dtype=torch.float16, device=cuda) for _ in range(2)]
    k, v = (w.as_strided((1, 1, page, d), (page * d + 3, 5, d, 1)) for w in wide)
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    n = torch.tensor([11], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    q = randn(r, 1, 1, d, dtype=torch.float16, device=cuda)
    into = torch.zeros(2 * d, dtype=torch.float16, device=cuda)
    out = into.as_strided((1, 1, d), (d + 1, 3, 1))
    want = A.paged_decode(q, k.contiguous(), v.contiguous(), table, n)
    assert torch.equal(A.paged_decode(q, k, v, table, n, out=out), want)
    check_attention(out, q, k, v, table, n)
    check_attention(A.paged_prefill(q, k, v, table, n, starts, out=out), q, k, v, table, n, starts)
    assert not into[d:].any()


# ------------------------------------------------- values that are not finite
INF, NAN = float("inf"), float("nan")


def place_of(table, b, key, page):
    return int(table[b, key // page]), key % page


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,length", [
    (2, 1, 64, 16, 1), (2, 2, 128, 16, 33), (4, 2, 80, 2, 200), (34, 2, 64, 16, 300),
    (4, 1, 256, 16, 300), (4, 2, 128, 16, 700), (2, 1, 96, 64, 5000), (6, 2, 256, 32, 2500)])
def test_decode_of_infinities_and_nans(cuda, h, g, d, page, length, dtype):
    """A visible value's infinity is the element's, whatever its weight; both
    signs, or a NaN, make it NaN; every other element and head keeps its bits,
    as does the sequence next to it.  Weights here are above 2^-40 of the
    largest, far from underflow."""
    note(f"decode non-finite {h} {g} {d} {page} {length} {dtype}")
    lengths, grp = [length, 77], h // g
    k, v, table = paged(length + d, lengths, g, d, page, dtype, cuda)
    q = randn(gen_of(d), 2, h, d, dtype=dtype, device=cuda)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    clean = A.paged_decode(q, k, v, table, n)
    check_attention(clean, q, k, v, table, n, what="clean")
    for key in sorted({0, length // 3, length - 1}):
        at, row = place_of(table, 0, key, page)
        bad = v.clone()
        for e, value in ((1, INF), (d // 2, -INF), (d - 1, NAN)):
            bad[at, 0, row, e] = value
        out = A.paged_decode(q, k, bad, table, n)
        assert (out[0, :grp, 1] == INF).all() and (out[0, :grp, d // 2] == -INF).all()
        assert torch.isnan(out[0, :grp, d - 1]).all()
        for e in (1, d // 2, d - 1):
            out[0, :grp, e] = clean[0, :grp, e]
        assert torch.equal(out, clean)
        if length > 1:
            at, row = place_of(table, 0, (key + length // 2) % length, page)
            bad[at, 0, row, 1] = -INF if (key + length // 2) % length != key else NAN
            assert torch.isnan(A.paged_decode(q, k, bad, table, n)[0, :grp, 1]).all()
        at, row = place_of(table, 0, key, page)
        bad = k.clone()
        bad[at, g - 1, row, 3] = NAN
        out = A.paged_decode(q, bad, v, table, n)
        assert torch.isnan(out[0, h - grp:]).all()
        out[0, h - grp:] = clean[0, h - grp:]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_keys(cuda, dtype):
    """An infinite key weighs nothing for a query that it scores -inf for, and
    makes the rows that it scores inf for NaN."""
    note(f"infinite keys {dtype}")
    h, d, length, key = 8, 64, 420, 200
    k, v, table = paged(2, [length], 1, d, 1, dtype, cuda)
    q = randn(gen_of(7), 1, h, d, dtype=dtype, device=cuda)
    q[..., 9] = torch.tensor([1.0, -1.0] * (h // 2)).to(dtype).to(cuda)
    n = torch.tensor([length], dtype=torch.int32, device=cuda)
    without = table.clone()
    without[0, key] = -1
    bad = k.clone()
    bad[int(table[0, key]), 0, 0, 9] = INF
    starts = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    for name, out in (("decode", A.paged_decode(q, bad, v, table, n)),
                      ("prefill", A.paged_prefill(q, bad, v, table, n, starts))):
        assert torch.isnan(out[0, ::2]).all(), name
        check_attention(out[:, 1::2], q[:, 1::2], k, v, without, n, what=name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,new,length", [
    (4, 2, 64, 16, 40, 40), (4, 2, 128, 16, 9, 3000), (4, 1, 64, 32, 7, 5000),
    (2, 1, 80, 8, 11, 2500), (2, 2, 256, 16, 6, 1800), (6, 2, 96, 4, 5, 1200),
    (2, 1, 24, 16, 20, 900), (3, 1, 192, 64, 30, 2100)])
def test_prefill_of_infinities_and_nans(cuda, h, g, d, page, new, length, dtype):
    """Rows recomputed key by key, whole tiles and tiles cut over the keys: an
    infinity that every row sees, a NaN among the newest tokens that only the
    later ones see, with and without a page that is unknown."""
    note(f"prefill non-finite {h} {g} {d} {page} {new} {length} {dtype}")
    grp = h // g
    k, v, table = paged(length + d, [length], g, d, page, dtype, cuda)
    q = randn(gen_of(d), new, h, d, dtype=dtype, device=cuda)
    n = torch.tensor([length], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, new], dtype=torch.int32, device=cuda)
    early, late = 2, length - new // 2          # keys; `late` is token new - new // 2
    for unknown in (False, True):
        if unknown:
            if length - new < 8 * page:
                continue
            table[0, (length // 2) // page] = -1
        clean = A.paged_prefill(q, k, v, table, n, starts)
        check_attention(clean, q, k, v, table, n, starts, what=f"clean {unknown}")
        bad = v.clone()
        at, row = place_of(table, 0, early, page)
        bad[at, 0, row, 1] = INF
        at, row = place_of(table, 0, late, page)
        bad[at, 0, row, 5] = NAN
        bad[at, 0, row, d - 1] = -INF
        out = A.paged_prefill(q, k, bad, table, n, starts)
        first = new - new // 2
        sees_early = 0 if new < length else early
        assert (out[sees_early:, :grp, 1] == INF).all()
        assert torch.isnan(out[first:, :grp, 5]).all()
        assert (out[first:, :grp, d - 1] == -INF).all()
        out[sees_early:, :grp, 1] = clean[sees_early:, :grp, 1]
        out[first:, :grp, 5] = clean[first:, :grp, 5]
        out[first:, :grp, d - 1] = clean[first:, :grp, d - 1]
        check_attention(out, q, k, v, table, n, starts, what=f"values {unknown}")
        assert torch.equal(out[:, grp:], clean[:, grp:])
        bad = k.clone()
        bad[at, g - 1, row, 3] = NAN
        out = A.paged_prefill(q, bad, v, table, n, starts)
        assert torch.isnan(out[first:, h - grp:]).all()
        out[first:, h - grp:] = clean[first:, h - grp:]
        check_attention(out, q, k, v, table, n, starts, what=f"key {unknown}")


def test_large_values_next_to_a_masked_nan(cuda):
    """bfloat16 values near the type's largest: 40 of them weigh alike, their
    mean is one of them, and a NaN that only the last row sees changes no row
    before it.  (Sums of 40 products of 2^-8 and 2e38 stay finite.)"""
    note("large values")
    n, d = 40, 64
    k, v, table = paged(1, [n], 1, d, 16, torch.bfloat16, cuda, poison=False)
    v.fill_(2e38)
    q = torch.zeros(n, 2, d, dtype=torch.bfloat16, device=cuda)
    lengths = torch.tensor([n], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    want = v[0, 0, 0, 0]
    assert (A.paged_prefill(q, k, v, table, lengths, starts) == want).all()
    assert (A.paged_decode(q[:1], k, v, table, lengths) == want).all()
    at, row = place_of(table, 0, n - 1, 16)
    v[at, 0, row] = NAN
    out = A.paged_prefill(q, k, v, table, lengths, starts)
    assert (out[:-1] == want).all() and torch.isnan(out[-1]).all()


# -------------------------------------------------- weights, and what sums them
@pytest.mark.parametrize("below", [10, 14, 20, 23, 26])
@pytest.mark.parametrize("dtype", DTYPES)
def test_numerator_and_denominator_hold_the_same_weights(cuda, dtype, below):
    """One key ahead of 20 thousand by about 2^below each, all of one value v:
    the result is v.  The weights lie just off a step of the 16-bit type, so
    that a denominator of unrounded ones would be off by half a step, and past
    2^-14 binary16 holds them in fewer bits or drops them.

    v has the mantissa next to 2, where half a step is e / 2 of it (e =
    finfo.eps / 2).  Sums: a piece has at most 20 units of 32 keys (32 pieces of
    626), so its denominator is at most 20 x 8 + 10 additions deep and its
    numerator 40 matrix instructions of at most 17, and a wavefront of a decode
    workgroup takes no more; 1100 u with the join's.  Decode's weights lose
    at most 2^-15 (bfloat16) or 2^-21, and 2^-24 of a scale of at least 2^7:
    n 2^-31.  All of it stays below e / 2, so the result is v exactly."""
    note(f"same weights {dtype} {below}")
    n, d, page = 20001, 64, 64
    e, u = torch.finfo(dtype).eps / 2, 2.0 ** -24
    lost = 2.0 ** -21 + n * 2.0 ** -31 if dtype == torch.float16 else 2.0 ** -15
    assert 1100 * u + lost < e / 2
    k, v, table = paged(31, [n], 1, d, page, dtype, cuda, poison=False)
    v.fill_(2.0 - torch.finfo(dtype).eps)
    k.zero_()
    k[table[0, 0].long(), 0, 0, 0] = 1.0
    q = torch.zeros(1, 2, d, dtype=dtype, device=cuda)
    q[..., 0] = 16.0
    scale = (below - math.log2(1.0 + 0.96 * e)) * math.log(2.0) / 16.0
    lengths = torch.tensor([n], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    for name, out in (("decode", A.paged_decode(q, k, v, table, lengths, scale=scale)),
                      ("prefill", A.paged_prefill(q, k, v, table, lengths, starts, scale=scale))):
        assert (out == v[0, 0, 0, 0]).all(), f"{name} {out.flatten()[0]} {v[0, 0, 0, 0]}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,lengths", [(8, 2, 128, [64, 33, 200]), (4, 4, 64, [600, 64]),
                                           (4, 1, 256, [90, 400])])
def test_decode_weights_keep_two_parts(cuda, h, g, d, lengths, dtype):
    """Decode's weights enter the product with more bits than the 16-bit type
    holds.  One element of a query is not zero, so a score is one product: with
    u = 2^-24, r = 2 (13 u |score| + 16 u) for both sums' weights, 2 n u for
    sums over n keys, 2^-15 (bfloat16: 8 + 8 bits cut off) or 2^-21 + n 2^-31
    (binary16: 11 + 11 bits, steps of 2^-24 at a scale of 2^7) for the two
    parts; e |out| for the result's rounding.  The definition with weights cut
    to the type misses this bound."""
    note(f"two parts {h} {g} {d} {lengths} {dtype}")
    k, v, table = paged(d, lengths, g, d, 16, dtype, cuda)
    q = torch.zeros(len(lengths), h, d, dtype=dtype, device=cuda)
    q[..., 2] = randn(gen_of(1), len(lengths), h, dtype=dtype, device=cuda, std=1.7 * d ** 0.5)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    want, size, dots = O.attention(q, k, v, table, n)
    u, e, most = 2.0 ** -24, torch.finfo(dtype).eps / 2, max(lengths)
    parts = 2.0 ** -21 + most * 2.0 ** -31 if dtype == torch.float16 else 2.0 ** -15
    tol = (2 * (13 * u * dots + 16 * u) + 2 * most * u + parts)[..., None] * size
    tol = tol + e * want.abs() + smallest(dtype)
    out = A.paged_decode(q, k, v, table, n).double().cpu()
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() - tol).max())
    # One part: the weights of the definition cut to the type's bits.
    bits, missed = (11 if dtype == torch.float16 else 8), 0
    for b, total in enumerate(lengths):
        for i in range(h):
            keys, _ = O.keys_of(k.cpu(), table.cpu(), b, i // (h // g), total)
            values, _ = O.keys_of(v.cpu(), table.cpu(), b, i // (h // g), total)
            s = keys @ q[b, i].double().cpu() * d ** -0.5
            p = torch.exp(s - s.max())
            m, x = torch.frexp(p)
            cut = torch.ldexp(torch.floor(m * 2.0 ** bits) * 2.0 ** -bits, x)
            missed += int((((cut @ values) / p.sum() - want[b, i]).abs() > tol[b, i]).sum())
    assert missed > 0


# ------------------------------------------------------- tables, strides, rows
@pytest.mark.parametrize("dtype", DTYPES)
def test_tables_wider_than_any_sequence(cuda, dtype):
    """A captured step's table has room to grow: 4096 keys and more where the
    sequences have at most 1590, the entries behind them unknown."""
    note(f"wide tables {dtype}")
    h, g, d, page = 8, 8, 64, 16
    lengths = [1590, 0, 1, 636, 1000, 31, 32, 1500] * 4
    k, v, table = paged(8, lengths, g, d, page, dtype, cuda)
    wide = torch.full((len(lengths), 640), 2 ** 31 - 1, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table
    q = randn(gen_of(9), len(lengths), h, d, dtype=dtype, device=cuda, std=1.7)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    check_attention(A.paged_decode(q, k, v, wide, n), q, k, v, table, n, what="decode")
    new = [9, 0, 1, 40, 130, 31, 1, 5]
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda)
    q = randn(gen_of(9), sum(new), h, d, dtype=dtype, device=cuda, std=1.7)
    check_attention(A.paged_prefill(q, k, v, wide[:8], n[:8], starts), q, k, v, table[:8], n[:8],
                    starts, what="prefill")


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_the_checks_make_contiguous(cuda, dtype):
    """Rows with scattered elements, a transposed table, lengths, positions and
    slots of every second place: the same bits as their copies, on values that
    all differ."""
    note(f"made contiguous {dtype}")
    h, g, d, page, lengths = 4, 2, 64, 16, [40, 300, 7]
    k, v, table = paged(12, lengths, g, d, page, dtype, cuda)
    r = gen_of(13)
    q = randn(r, 3, h, d, dtype=dtype, device=cuda)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)

    def every_second(x):
        wide = torch.full((2 * len(x),), 10 ** 6, dtype=x.dtype, device=cuda)
        wide[::2] = x
        return wide[::2]

    columns = table.T.contiguous().T
    want = A.paged_decode(q, k, v, table, n)
    check_attention(want, q, k, v, table, n, what="decode")
    assert torch.equal(A.paged_decode(turned, k, v, columns, every_second(n)), want)
    starts = torch.tensor([0, 1, 3, 3], dtype=torch.int32, device=cuda)
    want = A.paged_prefill(q, k, v, table, n, starts)
    check_attention(want, q, k, v, table, n, starts, what="prefill")
    assert torch.equal(A.paged_prefill(turned, k, v, columns, every_second(n),
                                       every_second(starts)), want)
    kv = [randn(r, 3, g, d, dtype=dtype, device=cuda) for _ in range(2)]
    positions, slots = (torch.tensor(x, device=cuda) for x in ([5, 900, 77], [3, 49, 18]))
    freq = A.rotary_frequencies(d, device=cuda).inv_freq
    got = []
    for rows, other, at, to, f in (
            (q, kv, positions, slots, freq),
            (turned, [x.transpose(1, 2).contiguous().transpose(1, 2) for x in kv],
             every_second(positions), every_second(slots), every_second(freq))):
        caches = torch.zeros(2, 4, g, page, d, dtype=dtype, device=cuda)
        out = A.rotary_store(rows, *other, at, to, f, caches[0], caches[1])
        got.append((out, caches, A.rotary(rows, at, f)))
    check_rotary(got[0][0], q, positions, freq, "half", 1.0)
    for a, b in zip(*got):
        assert a.any() and torch.equal(a, b)


@pytest.mark.parametrize("h,g,d,page,before,new,lengths,behind", [
    (4, 2, 64, 16, 0, [5, 20], [5, 90], 1), (8, 2, 128, 16, 3, [17, 0, 40], [30, 9, 40], 2100),
    (4, 4, 64, 16, 129, [128], [128], 0), (4, 1, 80, 8, 1, [3], [5000], 7),
    (2, 1, 24, 4, 2, [0, 0], [9, 0], 30), (3, 3, 256, 32, 0, [64, 64], [64, 200], 640),
    (8, 1, 64, 16, 0, [1 + i % 3 for i in range(70)], [9 + i for i in range(70)], 300)])
def test_padded_prompt_rows_are_zeros(cuda, h, g, d, page, before, new, lengths, behind):
    """Rows of no sequence, before the first one's and behind the last one's, in
    a tensor that the call allocates (of memory that held NaN), and nothing of
    them in a given one."""
    note(f"padded rows {h} {g} {d} {page} {before} {new[:4]} {behind}")
    for dtype in DTYPES:
        k, v, table = paged(h + d, lengths, g, d, page, dtype, cuda)
        starts = torch.tensor([before] + new).cumsum(0).to(torch.int32).to(cuda)
        t = before + sum(new) + behind
        q = randn(gen_of(t), t, h, d, dtype=dtype, device=cuda)
        n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        for _ in range(2):
            junk = [torch.full((t, h, d), NAN, dtype=dtype, device=cuda) for _ in range(8)]
            places = {x.data_ptr() for x in junk}
            del junk
            out = A.paged_prefill(q, k, v, table, n, starts)
            assert out.data_ptr() in places  # the NaNs' memory, or this shows nothing
            assert (out[:before] == 0).all() and (out[t - behind:] == 0).all()
            check_attention(out, q, k, v, table, n, starts)
        into = torch.full((t, h, d), 7.0, dtype=dtype, device=cuda)
        A.paged_prefill(q, k, v, table, n, starts, out=into)
        assert (into[:before] == 7.0).all() and (into[t - behind:] == 7.0).all()
        assert torch.equal(into[before:t - behind], out[before:t - behind])
    none = A.paged_prefill(q, k, v, table[:0], n[:0], starts[:1])
    assert none.shape == q.shape and not none.any()


def test_core_of_padded_steps(cuda):
    """Padded rows behind a step's chunks come out as zeros, with and without
    decode rows before them, whatever the memory held."""
    note("core padded")
    h, g, d, page, dtype = 4, 2, 64, 16, torch.float16
    cache = A.PagedKVCache(1, 8, g, d, page_size=page, dtype=dtype, device=cuda)
    core = A.PagedAttentionCore(cache, A.rotary_frequencies(d, device=cuda))
    r = gen_of(5)
    for pages, lengths, new, pad in (([[0, 1], [2]], [20, 9], [20, 9], 5),
                                     ([[0, 1], [2]], [21, 12], [1, 3], 6),
                                     ([[0, 1]], [22], [1], 0)):
        state = A.AttentionState.build(pages, lengths, new, page, device=cuda)
        rows = sum(new)
        x = [randn(r, rows + pad, n, d, dtype=dtype, device=cuda) for n in (h, g, g)]
        want = core(*[y[:rows] for y in x], 0, state)
        state.positions = torch.cat((state.positions, state.positions.new_zeros(pad)))
        state.slots = torch.cat((state.slots, state.slots.new_full((pad,), -1)))
        junk = [torch.full((rows + pad, h, d), NAN, dtype=dtype, device=cuda) for _ in range(8)]
        del junk
        out = core(*x, 0, state)
        assert out.shape == (rows + pad, h * d)
        assert torch.equal(out[:rows], want) and not out[rows:].any()


def test_core_of_empty_steps(cuda):
    """A step of no row is one, with sequences or without."""
    note("core empty")
    h, g, d, page = 4, 2, 64, 16
    cache = A.PagedKVCache(1, 8, g, d, page_size=page, device=cuda)
    core = A.PagedAttentionCore(cache, A.rotary_frequencies(d, device=cuda))
    q, k, v = (torch.empty(0, n, d, dtype=torch.float16, device=cuda) for n in (h, g, g))
    for pages, lengths, new in (([], [], []), ([[0, 1]], [22], [0])):
        state = A.AttentionState.build(pages, lengths, new, page, device=cuda)
        assert core(q, k, v, 0, state).shape == (0, h * d)


@pytest.mark.parametrize("h,g,d,page,new,lengths", [
    (8, 2, 128, 16, [4], [510]), (8, 2, 128, 16, [4], [512]), (8, 2, 128, 16, [4], [513]),
    (8, 8, 64, 16, [150, 4], [650, 604]), (4, 4, 96, 32, [520], [520]),
    (4, 1, 256, 16, [3, 0, 40], [700, 3, 41]), (3, 1, 80, 8, [760], [760])])
def test_prompts_cut_into_a_few_pieces(cuda, h, g, d, page, new, lengths):
    note(f"few pieces {h} {g} {d} {new} {lengths}")
    for dtype in DTYPES:
        k, v, table = paged(h + d, lengths, g, d, page, dtype, cuda)
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda)
        q = randn(gen_of(d), sum(new), h, d, dtype=dtype, device=cuda, std=1.7)
        n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        check_attention(A.paged_prefill(q, k, v, table, n, starts), q, k, v, table, n, starts)
