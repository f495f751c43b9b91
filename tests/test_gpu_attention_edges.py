"""Calls of the attention core that its documentation allows at the edges:
addresses, tables, padded rows, values that are not finite.

Tolerances as in test_gpu_attention.py where its check is used; others are
derived at the test."""
from __future__ import annotations

import pytest
import torch

from nanopointllm_amd import attention as A
from test_gpu_attention import DTYPES, check_attention, gen_of, note, paged, randn

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
