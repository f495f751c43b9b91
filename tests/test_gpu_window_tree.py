"""Attention with windows and sinks, trees of drafted tokens and accepted paths
on the GPU against their definitions in binary64 (oracle/drafts_oracle.py).

Tolerances as derived in test_gpu_attention.py: scores, probabilities and sums
are formed by the same arithmetic, over the keys that a row sees.  Keys and pages
that no row sees hold NaN and infinities.
"""
from __future__ import annotations

import math

import pytest
import torch

import test_gpu_attention as G
from nanopointllm_amd import attention as A
from nanopointllm_amd.runner import DecodeGraphBucket
from oracle import drafts_oracle as O

pytestmark = pytest.mark.gpu

U, DTYPES = G.U, G.DTYPES


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def check(out, q, k, v, table, lengths, starts, sight, what="", scale=None):
    want, size, dots = O.attention(q, k, v, table, lengths, starts, sight, scale)
    owned = ~torch.isnan(want)
    d, e, n = q.shape[2], G.half_step(q.dtype), int(lengths.max()) if lengths.numel() else 0
    finite = v.float().cpu()
    most = float(finite[torch.isfinite(finite)].abs().max()) if finite.numel() else 0.0
    rel = 2 * ((d + 12) * U * dots + 16 * U) + 2 * e + 2 * n * U
    tol = rel[..., None] * size + n * 2.0 ** -25 * most * (size > 0) + e * want.abs() \
        + G.smallest(q.dtype)
    err = (out.double().cpu() - want).abs()
    bad = owned & ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} off, worst {err[bad].max()} "
                           f"at {bad.nonzero()[0].tolist()}")
    return owned


def poison(k, v, table, lengths, seen_by_any, page):
    """NaN and infinities in every row of a sequence that no query sees, and page
    numbers that do not exist where a page holds no seen key."""
    pages = k.shape[0]
    for b, n in enumerate(lengths):
        seen = seen_by_any(b)
        for at in range(-(-n // page)):
            rows = seen[at * page:(at + 1) * page]
            e = int(table[b, at])
            hide = torch.zeros(page, dtype=torch.bool)
            hide[:len(rows)] = ~rows
            k[e, :, hide.to(k.device)] = math.nan
            v[e, :, hide.to(k.device)] = math.inf if at % 2 else math.nan
            if not rows.any():
                table[b, at] = (-1, pages + 7, 2 ** 31 - 1)[at % 3]


DECODE = [
    # heads, kv heads, dim, page, window, sinks, lengths
    (32, 8, 128, 16, 100, 4, [1, 2, 99, 100, 101, 104, 105, 131, 132, 133, 700, 0]),
    (4, 4, 64, 32, 1, 0, [1, 2, 31, 32, 33, 34, 35, 64, 65, 200]),
    (4, 4, 64, 8, 1, 1, [1, 2, 31, 32, 33, 34, 66, 67, 300]),
    (8, 2, 80, 8, 33, 40, [30, 70, 73, 74, 75, 106, 500]),
    (6, 2, 96, 1, 7, 3, [5, 9, 10, 11, 40]), (6, 2, 96, 2, 2, 33, [5, 36, 64, 65, 66, 67]),
    (16, 1, 128, 64, 500, 0, [3000, 600]), (40, 2, 8, 16, 64, 64, [50, 128, 129, 500]),
    (8, 2, 256, 16, 200, 10, [333, 64]), (28, 4, 128, 128, 10000, 4, [700, 3]),
    (8, 1, 128, 16, 2900, 4, [9000, 2901]), (2, 2, 64, 4, 20, 0, [1000, 21, 22, 23, 19]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,window,sinks,lengths", DECODE)
def test_window_decode_against_the_definition(cuda, h, g, d, page, window, sinks, lengths, dtype):
    G.note(f"window decode {h} {g} {d} {page} {window} {sinks} {lengths} {dtype}")
    k, v, table = G.paged(h + d, lengths, g, d, page, dtype, cuda)
    q = G.randn(G.gen_of(d), len(lengths), h, d, dtype=dtype, device=cuda, std=1.7)
    n = i32(lengths, cuda)

    def sight(b, rows, total):
        return O.window_sight(rows, total, window, sinks)

    poison(k, v, table, lengths, lambda b: sight(b, 1, lengths[b])[0] if lengths[b] else
           torch.zeros(0, dtype=torch.bool), page)
    starts = torch.arange(len(lengths) + 1)
    out = A.paged_decode(q, k, v, table, n, window=window, sinks=sinks)
    check(out, q, k, v, table, n, starts, sight)
    assert (out[n <= 0] == 0).all()
    assert torch.equal(out, A.paged_decode(q, k, v, table, n, window=window, sinks=sinks))
    # Heads inside tokens, rows and results inside larger tensors.
    k2, v2 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    rows = torch.zeros(len(lengths), h + 2, d, dtype=dtype, device=cuda)
    rows[:, 1:-1] = q
    into = torch.full((len(lengths), h + 1, d), 7.0, dtype=dtype, device=cuda)
    A.paged_decode(rows[:, 1:-1], k2, v2, table, n, window=window, sinks=sinks, out=into[:, :h])
    assert torch.equal(into[:, :h], out) and (into[:, h] == 7.0).all()


@pytest.mark.parametrize("batch,h,g,d,page,longest,window", [
    (130, 2, 2, 128, 16, 4000, 200), (260, 2, 2, 64, 64, 300, 50), (37, 8, 8, 128, 16, 5000, 1500),
    (70, 34, 2, 96, 8, 500, 17)])
def test_window_decode_of_large_batches(cuda, batch, h, g, d, page, longest, window):
    G.note(f"window decode batch {batch} {h} {g} {d} {page} {longest} {window}")
    r = G.gen_of(batch)
    lengths = torch.randint(0, longest, (batch,), generator=r).tolist()
    lengths[0], lengths[1], lengths[2] = longest, 0, 1
    dtype = DTYPES[batch % 2]
    k, v, table = G.paged(batch + d, lengths, g, d, page, dtype, cuda)
    q = G.randn(r, batch, h, d, dtype=dtype, device=cuda, std=1.7)
    n = i32(lengths, cuda)
    out = A.paged_decode(q, k, v, table, n, window=window, sinks=4)
    check(out, q, k, v, table, n, torch.arange(batch + 1),
          lambda b, rows, total: O.window_sight(rows, total, window, 4))


PREFILL = [
    # heads, kv heads, dim, page, window, sinks, new tokens, lengths
    (4, 4, 128, 16, 64, 4, [560], [560]),
    (8, 2, 128, 16, 33, 2, [1, 2, 31, 32, 33, 64, 0, 65, 127, 128, 129], None),
    (4, 1, 64, 32, 40, 50, [5, 100, 0, 3], [300, 100, 50, 90]),
    (7, 1, 80, 8, 1, 0, [40, 130], [41, 400]), (2, 2, 96, 1, 3, 1, [17, 33], [17, 80]),
    (4, 2, 256, 16, 50, 5, [70, 9], [70, 350]), (3, 3, 8, 4, 6, 6, [21], [30]),
    (2, 1, 192, 64, 100, 0, [140], [700]),
    # fewer keys than rows: the first see none
    (4, 2, 128, 16, 8, 2, [10, 50, 4], [3, 0, 4]), (2, 2, 64, 16, 30, 3, [200], [70]),
    # a few rows far behind, whose window is cut over its length
    (8, 2, 128, 64, 2000, 4, [3], [5000]), (4, 4, 64, 16, 1500, 70, [40, 1], [3333, 2000]),
    (2, 1, 128, 16, 1000, 1, [300], [4400]),
    # sinks and windows that meet, overlap, and leave one key between
    (2, 2, 64, 16, 96, 32, [64], [192]), (2, 2, 64, 16, 97, 33, [64], [192]),
    (2, 2, 64, 8, 60, 69, [1, 2], [130, 131]), (2, 2, 64, 8, 32, 96, [70], [200]),
    (16, 2, 96, 32, 5000, 4, [200, 0, 77, 31, 130], [200, 40, 500, 31, 300]),
    (200, 1, 64, 16, 5, 2, [3, 0, 70], [40, 9, 70]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,window,sinks,new,lengths", PREFILL)
def test_window_prefill_against_the_definition(cuda, h, g, d, page, window, sinks, new, lengths,
                                               dtype):
    G.note(f"window prefill {h} {g} {d} {page} {window} {sinks} {new} {lengths} {dtype}")
    lengths = new if lengths is None else lengths
    k, v, table = G.paged(h + d + len(new), lengths, g, d, page, dtype, cuda)

    def sight(b, rows, total):
        return O.window_sight(rows, total, window, sinks)

    poison(k, v, table, lengths, lambda b: sight(b, new[b], lengths[b]).any(0), page)
    before, behind = 3, 5
    starts = torch.tensor([before] + new).cumsum(0).to(torch.int32).to(cuda)
    rows = before + sum(new) + behind
    q = G.randn(G.gen_of(d + h), rows, h, d, dtype=dtype, device=cuda, std=1.7)
    n = i32(lengths, cuda)
    into = torch.full((rows, h, d), 7.0, dtype=dtype, device=cuda)
    out = A.paged_prefill(q, k, v, table, n, starts, window=window, sinks=sinks, out=into)
    assert out is into
    check(out, q, k, v, table, n, starts, sight)
    assert (out[:before] == 7.0).all() and (out[rows - behind:] == 7.0).all()
    fresh = A.paged_prefill(q, k, v, table, n, starts, window=window, sinks=sinks)
    assert torch.equal(fresh[before:rows - behind], out[before:rows - behind])
    assert (fresh[:before] == 0).all() and (fresh[rows - behind:] == 0).all()
    k2, v2 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    again = A.paged_prefill(q, k2, v2, table, n, starts, window=window, sinks=sinks)
    assert torch.equal(again, fresh)


def test_a_window_past_the_table_is_none(cuda):
    """The bits of the calls without one; sinks add nothing then."""
    G.note("wide windows")
    lengths = [300, 77]
    k, v, table = G.paged(4, lengths, 2, 64, 16, torch.float16, cuda)
    n = i32(lengths, cuda)
    most = table.shape[1] * 16
    q = G.randn(G.gen_of(1), 2, 4, 64, dtype=torch.float16, device=cuda)
    for window in (most, most + 1, 2 ** 40):
        assert torch.equal(A.paged_decode(q, k, v, table, n),
                           A.paged_decode(q, k, v, table, n, window=window, sinks=9))
    q = G.randn(G.gen_of(2), 60, 4, 64, dtype=torch.float16, device=cuda)
    starts = i32([0, 50, 60], cuda)
    assert torch.equal(A.paged_prefill(q, k, v, table, n, starts),
                       A.paged_prefill(q, k, v, table, n, starts, window=most))


def random_trees(seed, sizes, back=6):
    g = G.gen_of(seed)
    trees = []
    for n in sizes:
        step = torch.randint(1, back + 1, (n,), generator=g).tolist()
        trees.append([max(-1, i - s) if i else -1 for i, s in enumerate(step)])
    return trees


TREES = [
    # heads, kv heads, dim, page, drafted tokens, lengths with them
    (32, 32, 128, 16, [26], [627]), (8, 2, 128, 16, [1, 2, 31, 32, 33, 0, 63, 64, 65], None),
    (4, 1, 64, 32, [5, 100, 0, 3], [300, 100, 50, 9]), (7, 1, 80, 8, [40, 130], [41, 400]),
    (2, 2, 96, 1, [17, 33], [17, 80]), (4, 2, 256, 16, [70, 9], [70, 150]),
    (3, 3, 8, 4, [21], [30]), (2, 1, 192, 64, [140], [200]),
    # more drafted rows than keys: the first have none of their own
    (4, 2, 128, 16, [10, 50, 4], [3, 0, 4]),
    # few rows behind a long cache, cut over it
    (8, 2, 128, 64, [3], [5000]), (4, 4, 64, 16, [40, 1], [3333, 2000]),
    (16, 16, 128, 16, [16, 7, 12], [1500, 1111, 64]), (32, 4, 64, 16, [2, 2, 1], [700, 33, 1]),
    (8, 1, 64, 16, [1 + 7 * i % 41 for i in range(70)], [50 + 11 * i % 60 for i in range(70)]),
    (200, 1, 64, 16, [3, 0, 70], [40, 9, 70]), (2, 2, 64, 8, [300], [305]),
    # 33 to 64 rows, cut and whole, narrow heads, pages copied through registers
    (3, 3, 64, 16, [40, 64, 33], [2500, 700, 40]), (4, 2, 80, 8, [32, 20], [3000, 1501]),
    (2, 2, 128, 4, [50, 64, 7], [1000, 65, 640]), (2, 2, 96, 2, [9, 14], [600, 700]),
    (64, 64, 64, 32, [36, 64, 40, 50], [500, 64, 333, 600]),
    # more sequences than a wavefront has lanes, cut and whole
    (2, 2, 64, 16, [i % 4 for i in range(90)], [i % 4 + 13 * i % 700 for i in range(90)]),
    (4, 4, 128, 64, [1 + i % 9 for i in range(130)], [9 + 7 * i % 300 for i in range(130)]),
    (4, 2, 128, 16, [5, 17, 1], [20000, 9000, 70]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,g,d,page,new,lengths", TREES)
def test_trees_against_the_definition(cuda, h, g, d, page, new, lengths, dtype):
    G.note(f"tree {h} {g} {d} {page} {new} {lengths} {dtype}")
    lengths = new if lengths is None else lengths
    k, v, table = G.paged(h + d + len(new), lengths, g, d, page, dtype, cuda)
    trees = random_trees(h + len(new), new)
    masks = A.tree_masks(trees, device=cuda)
    before, behind = 2, 3
    starts = torch.tensor([before] + new).cumsum(0).to(torch.int32).to(cuda)
    rows = before + sum(new) + behind
    padded = torch.full((rows, masks.shape[1]), -1, dtype=torch.int64, device=cuda)
    padded[before:rows - behind] = masks
    q = G.randn(G.gen_of(d + h), rows, h, d, dtype=dtype, device=cuda, std=1.7)
    n = i32(lengths, cuda)

    def sight(b, count, total):
        return O.tree_sight(padded[int(starts[b]):int(starts[b + 1])].cpu(), total)

    into = torch.full((rows, h, d), 7.0, dtype=dtype, device=cuda)
    out = A.paged_tree(q, k, v, table, n, starts, padded, out=into)
    assert out is into
    check(out, q, k, v, table, n, starts, sight)
    assert (out[:before] == 7.0).all() and (out[rows - behind:] == 7.0).all()
    fresh = A.paged_tree(q, k, v, table, n, starts, padded)
    assert torch.equal(fresh[before:rows - behind], out[before:rows - behind])
    assert (fresh[:before] == 0).all() and (fresh[rows - behind:] == 0).all()
    # Masks inside a wider tensor, a cache in the other order.
    wide = torch.full((rows, masks.shape[1] + 2), -1, dtype=torch.int64, device=cuda)
    wide[:, :-2] = padded
    k2, v2 = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    assert torch.equal(A.paged_tree(q, k2, v2, table, n, starts, wide[:, :-2]), fresh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cached", [0, 1, 45, 700])
def test_masks_of_any_bits(cuda, cached, dtype):
    """Random bits, rows that see nothing but the cache, only later tokens, or
    (without a cache) nothing at all; too few words; NaN where nobody looks."""
    G.note(f"tree masks {cached} {dtype}")
    h, g, d, page, n = 4, 2, 64, 16, 75
    total = cached + n
    k, v, table = G.paged(3 + cached, [total], g, d, page, dtype, cuda)
    r = G.gen_of(cached)
    masks = torch.randint(-2 ** 62, 2 ** 62, (n, 2), generator=r, dtype=torch.int64)
    masks[3] = 0
    masks[4] = torch.tensor([-2 ** 63, 0])
    masks[:, 0] &= ~(1 << 20)          # nobody sees drafted tokens 20 and 70
    masks[:, 1] &= ~(1 << 6)
    for j in (20, 70):
        e = int(table[0, (cached + j) // page])
        k[e, :, (cached + j) % page] = math.nan
        v[e, :, (cached + j) % page] = math.inf
    q = G.randn(r, n, h, d, dtype=dtype, device=cuda, std=1.5)
    lengths, starts = i32([total], cuda), i32([0, n], cuda)
    for words in (2, 1, 0):
        m = masks[:, :words].contiguous()
        out = A.paged_tree(q, k, v, table, lengths, starts, m.to(cuda))
        check(out, q, k, v, table, lengths, starts, lambda b, c, t: O.tree_sight(m, t))
        if cached == 0:
            assert (out[3] == 0).all()


def test_values_that_only_some_rows_see(cuda):
    """A NaN and an infinity among the drafted tokens reach the rows that see
    them, and no others; so do those of a window."""
    G.note("special values")
    h = g = 2
    d, page, cached, n = 64, 16, 100, 20
    for dtype in DTYPES:
        k, v, table = G.paged(8, [cached + n], g, d, page, dtype, cuda)
        e = int(table[0, (cached + 5) // page])
        v[e, :, (cached + 5) % page, 3] = math.inf
        v[e, :, (cached + 5) % page, 7] = math.nan
        q = G.randn(G.gen_of(2), n, h, d, dtype=dtype, device=cuda)
        lengths, starts = i32([cached + n], cuda), i32([0, n], cuda)
        tree = [-1, 0, 1, 2, 3] + [4 if i % 2 else i - 1 for i in range(5, n)]
        sees = O.tree_sight(A.tree_masks([tree], device="cpu"), cached + n)[:, cached + 5]
        out = A.paged_tree(q, k, v, table, lengths, starts, A.tree_masks([tree], device=cuda))
        assert 0 < int(sees.sum()) < n
        assert (out[sees.to(cuda)][..., 3] == math.inf).all()
        assert out[sees.to(cuda)][..., 7].isnan().all()
        assert torch.isfinite(out[~sees.to(cuda)]).all()
        keep = [i for i in range(d) if i not in (3, 7)]
        assert torch.isfinite(out[..., keep]).all()
        sees = O.window_sight(n, cached + n, 6, 2)[:, cached + 5]
        out = A.paged_prefill(q, k, v, table, lengths, starts, window=6, sinks=2)
        assert torch.equal(out[..., 3].isinf().all(1).cpu(), sees)
        assert torch.equal(out[..., 7].isnan().all(1).cpu(), sees)
        assert torch.isfinite(out[..., keep]).all()
        one = A.paged_decode(q[-1:], k, v, table, lengths, window=n - 5, sinks=1)
        assert (one[..., 3] == math.inf).all() and one[..., 7].isnan().all()
        one = A.paged_decode(q[-1:], k, v, table, lengths, window=n - 6, sinks=1)
        assert torch.isfinite(one).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers,g,d,page,lengths,steps", [
    (3, 2, 128, 16, [0, 5, 15, 16, 17, 100], 5), (1, 1, 8, 1, [3, 0], 3), (2, 5, 80, 8, [7], 1),
    (4, 8, 64, 64, [63, 64, 1], 19), (2, 3, 256, 4, [2, 9, 30], 8)])
def test_accepted_paths(cuda, layers, g, d, page, lengths, steps, dtype):
    """Every layer's rows, to the bit; the rest of the cache keeps its own."""
    G.note(f"accept {layers} {g} {d} {page} {lengths} {steps} {dtype}")
    r = G.gen_of(steps + d)
    drafted = steps + 11
    k, v, table = G.paged(d, [n + drafted for n in lengths], g, d, page, dtype, cuda, spare=1)
    pages = k.shape[0]
    path = torch.full((len(lengths), steps), -1, dtype=torch.int32)
    for b in range(len(lengths)):
        n = steps if b == 0 else int(torch.randint(0, steps + 1, (1,), generator=r))
        path[b, :n] = torch.randperm(drafted, generator=r)[:n].sort()[0].to(torch.int32)
    n = i32(lengths, cuda)
    store = torch.randn(layers, 2, pages, g, page, d, generator=r).to(dtype).to(cuda)
    want = [O.accept(store[:, i], table, n.cpu(), path) for i in range(2)]
    kept = store.clone()
    A.paged_accept(kept[:, 0], kept[:, 1], table, n, path.to(cuda))
    assert torch.equal(kept[:, 0].cpu(), want[0]) and torch.equal(kept[:, 1].cpu(), want[1])
    one = store[0].clone()
    A.paged_accept(one[0], one[1], table, n, path.to(cuda))
    assert torch.equal(one[0].cpu(), want[0][0]) and torch.equal(one[1].cpu(), want[1][0])
    # The layers as the innermost axis, heads inside tokens.
    other = [store[:, i].permute(1, 3, 2, 0, 4).contiguous().permute(3, 0, 2, 1, 4)
             for i in range(2)]
    A.paged_accept(*other, table, n, path.to(cuda))
    assert torch.equal(other[0].cpu(), want[0]) and torch.equal(other[1].cpu(), want[1])


def test_accepted_places_outside_the_cache(cuda):
    """Pages that do not exist, places past the table, entries that do not rise
    past their place, negative lengths: nothing but the rest moves."""
    G.note("accept outside")
    g, d, page = 2, 16, 4
    k = torch.randn(6, g, page, d, generator=G.gen_of(1)).half().to(cuda)
    v = torch.randn(6, g, page, d, generator=G.gen_of(2)).half().to(cuda)
    table = i32([[0, 2], [1, 9], [-1, 3], [4, 5]], cuda)
    n = i32([6, 2, 1, -3], cuda)
    path = i32([[1, 2, 2 ** 31 - 1], [1, 2, 3], [2, 5, 1], [0, 0, 2]], cuda)
    want = [O.accept(c, table, n.cpu(), path.cpu()) for c in (k, v)]
    A.paged_accept(k, v, table, n, path)
    assert torch.equal(k.cpu(), want[0]) and torch.equal(v.cpu(), want[1])


def test_captured_steps_on_two_streams(cuda):
    """Two captured graphs of windowed and tree attention, replayed by turns with
    eager work between and refilled inputs, and a call on a side stream."""
    G.note("graphs")
    h, g, d, page, dtype = 8, 2, 128, 16, torch.float16
    lengths = [900, 333]
    k, v, table = G.paged(1, [1200, 500], g, d, page, dtype, cuda, poison=False)
    n, starts = i32(lengths, cuda), i32([0, 9, 16], cuda)
    q = G.randn(G.gen_of(3), 16, h, d, dtype=dtype, device=cuda)
    masks = A.tree_masks(random_trees(5, [9, 7]), device=cuda)

    def step():
        return torch.cat((A.paged_decode(q[:2], k, v, table, n, window=700, sinks=4),
                          A.paged_prefill(q, k, v, table, n, starts, window=500, sinks=4),
                          A.paged_tree(q, k, v, table, n, starts, masks)))

    buckets = [DecodeGraphBucket(cuda), DecodeGraphBucket(cuda)]
    for b in buckets:
        b.capture(step)
    for turn in range(4):
        q.copy_(G.randn(G.gen_of(10 + turn), 16, h, d, dtype=dtype, device=cuda))
        n.copy_(i32([900 + 70 * turn, 400 - 90 * turn], cuda))
        want = step()
        torch.cuda.synchronize()
        for b in buckets:
            got = b.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert torch.equal(got, want)


def test_starts_that_decrease_stay_inside(cuda):
    """Not a batch that the call allows: two sequences have the same rows.  Each
    row is one of theirs."""
    G.note("decreasing starts")
    lengths = [700, 650, 600, 640]
    for dtype in DTYPES:
        k, v, table = G.paged(2, lengths, 2, 64, 16, dtype, cuda, poison=False)
        q = G.randn(G.gen_of(4), 40, 4, 64, dtype=dtype, device=cuda)
        n, starts = i32(lengths, cuda), i32([0, 40, 0, 40, 20], cuda)
        masks = torch.full((40, 1), -1, dtype=torch.int64, device=cuda)
        out = A.paged_tree(q, k, v, table, n, starts, masks)
        assert torch.isfinite(out).all()


# few rows of a sequence, in one piece and in several; many rows
NEW = [[9, 3], [40, 1], [200, 30]]


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("new", NEW)
def test_given_scales(cuda, new, scale):
    G.note(f"scale {scale} {new}")
    lengths, dtype = [900, 230], torch.float16
    k, v, table = G.paged(5, lengths, 2, 64, 16, dtype, cuda)
    n, starts = i32(lengths, cuda), i32([0, new[0], sum(new)], cuda)
    q = G.randn(G.gen_of(1), sum(new), 4, 64, dtype=dtype, device=cuda)
    masks = A.tree_masks(random_trees(3, new), device=cuda)
    out = A.paged_tree(q, k, v, table, n, starts, masks, scale=scale)
    check(out, q, k, v, table, n, starts, lambda b, c, t: O.tree_sight(
        masks[int(starts[b]):int(starts[b + 1])].cpu(), t), scale=scale)

    def sight(b, rows, total):
        return O.window_sight(rows, total, 77, 3)

    out = A.paged_prefill(q, k, v, table, n, starts, scale=scale, window=77, sinks=3)
    check(out, q, k, v, table, n, starts, sight, scale=scale)
    out = A.paged_decode(q[:2], k, v, table, n, scale=scale, window=77, sinks=3)
    check(out, q[:2], k, v, table, n, torch.arange(3), sight, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", NEW)
def test_sharp_and_flat_rows(cuda, new, dtype):
    """Scores hundreds apart, all equal, a first key far above or far below the
    rest, and a drafted key that takes all where it is seen."""
    G.note(f"sharp trees {new} {dtype}")
    lengths = [900, 230]
    k, v, table = G.paged(9, lengths, 1, 64, 16, dtype, cuda, poison=False)
    q = G.randn(G.gen_of(3), sum(new), 4, 64, dtype=dtype, device=cuda)
    first = k[table[0, 0].long(), 0, 0]
    first *= 8.0
    place = lengths[0] - new[0] + 1
    drafted = k[table[0, place // 16].long(), 0, place % 16]
    drafted *= 8.0
    q[0] *= 60.0
    q[1], q[2], q[3], q[4] = 0.0, first * 0.5, -first * 0.5, drafted * 0.5
    q[5], q[6] = drafted * 0.5, -drafted * 0.5
    n, starts = i32(lengths, cuda), i32([0, new[0], sum(new)], cuda)
    masks = A.tree_masks(random_trees(3, new), device=cuda)
    masks[4] |= 2
    masks[5] &= ~2
    out = A.paged_tree(q, k, v, table, n, starts, masks)
    check(out, q, k, v, table, n, starts, lambda b, c, t: O.tree_sight(
        masks[int(starts[b]):int(starts[b + 1])].cpu(), t))
    out = A.paged_prefill(q, k, v, table, n, starts, window=100, sinks=1)
    check(out, q, k, v, table, n, starts, lambda b, c, t: O.window_sight(c, t, 100, 1))


@pytest.mark.parametrize("new", NEW)
def test_lengths_past_the_table_are_cut(cuda, new):
    G.note(f"long lengths {new}")
    k, v, table = G.paged(7, [640, 640], 2, 64, 16, torch.float16, cuda)
    table = table[:, :40]
    q = G.randn(G.gen_of(2), sum(new), 4, 64, dtype=torch.float16, device=cuda)
    masks = A.tree_masks(random_trees(3, new), device=cuda)
    starts = i32([0, new[0], sum(new)], cuda)
    for given, cut in ([2 ** 31 - 1, -5], [640, 0]), ([10 ** 9, 641], [640, 640]):
        n, m = i32(given, cuda), i32(cut, cuda)
        out = A.paged_tree(q, k, v, table, n, starts, masks)
        assert torch.equal(out, A.paged_tree(q, k, v, table, m, starts, masks))
        check(out, q, k, v, table, m, starts, lambda b, c, t: O.tree_sight(
            masks[int(starts[b]):int(starts[b + 1])].cpu(), t))
        assert torch.equal(A.paged_prefill(q, k, v, table, n, starts, window=70, sinks=2),
                           A.paged_prefill(q, k, v, table, m, starts, window=70, sinks=2))
        assert torch.equal(A.paged_decode(q[:2], k, v, table, n, window=70, sinks=2),
                           A.paged_decode(q[:2], k, v, table, m, window=70, sinks=2))


def test_empty_calls(cuda):
    G.note("empty")
    k, v, table = G.paged(7, [64], 2, 64, 16, torch.float16, cuda)
    none = torch.empty(0, 4, 64, dtype=torch.float16, device=cuda)
    no_rows = torch.zeros(0, 1, dtype=torch.int64, device=cuda)
    no_seqs, n, zero = i32([], cuda), i32([64], cuda), i32([0, 0], cuda)
    assert A.paged_decode(none, k, v, table[:0], no_seqs, window=3, sinks=1).shape == none.shape
    assert A.paged_prefill(none, k, v, table, n, zero, window=3, sinks=1).shape == none.shape
    assert A.paged_tree(none, k, v, table, n, zero, no_rows).shape == none.shape
    kept = k.clone(), v.clone()
    A.paged_accept(k, v, table[:0], no_seqs, torch.zeros(0, 3, dtype=torch.int32, device=cuda))
    A.paged_accept(k, v, table, n, torch.zeros(1, 0, dtype=torch.int32, device=cuda))
    A.paged_accept(k, v, table[:, :0], n, i32([[1, 2]], cuda))
    A.paged_accept(k[:0], v[:0], table, n, i32([[1, 2]], cuda))
    for now, then in zip((k, v), kept):
        assert torch.equal(now.view(torch.int16), then.view(torch.int16))
    # Rows of no sequence, no page, no sequence.
    q = torch.ones(3, 4, 64, dtype=torch.float16, device=cuda)
    masks = torch.full((3, 1), -1, dtype=torch.int64, device=cuda)
    for rows, seqs, pages in ((zero, n, table), (i32([0, 3], cuda), n, table[:, :0]),
                              (i32([0], cuda), no_seqs, table[:0])):
        assert (A.paged_tree(q, k, v, pages, seqs, rows, masks) == 0).all()
        assert (A.paged_prefill(q, k, v, pages, seqs, rows, window=2) == 0).all()
    assert (A.paged_tree(q, k[:0], v[:0], table, n, i32([0, 3], cuda), masks) == 0).all()


def test_offsets_past_32_bits(cuda):
    """Pages more than 2^32 elements into the cache, and layers as far apart."""
    G.note("far pages")
    g, page, d, dtype = 2, 64, 128, torch.bfloat16
    pages = (1 << 32) // (g * page * d) + 40
    store = torch.empty(1, 2, pages, g, page, d, dtype=dtype, device=cuda)
    k, v = store[0]
    lengths, r = [150, 70], G.gen_of(5)
    table = i32([[pages - 1, 3, pages - 30], [pages - 7, pages - 2, -1]], cuda)
    at = table.flatten()[:5].long()
    for c in (k, v):
        c[at] = G.randn(r, 5, g, page, d, dtype=dtype, device=cuda)
    small = i32([[0, 1, 2], [3, 4, -1]], cuda)
    ks, vs, n = k[at], v[at], i32(lengths, cuda)
    for new in ([20, 9], [140, 60]):
        q = G.randn(r, sum(new), 4, d, dtype=dtype, device=cuda)
        starts = i32([0, new[0], sum(new)], cuda)
        masks = A.tree_masks(random_trees(3, new), device=cuda)
        assert torch.equal(A.paged_tree(q, k, v, table, n, starts, masks),
                           A.paged_tree(q, ks, vs, small, n, starts, masks))
        assert torch.equal(A.paged_prefill(q, k, v, table, n, starts, window=30, sinks=2),
                           A.paged_prefill(q, ks, vs, small, n, starts, window=30, sinks=2))
        assert torch.equal(A.paged_decode(q[:2], k, v, table, n, window=30, sinks=2),
                           A.paged_decode(q[:2], ks, vs, small, n, window=30, sinks=2))
    before, path = i32([100, 62], cuda), i32([[3, 30, 49], [0, 5, -1]], cuda)
    A.paged_accept(store[:, 0], store[:, 1], table, before, path)
    A.paged_accept(ks, vs, small, before, path)
    assert torch.equal(k[at], ks) and torch.equal(v[at], vs)
    # One page per layer, the layers far apart.
    layers = store.flatten()[:2 << 32].view(2, 1 << 32)[:, :2 * g * page * d]
    layers = layers.view(2, 2, 1, g, page, d)
    layers.copy_(G.randn(r, *layers.shape, dtype=dtype, device=cuda))
    near = layers.contiguous()
    assert layers.stride(0) == 1 << 32 and near.stride(0) < 1 << 32
    for c in (layers, near):
        A.paged_accept(c[:, 0], c[:, 1], i32([[0]], cuda), i32([9], cuda), i32([[2, 5]], cuda))
    assert torch.equal(layers, near) and not torch.equal(near[1, 0, 0, :, 9], near[1, 0, 0, :, 10])
    assert torch.equal(near[1, 0, 0, :, 9], near[1, 0, 0, :, 11])
