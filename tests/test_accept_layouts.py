"""Accepted paths in caches of any order of axes: keys and values apart, or side
by side within layers, pages, heads or tokens of one tensor.

Without a GPU a call whose arguments are taken gets as far as its launch, which
reports that there is no device; refused ones do not.
"""
from __future__ import annotations

import itertools

import pytest
import torch

import test_drafts_host as H
from nanopointllm_amd import _lib, attention as A
from oracle import drafts_oracle as O

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")


def rows_share(axes, off, dim):
    """Whether rows at [0, dim) and [off, off + dim) plus any indexes of the axes
    (stride, count) share an element."""
    at = {sum(i * s for i, (s, _) in zip(index, axes))
          for index in itertools.product(*[range(n) for _, n in axes])}
    return any(x + off + d in at for x in at for d in range(-dim + 1, dim))


def strides_of(order, sizes, dim):
    """Element strides of the axes of a dense tensor with the axes in ``order``
    before the row."""
    strides, step = {}, dim
    for name in reversed(order):
        strides[name] = step
        step *= sizes[name]
    return strides, step


@no_gpu
def test_caches_that_share_no_element_reach_the_launch():
    """Every order of layers, keys and values, pages, heads and tokens."""
    sizes = {"layers": 2, "kv": 2, "pages": 3, "heads": 2, "page": 4}
    for order in itertools.permutations(sizes):
        s, _ = strides_of(order, sizes, 64)
        for pair in ((H.KC, H.KC + 2 * s["kv"]), (H.KC + 2 * s["kv"], H.KC)):
            got = H._accept(kc=pair[0], vc=pair[1], cl=s["layers"], layers=2, pages=3, page=4,
                            cs=(s["pages"], s["heads"], s["page"]))
            assert got == _lib.ERR_HIP, (order, got)
    # One layer, keys and values in each page; far apart; a stride of an axis of one.
    assert H._accept(vc=H.KC + 2 * 2048, cs=(4096, 1024, 64), layers=1, cl=0) == _lib.ERR_HIP
    assert H._accept(vc=H.KC + 2 * 2048, cs=(4096, 1024, 64), layers=1, cl=64) == _lib.ERR_HIP
    assert H._accept(vc=H.KC + (1 << 40)) == _lib.ERR_HIP


@no_gpu
@pytest.mark.parametrize("gap", [0, 8, 64, 200])
def test_caches_at_any_distance(gap):
    """Taken exactly where no row of the keys meets one of the values, by counting
    them all; axes with gaps between them."""
    dim, heads, page, pages, layers = 16, 2, 2, 2, 2
    tok = dim + gap % 16
    head = page * tok + gap // 2 * 2
    one = heads * head + gap
    layer = pages * one + 2 * gap
    axes = [(layer, layers), (one, pages), (head, heads), (tok, page)]
    span = layers * layer
    seen = set()
    for off in range(-span - 64, span + 72, 8):
        meets = rows_share(axes, off, dim)
        got = H._accept(kc=H.KC, vc=H.KC + 2 * off, cl=layer, layers=layers, pages=pages, page=page,
                        cs=(one, head, tok), g=heads, d=dim, n=4, ld=4)
        assert got == (_lib.ERR_OVERLAP if meets else _lib.ERR_HIP), (off, meets, got)
        seen.add(meets)
    assert seen == {True, False}


@pytest.mark.gpu
@pytest.mark.parametrize("layers", [1, 3])
def test_accepted_paths_in_every_order_of_axes(cuda, layers):
    g, d, page, pages = 2, 16, 4, 5
    r = torch.Generator().manual_seed(layers)
    table = torch.tensor([[3, 0, -1], [4, 1, 2]], dtype=torch.int32, device=cuda)
    n = torch.tensor([1, 5], dtype=torch.int32, device=cuda)
    path = torch.tensor([[0, 2, 6], [1, 3, -1]], dtype=torch.int32, device=cuda)
    base = torch.randn(layers, 2, pages, g, page, d, generator=r).half()
    want = [O.accept(base[:, i], table, n.cpu(), path.cpu()) for i in range(2)]
    for order in itertools.permutations(range(5)):
        back = [order.index(i) for i in range(5)] + [5]
        store = base.permute(*order, 5).contiguous().to(cuda).permute(back)
        A.paged_accept(store[:, 0], store[:, 1], table, n, path)
        assert torch.equal(store[:, 0].cpu(), want[0]), order
        assert torch.equal(store[:, 1].cpu(), want[1]), order
    # One layer's caches inside the pages of one tensor, as the other calls take them.
    store = base[0].transpose(0, 1).contiguous().to(cuda)        # [pages, 2, heads, page, dim]
    A.paged_accept(store[:, 0], store[:, 1], table, n, path)
    assert torch.equal(store[:, 0].cpu(), want[0][0]) and torch.equal(store[:, 1].cpu(), want[1][0])
    with pytest.raises(Exception, match="overlap"):
        A.paged_accept(store[:, 0], store[:, 0], table, n, path)


def test_launches_past_32_bits_of_threads_are_refused():
    """2^24 workgroups of 256 threads; with no page a call that is taken does
    nothing."""
    def call(**kw):
        return H._accept(pages=0, cl=1 << 30, cs=(1 << 20, 1 << 10, 64), **kw)

    assert call(b=65535, layers=64, g=32, d=128) == _lib.OK
    assert call(b=65535, layers=65, g=32, d=128) == _lib.ERR_SHAPE
    assert call(b=65535, layers=128, g=8, d=128) == _lib.OK
    assert call(b=65535, layers=129, g=8, d=128) == _lib.ERR_SHAPE
    assert call(b=65535, layers=64, g=33, d=128) == _lib.ERR_SHAPE
    assert call(b=1, layers=32767, g=4096, d=256) == _lib.ERR_SHAPE
    assert call(b=65535, layers=32767, g=1, d=8) == _lib.ERR_SHAPE


@no_gpu
def test_tables_that_end_where_a_cache_begins():
    """The last columns of a wide table or path: their last row ends with its own
    entries, a whole row further would be inside the cache."""
    n, ld, b = 4, 1000, 3
    last = 4 * ((b - 1) * ld + n)
    for cache in (H.KC, H.VC):
        assert H._accept(table=cache - last, ld=ld, n=n, b=b) == _lib.ERR_HIP
        assert H._accept(table=cache - last + 4, ld=ld, n=n, b=b) == _lib.ERR_OVERLAP
        assert H._accept(path=cache - last, ld_path=ld, steps=n, b=b) == _lib.ERR_HIP
        assert H._accept(path=cache - last + 4, ld_path=ld, steps=n, b=b) == _lib.ERR_OVERLAP
        assert H._accept(lengths=cache - 4 * b, b=b) == _lib.ERR_HIP
        assert H._accept(lengths=cache - 4 * b + 4, b=b) == _lib.ERR_OVERLAP


@pytest.mark.gpu
def test_accepted_paths_with_a_table_right_before_the_cache(cuda):
    """Table and caches in one allocation, the table the last columns of a wide one."""
    g, d, page, pages, ld, b = 2, 16, 4, 5, 1000, 2
    cells = pages * g * page * d
    room = torch.zeros(ld * 4 + 4 * cells, dtype=torch.uint8, device=cuda)
    table = room[:ld * 4].view(torch.int32).as_strided((b, 3), (ld - 3, 1), 0)
    table.copy_(torch.tensor([[3, 0, -1], [4, 1, 2]], dtype=torch.int32))
    assert table.data_ptr() + 4 * ((b - 1) * (ld - 3) + 3) == room.data_ptr() + ld * 4
    caches = room[ld * 4:].view(torch.float16).view(2, pages, g, page, d)
    caches.copy_(torch.randn(caches.shape, generator=torch.Generator().manual_seed(1)))
    n = torch.tensor([1, 5], dtype=torch.int32, device=cuda)
    path = torch.tensor([[0, 2, 6], [1, 3, -1]], dtype=torch.int32, device=cuda)
    want = [O.accept(c, table, n.cpu(), path.cpu()) for c in caches]
    A.paged_accept(caches[0], caches[1], table, n, path)
    assert torch.equal(caches[0].cpu(), want[0]) and torch.equal(caches[1].cpu(), want[1])
