"""Attention's rows and caches at addresses and strides that its 16-byte
accesses do not take, without a GPU: what is copied, and which strides are
never multiplied by anything but zero."""
from __future__ import annotations

import pytest
import torch

from nanopointllm_amd import _lib, attention as A
from test_attention_host import _decode, _prefill


def taken(q: torch.Tensor) -> torch.Tensor:
    got, strides = A._queries(q)
    assert got.data_ptr() % 16 == 0 and strides == got.stride()
    assert strides[2] == 1 and strides[0] % 8 == 0 and strides[1] % 8 == 0
    assert torch.equal(got, q)
    return got


def test_queries_are_copied_where_contiguous_means_nothing():
    flat = torch.randn(5 * 64 + 8, dtype=torch.float32).half()
    for offset in (1, 2, 4, 7):
        taken(flat[offset:offset + 4 * 64].view(2, 2, 64))      # contiguous, misaligned
    wide = torch.randn(3, 4 * 64 + 3).half()
    for q in (wide[:1, :256].view(1, 4, 64),                     # one row, a stride of 259
              wide[1:2, 1:257].view(1, 4, 64), wide[:, :64].view(3, 1, 64),
              wide[:, :256].view(3, 4, 64), wide[:, :64].T.contiguous().T.view(3, 1, 64)):
        taken(q)
    aligned = torch.zeros(3, 4, 64, dtype=torch.float16)
    assert A._queries(aligned)[0] is aligned                     # nothing copied


# No launch: a call that passes every check up to the workspace's, which is missing.
WIDE = {"n": 64, "ld": 64, "ws": None, "wb": 0}


@pytest.mark.parametrize("call, one", [(_decode, {"b": 1}), (_prefill, {"t": 1, "b": 1})])
def test_strides_of_axes_of_one_are_not_used(call, one):
    passed, align = _lib.ERR_WORKSPACE, _lib.ERR_ALIGN
    assert call(**WIDE) == passed
    assert call(qs=(259, 64), os=(261, 64), **one, **WIDE) == passed
    single = {"h": 1, "g": 1, "qs": (64, 3), "os": (64, 5), "cs": (1024, 7, 64)}
    assert call(**single, **WIDE) == passed
    assert call(pages=1, cs=(2049, 1024, 64), **WIDE) == passed
    assert call(page=1, n=1024, ld=1024, ws=None, wb=0, cs=(128, 64, 3)) == passed
    # The same strides where the axis is longer.
    assert call(qs=(259, 64), **WIDE) == align and call(os=(261, 64), **WIDE) == align
    assert call(qs=(256, 67), **one, **WIDE) == align
    assert call(cs=(2049, 1024, 64), **WIDE) == align
    assert call(cs=(2048, 1025, 64), **WIDE) == align
    assert call(cs=(2048, 1024, 65), **WIDE) == align


def test_caches_may_differ_in_unused_strides():
    q = torch.zeros(1, 2, 8, dtype=torch.float16)
    k = torch.zeros(1, 2, 4, 8, dtype=torch.float16)
    v = torch.zeros(2 * 77, dtype=torch.float16).as_strided((1, 2, 4, 8), (77, 32, 8, 1))
    shape, strides = A._cache(k, v, q, 8)
    assert shape == k.shape and strides == k.stride()
    with pytest.raises(ValueError, match="equal strides"):
        A._cache(k, torch.zeros(1, 4, 2, 8, dtype=torch.float16).transpose(1, 2), q, 8)
    with pytest.raises(ValueError, match="equal strides"):
        A._cache(k.expand(2, 2, 4, 8), torch.zeros(2, 2, 4, 8, dtype=torch.float16), q, 8)
