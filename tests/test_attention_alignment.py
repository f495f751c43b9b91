"""Attention's rows at addresses and strides that its 16-byte accesses do not
take, without a GPU: what is copied."""
from __future__ import annotations

import torch

from nanopointllm_amd import attention as A


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
