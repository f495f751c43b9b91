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
