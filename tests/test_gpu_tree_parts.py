"""Trees of up to 64 rows per sequence and key head on average carry their
probabilities as two 16-bit parts into the second product, as decode does.

Tolerances as in test_gpu_attention.py, without a rounding of the probabilities to
the 16-bit type: two parts that are cut off leave less than h = 2^-21 of a binary16
probability and 2^-15 of a bfloat16 one, in the numerator alone: (r + h + 2 n u) sum
p |v| + n 2^-25 max|v| + e |out| (+ the smallest step).  Few keys, small scores and
values that nearly cancel make e |out| and r small: a single rounding, e = 2^-11 or
2^-8 of each probability, misses this.
"""
from __future__ import annotations

import math

import pytest
import torch

import test_gpu_attention as G
from nanopointllm_amd import attention as A
from oracle import drafts_oracle as O

pytestmark = pytest.mark.gpu

U = G.U


@pytest.mark.parametrize("dtype", G.DTYPES)
@pytest.mark.parametrize("h,g,d,page,new,cached", [
    (2, 2, 128, 16, [64], [0]), (8, 2, 128, 16, [16, 9], [5, 30]), (4, 4, 64, 16, [40, 60], [7, 0]),
    (4, 1, 96, 8, [10, 12], [20, 3]), (2, 2, 128, 4, [50], [9]), (2, 2, 128, 16, [20, 3], [0, 40]),
    # cut over the keys and joined
    (2, 2, 128, 16, [48], [900]), (2, 2, 64, 16, [33], [900])])
def test_probabilities_keep_two_parts(cuda, h, g, d, page, new, cached, dtype):
    G.note(f"tree parts {h} {g} {d} {page} {new} {cached} {dtype}")
    lengths = [n + c for n, c in zip(new, cached)]
    k, v, table = G.paged(h + d, lengths, g, d, page, dtype, cuda, poison=False)
    starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    trees = [[(i - 1) // 2 if i else -1 for i in range(n)] for n in new]
    masks = A.tree_masks(trees, device="cpu")
    q = G.randn(G.gen_of(d + h), sum(new), h, d, dtype=dtype, device=cuda, std=0.02)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    out = A.paged_tree(q, k, v, table, n, starts.to(cuda), masks.to(cuda))
    want, size, dots = O.attention(q, k, v, table, n, starts, lambda b, count, total: O.tree_sight(
        masks[int(starts[b]):int(starts[b + 1])], total))
    e, most, keys = G.half_step(dtype), float(v.float().abs().max()), max(lengths)
    parts = 2.0 ** -21 if dtype == torch.float16 else 2.0 ** -15
    rel = 2 * ((d + 12) * U * dots + 16 * U) + parts + 2 * keys * U
    tol = rel[..., None] * size + keys * 2.0 ** -25 * most + e * want.abs() + G.smallest(dtype)
    err = (out.double().cpu() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max())}"


@pytest.mark.parametrize("dtype", G.DTYPES)
@pytest.mark.parametrize("cached,n", [(100, 50), (700, 64), (0, 40)])
def test_values_that_only_some_of_many_rows_see(cuda, cached, n, dtype):
    """An infinity and a NaN among the drafted values, and an infinite and a NaN key
    that no row sees: they reach the rows that see them, and no others, in one piece
    and in several."""
    G.note(f"tree parts special values {cached} {n} {dtype}")
    h = g = 2
    d, page = 64, 16
    k, v, table = G.paged(8, [cached + n], g, d, page, dtype, cuda)

    def row(cache, node):
        at = cached + node
        return cache[int(table[0, at // page]), :, at % page]

    row(v, 5)[:, 3], row(v, 5)[:, 7] = math.inf, math.nan
    row(k, 9)[:, 1], row(k, 11)[:, 2] = math.inf, math.nan
    row(v, 9)[:], row(v, 11)[:] = math.nan, -math.inf
    masks = A.tree_masks([[-1, 0, 1, 2, 3] + [4 if i % 2 else i - 1 for i in range(5, n)]],
                         device="cpu")
    masks &= ~(1 << 9 | 1 << 11)
    q = G.randn(G.gen_of(2), n, h, d, dtype=dtype, device=cuda)
    lengths = torch.tensor([cached + n], dtype=torch.int32, device=cuda)
    starts = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    out = A.paged_tree(q, k, v, table, lengths, starts, masks.to(cuda))
    sees = O.tree_sight(masks, cached + n)[:, cached + 5].to(cuda)
    assert 0 < int(sees.sum()) < n
    assert (out[sees][..., 3] == math.inf).all() and out[sees][..., 7].isnan().all()
    assert torch.isfinite(out[~sees]).all()
    keep = [i for i in range(d) if i not in (3, 7)]
    assert torch.isfinite(out[..., keep]).all()
    # The others to the bit what they are without those values.
    row(v, 5)[:, 3], row(v, 5)[:, 7] = 0.25, -0.5
    want = A.paged_tree(q, k, v, table, lengths, starts, masks.to(cuda))
    assert torch.isfinite(want).all() and torch.equal(out[~sees], want[~sees])
