"""States of drafted tokens through the runner's attention core: steps that mix
single new tokens with trees, and stacks that take none."""
from __future__ import annotations

import pytest
import torch

import test_gpu_attention as G
import test_gpu_window_tree as W
from nanopointllm_amd import attention as A
from oracle import drafts_oracle as O


def test_a_stack_with_one_windowed_layer_refuses_at_its_first(monkeypatch):
    """Whichever layer asks, before anything is stored."""
    def stored(*args, **kw):
        raise AssertionError("stored")

    monkeypatch.setattr(A, "rotary_store", stored)
    cache = A.PagedKVCache(3, 1, 1, 64, device="cpu")
    state = A.AttentionState.build_drafts([[0]], [3], [[-1, 0]], 16, device="cpu")
    q = torch.zeros(2, 1, 64, dtype=torch.float16)
    for window in ([None, None, 4], [4, None, None], [8, 4, 2], 5):
        core = A.PagedAttentionCore(cache, None, window=window, sinks=2)
        for layer in range(3):
            with pytest.raises(ValueError, match="without a window"):
                core(q, q, q, layer, state)
    frequencies = A.rotary_frequencies(64, device="cpu")
    for window in (None, [None, None, None]):
        core = A.PagedAttentionCore(cache, frequencies, window=window)
        with pytest.raises(AssertionError, match="stored"):
            core(q, q, q, 0, state)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", G.DTYPES)
def test_single_tokens_and_trees_in_one_step(cuda, dtype):
    """Sequences of one new token first, then trees, then padded rows: to the bit
    what the single calls give, and what a tree of one gives for the tokens."""
    G.note(f"mixed drafts {dtype}")
    h, g, d, page, ones, padded = 4, 2, 64, 8, 3, 4
    cached, trees = [30, 7, 0, 21, 40], [[-1, 0, 0, 1, 1], [-1, 0, 1, 1, 2, 0, 3]]
    new = [1, 1, 1] + [len(t) for t in trees]
    lengths = [n + m for n, m in zip(cached, new)]
    pages = [[4 * b + 20 * i for i in range(6)] for b in range(5)]
    cache = A.PagedKVCache(2, 128, g, d, page_size=page, dtype=dtype, device=cuda)
    r = G.gen_of(6)
    for c in cache.k + cache.v:
        c.copy_(G.randn(r, *c.shape, dtype=dtype, device=cuda))
    before = [c.clone() for c in cache.k + cache.v]
    state = A.AttentionState.build(pages, lengths, new, page, device=cuda)
    assert state.decode_rows == ones
    drafts = A.AttentionState.build_drafts(pages[ones:], cached[ones:], trees, page, device=cuda)
    state.positions[ones:] = drafts.positions
    # Padded rows: no sequence's, not stored, masks that show everything.
    total = sum(new) + padded
    state.positions = torch.cat((state.positions, torch.zeros(padded, dtype=torch.int64, device=cuda)))
    state.slots = torch.cat((state.slots, torch.full((padded,), -1, device=cuda)))
    state.masks = torch.full((total - ones, 1), -1, dtype=torch.int64, device=cuda)
    state.masks[:-padded] = drafts.masks
    frequencies = A.rotary_frequencies(d, device=cuda)
    core = A.PagedAttentionCore(cache, frequencies)
    q, k, v = (G.randn(r, total, n, d, dtype=dtype, device=cuda) for n in (h, g, g))
    out = core(q, k, v, 1, state).view(total, h, d)

    assert all(torch.equal(a, b) for a, b in zip((cache.k[0], cache.v[0]), (before[0], before[2])))
    kc, vc = before[1], before[3]
    turned = A.rotary_store(q, k, v, state.positions, state.slots, frequencies.inv_freq, kc, vc)
    assert torch.equal(cache.k[1], kc) and torch.equal(cache.v[1], vc)
    table, n = state.page_table, state.lengths
    assert torch.equal(out[:ones], A.paged_decode(turned[:ones], kc, vc, table[:ones], n[:ones]))
    assert torch.equal(out[ones:], A.paged_tree(turned[ones:], kc, vc, table[ones:], n[ones:],
                                                state.q_starts, state.masks))
    assert (out[-padded:] == 0).all() and out[:-padded].abs().sum(-1).min() > 0
    # And the definition, a single token as a tree of one.
    starts = torch.tensor([0, 1, 2, 3] + [3 + m for m in (5, 12)], dtype=torch.int32)
    masks = torch.cat((torch.ones(ones, 1, dtype=torch.int64), state.masks.cpu()))
    owned = W.check(out, turned, kc, vc, table, n, starts, lambda b, count, keys: O.tree_sight(
        masks[int(starts[b]):int(starts[b + 1])], keys))
    assert owned[:-padded].all() and not owned[-padded:].any()
