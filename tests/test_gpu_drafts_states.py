"""States of drafted tokens through the runner's attention core."""
from __future__ import annotations

import pytest
import torch

from nanopointllm_amd import attention as A


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
