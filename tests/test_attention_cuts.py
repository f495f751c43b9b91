"""Which calls of the attention core may be cut over the keys, by their
workspace: a call that is never cut needs none."""
from __future__ import annotations

from nanopointllm_amd import _lib


def test_few_rows_are_cut_from_two_pieces_of_256_keys_on():
    size = _lib.load().w8a8_paged_prefill_workspace_bytes
    for tokens, heads, kv in ((4, 32, 8), (150, 32, 8), (4, 8, 8), (40, 32, 32)):
        assert size(tokens, 1, heads, kv, 128, 480) == 0
        assert size(tokens, 1, heads, kv, 128, 512) > 0
    # A row tile for every second CU: whole up to pieces of 512 keys.
    assert size(560, 1, 32, 32, 128, 992) == 0 and size(560, 1, 32, 32, 128, 1024) > 0
    assert size(8192, 1, 32, 32, 128, 8192) == 0      # workgroups enough
