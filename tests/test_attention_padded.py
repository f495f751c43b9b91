"""Prompts in a padded buffer, without a GPU: refusals before any launch."""
from __future__ import annotations

from nanopointllm_amd import _lib
from test_attention_host import AUX, KC, OUT, Q, VC, WS, _p


def padded(*, t=5, b=3, starts=AUX, wb=1 << 30, n=4, os=(256, 64)):
    return _lib.load().w8a8_paged_prefill_padded(
        _p(Q), 256, 64, _p(KC), _p(VC), 2048, 1024, 64, 4, 16, _p(AUX), n, n, _p(AUX), _p(starts),
        _lib.F16, 0.125, _p(OUT), *os, t, b, 4, 2, 64, _p(WS), wb, None)


def test_refusals():
    assert padded(t=-1) == _lib.ERR_SHAPE and padded(b=-1) == _lib.ERR_SHAPE
    assert padded(starts=None) == _lib.ERR_NULL and padded(starts=AUX + 2) == _lib.ERR_ALIGN
    assert padded(os=(64, 64)) == _lib.ERR_OVERLAP
    assert padded(n=64, wb=0) == _lib.ERR_WORKSPACE
    # No sequence, so no workgroup that could clear the rows.
    assert padded(b=0) == _lib.ERR_SHAPE
    assert padded(t=0) == _lib.OK and padded(t=0, b=0) == _lib.OK
