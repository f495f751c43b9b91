"""The attention core without a GPU: rotary frequencies against their
formulas, the state of a step, and refusals before any launch."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nanopointllm_amd import _lib, attention as A


# ------------------------------------------------------------- frequencies
def test_plain_frequencies():
    f, a = A.rotary_frequencies(128, base=10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (64,) and a == 1.0
    for i in (0, 1, 17, 63):
        assert math.isclose(f[i], 10000.0 ** (-2 * i / 128), rel_tol=1e-14)
    assert A.rotary_frequencies(0, device="cpu").inv_freq.shape == (0,)


def test_linear_and_ntk_scaling():
    plain = A.rotary_frequencies(64, device="cpu").inv_freq
    lin, a = A.rotary_frequencies(64, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(lin, plain / 4.0) and a == 1.0
    ntk, _ = A.rotary_frequencies(64, scaling={"rope_type": "ntk", "factor": 4.0}, device="cpu")
    # The base is chosen so that the slowest pair slows by the factor exactly
    # and the fastest not at all.
    assert math.isclose(ntk[0], plain[0], rel_tol=1e-14)
    assert math.isclose(ntk[-1], plain[-1] / 4.0, rel_tol=1e-12)


def test_llama3_scaling():
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    plain = A.rotary_frequencies(128, base=500000.0, device="cpu").inv_freq
    got, a = A.rotary_frequencies(128, base=500000.0, scaling=cfg, device="cpu")
    assert a == 1.0
    kinds = set()
    for f, g in zip(plain.tolist(), got.tolist()):
        wave = 2 * math.pi / f
        if wave < 8192 / 4.0:
            want, kind = f, "kept"
        elif wave > 8192 / 1.0:
            want, kind = f / 8.0, "slowed"
        else:
            s = (8192 / wave - 1.0) / 3.0
            want, kind = (1 - s) * f / 8.0 + s * f, "blended"
        kinds.add(kind)
        assert math.isclose(g, want, rel_tol=1e-12)
    assert kinds == {"kept", "slowed", "blended"}


def test_yarn_scaling():
    cfg = {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    plain = A.rotary_frequencies(128, device="cpu").inv_freq
    got, a = A.rotary_frequencies(128, scaling=cfg, device="cpu")
    assert math.isclose(a, 0.1 * math.log(16.0) + 1.0)
    turns = (plain * 4096 / (2 * math.pi)).tolist()
    for i, t in enumerate(turns):
        if t > 64:      # well above beta_fast = 32 turns: kept
            assert got[i] == plain[i]
        elif t < 0.5:   # well below beta_slow = 1: slowed by the factor
            assert math.isclose(got[i], plain[i] / 16.0, rel_tol=1e-14)
    ratio = (got / plain).tolist()
    assert all(x >= y - 1e-15 for x, y in zip(ratio, ratio[1:]))   # monotone blend
    low = math.floor(128 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    high = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    i = (low + high) // 2
    slowed = (i - low) / (high - low)
    assert math.isclose(ratio[i], 1 - slowed + slowed / 16.0, rel_tol=1e-12)
    assert A.rotary_frequencies(128, scaling={**cfg, "attention_factor": 1.25},
                                device="cpu").attention_factor == 1.25


@pytest.mark.parametrize("call, message", [
    (lambda: A.rotary_frequencies(7, device="cpu"), "even"),
    (lambda: A.rotary_frequencies(8, base=0.0, device="cpu"), "base"),
    (lambda: A.rotary_frequencies(8, scaling={"type": "unheard"}, device="cpu"), "unknown"),
    (lambda: A.rotary_frequencies(8, scaling={"type": "linear", "factor": 0.5}, device="cpu"),
     "factor"),
    (lambda: A.rotary_frequencies(8, scaling={
        "type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
        "original_max_position_embeddings": 64}, device="cpu"), "low_freq_factor"),
    (lambda: A.PagedAttentionCore(None, None, layout="quarter"), "layout"),
    (lambda: A.PagedKVCache(1, 1, 1, 64, page_size=12, device="cpu"), "power of two"),
    (lambda: A.PagedKVCache(1, 1, 1, 60, device="cpu"), "multiple of 8"),
    (lambda: A.PagedKVCache(1, 1, 1, 64, dtype=torch.float32, device="cpu"), "float16"),
])
def test_python_refusals(call, message):
    with pytest.raises(ValueError, match=message):
        call()


# -------------------------------------------------------------------- state
def test_state_of_a_mixed_step():
    s = A.AttentionState.build([[3], [5, 1], [2, 0, 4]], [4, 5, 9], [1, 1, 3], 4, device="cpu")
    assert s.decode_rows == 2
    assert s.positions.tolist() == [3, 4, 6, 7, 8]
    assert s.slots.tolist() == [3 * 4 + 3, 1 * 4 + 0, 0 * 4 + 2, 0 * 4 + 3, 4 * 4 + 0]
    assert s.page_table.tolist() == [[3, -1, -1], [5, 1, -1], [2, 0, 4]]
    assert s.lengths.tolist() == [4, 5, 9] and s.q_starts.tolist() == [0, 3]
    only = A.AttentionState.build([[0], [1]], [1, 2], [1, 1], 4, device="cpu")
    assert only.q_starts is None and only.decode_rows == 2
    with pytest.raises(ValueError, match="hold"):
        A.AttentionState.build([[0]], [5], [1], 4, device="cpu")
    with pytest.raises(ValueError, match="negative"):
        A.AttentionState.build([[-1]], [2], [1], 4, device="cpu")
    with pytest.raises(ValueError, match="one entry"):
        A.AttentionState.build([[0]], [2, 3], [1], 4, device="cpu")


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 8, dtype=torch.float16)
    c = torch.zeros(1, 2, 4, 8, dtype=torch.float16)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        A.paged_decode(q, c, c, one.reshape(1, 1), one)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        A.rotary(q, one.long(), torch.ones(4, dtype=torch.float64))


# ----------------------------------------------------- the C ABI's refusals
def _p(addr):
    return None if addr is None else ctypes.c_void_p(addr)


Q, K, V, OUT = 0x1000000, 0x2000000, 0x3000000, 0x4000000
KC, VC, AUX, WS = 0x10000000, 0x20000000, 0x5000000, 0x6000000


def _store(*, q=Q, qs=(256, 64), k=K, v=V, ks=(128, 64), dtype=_lib.F16, positions=AUX, slots=AUX,
           freq=AUX, rot=64, layout=0, factor=1.0, out=OUT, os=(256, 64), kc=KC, vc=VC,
           cs=(2048, 1024, 64), pages=4, page=16, t=3, h=4, g=2, d=64):
    return _lib.load().w8a8_rotary_store(
        _p(q), *qs, _p(k), *ks, _p(v), *ks, dtype, _p(positions), _p(slots), _p(freq), rot, layout,
        factor, _p(out), *os, _p(kc), _p(vc), *cs, pages, page, t, h, g, d, None)


def test_rotary_store_refusals():
    S, N, D, AL, O = (_lib.ERR_SHAPE, _lib.ERR_NULL, _lib.ERR_DTYPE, _lib.ERR_ALIGN,
                      _lib.ERR_OVERLAP)
    assert _store(dtype=_lib.F32) == D
    assert _store(layout=2) == D
    assert _store(d=60) == S and _store(d=264) == S and _store(d=0) == S
    assert _store(rot=65) == S and _store(rot=66) == S and _store(rot=-2) == S
    assert _store(t=-1) == S and _store(h=-1) == S and _store(t=1 << 31) == S
    assert _store(page=12) == S and _store(page=0) == S and _store(pages=-1) == S
    assert _store(factor=math.inf) == S and _store(factor=math.nan) == S
    assert _store(qs=(-256, 64)) == S and _store(cs=(2048, -1024, 64)) == S
    assert _store(qs=(1 << 60, 64), t=100) == S              # past any address
    for name in ("q", "k", "v", "positions", "slots", "freq", "out", "kc", "vc"):
        assert _store(**{name: None}) == N, name
    for name in ("q", "k", "v", "out", "kc", "vc"):
        assert _store(**{name: 0x7000001}) == AL, name
    assert _store(positions=AUX + 4) == AL and _store(slots=AUX + 4) == AL
    # q_out over other rows of q, over k, over the cache; over itself
    assert _store(out=Q + 512) == O and _store(out=K) == O and _store(out=KC) == O
    assert _store(out=Q, os=(512, 64)) == O
    assert _store(os=(64, 64)) == O and _store(os=(256, 32)) == O
    # k from the cache; both caches one; a cache whose rows overlap
    assert _store(k=KC + 64) == O and _store(vc=KC) == O
    assert _store(cs=(2048, 1024, 32)) == O and _store(cs=(0, 1024, 64)) == O
    # columns of one matrix: q in place next to k and v is fine, q over k is not
    row = (512, 64)
    assert _store(q=Q, qs=row, k=Q + 512, v=Q + 768, ks=row, out=Q, os=row, t=0) == _lib.OK
    assert _store(q=Q, qs=row, k=Q + 384, v=Q + 768, ks=row, out=Q, os=row) == O
    # nothing to do
    assert _store(t=0, q=None, out=None) == _lib.OK


def test_more_rows_than_a_launch_takes():
    """A launch's threads are counted in 32 bits: 2^24 workgroups of 256 are one
    too many."""
    many, S = 1 << 24, _lib.ERR_SHAPE
    assert _store(t=many) == S
    assert _lib.load().w8a8_rotary(Q, 8, 8, _lib.F16, AUX, AUX, 8, 0, 1.0, OUT, 8, 8, many, 1, 8,
                                   None) == S
    row = {"d": 8, "cs": (256, 128, 8), "qs": (8, 8), "os": (8, 8), "h": 1, "g": 1}
    assert _decode(b=many, **row) == S and _prefill(t=5, b=many, **row) == S
    assert _decode(b=1 << 20, **{**row, "h": 32, "g": 32, "os": (256, 8)}) == S
    assert _prefill(t=1 << 27, **{**row, "h": 32, "g": 32, "os": (256, 8)}) == S
    lib = _lib.load()
    assert lib.w8a8_paged_decode_workspace_bytes(many, 1, 1, 8, 64) == -1
    assert lib.w8a8_paged_prefill_workspace_bytes(1 << 27, 1, 32, 32, 8, 64) == -1


def _decode(*, q=Q, qs=(256, 64), kc=KC, vc=VC, cs=(2048, 1024, 64), pages=4, page=16, table=AUX,
            ld=4, n=4, lengths=AUX, dtype=_lib.F16, scale=0.125, out=OUT, os=(256, 64), b=3, h=4,
            g=2, d=64, ws=WS, wb=1 << 30):
    return _lib.load().w8a8_paged_decode(
        _p(q), *qs, _p(kc), _p(vc), *cs, pages, page, _p(table), ld, n, _p(lengths), dtype, scale,
        _p(out), *os, b, h, g, d, _p(ws), wb, None)


def _prefill(*, q=Q, qs=(256, 64), kc=KC, vc=VC, cs=(2048, 1024, 64), pages=4, page=16, table=AUX,
             ld=4, n=4, lengths=AUX, starts=AUX, dtype=_lib.F16, scale=0.125, out=OUT,
             os=(256, 64), t=5, b=3, h=4, g=2, d=64, ws=WS, wb=1 << 30):
    return _lib.load().w8a8_paged_prefill(
        _p(q), *qs, _p(kc), _p(vc), *cs, pages, page, _p(table), ld, n, _p(lengths), _p(starts),
        dtype, scale, _p(out), *os, t, b, h, g, d, _p(ws), wb, None)


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_attention_refusals(call):
    S, N, D, AL, O = (_lib.ERR_SHAPE, _lib.ERR_NULL, _lib.ERR_DTYPE, _lib.ERR_ALIGN,
                      _lib.ERR_OVERLAP)
    assert call(dtype=_lib.F32) == D
    assert call(d=60) == S and call(d=264) == S
    assert call(h=5) == S and call(h=0) == S and call(g=0) == S
    assert call(page=24) == S and call(pages=-1) == S
    assert call(ld=3) == S and call(n=1 << 30, ld=1 << 30) == S
    assert call(b=-1) == S and call(scale=math.nan) == S
    many = {"t": 1 << 24} if call is _prefill else {"b": 1 << 24}
    assert call(h=256, g=1, **many) == S      # rows of one key head past 32 bits
    for name in ("q", "kc", "vc", "table", "lengths", "out"):
        assert call(**{name: None}) == N, name
    for name in ("q", "kc", "vc", "out"):
        assert call(**{name: 0x7000008}) == AL, name
    assert call(qs=(260, 64)) == AL and call(cs=(2048, 1024, 68)) == AL
    assert call(table=AUX + 2) == AL and call(lengths=AUX + 2) == AL
    assert call(out=Q) == O and call(out=KC) == O and call(os=(64, 64)) == O
    assert call(b=0, q=None, out=None) == _lib.OK
    if call is _prefill:
        assert call(starts=None) == N and call(starts=AUX + 2) == AL
        assert call(t=0, q=None) == _lib.OK and call(t=-1) == S


def test_workspace_sizes():
    lib = _lib.load()
    dec, pre = lib.w8a8_paged_decode_workspace_bytes, lib.w8a8_paged_prefill_workspace_bytes
    assert dec(1, 4, 3, 64, 100) == -1 and dec(1, 4, 2, 60, 100) == -1
    assert pre(5, 1, 4, 2, 264, 100) == -1 and pre(-1, 1, 4, 2, 64, 100) == -1
    assert dec(0, 4, 2, 64, 100) == 0 and pre(0, 0, 4, 2, 64, 100) == 0
    assert dec(1, 32, 32, 128, 4096) >= 0 and pre(16, 1, 32, 8, 128, 1 << 17) >= 0
