"""Windows, trees of drafted tokens, accepted paths and log probabilities
without a GPU: masks and states, and refusals before any launch."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nanopointllm_amd import _lib, attention as A, lm_head as L
from oracle import drafts_oracle as O

S, N, D, AL, OV, WS_ = (_lib.ERR_SHAPE, _lib.ERR_NULL, _lib.ERR_DTYPE, _lib.ERR_ALIGN,
                        _lib.ERR_OVERLAP, _lib.ERR_WORKSPACE)
Q, K, OUT = 0x1000000, 0x2000000, 0x4000000
KC, VC, AUX, WS = 0x10000000, 0x20000000, 0x5000000, 0x6000000


def _p(addr):
    return None if addr is None else ctypes.c_void_p(addr)


# -------------------------------------------------------------------- masks
def test_masks_of_trees():
    chain = A.tree_masks([[-1, 0, 1, 2]], device="cpu")
    assert chain.dtype == torch.int64 and chain[:, 0].tolist() == [1, 3, 7, 15]
    forest = A.tree_masks([[-1, -1, 0, 1, 2], [], [-1]], device="cpu")
    assert forest[:, 0].tolist() == [1, 2, 5, 10, 21, 1]
    assert A.tree_masks([], device="cpu").shape == (0, 1)
    long = A.tree_masks([list(range(-1, 199)), [-1, 0]], device="cpu")
    assert long.shape == (202, 4)
    # Chains see as prompts do.
    assert torch.equal(O.tree_sight(long[:200], 230), O.window_sight(200, 230, None, 0))
    assert long[63].tolist() == [-1, 0, 0, 0] and long[199].tolist() == [-1, -1, -1, 255]
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1, 0, 3]]):
        with pytest.raises(ValueError, match="parent"):
            A.tree_masks(bad, device="cpu")


def test_state_of_drafts():
    s = A.AttentionState.build_drafts([[3, 1], [2], [0]], [5, 2, 7], [[-1, 0, 0, 1], [-1], []], 8,
                                      device="cpu")
    assert s.positions.tolist() == [5, 6, 6, 7, 2]
    assert s.slots.tolist() == [3 * 8 + 5, 3 * 8 + 6, 3 * 8 + 7, 8, 2 * 8 + 2]
    assert s.lengths.tolist() == [9, 3, 7] and s.q_starts.tolist() == [0, 4, 5, 5]
    assert s.decode_rows == 0 and s.masks[:, 0].tolist() == [1, 3, 5, 11, 1]
    # One drafted token each is a tree too, not a decode step.
    one = A.AttentionState.build_drafts([[0], [1]], [3, 4], [[-1], [-1]], 8, device="cpu")
    assert one.decode_rows == 0 and one.q_starts.tolist() == [0, 1, 2]
    with pytest.raises(ValueError, match="hold"):
        A.AttentionState.build_drafts([[0]], [7], [[-1, 0]], 8, device="cpu")
    with pytest.raises(ValueError, match="one entry"):
        A.AttentionState.build_drafts([[0]], [7], [], 8, device="cpu")


# ------------------------------------------------------- refusals in Python
@pytest.mark.parametrize("window,sinks", [(8, 2 ** 64), (8, 2 ** 64 + 3), (2 ** 64 + 8, 2)])
def test_numbers_past_64_bits_are_refused(window, sinks):
    """Not cut to their lower bits."""
    cache = A.PagedKVCache(1, 1, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="sinks" if sinks > 8 else "window"):
        A.PagedAttentionCore(cache, None, window=window, sinks=sinks)


def test_windows_refused():
    cache = A.PagedKVCache(2, 1, 1, 64, device="cpu")
    for window, sinks, message in ((0, 0, "window"), (-3, 0, "window"), (2.0, 0, "window"),
                                   (True, 0, "window"), (5, -1, "sinks"), (5, 1.0, "sinks"),
                                   (None, 3, "sinks"), ([4], 0, "each"), ([4, 0], 0, "window"),
                                   ([None, None], 2, "sinks")):
        with pytest.raises(ValueError, match=message):
            A.PagedAttentionCore(cache, None, window=window, sinks=sinks)
    core = A.PagedAttentionCore(cache, None, window=[None, 4], sinks=2)
    state = A.AttentionState.build_drafts([[0]], [3], [[-1]], 16, device="cpu")
    q = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="without a window"):
        core(q, q, q, 1, state)
    state.q_starts = None
    with pytest.raises(ValueError, match="q_starts"):
        core(q, q, q, 0, state)
    with pytest.raises(ValueError, match="sinks"):
        A.paged_prefill(q, *[None] * 5, sinks=1)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 8, dtype=torch.float16)
    c = torch.zeros(1, 2, 4, 8, dtype=torch.float16)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        A.paged_tree(q, c, c, one[None], one, one, one.long()[None])
    with pytest.raises(RuntimeError, match="only on the GPU"):
        A.paged_accept(c, c, one[None], one, one[None])
    with pytest.raises(RuntimeError, match="only on the GPU"):
        A.paged_decode(q, c, c, one[None], one, window=4)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        L.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))


# ----------------------------------------------------- the C ABI's refusals
def _attend(name, extra, *, q=Q, qs=(256, 64), kc=KC, vc=VC, cs=(2048, 1024, 64), pages=4,
            page=16, table=AUX, ld=4, n=4, lengths=AUX, starts=AUX, dtype=_lib.F16, scale=0.125,
            out=OUT, os=(256, 64), t=5, b=3, h=4, g=2, d=64, ws=WS, wb=1 << 30):
    lib = _lib.load()
    head = (_p(q), *qs, _p(kc), _p(vc), *cs, pages, page, _p(table), ld, n, _p(lengths))
    tail = (dtype, scale, _p(out), *os)
    if name == "w8a8_paged_decode_window":
        return getattr(lib, name)(*head, *extra, *tail, b, h, g, d, _p(ws), wb, None)
    return getattr(lib, name)(*head, _p(starts), *extra, *tail, t, b, h, g, d, _p(ws), wb, None)


def _decode(*, window=7, sinks=1, t=None, starts=None, **kw):
    return _attend("w8a8_paged_decode_window", (window, sinks), **kw)


def _prefill(*, window=7, sinks=1, clear=0, **kw):
    return _attend("w8a8_paged_prefill_window", (window, sinks, clear), **kw)


def _tree(*, masks=AUX, ld_masks=2, words=2, clear=0, **kw):
    return _attend("w8a8_paged_tree", (_p(masks), ld_masks, words, clear), **kw)


@pytest.mark.parametrize("call", [_decode, _prefill, _tree])
def test_attention_refusals(call):
    assert call(dtype=_lib.F32) == D
    assert call(d=60) == S and call(d=264) == S and call(h=5) == S and call(g=0) == S
    assert call(page=24) == S and call(pages=-1) == S and call(ld=3) == S
    assert call(b=-1) == S and call(scale=math.nan) == S
    for name in ("q", "kc", "vc", "table", "lengths", "out"):
        assert call(**{name: None}) == N, name
    for name in ("q", "kc", "vc", "out"):
        assert call(**{name: 0x7000008}) == AL, name
    assert call(qs=(260, 64)) == AL and call(cs=(2048, 1024, 68)) == AL
    assert call(out=Q) == OV and call(out=KC) == OV and call(os=(64, 64)) == OV
    assert call(b=0, t=0, q=None, out=None) == _lib.OK
    if call is not _tree:
        assert call(window=0) == S and call(window=-1) == S and call(sinks=-1) == S
    if call is not _decode:
        assert call(starts=None) == N and call(starts=AUX + 2) == AL
        assert call(t=0, q=None) == _lib.OK and call(t=-1) == S
        assert call(b=0, clear=1) == S
    if call is _tree:
        assert call(words=-1) == S and call(ld_masks=1) == S and call(words=1 << 31,
                                                                     ld_masks=1 << 31) == S
        assert call(masks=None) == N and call(masks=AUX + 4) == AL and call(masks=OUT) == OV


def test_workspaces():
    lib = _lib.load()
    dec, pre, tree = (lib.w8a8_paged_decode_window_workspace_bytes,
                      lib.w8a8_paged_prefill_window_workspace_bytes,
                      lib.w8a8_paged_tree_workspace_bytes)
    assert dec(1, 4, 3, 64, 100, 5, 0) == -1 and dec(1, 4, 2, 64, 100, 0, 0) == -1
    assert pre(5, 1, 4, 2, 264, 100, 5, 0) == -1 and pre(5, 1, 4, 2, 64, 100, 5, -1) == -1
    assert tree(-1, 1, 4, 2, 64, 100) == -1 and tree(5, 1, 4, 2, 60, 100) == -1
    assert tree(5, 1, 4, 2, 64, -1) == -1 and tree(5, 1, 4, 2, 64, 1 << 32) == -1
    assert tree(0, 0, 4, 2, 64, 64) == 0 < tree(300, 1, 8, 2, 64, 1 << 14)
    assert tree(5, 1, 4, 2, 64, 128) == 0 < tree(5, 1, 4, 2, 64, 1 << 14)
    # By what is seen, not by the table's width; all of it for a wide window.
    assert dec(1, 32, 8, 128, 1 << 17, 100, 4) == 0 < dec(1, 32, 8, 128, 1 << 17, 1 << 16, 4)
    assert dec(1, 32, 8, 128, 1 << 17, 1 << 17, 4) == \
        lib.w8a8_paged_decode_workspace_bytes(1, 32, 8, 128, 1 << 17)
    assert pre(16, 1, 32, 8, 128, 1 << 17, 100, 4) == 0 < pre(16, 1, 32, 8, 128, 1 << 17, 9999, 4)
    long = dict(n=1 << 13, ld=1 << 13, b=1, wb=16)
    assert _decode(window=1 << 16, **long) == WS_ and _prefill(window=1 << 16, **long) == WS_
    assert _tree(**long) == WS_ and _tree(**{**long, "wb": 1 << 30}, ws=WS + 8) == AL


def _accept(*, kc=KC, vc=VC, cl=1 << 20, cs=(2048, 1024, 64), layers=2, pages=4, page=16,
            table=AUX, ld=4, n=4, lengths=AUX, path=AUX, ld_path=5, steps=5, dtype=_lib.F16, b=3,
            g=2, d=64):
    return _lib.load().w8a8_cache_accept(
        _p(kc), _p(vc), cl, *cs, layers, pages, page, _p(table), ld, n, _p(lengths), _p(path),
        ld_path, steps, dtype, b, g, d, None)


def test_accept_refusals():
    assert _accept(dtype=_lib.F32) == D
    assert _accept(d=60) == S and _accept(d=264) == S and _accept(g=0) == S
    assert _accept(page=24) == S and _accept(pages=-1) == S and _accept(ld=3) == S
    assert _accept(b=-1) == S and _accept(b=65536) == S and _accept(layers=32768) == S
    assert _accept(steps=-1) == S and _accept(ld_path=4) == S and _accept(cl=-8) == S
    for name in ("kc", "vc", "table", "lengths", "path"):
        assert _accept(**{name: None}) == N, name
        assert _accept(**{name: 0x7000002 if name in ("kc", "vc") else AUX + 2}) == AL, name
    assert _accept(cl=(1 << 20) + 4) == AL and _accept(cs=(2048, 1024, 60)) == AL
    assert _accept(vc=KC) == OV and _accept(cl=64) == OV and _accept(cs=(1024, 1024, 64)) == OV
    assert _accept(path=KC + 64) == OV and _accept(table=VC) == OV
    # A layer's k and v side by side, and k and v that meet between the layers.
    assert _accept(vc=KC + 2 * 8192, cl=16384, b=0) == _lib.OK
    assert _accept(vc=KC + 2 * 4096, cl=16384) == OV
    for nothing in ("b", "layers", "pages", "n", "steps"):
        assert _accept(**{nothing: 0}, kc=None) == _lib.OK, nothing


def _logprobs(*, x=Q, ld=1000, dtype=_lib.F16, tokens=K, ld_tokens=2, given=2, top=3, y=OUT,
              entropy=OUT + 0x10000, best=OUT + 0x20000, ids=OUT + 0x30000, rows=5, vocab=1000,
              ws=WS, wb=1 << 30):
    return _lib.load().w8a8_token_logprobs(
        _p(x), ld, dtype, _p(tokens), ld_tokens, given, top, _p(y), _p(entropy), _p(best), _p(ids),
        rows, vocab, _p(ws), wb, None)


def test_logprobs_refusals():
    assert _logprobs(dtype=_lib.I8) == D
    assert _logprobs(vocab=0) == S and _logprobs(vocab=(1 << 20) + 1) == S
    assert _logprobs(top=65) == S and _logprobs(top=-1) == S and _logprobs(vocab=2) == S
    assert _logprobs(rows=-1) == S and _logprobs(rows=1 << 22) == S and _logprobs(given=-1) == S
    assert _logprobs(ld=-1) == S and _logprobs(ld_tokens=-1) == S
    for name in ("x", "tokens", "y", "best", "ids"):
        assert _logprobs(**{name: None}) == N, name
    for name in ("x", "tokens", "y", "entropy", "best", "ids"):
        assert _logprobs(**{name: 0x7000001}) == AL, name
    assert _logprobs(y=Q) == OV and _logprobs(entropy=K) == OV and _logprobs(ids=OUT) == OV
    assert _logprobs(rows=0, x=None) == _lib.OK
    sizes = _lib.load().w8a8_token_logprobs_workspace_bytes
    assert sizes(5, 0, 0, _lib.F16) == -1 and sizes(5, 100, 101, _lib.F16) == -1
    assert sizes(5, 100, 5, _lib.I8) == -1 and sizes(5, 100, 5, _lib.F16) >= 0


def test_logprobs_shapes_are_checked():
    x, t = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)

    class OnGpu(torch.Tensor):
        is_cuda = True

    for bad_x, bad_t, top, message in (
            (x.double(), t, 0, "float16"), (x, t.int(), 0, "int64"), (x, t[:1], 0, "int64"),
            (x, t[..., None, None], 0, "int64"), (x, t, 6, "top"), (x, t, -1, "top"),
            (x, t, True, "top"), (x[..., :0], t, 0, "vocabulary")):
        with pytest.raises(ValueError, match=message):
            L.token_logprobs(bad_x.as_subclass(OnGpu), bad_t.as_subclass(OnGpu), top=top)
