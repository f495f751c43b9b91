"""The attention core of a decoder stack on the GPU: rotary positions, a paged
key-value cache, and attention over it.

The counterpart of the precomputed branch of ``PagedLlamaAttention.forward``
(nanopointllm/llama/paged_attention.py:1284-1307, 1354-1440):

* :func:`rotary` and :func:`rotary_store` - rotary positions (half or
  interleaved pairs, all or part of a head, frequencies scaled for long
  contexts by :func:`rotary_frequencies`), the second with the store of the
  rotated keys and the values into the cache in the same launch;
* :func:`paged_decode` - attention of one new token per sequence, split over
  the cache's length where there are few sequences;
* :func:`paged_prefill` - causal attention of prompts, or of chunks of them
  behind a cached part, in a ragged batch; both also with a sliding window and
  sinks, whose keys are the only ones read;
* :func:`paged_tree` - attention of trees of drafted tokens (:func:`tree_masks`)
  and :func:`paged_accept`, which keeps their accepted paths in the cache;
* :class:`PagedAttentionCore` - these as the attention core that
  :class:`nanopointllm_amd.runner.W8A8LlamaRunner` calls, with
  :class:`PagedKVCache` and :class:`AttentionState`.

A cache is a pair of tensors ``[pages, kv_heads, page_size, head_dim]`` with
equal strides, the last axis contiguous and the others in any order (a
``[pages, page_size, kv_heads, head_dim]`` cache goes in as
``cache.transpose(1, 2)``).  Rows are float16 or bfloat16, as the runner's.
Every call enqueues on torch's current stream, allocates from torch's caching
allocator only and never synchronizes, so it can be captured into a HIP graph;
lengths, positions, slots and the page table are read on the device and may
change between replays.  There is no CPU path and no autograd.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from functools import lru_cache
from typing import Any, NamedTuple, Sequence

import torch

from . import _lib

MAX_HEAD_DIM = 256

_LAYOUTS = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}


# ------------------------------------------------------------- frequencies
class RotaryFrequencies(NamedTuple):
    inv_freq: torch.Tensor    # float64 [rotary_dim / 2], radians per position
    attention_factor: float   # amplitude of cos and sin


# The keys of a scaling dictionary that each kind needs, and those that it may
# have besides its name and the base.
_SCALING_KEYS = {
    "default": ((), ("factor",)),
    "linear": (("factor",), ()),
    "ntk": (("factor",), ()),
    "llama3": (("factor", "original_max_position_embeddings", "low_freq_factor",
                "high_freq_factor"), ()),
    "yarn": (("factor", "original_max_position_embeddings"),
             ("beta_fast", "beta_slow", "truncate", "attention_factor", "mscale",
              "mscale_all_dim")),
}


def _scaling_of(scaling: dict[str, Any] | None, base: float) -> tuple[str, dict[str, Any]]:
    """(kind, its values as numbers); a key of None is one left out."""
    given = {k: v for k, v in (scaling or {}).items() if v is not None}
    kind = given.pop("rope_type", given.get("type", "default"))
    if given.pop("type", kind) != kind:
        raise ValueError("rope_type and type of the rotary scaling differ")
    if kind not in _SCALING_KEYS:
        raise ValueError(f"unknown rotary scaling {kind!r}")
    if given.pop("rope_theta", base) != base:
        raise ValueError("rope_theta of the rotary scaling is not the given base")
    needed, optional = _SCALING_KEYS[kind]
    for key in needed:
        if key not in given:
            raise ValueError(f"{kind} rotary scaling needs {key}")
    for key, value in given.items():
        if key not in needed + optional:
            raise ValueError(f"{kind} rotary scaling does not use {key}")
        if key == "truncate":
            if not isinstance(value, bool):
                raise ValueError("truncate of the rotary scaling must be a truth value")
            continue
        try:
            given[key] = float(value)
        except (TypeError, ValueError):
            given[key] = math.nan
        if not 0.0 < given[key] < math.inf:
            raise ValueError(f"{key} of the rotary scaling must be a positive number")
    return kind, given


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0,
                       scaling: dict[str, Any] | None = None,
                       device: torch.device | str = "cuda") -> RotaryFrequencies:
    """``base ** (-2 i / rotary_dim)`` for the pairs of ``rotary_dim`` elements,
    optionally scaled for contexts longer than the model was trained on.

    ``scaling`` is a ``rope_scaling`` dictionary of a Hugging Face config; its
    ``rope_type`` (or ``type``) is one of

    * ``"default"``: unscaled;
    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: the base raised to ``base * factor ** (d / (d - 2))``;
    * ``"llama3"``: frequencies whose wavelength is past
      ``original_max_position_embeddings / low_freq_factor`` divided by
      ``factor``, those below ``.../high_freq_factor`` kept, blended between;
    * ``"yarn"``: blended by the number of turns over
      ``original_max_position_embeddings``, from ``beta_fast`` (32) to
      ``beta_slow`` (1), the pairs of both as whole numbers outwards unless
      ``truncate`` is False; with the amplitude ``attention_factor``, else
      ``s(mscale) / s(mscale_all_dim)`` where both are given, else ``s(1)``, of
      ``s(m) = 0.1 m ln(factor) + 1``.

    A key that is missing, or that the kind does not use, is refused, and so
    is a ``rope_theta`` that is not ``base``."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    if not 0 < base < math.inf:
        raise ValueError("the rotary base must be positive")
    kind, given = _scaling_of(scaling, base)
    factor = given.get("factor", 1.0)
    if not factor >= 1.0:
        raise ValueError("the rotary scaling factor must be at least 1")
    if kind == "default" and factor != 1.0:
        raise ValueError("unscaled rotary frequencies do not use factor")
    d = rotary_dim
    if kind == "ntk" and d > 2:
        base = base * factor ** (d / (d - 2))
    i = torch.arange(d // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / max(d, 1))
    amplitude = 1.0
    if kind == "linear":
        freq = freq / factor
    elif kind == "llama3":
        context = given["original_max_position_embeddings"]
        low, high = given["low_freq_factor"], given["high_freq_factor"]
        if not low < high:
            raise ValueError("llama3 scaling needs 0 < low_freq_factor < high_freq_factor")
        kept = ((context * freq / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (kept + (1.0 - kept) / factor)
    elif kind == "yarn":
        context = given["original_max_position_embeddings"]
        fast, slow = given.get("beta_fast", 32.0), given.get("beta_slow", 1.0)
        if fast < slow:
            raise ValueError("yarn scaling needs beta_slow <= beta_fast")
        if not base > 1.0:
            raise ValueError("yarn scaling needs a rotary base above 1")

        def pair_of(turns: float) -> float:   # the pair that turns so often in the context
            return d * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = pair_of(fast), pair_of(slow)
        if given.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, d - 1)
        slowed = ((i - low) / (high - low if high != low else 0.001)).clamp(0.0, 1.0)
        freq = freq * (1.0 - slowed + slowed / factor)

        def size(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0

        if ("mscale" in given) != ("mscale_all_dim" in given):
            raise ValueError("yarn scaling takes mscale and mscale_all_dim together")
        amplitude = given.get("attention_factor")
        if amplitude is None:
            amplitude = (size(given["mscale"]) / size(given["mscale_all_dim"])
                         if "mscale" in given else size(1.0))
    return RotaryFrequencies(freq.to(device), amplitude)


# ------------------------------------------------------- checks and launches
# A decode step runs every call here once per layer, eagerly bounded by the
# host: each wrapper reads an attribute once and compares devices by number
# (a small call takes 11 us in all, with general helpers 15).
_CODES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _gpu(*tensors: torch.Tensor | None) -> int:
    """The number of the one GPU that the tensors are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index or index < 0:
            _lib.require_cuda(*tensors)    # raises, naming the reason
    return index


def _rows(x: torch.Tensor, name: str) -> int:
    """The dtype code of 16-bit ``[tokens, heads, head_dim]`` rows."""
    code = _CODES.get(x.dtype)
    if code is None or x.dim() != 3:
        raise ValueError(f"{name} must be float16 / bfloat16 [tokens, heads, head_dim]")
    return code


def _out_like(out: torch.Tensor | None, q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have the queries' shape, dtype and device")
    if out.stride(2) != 1 and out.shape[2] > 1:
        raise ValueError("out must have contiguous heads")
    return out


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, q: torch.Tensor, d: int
           ) -> tuple[tuple[int, ...], tuple[int, ...]]:
    """(shape, strides) of the two cache tensors."""
    shape, strides = k_cache.shape, k_cache.stride()
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be [pages, kv_heads, page_size, head_dim]")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("the cache must have the rows' dtype")
    if shape[3] != d:
        raise ValueError("the cache and the rows must have one head_dim")
    if strides[3] != 1 or strides != v_cache.stride() and any(
            n > 1 and a != b for n, a, b in zip(shape, strides, v_cache.stride())):
        raise ValueError("k_cache and v_cache must have equal strides and contiguous heads")
    return shape, strides


def _index(t: torch.Tensor, dtype: torch.dtype, count: int, name: str) -> torch.Tensor:
    if t.dtype != dtype or t.shape != (count,):
        raise ValueError(f"{name} must be {str(dtype)[6:]} with {count} values")
    return t if t.is_contiguous() else t.contiguous()


def _frequencies(inv_freq: torch.Tensor, head_dim: int) -> torch.Tensor:
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1:
        raise ValueError("inv_freq must be a float64 vector (rotary_frequencies)")
    if 2 * inv_freq.shape[0] > head_dim:
        raise ValueError("inv_freq has more pairs than a head")
    return inv_freq if inv_freq.is_contiguous() else inv_freq.contiguous()


def _layout(layout: str) -> int:
    try:
        return _LAYOUTS[layout]
    except KeyError:
        raise ValueError("rotary layout must be 'half' or 'interleaved'") from None


# ------------------------------------------------------------------- rotary
def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
           layout: str = "half", attention_factor: float = 1.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows ``x [tokens, heads, head_dim]`` turned to their ``positions``
    (int64 ``[tokens]``): pair ``i`` of the first ``2 * len(inv_freq)``
    elements by ``positions * inv_freq[i]`` radians, times
    ``attention_factor``; the rest of each head is copied.  ``layout``:
    ``"half"`` pairs elements ``(i, i + len(inv_freq))``, ``"interleaved"``
    neighbours.  ``out`` may be ``x`` itself."""
    index = _gpu(x, positions, inv_freq, out)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return rotary(x, positions, inv_freq, layout=layout,
                          attention_factor=attention_factor, out=out)
    code = _rows(x, "x")
    if out is not x and x.stride(2) != 1 and x.shape[2] > 1:
        x = x.contiguous()
    t, h, d = x.shape
    positions = _index(positions, torch.int64, t, "positions")
    freq = _frequencies(inv_freq, d)
    out = _out_like(out, x)
    xs, os = x.stride(), out.stride()
    _lib.check(_lib.load().w8a8_rotary(
        x.data_ptr(), xs[0], xs[1], code, positions.data_ptr(), freq.data_ptr(),
        2 * freq.shape[0], _layout(layout), attention_factor, out.data_ptr(), os[0], os[1], t, h,
        d, torch._C._cuda_getCurrentRawStream(index)), "w8a8_rotary")
    return out


def rotary_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                 slots: torch.Tensor, inv_freq: torch.Tensor, k_cache: torch.Tensor,
                 v_cache: torch.Tensor, *, layout: str = "half", attention_factor: float = 1.0,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`rotary` of ``q``, returned (``out`` may be ``q`` itself), and in
    the same launch the rotated ``k`` and the values ``v`` (both ``[tokens,
    kv_heads, head_dim]``) into the cache: token ``t`` at row
    ``slots[t] % page_size`` of page ``slots[t] // page_size`` (int64
    ``[tokens]``, distinct; a slot outside the cache, such as a padded row's
    -1, is not written).  q, k and v may be views of one packed matrix."""
    index = _gpu(q, k, v, positions, slots, inv_freq, k_cache, v_cache, out)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return rotary_store(q, k, v, positions, slots, inv_freq, k_cache, v_cache,
                                layout=layout, attention_factor=attention_factor, out=out)
    code = _CODES.get(q.dtype)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    if code is None or not len(qs) == len(ks) == len(vs) == 3:
        raise ValueError("q, k and v must be float16 / bfloat16 [tokens, heads, head_dim]")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have one dtype")
    t, h, d = q.shape
    shape = k.shape
    if shape != v.shape or shape[0] != t or shape[2] != d:
        raise ValueError("k and v must be [tokens, kv_heads, head_dim] rows of q's tokens")
    if not qs[2] == ks[2] == vs[2] == 1 and d > 1:
        if out is not q:
            q = q.contiguous()
        k, v = k.contiguous(), v.contiguous()
        qs, ks, vs = q.stride(), k.stride(), v.stride()
    (pages, g, page_size, _), cs = _cache(k_cache, v_cache, q, d)
    if g != shape[1]:
        raise ValueError("the cache and k must have the same heads")
    positions = _index(positions, torch.int64, t, "positions")
    slots = _index(slots, torch.int64, t, "slots")
    freq = _frequencies(inv_freq, d)
    out = _out_like(out, q)
    os = out.stride()
    _lib.check(_lib.load().w8a8_rotary_store(
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], code,
        positions.data_ptr(), slots.data_ptr(), freq.data_ptr(), 2 * freq.shape[0],
        _layout(layout), attention_factor, out.data_ptr(), os[0], os[1], k_cache.data_ptr(),
        v_cache.data_ptr(), cs[0], cs[1], cs[2], pages, page_size, t, h, g, d,
        torch._C._cuda_getCurrentRawStream(index)), "w8a8_rotary_store")
    return out


# ---------------------------------------------------------------- attention
@lru_cache(maxsize=1024)
def _decode_workspace(batch: int, heads: int, kv_heads: int, dim: int, max_keys: int) -> int:
    return int(_lib.load().w8a8_paged_decode_workspace_bytes(batch, heads, kv_heads, dim,
                                                             max_keys))


@lru_cache(maxsize=1024)
def _prefill_workspace(tokens: int, batch: int, heads: int, kv_heads: int, dim: int,
                       max_keys: int) -> int:
    return int(_lib.load().w8a8_paged_prefill_workspace_bytes(tokens, batch, heads, kv_heads,
                                                              dim, max_keys))


@lru_cache(maxsize=1024)
def _decode_window_workspace(batch: int, heads: int, kv_heads: int, dim: int, max_keys: int,
                             window: int, sinks: int) -> int:
    return int(_lib.load().w8a8_paged_decode_window_workspace_bytes(
        batch, heads, kv_heads, dim, max_keys, window, sinks))


@lru_cache(maxsize=1024)
def _prefill_window_workspace(tokens: int, batch: int, heads: int, kv_heads: int, dim: int,
                              max_keys: int, window: int, sinks: int) -> int:
    return int(_lib.load().w8a8_paged_prefill_window_workspace_bytes(
        tokens, batch, heads, kv_heads, dim, max_keys, window, sinks))


@lru_cache(maxsize=1024)
def _tree_workspace(tokens: int, batch: int, heads: int, kv_heads: int, dim: int,
                    max_keys: int) -> int:
    return int(_lib.load().w8a8_paged_tree_workspace_bytes(tokens, batch, heads, kv_heads, dim,
                                                           max_keys))


def _window(window: int | None, sinks: int) -> None:
    if type(sinks) is not int or not 0 <= sinks < 1 << 62:
        raise ValueError("sinks must be a whole number of at least 0")
    if window is None:
        if sinks:
            raise ValueError("sinks need a window")
    elif type(window) is not int or not 1 <= window < 1 << 62:
        raise ValueError("window must be a whole number of at least 1, or None")


def _queries(q: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """Query rows whose addresses the kernels' 16-byte loads take: a copy where
    q's are not (not by contiguous(), which returns a contiguous view at an odd
    address, or of one row with a stride of its own, as it is)."""
    strides = q.stride()
    if strides[2] != 1 or strides[0] % 8 or strides[1] % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        strides = q.stride()
    return q, strides


def _table(page_table: torch.Tensor, batch: int) -> tuple[torch.Tensor, int, int]:
    """(table, its row stride, pages per row)."""
    shape = page_table.shape
    if page_table.dtype != torch.int32 or len(shape) != 2 or shape[0] != batch:
        raise ValueError("page_table must be int32 [batch, pages of the longest sequence]")
    strides = page_table.stride()
    if strides[0] < shape[1] or strides[1] != 1 and shape[1] > 1:
        page_table = page_table.contiguous()
        strides = page_table.stride()
    return page_table, max(strides[0], shape[1]), shape[1]


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, *,
                 scale: float | None = None, window: int | None = None, sinks: int = 0,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence, ``q [batch, heads, head_dim]``,
    over the first ``lengths[b]`` keys of the cache (the new one is already in
    it).  ``page_table`` int32 ``[batch, n]`` names each sequence's pages,
    ``lengths`` int32 ``[batch]``; a length of zero (a padded row) gives zeros,
    table entries past a sequence's pages are not used.  ``heads`` is a
    multiple of the cache's heads, which consecutive queries share.  ``scale``
    defaults to ``head_dim ** -0.5``.  A NaN or infinite value among a row's
    keys makes the elements that it enters NaN or infinite, one behind its
    length does nothing.

    With a ``window`` a sequence's row sees its last ``window`` keys and its
    first ``sinks`` only; the keys between are not read, and pages that hold no
    others may be gone (their table entries are not used)."""
    index = _gpu(q, k_cache, v_cache, page_table, lengths, out)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return paged_decode(q, k_cache, v_cache, page_table, lengths, scale=scale,
                                window=window, sinks=sinks, out=out)
    if window is not None or sinks:
        _window(window, sinks)
    code = _rows(q, "q")
    q, qs = _queries(q)
    b, h, d = q.shape
    (pages, g, page_size, _), cs = _cache(k_cache, v_cache, q, d)
    page_table, ld, width = _table(page_table, b)
    lengths = _index(lengths, torch.int32, b, "lengths")
    out = _out_like(out, q)
    os = out.stride()
    if window is not None:
        need = _decode_window_workspace(b, h, g, d, width * page_size, window, sinks)
        ws = q.new_empty(((need + 1) // 2,)) if need > 0 else None
        _lib.check(_lib.load().w8a8_paged_decode_window(
            q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1],
            cs[2], pages, page_size, page_table.data_ptr(), ld, width, lengths.data_ptr(), window,
            sinks, code, d ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1], b, h,
            g, d, None if ws is None else ws.data_ptr(), need,
            torch._C._cuda_getCurrentRawStream(index)), "w8a8_paged_decode_window")
        return out
    need = _decode_workspace(b, h, g, d, width * page_size)
    ws = q.new_empty(((need + 1) // 2,)) if need > 0 else None
    _lib.check(_lib.load().w8a8_paged_decode(
        q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2],
        pages, page_size, page_table.data_ptr(), ld, width, lengths.data_ptr(), code,
        d ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1], b, h, g, d,
        None if ws is None else ws.data_ptr(), need, torch._C._cuda_getCurrentRawStream(index)),
        "w8a8_paged_decode")
    return out


def paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  page_table: torch.Tensor, lengths: torch.Tensor, q_starts: torch.Tensor, *,
                  scale: float | None = None, window: int | None = None, sinks: int = 0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of prompts or prompt chunks in a ragged batch: rows
    ``q_starts[b] .. q_starts[b + 1] - 1`` of ``q [tokens, heads, head_dim]``
    (int32 ``[batch + 1]``, not decreasing) are the newest tokens of sequence
    ``b``, whose ``lengths[b]`` keys, theirs among them, are in the cache.  The
    last row sees all of them, each row before it one fewer; a row that sees
    none is zeros.  Rows of no sequence (a padded batch's) are zeros too, but
    in a given ``out`` they keep what they hold.  With a ``window`` a row sees,
    of these, its own key and the ``window - 1`` before it, and the sequence's
    first ``sinks``.  Otherwise as :func:`paged_decode`."""
    if window is not None or sinks:
        _window(window, sinks)
    return _prefill(q, k_cache, v_cache, page_table, lengths, q_starts, scale, out, out is None,
                    window, sinks)


def paged_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               page_table: torch.Tensor, lengths: torch.Tensor, q_starts: torch.Tensor,
               masks: torch.Tensor, *, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of trees of drafted tokens: rows ``q_starts[b] .. q_starts[b +
    1] - 1`` of ``q`` are the ``n`` drafted tokens of sequence ``b``, whose keys
    are the last ``n`` of its ``lengths[b]`` in the cache.  Each row sees all
    keys before those, and of the drafted ones key ``j`` where bit ``j % 64`` of
    ``masks[row, j // 64]`` is set (int64 ``[tokens, words]``, see
    :func:`tree_masks`; a row sees itself only if its own bit is set, and no key
    past the words).  A row that sees no key is zeros.

    Trees of at most 64 rows (tokens x query heads of a key head) per sequence, on
    the call's average, and heads of at most 128 have :func:`paged_decode`'s
    arithmetic, others :func:`paged_prefill`'s, whose probabilities are rounded to
    the rows' type: a tree's last bits, and how fast it runs, depend on the trees
    that it is called with.  Otherwise as :func:`paged_prefill`."""
    return _prefill(q, k_cache, v_cache, page_table, lengths, q_starts, scale, out, out is None,
                    None, 0, masks)


def _masks(masks: torch.Tensor, tokens: int) -> tuple[torch.Tensor, int, int]:
    """(masks, their row stride, words per row)."""
    shape = masks.shape
    if masks.dtype != torch.int64 or len(shape) != 2 or shape[0] != tokens:
        raise ValueError("masks must be int64 [tokens, words]")
    if masks.stride(0) < shape[1] or masks.stride(1) != 1 and shape[1] > 1:
        masks = masks.contiguous()
    return masks, max(masks.stride(0), shape[1]), shape[1]


def _prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             page_table: torch.Tensor, lengths: torch.Tensor, q_starts: torch.Tensor,
             scale: float | None, out: torch.Tensor | None, clear: bool,
             window: int | None = None, sinks: int = 0, masks: torch.Tensor | None = None
             ) -> torch.Tensor:
    """:func:`paged_prefill` and, with masks, :func:`paged_tree`; ``clear``: rows
    of no sequence become zeros."""
    index = _gpu(q, k_cache, v_cache, page_table, lengths, q_starts, out, masks)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _prefill(q, k_cache, v_cache, page_table, lengths, q_starts, scale, out, clear,
                            window, sinks, masks)
    code = _rows(q, "q")
    q, qs = _queries(q)
    t, h, d = q.shape
    (pages, g, page_size, _), cs = _cache(k_cache, v_cache, q, d)
    b = lengths.shape[0] if lengths.dim() == 1 else -1
    page_table, ld, width = _table(page_table, b)
    lengths = _index(lengths, torch.int32, b, "lengths")
    q_starts = _index(q_starts, torch.int32, b + 1, "q_starts")
    out = _out_like(out, q)
    os = out.stride()
    if masks is not None or window is not None:
        return _prefill_masked(q, k_cache, v_cache, page_table, lengths, q_starts, scale, out,
                               clear, window, sinks, masks, ld, width, code, index)
    need = _prefill_workspace(t, b, h, g, d, width * page_size)
    ws = q.new_empty(((need + 1) // 2,)) if need > 0 else None
    if clear and b == 0:
        return out.zero_()
    lib = _lib.load()
    _lib.check((lib.w8a8_paged_prefill_padded if clear else lib.w8a8_paged_prefill)(
        q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1], cs[2],
        pages, page_size, page_table.data_ptr(), ld, width, lengths.data_ptr(),
        q_starts.data_ptr(), code, d ** -0.5 if scale is None else scale, out.data_ptr(), os[0],
        os[1], t, b, h, g, d, None if ws is None else ws.data_ptr(), need,
        torch._C._cuda_getCurrentRawStream(index)), "w8a8_paged_prefill")
    return out


def _prefill_masked(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, q_starts: torch.Tensor,
                    scale: float | None, out: torch.Tensor, clear: bool, window: int | None,
                    sinks: int, masks: torch.Tensor | None, ld: int, width: int, code: int,
                    index: int) -> torch.Tensor:
    """The windowed and the tree call of :func:`_prefill`, whose arguments are
    checked."""
    (t, h, d), (pages, g, page_size, _), b = q.shape, k_cache.shape, lengths.shape[0]
    qs, cs, os = q.stride(), k_cache.stride(), out.stride()
    if masks is not None:
        masks, ld_masks, words = _masks(masks, t)
        need = _tree_workspace(t, b, h, g, d, width * page_size)
    else:
        need = _prefill_window_workspace(t, b, h, g, d, width * page_size, window, sinks)
    if clear and b == 0:
        return out.zero_()
    ws = q.new_empty(((need + 1) // 2,)) if need > 0 else None
    given = (q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), cs[0], cs[1],
             cs[2], pages, page_size, page_table.data_ptr(), ld, width, lengths.data_ptr(),
             q_starts.data_ptr())
    rest = (clear, code, d ** -0.5 if scale is None else scale, out.data_ptr(), os[0], os[1], t, b,
            h, g, d, None if ws is None else ws.data_ptr(), need,
            torch._C._cuda_getCurrentRawStream(index))
    lib = _lib.load()
    if masks is not None:
        _lib.check(lib.w8a8_paged_tree(*given, masks.data_ptr(), ld_masks, words, *rest),
                   "w8a8_paged_tree")
    else:
        _lib.check(lib.w8a8_paged_prefill_window(*given, window, sinks, *rest),
                   "w8a8_paged_prefill_window")
    return out


# ------------------------------------------------------------ drafted tokens
def tree_masks(parents: Sequence[Sequence[int]], *, device: torch.device | str = "cuda"
               ) -> torch.Tensor:
    """The masks of :func:`paged_tree` for a batch of trees: ``parents[b][i]`` is
    the parent of sequence ``b``'s drafted token ``i``, one of those before it
    (a chain: ``i - 1``), or -1 for one that follows the cached tokens; each
    token sees its ancestors and itself.  int64 ``[tokens, words]`` with as many
    words as the longest tree needs."""
    rows: list[int] = []
    for tree in parents:
        own: list[int] = []
        for i, parent in enumerate(tree):
            if not -1 <= parent < i:
                raise ValueError("a drafted token's parent must be one before it, or -1")
            own.append(1 << i | (own[parent] if parent >= 0 else 0))
        rows += own
    words = max(1, -(-max(map(len, parents), default=0) // 64))
    low = (1 << 64) - 1
    signed = [[((m >> 64 * w & low) ^ 1 << 63) - (1 << 63) for w in range(words)] for m in rows]
    return torch.tensor(signed, dtype=torch.int64).reshape(len(rows), words).to(device)


def paged_accept(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                 lengths: torch.Tensor, path: torch.Tensor) -> None:
    """Keeps accepted drafted tokens in the cache, in place: the key and value of
    sequence ``b``'s drafted token ``path[b, i]`` (int32 ``[batch, steps]``,
    rising; -1 behind the path's end) go to place ``lengths[b] + i``, where
    ``lengths[b]`` (int32) keys were cached before the drafted ones.  The caches
    are one layer's, or ``[layers, pages, kv_heads, page_size, head_dim]``: all
    layers in one launch (:meth:`PagedKVCache.accept`); keys and values may be
    views of one tensor, in any order of its axes.  An entry below its
    ``i`` moves nothing, as does a place outside the table or the cache.  The
    pages of the drafted tokens belong to one sequence only."""
    index = _gpu(k_cache, v_cache, page_table, lengths, path)
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return paged_accept(k_cache, v_cache, page_table, lengths, path)
    code = _CODES.get(k_cache.dtype)
    if code is None or v_cache.dtype != k_cache.dtype:
        raise ValueError("the cache must be float16 / bfloat16")
    shape, strides, other = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) not in (4, 5) or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must be [pages, kv_heads, page_size, head_dim] "
                         "or [layers, ...] of these")
    if strides[-1] != 1 or strides != other and any(
            n > 1 and x != y for n, x, y in zip(shape, strides, other)):
        raise ValueError("k_cache and v_cache must have equal strides and contiguous heads")
    layers, ls = (shape[0], strides[0]) if len(shape) == 5 else (1, 0)
    pages, g, page_size, d = shape[-4:]
    b = lengths.shape[0] if lengths.dim() == 1 else -1
    page_table, ld, width = _table(page_table, b)
    lengths = _index(lengths, torch.int32, b, "lengths")
    if path.dtype != torch.int32 or path.dim() != 2 or path.shape[0] != b:
        raise ValueError("path must be int32 [batch, steps]")
    path = path if path.is_contiguous() else path.contiguous()
    steps = path.shape[1]
    _lib.check(_lib.load().w8a8_cache_accept(
        k_cache.data_ptr(), v_cache.data_ptr(), ls, *strides[-4:-1], layers, pages, page_size,
        page_table.data_ptr(), ld, width, lengths.data_ptr(), path.data_ptr(), steps, steps, code,
        b, g, d, torch._C._cuda_getCurrentRawStream(index)), "w8a8_cache_accept")


# --------------------------------------------------------- the runner's core
class PagedKVCache:
    """Keys and values of a decoder stack in pages of ``page_size`` tokens (a
    power of two), ``k[layer]`` and ``v[layer]`` of shape ``[pages, kv_heads,
    page_size, head_dim]``.  Which pages a sequence owns is the caller's
    bookkeeping (the reference's block manager)."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *,
                 page_size: int = 16, dtype: torch.dtype = torch.float16,
                 device: torch.device | str = "cuda") -> None:
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("the cache is float16 / bfloat16")
        if head_dim < 8 or head_dim % 8 or head_dim > MAX_HEAD_DIM:
            raise ValueError(f"head_dim must be a multiple of 8, at most {MAX_HEAD_DIM}")
        self.page_size = page_size
        store = torch.zeros((layers, 2, pages, kv_heads, page_size, head_dim), dtype=dtype,
                            device=device)
        self.k = [store[i, 0] for i in range(layers)]
        self.v = [store[i, 1] for i in range(layers)]
        self._store = store

    def accept(self, page_table: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor) -> None:
        """:func:`paged_accept` in every layer, one launch."""
        paged_accept(self._store[:, 0], self._store[:, 1], page_table, lengths, path)


@dataclass
class AttentionState:
    """What one step of the stack attends to, all on the GPU: per row its
    position and its slot in the cache (-1: a padded row, not stored; behind
    the chunks' rows it belongs to no sequence, and its result is zeros), per
    sequence its pages and its length with this step's tokens.  The first
    ``decode_rows`` rows are one new token each of the first ``decode_rows``
    sequences; the others are chunks, ``q_starts`` giving where each of the
    remaining sequences' rows start, counted from the first of them.  With
    ``masks`` those chunks are trees of drafted tokens (:meth:`build_drafts`)."""

    positions: torch.Tensor            # int64 [rows]
    slots: torch.Tensor                # int64 [rows]
    page_table: torch.Tensor           # int32 [sequences, pages]
    lengths: torch.Tensor              # int32 [sequences]
    q_starts: torch.Tensor | None = None   # int32 [sequences - decode_rows + 1]
    decode_rows: int = 0
    masks: torch.Tensor | None = None      # int64 [rows - decode_rows, words]

    @classmethod
    def build_drafts(cls, pages: Sequence[Sequence[int]], lengths: Sequence[int],
                     parents: Sequence[Sequence[int]], page_size: int, *,
                     device: torch.device | str = "cuda") -> "AttentionState":
        """The state of a step that verifies a tree of drafted tokens per
        sequence: sequence ``b``, which owns ``pages[b]`` in order and has
        ``lengths[b]`` cached tokens, gets the drafted tokens whose parents are
        ``parents[b]`` (:func:`tree_masks`).  Token ``i`` is stored at place
        ``lengths[b] + i`` and turned to the position of its depth in the tree;
        :meth:`PagedKVCache.accept` moves the accepted ones to their places."""
        if not len(pages) == len(lengths) == len(parents):
            raise ValueError("pages, lengths and parents must have one entry per sequence")
        state = cls.build(pages, [n + len(tree) for n, tree in zip(lengths, parents)],
                          [len(tree) for tree in parents], page_size, device=device)
        masks = tree_masks(parents, device=device)
        positions: list[int] = []
        for n, tree in zip(lengths, parents):
            own: list[int] = []
            for parent in tree:
                own.append(own[parent] + 1 if parent >= 0 else n)
            positions += own
        starts = [0]
        for tree in parents:
            starts.append(starts[-1] + len(tree))
        state.positions = torch.tensor(positions, dtype=torch.int64, device=device)
        state.q_starts = torch.tensor(starts, dtype=torch.int32, device=device)
        state.decode_rows, state.masks = 0, masks
        return state

    @classmethod
    def build(cls, pages: Sequence[Sequence[int]], lengths: Sequence[int],
              new_tokens: Sequence[int], page_size: int, *,
              device: torch.device | str = "cuda") -> "AttentionState":
        """The state of a step in which sequence ``b``, which owns ``pages[b]``
        in order, gets its ``new_tokens[b]`` newest tokens, ``lengths[b]`` in
        all.  Sequences of one new token come first and run as decode."""
        if not len(pages) == len(lengths) == len(new_tokens):
            raise ValueError("pages, lengths and new_tokens must have one entry per sequence")
        decode = 0
        for n in new_tokens:
            if n != 1:
                break
            decode += 1
        positions, slots = [], []
        for own, total, n in zip(pages, lengths, new_tokens):
            if n < 0 or n > total or total > len(own) * page_size:
                raise ValueError("a sequence's pages must hold its tokens")
            if any(p < 0 for p in own):
                raise ValueError("a page must not be negative")
            for at in range(total - n, total):
                positions.append(at)
                slots.append(own[at // page_size] * page_size + at % page_size)
        width = max((len(own) for own in pages), default=0)
        table = [list(own) + [-1] * (width - len(own)) for own in pages]
        starts = None
        if decode < len(pages):
            starts = [0]
            for n in new_tokens[decode:]:
                starts.append(starts[-1] + n)
            starts = torch.tensor(starts, dtype=torch.int32, device=device)
        return cls(torch.tensor(positions, dtype=torch.int64, device=device),
                   torch.tensor(slots, dtype=torch.int64, device=device),
                   torch.tensor(table, dtype=torch.int32, device=device).reshape(len(table), width),
                   torch.tensor(list(lengths), dtype=torch.int32, device=device), starts, decode)


class PagedAttentionCore:
    """The attention core of :class:`~nanopointllm_amd.runner.W8A8LlamaRunner`:
    rotary positions with the store into ``cache``, then attention over it.

    ``runner = W8A8LlamaRunner(model, PagedAttentionCore(cache, frequencies))``
    and ``runner(ids, attention_state=AttentionState.build(...))``; a decode
    step is captured with :class:`~nanopointllm_amd.runner.DecodeGraphBucket`
    on a state whose tensors are then refilled in place between replays.
    ``window`` (one for all layers, or one or None for each) and ``sinks``
    limit what a row sees as in :func:`paged_decode`; sequences keep their own
    positions, sinks included.  Where any layer has a window, trees of drafted
    tokens are refused, by each layer before it stores anything."""

    def __init__(self, cache: PagedKVCache, frequencies: RotaryFrequencies, *,
                 layout: str = "half", scale: float | None = None,
                 window: int | None | Sequence[int | None] = None, sinks: int = 0) -> None:
        _layout(layout)
        self.cache, self.frequencies = cache, frequencies
        self.layout, self.scale = layout, scale
        if not isinstance(window, Sequence):
            _window(window, sinks)
        else:
            window = list(window)
            if len(window) != len(cache.k):
                raise ValueError("window must be one for all layers, or one for each")
            for w in window:
                _window(w, sinks if w is not None else 0)
            _window(max((w for w in window if w is not None), default=None), sinks)
        self.window, self.sinks = window, sinks

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layer_index: int,
                 state: AttentionState) -> torch.Tensor:
        k_cache, v_cache = self.cache.k[layer_index], self.cache.v[layer_index]
        window = self.window[layer_index] if isinstance(self.window, list) else self.window
        sinks = 0 if window is None else self.sinks
        table, lengths, n = state.page_table, state.lengths, state.decode_rows
        if state.masks is not None:
            if state.q_starts is None:
                raise ValueError("masks need the q_starts of their trees")
            # Of all layers, so that none has stored a step that a later one refuses.
            windows = self.window if isinstance(self.window, list) else [self.window]
            if any(w is not None for w in windows):
                raise ValueError("trees of drafted tokens run on stacks without a window")
        q = rotary_store(q, k, v, state.positions, state.slots, self.frequencies.inv_freq,
                         k_cache, v_cache, layout=self.layout,
                         attention_factor=self.frequencies.attention_factor)
        if state.q_starts is None:
            out = paged_decode(q, k_cache, v_cache, table, lengths, scale=self.scale,
                               window=window, sinks=sinks)
        elif n == 0:
            out = _prefill(q, k_cache, v_cache, table, lengths, state.q_starts, self.scale, None,
                           True, window, sinks, state.masks)
        else:
            out = torch.empty_like(q)
            paged_decode(q[:n], k_cache, v_cache, table[:n], lengths[:n], scale=self.scale,
                         window=window, sinks=sinks, out=out[:n])
            _prefill(q[n:], k_cache, v_cache, table[n:], lengths[n:], state.q_starts,
                     self.scale, out[n:], True, window, sinks, state.masks)
        return out.flatten(1)
