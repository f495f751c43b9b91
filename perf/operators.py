"""Performance cases of the attention core's operators: rotary positions with
the store into a paged key-value cache, attention of one new token per
sequence over that cache, and attention of prompts and prompt chunks over it.

Sizes are the repository's own workload (32 heads of 128, about 560 prompt
rows, decode batches up to 64) and generic decoder shapes around it: shared
key-value heads, heads of 64 to 128, pages of 8 to 128 tokens, contexts up to
131071.  ``run`` computes the operators in their plain form, or where ``own``
is true makes the framework's calls.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "nano-pointllm_amd"))

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
DEVICE = "cuda"


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # One token of single-stream decode: launch latency.
        {"name": "rotary_t1", "kind": "rotary", "tokens": 1, "heads": 32, "kv_heads": 32,
         "dim": 128, "rotary_dim": 128, "layout": "half", "factor": 1.0, "start": 600, "page": 16,
         "dtype": "float16"},
        # The prompt of the workload: 513 point tokens and text.
        {"name": "rotary_t560", "kind": "rotary", "tokens": 560, "heads": 32, "kv_heads": 32,
         "dim": 128, "rotary_dim": 128, "layout": "half", "factor": 1.0, "start": 0, "page": 16,
         "dtype": "float16"},
        # A chunk far into a long context whose frequencies and amplitude are
        # scaled; half of each head turns, neighbours paired, shared heads.
        {"name": "rotary_far_chunk", "kind": "rotary", "tokens": 4097, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary_dim": 64, "layout": "interleaved", "factor": 1.13, "start": 120001,
         "page": 64, "dtype": "bfloat16"},
        # Single-stream decode right behind the workload's prompt.
        {"name": "decode_b1", "kind": "decode", "batch": 1, "heads": 32, "kv_heads": 32,
         "dim": 128, "length": 601, "spread": 0.0, "page": 16, "dtype": "float16"},
        # The workload's decode batch, sequences of uneven age.
        {"name": "decode_b8", "kind": "decode", "batch": 8, "heads": 32, "kv_heads": 32,
         "dim": 128, "length": 1590, "spread": 0.6, "page": 16, "dtype": "float16"},
        # One conversation over a very long context with shared heads.
        {"name": "decode_b1_long", "kind": "decode", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "length": 131071, "spread": 0.0, "page": 16, "dtype": "bfloat16"},
        # A large batch of very uneven lengths, four queries to a key head.
        {"name": "decode_b64", "kind": "decode", "batch": 64, "heads": 32, "kv_heads": 8,
         "dim": 128, "length": 8190, "spread": 0.98, "page": 64, "dtype": "bfloat16"},
        # Narrow heads, six queries to a key head, an odd batch.
        {"name": "decode_b33_d64", "kind": "decode", "batch": 33, "heads": 24, "kv_heads": 4,
         "dim": 64, "length": 3001, "spread": 0.5, "page": 32, "dtype": "float16"},
        # The workload's prompt.
        {"name": "prefill_560", "kind": "prefill", "batch": 1, "heads": 32, "kv_heads": 32,
         "dim": 128, "new": 560, "spread": 0.0, "prefix": 0, "page": 16, "dtype": "float16"},
        # A batch of uneven prompts, some behind a cached prefix.
        {"name": "prefill_ragged", "kind": "prefill", "batch": 7, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 777, "spread": 0.95, "prefix": 300, "page": 16, "dtype": "bfloat16"},
        # One chunk of a long prompt whose beginning is in the cache.
        {"name": "prefill_chunk", "kind": "prefill", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 512, "spread": 0.0, "prefix": 7680, "page": 64, "dtype": "bfloat16"},
        # A long prompt at once: the largest call.
        {"name": "prefill_8k", "kind": "prefill", "batch": 1, "heads": 32, "kv_heads": 32,
         "dim": 128, "new": 8192, "spread": 0.0, "prefix": 0, "page": 16, "dtype": "float16"},
    ]


HEADS = ((32, 32), (40, 40), (16, 16), (32, 8), (20, 4), (28, 4), (16, 2), (8, 1))


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """Another case of the listed ones' ranges; tokens, batch and length are
    spread over their logarithm, and a case that would cost more than the
    largest of its kind is cut down."""
    kind = rng.choice(("rotary", "decode", "prefill"))
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice((64, 80, 96, 128, 128))
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice((8, 16, 32, 64, 128)), "dtype": rng.choice(sorted(DTYPES))}
    if kind == "rotary":
        case.update(tokens=_log_int(rng, 1, 4097), rotary_dim=rng.choice((dim, dim, dim // 2, 24)),
                    layout=rng.choice(("half", "interleaved")),
                    factor=rng.choice((1.0, round(rng.uniform(1.0, 1.4), 3))),
                    start=_log_int(rng, 1, 200000) - 1)
        return case
    if kind == "decode":
        case.update(batch=_log_int(rng, 1, 64), length=_log_int(rng, 1, 131071),
                    spread=round(rng.choice((0.0, rng.uniform(0.0, 0.98))), 2))
        while work(case)["bytes"] > 1.3e9 or case["batch"] * case["length"] > 64 * 8190:
            case["length"] = case["length"] * 3 // 4
        return case
    case.update(batch=_log_int(rng, 1, 16), new=_log_int(rng, 1, 8192),
                spread=round(rng.choice((0.0, rng.uniform(0.0, 0.98))), 2),
                prefix=rng.choice((0, _log_int(rng, 1, 16000))))
    while heads * case["batch"] * case["new"] * (case["new"] + case["prefix"]) > 32 * 8192 ** 2:
        key = "prefix" if case["prefix"] > case["new"] else "new"
        case[key] = case[key] * 3 // 4
    return case


def _shares(batch: int, spread: float) -> list[float]:
    """Each sequence's part of the longest: 1 for the first, the others spread
    evenly (the golden ratio's multiples) over the last ``spread``."""
    return [1.0 - spread * ((i * 0.6180339887498949) % 1.0) for i in range(batch)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, cached and new tokens) of each sequence."""
    part = _shares(case["batch"], case["spread"])
    if case["kind"] == "decode":
        return [1] * case["batch"], [max(1, int(case["length"] * p)) for p in part]
    new = [max(1, int(case["new"] * p)) for p in part]
    # The shorter prompts are the ones with a longer cached part.
    return new, [n + int(case["prefix"] * (2.0 - p) / 2.0 if case["spread"] else case["prefix"])
                 for n, p in zip(new, part)]


# ------------------------------------------------------------ inputs and state
def _rows(gen, dtype, *shape: int, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, device=DEVICE, dtype=dtype).normal_(0.0, std, generator=gen)


def _packed_rows(gen, case: dict, tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q, k and v as the packed projection leaves them: views of one matrix's
    rows, a few channels larger than the others."""
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    rows = _rows(gen, DTYPES[case["dtype"]], tokens, (h + 2 * g) * d)
    loud = torch.randperm(rows.shape[1], generator=gen, device=DEVICE)[:max(1, h // 8)]
    rows[:, loud] *= 4.0
    q, k, v = rows.split((h * d, g * d, g * d), dim=1)
    return q.view(tokens, h, d), k.view(tokens, g, d), v.view(tokens, g, d)


def _state(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(1000003 * seed + 29)
    dtype, page, g, d = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["dim"]
    if case["kind"] == "rotary":
        tokens = case["tokens"]
        q, k, v = _packed_rows(gen, case, tokens)
        pages = -(-tokens // page) + 2
        at = torch.randperm(pages, generator=gen, device=DEVICE)
        place = torch.arange(tokens, device=DEVICE)
        half = torch.arange(case["rotary_dim"] // 2, device=DEVICE, dtype=torch.float64)
        return {"case": case, "q": q, "k": k, "v": v, "positions": place + case["start"],
                "slots": at[place // page] * page + place % page,
                "inv_freq": 10000.0 ** (-2.0 * half / case["rotary_dim"]),
                "k_cache": _rows(gen, dtype, pages, g, page, d),
                "v_cache": _rows(gen, dtype, pages, g, page, d)}
    new, lengths = _lengths(case)
    needs = [-(-n // page) for n in lengths]
    pages = sum(needs) + 3
    at = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    used = torch.arange(max(needs)) < torch.tensor(needs)[:, None]
    table = torch.full(used.shape, -1, device=DEVICE, dtype=torch.int32)
    table[used.to(DEVICE)] = at[:sum(needs)]
    q = _packed_rows(gen, case, sum(new))[0]
    starts = torch.zeros(len(new) + 1, dtype=torch.int32)
    starts[1:] = torch.tensor(new).cumsum(0)
    return {"case": case, "q": q * 1.5, "k_cache": _rows(gen, dtype, pages, g, page, d),
            "v_cache": _rows(gen, dtype, pages, g, page, d, std=0.7), "table": table,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
            "starts": starts.to(DEVICE), "most": max(new),
            # The sequence of each query row.
            "owner": torch.arange(len(new)).repeat_interleave(torch.tensor(new)).to(DEVICE)}


def prepare(case: dict, seed: int) -> dict:
    return _state(case, seed)


# -------------------------------------------------------------- the operators
def run(state: dict):
    case = state["case"]
    if own:
        from nanopointllm_amd import attention

        if case["kind"] == "rotary":
            q = attention.rotary_store(
                state["q"], state["k"], state["v"], state["positions"], state["slots"],
                state["inv_freq"], state["k_cache"], state["v_cache"], layout=case["layout"],
                attention_factor=case["factor"])
            return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
        if case["kind"] == "decode":
            return attention.paged_decode(state["q"], state["k_cache"], state["v_cache"],
                                          state["table"], state["lengths"])
        return attention.paged_prefill(state["q"], state["k_cache"], state["v_cache"],
                                       state["table"], state["lengths"], state["starts"])
    if case["kind"] == "rotary":
        return _plain_rotary_store(state)
    return _plain_attention(state)


def _turn(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, layout: str) -> torch.Tensor:
    width = 2 * cos.shape[-1]
    turned, rest = x[..., :width].float(), x[..., width:]
    if layout == "half":
        a, b = turned.chunk(2, dim=-1)
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    return torch.cat((out.to(x.dtype), rest), dim=-1)


def _plain_rotary_store(state: dict) -> dict:
    case, page = state["case"], state["case"]["page"]
    angle = state["positions"].double()[:, None, None] * state["inv_freq"]
    cos = (case["factor"] * angle.cos()).float()
    sin = (case["factor"] * angle.sin()).float()
    q = _turn(state["q"], cos, sin, case["layout"])
    pages, offsets = state["slots"] // page, state["slots"] % page
    state["k_cache"][pages, :, offsets] = _turn(state["k"], cos, sin, case["layout"])
    state["v_cache"][pages, :, offsets] = state["v"]
    return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _gathered(cache: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """[batch, kv heads, keys, dim] in 32 bits."""
    pages = cache[table.clamp_min(0).long()]
    return pages.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _plain_attention(state: dict) -> torch.Tensor:
    """Padded to the longest sequence: queries [batch, kv heads, group x new,
    dim] against the gathered keys, softmax over those that each may see."""
    q, starts, lengths = state["q"], state["starts"].long(), state["lengths"].long()
    h, d = q.shape[1:]
    g, most = state["k_cache"].shape[1], state["most"]
    k, v = _gathered(state["k_cache"], state["table"]), _gathered(state["v_cache"], state["table"])
    new = starts[1:] - starts[:-1]
    step = torch.arange(most, device=q.device)
    rows = (starts[:-1, None] + step).clamp_max(q.shape[0] - 1)
    padded = q[rows].float() * d ** -0.5                        # [batch, most, heads, dim]
    padded = padded.view(-1, most, g, h // g, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = padded @ k.transpose(-1, -2).contiguous()          # [batch, kv, group x most, keys]
    last = (lengths - new)[:, None] + step                      # [batch, most]
    hidden = torch.arange(k.shape[2], device=q.device) > last[..., None]
    scores = scores.view(*scores.shape[:2], h // g, most, -1)
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    peak = scores.amax(-1, keepdim=True)
    scores.sub_(peak.masked_fill(peak == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ v).view(*scores.shape[:-1], d)
    out = out / total.masked_fill(total == 0.0, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(-1, most, h, d)    # [batch, most, heads, dim]
    owner = state["owner"]
    place = torch.arange(q.shape[0], device=q.device) - starts[owner]
    return out[owner, place].to(q.dtype)


# ---------------------------------------------------------------------- work
def work(case: dict) -> dict:
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "rotary":
        rows = case["tokens"] * (h + 2 * g) * d
        return {"bytes": 2 * 2 * rows + 16 * case["tokens"],
                "flops": 3 * case["tokens"] * (h + g) * case["rotary_dim"]}
    new, lengths = _lengths(case)
    seen = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, lengths))
    table = 4 * sum(-(-t // case["page"]) for t in lengths)
    return {"bytes": 4 * sum(new) * h * d + 4 * sum(lengths) * g * d + table,
            "flops": 4 * seen * h * d}


# --------------------------------------------------- the definition in 64 bits
def _exact_rotary(case: dict, s: dict) -> dict:
    """Each pair, as a complex number, times factor * exp(i position frequency)."""
    spin = torch.polar(
        torch.full((), case["factor"], dtype=torch.float64, device=DEVICE),
        torch.outer(s["positions"].double(), s["inv_freq"]))[:, None]
    first = torch.arange(case["rotary_dim"] // 2, device=DEVICE)
    second = first + case["rotary_dim"] // 2
    if case["layout"] == "interleaved":
        first, second = 2 * first, 2 * first + 1

    def turned(x):
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * spin
        x[..., first], x[..., second] = z.real, z.imag
        return x

    caches = {}
    for name, rows in (("k_cache", turned(s["k"])), ("v_cache", s["v"].double())):
        # One row per slot: [pages, heads, page, dim] seen as [pages x page, heads, dim].
        flat = s[name].double().transpose(1, 2).flatten(0, 1)
        flat[s["slots"]] = rows
        caches[name] = flat.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous()
    return {"q": turned(s["q"]), **caches}


def exact(case: dict, seed: int):
    """Rotary as complex numbers; attention sequence by sequence and head by head."""
    s = _state(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, s)
    new, lengths = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at = 0
    for b, (n, t) in enumerate(zip(new, lengths)):
        pages = s["table"][b, :-(-t // case["page"])].long()
        for head in range(case["kv_heads"]):
            k = s["k_cache"][pages, head].flatten(0, 1)[:t].double()
            v = s["v_cache"][pages, head].flatten(0, 1)[:t].double()
            for i in range(head * group, (head + 1) * group):
                logits = s["q"][at:at + n, i].double() @ k.T.contiguous() / math.sqrt(case["dim"])
                logits += torch.full((n, t), -math.inf, dtype=torch.float64,
                                     device=DEVICE).triu_(t - n + 1)
                out[at:at + n, i] = torch.softmax(logits, -1) @ v
        at += n
    return out
