"""Windows, trees of drafted tokens, accepted paths and log probabilities
together, as a serving loop runs them through W8A8LlamaRunner.

Logits of a step are compared with those of the same tokens run as one prompt:
within the W8A8 stack's sensitivity to the 16-bit rounding of the attention's
rows, as in test_gpu_attention.py.
"""
from __future__ import annotations

import pytest
import torch

import test_gpu_attention as G
from nanopointllm_amd import attention as A
from nanopointllm_amd import lm_head as L
from nanopointllm_amd.runner import DecodeGraphBucket, W8A8LlamaRunner

pytestmark = pytest.mark.gpu

HEADS, KV, HIDDEN, PAGE, VOCAB, LAYERS = 4, 2, 256, 8, 512, 2


def model_of(cuda):
    from workloads import llama_model

    return llama_model(cuda, layers=LAYERS, hidden=HIDDEN, heads=HEADS, kv_heads=KV,
                       intermediate=384, vocab=VOCAB)


def cache_of(cuda, pages=20):
    return A.PagedKVCache(LAYERS, pages, KV, HIDDEN // HEADS, page_size=PAGE, device=cuda)


def close(got, want):
    off = float((got.double() - want.double()).norm() / want.double().norm())
    assert off < 0.05, off


def test_drafts_verified_and_accepted(cuda):
    G.note("drafts through the runner")
    freq = A.rotary_frequencies(HIDDEN // HEADS, device=cuda)
    runner = W8A8LlamaRunner(model_of(cuda), A.PagedAttentionCore(cache_of(cuda), freq))
    g = G.gen_of(3)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (29, 14)]
    pages = [[5, 2, 9, 0, 7, 12], [1, 8, 3, 10]]
    state = A.AttentionState.build(pages, [29, 14], [29, 14], PAGE, device=cuda)
    runner(torch.cat(prompts)[None].to(cuda), attention_state=state)

    # A tree and a chain; the root is the token that the prompt's last row chose.
    parents = [[-1, 0, 0, 1, 1, 2, 3], [-1, 0, 1]]
    tokens = [torch.randint(0, VOCAB, (len(p),), generator=g) for p in parents]
    drafts = A.AttentionState.build_drafts(pages, [29, 14], parents, PAGE, device=cuda)
    ids = torch.cat(tokens)[None].to(cuda)
    # The drafted children of every node, -1 where it has fewer.
    children = torch.full((1, 10, 2), -1, dtype=torch.int64)
    at = 0
    for p, t in zip(parents, tokens):
        for i, parent in enumerate(p[1:], 1):
            row = children[0, at + parent]
            row[int(row[0] >= 0)] = t[i]
        at += len(p)
    children = children.to(cuda)
    logits = runner(ids, attention_state=drafts)
    scores = runner.score(ids, tokens=children, top=3, attention_state=drafts)
    again = L.token_logprobs(logits, children, top=3)
    assert all(torch.equal(a, b) for a, b in zip(scores, again))
    want = torch.log_softmax(logits.double(), -1)
    taken = want.gather(-1, children.clamp_min(0)).masked_fill(children < 0, 0.0)
    assert (scores.logprobs.double() - taken).abs().max() < 1e-5
    assert torch.equal(scores.top_tokens[..., 0], logits.float().argmax(-1))

    def alone(tokens_of_path, b):
        """The logits of a prompt with a path behind it, all as one prompt."""
        whole = torch.cat((prompts[b], tokens_of_path))
        fresh = cache_of(cuda)
        for layer in runner.layers:
            layer.attention_core.cache = fresh
        n = len(whole)
        own = A.AttentionState.build([list(range(6))], [n], [n], PAGE, device=cuda)
        out = runner(whole[None].to(cuda), attention_state=own)
        for layer in runner.layers:
            layer.attention_core.cache = kept
        return out[0, len(prompts[b]):]

    kept = runner.layers[0].attention_core.cache
    for path in ([0, 1, 3, 6], [0, 1, 4], [0, 2, 5]):
        close(logits[0, path], alone(tokens[0][path], 0))
    close(logits[0, 7:], alone(tokens[1], 1))

    # The tree's path 0, 2, 5 and two of the chain are kept; the step behind them.
    accepted = torch.tensor([[0, 2, 5], [0, 1, -1]], dtype=torch.int32, device=cuda)
    before = [c.clone() for c in kept.k + kept.v]
    cached = torch.tensor([29, 14], dtype=torch.int32, device=cuda)
    kept.accept(drafts.page_table, cached, accepted)
    for old, new in zip(before, kept.k + kept.v):
        for b, (n, path) in enumerate(zip((29, 14), ([0, 2, 5], [0, 1]))):
            for i, node in enumerate(path):
                to, source = n + i, n + node
                assert torch.equal(new[pages[b][to // PAGE], :, to % PAGE],
                                   old[pages[b][source // PAGE], :, source % PAGE])
    follow = torch.randint(0, VOCAB, (2,), generator=g)
    step = A.AttentionState.build(pages, [33, 17], [1, 1], PAGE, device=cuda)
    got = runner(follow[None].to(cuda), attention_state=step)
    close(got[0, 0], alone(torch.cat((tokens[0][[0, 2, 5]], follow[:1])), 0)[-1])
    close(got[0, 1], alone(torch.cat((tokens[1][:2], follow[1:])), 1)[-1])


def test_windowed_layers(cuda):
    """A layer of full attention and one of a window with sinks: a prompt, then
    captured decode steps whose pages behind the window are given back."""
    G.note("windowed layers through the runner")
    freq = A.rotary_frequencies(HIDDEN // HEADS, device=cuda)
    model = model_of(cuda)
    total, start, window, sinks = 47, 40, 10, 3
    ids = torch.randint(0, VOCAB, (1, total), generator=G.gen_of(4)).to(cuda)
    pages = [[4, 1, 6, 3, 0, 2]]

    def run(**kw):
        runner = W8A8LlamaRunner(model, A.PagedAttentionCore(cache_of(cuda), freq, **kw),
                                 inject=not hasattr(model.model.layers[0].self_attn, "w8a8_qkv"))
        embeds = runner.embed_tokens(ids)
        whole = runner(inputs_embeds=embeds, attention_state=A.AttentionState.build(
            pages, [total], [total], PAGE, device=cuda))
        for layer in runner.layers:
            layer.attention_core.cache = cache_of(cuda)
        logits = [runner(inputs_embeds=embeds[:, :start], attention_state=A.AttentionState.build(
            pages, [start], [start], PAGE, device=cuda))]
        state = A.AttentionState.build(pages, [start + 1], [1], PAGE, device=cuda)
        if kw.get("window") == window:
            # Places 8 .. 30 are in no row's window from place 41 on, nor sinks.
            state.page_table[0, 1:3] = torch.tensor([-1, 2 ** 30], dtype=torch.int32)
        token = embeds[:, start:start + 1].clone()
        bucket = DecodeGraphBucket(cuda)
        static = bucket.capture(lambda: runner(inputs_embeds=token, attention_state=state))
        for i in range(start, total):
            now = A.AttentionState.build(pages, [i + 1], [1], PAGE, device=cuda)
            token.copy_(embeds[:, i:i + 1])
            for name in ("positions", "slots", "lengths"):
                getattr(state, name).copy_(getattr(now, name))
            bucket.replay()
            logits.append(static.clone())
            assert torch.equal(static, runner(inputs_embeds=token, attention_state=state))
        close(torch.cat(logits, 1), whole)
        return whole

    full = run()
    assert torch.equal(run(window=[None, 1000], sinks=2), full)
    mixed = run(window=[None, window], sinks=sinks)
    both = run(window=window, sinks=sinks)
    # The first rows are inside every window, the others are not.
    assert torch.equal(mixed[:, :window], full[:, :window])
    assert not torch.equal(mixed[:, window:], full[:, window:])
    assert not torch.equal(both, mixed)
