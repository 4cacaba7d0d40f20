# SPDX-License-Identifier: MIT
"""examples/beam_decode.py: the search, the cache and its attention together, against the same model
run without a cache (every sequence from its first token on, plain attention in 32 bits)."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from beamgrad_b200.search import DeviceSearch

ROOT = Path(__file__).resolve().parents[1]


def example():
    spec = importlib.util.spec_from_file_location("beam_decode", ROOT / "examples" / "beam_decode.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_logits(model, tokens):
    """The logits behind each token of sequences tokens [S, T], without a cache."""
    S, T = tokens.shape
    x = model.embed[tokens] + model.place[torch.arange(T, device=tokens.device)]
    causal = torch.ones((T, T), dtype=torch.bool, device=tokens.device).tril()
    for i in range(model.layers):
        y = F.linear(F.layer_norm(x, x.shape[-1:]), model.qkv[i]).unflatten(-1, (-1, model.head_dim))
        q, k, v = y.split((model.heads, model.kv_heads, model.kv_heads), -2)
        k, v = (z.repeat_interleave(model.heads // model.kv_heads, 2) for z in (k, v))
        s = torch.einsum("sihd,sjhd->shij", q, k) * model.head_dim**-0.5
        a = torch.softmax(s.masked_fill(~causal, float("-inf")), -1)
        x = x + F.linear(torch.einsum("shij,sjhd->sihd", a, v).flatten(-2), model.out[i])
        x = x + F.linear(F.gelu(F.linear(F.layer_norm(x, x.shape[-1:]), model.up[i])), model.down[i])
    return F.linear(F.layer_norm(x, x.shape[-1:]), model.embed) * x.shape[-1] ** -0.5


@pytest.mark.gpu
def test_beam_search_with_the_cache_equals_the_search_without():
    ex = example()
    model = ex.TinyLM(vocab=200, layers=2, dtype=torch.float32, seed=3)
    B, K, T, steps = 3, 4, 21, 20
    prompt = torch.randint(0, model.vocab, (B, T), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    result, cache = ex.beam_decode(model, prompt, K, steps, eos=7)
    cache.check()
    search = DeviceSearch(B, K, model.vocab, steps, from_logits=True, eos_token=7, length_penalty_alpha=0.6)
    for t in range(steps):
        if t == 0:
            rows = plain_logits(model, prompt)[:, -1][:, None].expand(B, K, -1)
        else:
            seq = search.state().sequences.clamp(min=0).reshape(B * K, t)
            rows = plain_logits(model, torch.cat([prompt.repeat_interleave(K, 0), seq], 1))[:, -1].view(B, K, -1)
        search.step(rows)
    want = search.result()
    assert torch.equal(result.sequences, want.sequences)
    assert float((result.scores - want.scores).abs().max()) < 1e-3
    # The beams share what they have in common: far fewer pages than beams times columns.
    assert int((cache.references > 0).sum()) < int((cache.table >= 0).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("good", [True, False])
def test_drafted_decoding_equals_greedy_decoding(good):
    ex = example()
    model = ex.TinyLM(vocab=100, layers=2, dtype=torch.float32, seed=5)
    B, T, steps = 2, 18, 12
    prompt = torch.randint(0, model.vocab, (B, T), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    greedy = prompt
    for _ in range(steps + 8):
        greedy = torch.cat([greedy, plain_logits(model, greedy)[:, -1:].argmax(-1)], 1)
    truth = greedy[:, T:]
    at = [0]

    def draft(last, width, depth):
        # A tree of 2 + 4 tokens behind the last one: the true continuation among wrong ones, or only wrong.
        step = at[0]
        nxt = truth[:, step + 1 : step + 3] if good else (truth[:, step + 1 : step + 3] + 1) % model.vocab
        wrong = (truth[:, step + 1 : step + 2] + 3) % model.vocab
        tokens = torch.cat([last[:, None], wrong, nxt[:, :1], wrong, wrong, nxt[:, 1:], nxt[:, 1:]], 1)
        at[0] += 3 if good else 1
        return tokens, [-1, 0, 0, 1, 1, 2, 2]

    tokens, passes = ex.drafted_decode(model, prompt, steps, draft)
    assert torch.equal(tokens[:, :steps], truth[:, :steps])
    assert passes <= (5 if good else steps)
