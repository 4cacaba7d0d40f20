# SPDX-License-Identifier: MIT
"""Beam search and drafted decoding of a small transformer on the paged beam cache.

    python examples/beam_decode.py [--batch 4] [--beams 8] [--prompt 100] [--steps 64] [--dtype bfloat16]

Random weights: the program shows how the pieces are used together, and times them.

* :func:`beam_decode` -- the prompt is written for beam 0 of each example and forked to all beams;
  then every step of :class:`beamgrad_b200.search.DeviceSearch` is followed by one
  ``PagedCache.fork`` with the parents it chose. Nothing waits for the host.
* :func:`drafted_decode` -- greedy decoding in which a tree of drafted tokens is checked in one pass
  of the model, the longest path that agrees is accepted with ``PagedCache.commit`` and the rest is
  dropped.
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch
import torch.nn.functional as F

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from beamgrad_b200.cache import PagedCache
from beamgrad_b200.search import DeviceSearch, SearchResult


class TinyLM:
    """A pre-norm transformer with grouped heads and learned positions; random weights."""

    def __init__(self, vocab=1000, width=256, layers=4, heads=8, kv_heads=2, head_dim=64, positions=4096,
                 dtype=torch.bfloat16, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *shape: (torch.randn(shape, generator=gen, device="cuda") / shape[-1] ** 0.5).to(dtype)  # noqa: E731
        self.vocab, self.layers, self.heads, self.kv_heads, self.head_dim = vocab, layers, heads, kv_heads, head_dim
        self.dtype = dtype
        self.embed, self.place = w(vocab, width) * width ** 0.5, w(positions, width)
        self.qkv = [w((heads + 2 * kv_heads) * head_dim, width) for _ in range(layers)]
        self.out = [w(width, heads * head_dim) for _ in range(layers)]
        self.up, self.down = [w(4 * width, width) for _ in range(layers)], [w(width, 4 * width) for _ in range(layers)]

    def new_cache(self, batch, beams, max_length, page_size=16) -> PagedCache:
        return PagedCache(batch, beams, max_length, num_layers=self.layers, num_kv_heads=self.kv_heads,
                          head_dim=self.head_dim, page_size=page_size, dtype=self.dtype)

    @torch.no_grad()
    def forward(self, tokens, positions, cache: PagedCache, mask=None) -> torch.Tensor:
        """tokens, positions [B, beams, N] -> logits [B, beams, N, vocab]. Keys and values of the tokens
        go to the cache behind each beam's committed ones."""
        x = self.embed[tokens] + self.place[positions]
        for i in range(self.layers):
            y = F.linear(F.layer_norm(x, x.shape[-1:]), self.qkv[i])
            q, k, v = y.unflatten(-1, (-1, self.head_dim)).split((self.heads, self.kv_heads, self.kv_heads), -2)
            x = x + F.linear(cache.attend(i, q, k, v, mask=mask).flatten(-2), self.out[i])
            x = x + F.linear(F.gelu(F.linear(F.layer_norm(x, x.shape[-1:]), self.up[i])), self.down[i])
        return F.linear(F.layer_norm(x, x.shape[-1:]), self.embed) * x.shape[-1] ** -0.5


def prefill(model: TinyLM, cache: PagedCache, prompt: torch.Tensor) -> torch.Tensor:
    """Writes prompt [B, T] for beam 0 of each example; the logits [B, vocab] behind it. The tokens become
    committed with the caller's next fork (``written``)."""
    B, T = prompt.shape
    room = torch.zeros((B, cache.beam_size), dtype=torch.int32, device=prompt.device)
    room[:, 0] = T
    cache.reserve(room)
    positions = torch.arange(T, device=prompt.device).expand(B, 1, T)
    return model.forward(prompt[:, None], positions, cache)[:, 0, -1]


def beam_decode(model: TinyLM, prompt: torch.Tensor, beams: int, steps: int, eos: int = -1,
                alpha: float = 0.6) -> tuple[SearchResult, PagedCache]:
    B, T = prompt.shape
    cache = model.new_cache(B, beams, T + steps + 1)
    search = DeviceSearch(B, beams, model.vocab, steps, dtype=torch.float32, from_logits=True, eos_token=eos,
                          length_penalty_alpha=alpha, device=prompt.device)
    rows = prefill(model, cache, prompt)[:, None].expand(B, beams, model.vocab)
    written = torch.zeros((B, beams), dtype=torch.int32, device=prompt.device)
    written[:, 0] = T
    for t in range(steps):
        search.step(rows.float())
        state = search.state()
        # Beams follow their parents, then there is room for the token that the step chose.
        cache.fork(state.parents, written=written if t == 0 else 1, room=1)
        if t + 1 < steps:
            tokens = state.tokens.clamp(min=0)[..., None]
            rows = model.forward(tokens, torch.full_like(tokens, T + t), cache)[:, :, 0]
    return search.result(), cache


def drafted_decode(model: TinyLM, prompt: torch.Tensor, steps: int, draft, width: int = 2, depth: int = 3):
    """Greedy decoding with drafts; the tokens [B, >= steps] and the passes of the model it took. ``draft(
    last, width, depth)`` proposes token trees: tokens [B, N] and each one's parent [N], the first one the
    last token chosen."""
    B, T = prompt.shape
    device = prompt.device
    cache = model.new_cache(B, 1, T + steps + 2 * width ** (depth + 1))
    last = prefill(model, cache, prompt).argmax(-1)  # [B]
    cache.fork(written=T, room=0)
    chosen, length = [last[:, None]], torch.full((B,), T, device=device)
    passes = 0
    while passes < steps and min(sum(int((c[b] >= 0).sum()) for c in chosen) for b in range(B)) < steps:
        tokens, parent = draft(last, width, depth)
        N = tokens.shape[1]
        ancestors = torch.eye(N, dtype=torch.bool, device=device)
        level = torch.zeros(N, dtype=torch.long, device=device)
        for i in range(1, N):
            ancestors[i] |= ancestors[parent[i]]
            level[i] = level[parent[i]] + 1
        cache.reserve(N)
        logits = model.forward(tokens[:, None], length[:, None, None] + level, cache, ancestors.expand(B, 1, N, N))
        best = logits[:, 0].argmax(-1)  # the model's choice behind every drafted token
        # A drafted token is right if its parent is and the model chose it there.
        right = torch.zeros((B, N), dtype=torch.bool, device=device)
        right[:, 0] = True
        for i in range(1, N):
            twin = (tokens[:, :i] == tokens[:, i : i + 1]) & (torch.tensor(parent[:i], device=device) == parent[i])
            right[:, i] = right[:, parent[i]] & (best[:, parent[i]] == tokens[:, i]) & ~(twin & right[:, :i]).any(1)
        counts = right.sum(1)
        path = torch.argsort(~right, dim=1, stable=True)  # the right ones, in order
        cache.commit(path[:, None].int(), counts[:, None].int())
        got = torch.where(torch.arange(N, device=device) < counts[:, None], best.gather(1, path), -1)
        chosen.append(got)
        last = got.gather(1, counts[:, None] - 1)[:, 0]
        length = length + counts
        passes += 1
    rows = torch.cat(chosen, 1)
    order = torch.argsort((rows < 0).int(), dim=1, stable=True)
    return rows.gather(1, order), passes


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("batch", 4), ("beams", 8), ("prompt", 100), ("steps", 64)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--dtype", choices=("float32", "float16", "bfloat16"), default="bfloat16")
    args = ap.parse_args()
    model = TinyLM(dtype=getattr(torch, args.dtype))
    prompt = torch.randint(0, model.vocab, (args.batch, args.prompt), device="cuda")
    for _ in range(2):  # the first time pays for the allocations
        torch.cuda.synchronize()
        start = time.perf_counter()
        result, cache = beam_decode(model, prompt, args.beams, args.steps)
        cache.check()
        seconds = time.perf_counter() - start
    used, full = int((cache.references > 0).sum()), args.batch * args.beams * -(-(args.prompt + args.steps) // cache.page_size)
    print(f"beam search: {args.steps / seconds:.0f} steps/s, {used} pages in use ({full} without sharing)")
    print("best scores:", [round(x, 3) for x in result.scores[:, 0].tolist()])
    cache.compact()
    draft = lambda last, width, depth: (  # noqa: E731  a chain of guesses: the last token again
        last[:, None].expand(-1, depth + 1).contiguous(), [-1, *range(depth)])
    tokens, passes = drafted_decode(model, prompt, 16, draft)
    print(f"drafted: {tokens.shape[1]} token columns in {passes} passes")


if __name__ == "__main__":
    main()
