"""Beam search over a paged cache, with W4A16 linears.

A small decoder with random int4 weights reads a prompt in chunks, and then keeps the `beams` likeliest
continuations: each step scores the next tokens (token_logprobs gives the top alternatives of every
beam), forks the rows of the beams that go on, frees the others' pages, and attends over what the rows
share.  At the end the pool is compacted.

    python examples/branching_decode.py
"""

from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pulsar_amd import ops  # noqa: E402
from pulsar_amd.linear import W4A16Linear, W4A16SiluGate  # noqa: E402
from pulsar_amd.paged import PagedKVCache, Step  # noqa: E402


class Decoder:
    """`layers` blocks of RMSNorm, q|k|v, RoPE, paged attention, o, RMSNorm and a SiLU-gated MLP."""

    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, inter=1024, vocab=1003, seed=0, device="cuda:0"):
        self.heads, self.kv_heads, self.dim = heads, kv_heads, hidden // heads
        gen = torch.Generator(device=device).manual_seed(seed)

        def linear(k: int, n: int) -> W4A16Linear:
            words = torch.randint(-(2 ** 31), 2 ** 31, (k // 8, n), dtype=torch.int32, device=device, generator=gen)
            scales = (torch.rand(k // 128, n, device=device, generator=gen) * 0.2 + 0.9) / (4.6 * math.sqrt(k))
            return W4A16Linear.from_gptq(words, scales.half(), 128)

        kv = kv_heads * self.dim
        self.layers = [{"qkv": W4A16Linear.concat([linear(hidden, hidden), linear(hidden, kv), linear(hidden, kv)]),
                        "o": linear(hidden, hidden),
                        "gate_up": W4A16SiluGate.from_members(linear(hidden, inter), linear(hidden, inter)),
                        "down": linear(inter, hidden)} for _ in range(layers)]
        self.embedding = torch.randn(vocab, hidden, device=device, generator=gen).half()
        self.head = (torch.randn(vocab, hidden, device=device, generator=gen) * 3 / math.sqrt(hidden)).half()

    def rope(self, x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        half = self.dim // 2
        angle = pos[:, None].float() * 10000.0 ** (-torch.arange(half, device=x.device) / half)
        cos, sin = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x.float().split(half, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(x.dtype)

    def forward(self, tokens: torch.Tensor, pos: torch.Tensor, attend) -> torch.Tensor:
        """Logits [T, vocab] of tokens at positions pos; attend(layer, q, k, v) -> [T, heads, dim]."""
        def norm(x):
            return torch.nn.functional.rms_norm(x.float(), x.shape[-1:]).half()

        x = self.embedding[tokens]
        split = [self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim]
        for i, layer in enumerate(self.layers):
            q, k, v = (t.unflatten(-1, (-1, self.dim)) for t in layer["qkv"](norm(x)).split(split, dim=-1))
            o = attend(i, self.rope(q, pos), self.rope(k, pos), v)
            x = x + layer["o"](o.flatten(1))
            x = x + layer["down"](layer["gate_up"](norm(x)))
        return norm(x) @ self.head.t()


def paged(cache: PagedKVCache, step: Step):
    def attend(layer, q, k, v):
        cache.write(layer, k, v, step)
        return cache.attend(layer, q, step)

    return attend


def room(missing: torch.Tensor, what: str) -> None:
    """Raises where the cache had no room: it took nothing then, and the rows are as they were."""
    if int(missing):
        raise RuntimeError(f"{what}: {int(missing)} pages (or table columns) too few")


def beam_search(model: Decoder, cache: PagedKVCache, prompt: torch.Tensor, beams: int, steps: int, chunk: int = 48):
    """The `beams` likeliest continuations found, [(log probability, tokens)], likeliest first, and the
    prompt's own log probabilities.  Uses rows 0 to 2 * beams - 1 of the cache."""
    dev, n = prompt.device, prompt.numel()
    scored = []
    for at in range(0, n, chunk):  # the prompt, in chunks, into row 0
        tokens = prompt[at:at + chunk]
        step = cache.extend([tokens.numel()] + [0] * (cache.rows - 1))
        room(step.missing, "prompt")
        logits = model.forward(tokens, torch.arange(at, at + tokens.numel(), device=dev), paged(cache, step))
        after = torch.full_like(tokens, -1)  # the token that follows each one, none behind the last
        after[:min(tokens.numel(), n - at - 1)] = prompt[at + 1:at + chunk + 1]
        lp, _, _, top, ids = ops.token_logprobs(logits, after, beams)
        scored.append(lp)
    alive = [(float(top[-1, j]), 0, [int(ids[-1, j])]) for j in range(beams)]  # (score, row that it continues, tokens)
    rows, spare = list(range(beams)), list(range(beams, 2 * beams))
    held = [0]
    for i in range(1, steps + 1):
        # every beam goes on in a row of its own, which shares its parent's full pages
        room(cache.fork([row for _, row, _ in alive], spare), "fork")
        cache.free(held)
        held, spare = spare, rows
        rows = held
        if i == steps:
            break
        step = cache.extend([1 if r in held else 0 for r in range(cache.rows)])
        room(step.missing, "next tokens")
        tokens = torch.tensor([t[-1] for _, _, t in alive], device=dev)
        logits = model.forward(tokens, torch.full((beams,), n + i - 1, device=dev), paged(cache, step))
        _, _, _, top, ids = ops.token_logprobs(logits, torch.full_like(tokens, -1), beams)
        top, ids = top.tolist(), ids.tolist()
        grown = [(s + top[b][j], held[b], t + [ids[b][j]]) for b, (s, _, t) in enumerate(alive) for j in range(beams)]
        alive = sorted(grown, key=lambda g: -g[0])[:beams]
    return [(s, t) for s, _, t in alive], torch.cat(scored)


def main() -> None:
    torch.manual_seed(1)
    model = Decoder()
    cache = PagedKVCache(layers=2, pages=256, page_size=16, kv_heads=2, head_dim=64, rows=8, max_seq_len=512,
                         dtype=torch.float16)
    prompt = torch.randint(0, 1003, (150,), device="cuda:0")
    found, scored = beam_search(model, cache, prompt, beams=4, steps=12)
    print(f"prompt: {prompt.numel()} tokens, mean log probability {float(scored[:-1].mean()):.3f}")
    for score, tokens in found:
        print(f"{score:9.3f}  {tokens}")
    used = cache.compact()
    print(f"pages in use: {int(used)} of {cache.ref_counts.numel()}, the pool's first ones after compacting")


if __name__ == "__main__":
    main()
