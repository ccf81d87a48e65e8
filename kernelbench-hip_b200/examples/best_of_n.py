"""Sampling n continuations of one prompt with the library's operators.

A small decoder with random weights (fp32): the prompt runs through it once, its slot of the paged cache is forked
for every sample, and each step decodes all samples together, the prompt's full pages read once for all of them.

    python kernelbench-hip_b200/examples/best_of_n.py --samples 8 --steps 32

Per layer: ops.rms_norm, ops.matmul, lm.qk_norm_rope, lm.cache_append, lm.shared_prefix_attention, ops.gelu_tanh;
per step: lm.cache_reserve, lm.penalize_logits, ops.softmax, ops.cumsum.  When a sample ends its slot is freed, and
at the end the live pages are compacted.  A sample that the cache refuses a place ends there, without the host: what
cache_reserve granted goes to cache_append, which leaves the slots of the others' requests alone.
"""
from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch  # noqa: E402

from kbb200 import lm, ops  # noqa: E402


@dataclass
class Sizes:
    vocab: int = 1000
    layers: int = 2
    heads_q: int = 8
    heads_kv: int = 2
    dim: int = 64
    hidden: int = 512
    page: int = 16
    longest: int = 1024


class Decoder:
    """Random weights of a decoder of the given sizes."""

    def __init__(self, sizes: Sizes, seed: int = 0, device="cuda"):
        self.s = s = sizes
        g = torch.Generator(device=device).manual_seed(seed)
        model = s.heads_q * s.dim

        def mat(rows, cols):
            return torch.randn(rows, cols, device=device, generator=g) / rows ** 0.5

        def gain(n):
            return 1 + 0.1 * torch.randn(n, device=device, generator=g)

        self.embedding = torch.randn(s.vocab, model, device=device, generator=g)
        self.layers = [{"norm": gain(model), "qkv": mat(model, (s.heads_q + 2 * s.heads_kv) * s.dim), "q_norm": gain(s.dim),
                        "k_norm": gain(s.dim), "out": mat(model, model), "norm2": gain(model), "up": mat(model, s.hidden),
                        "down": mat(s.hidden, model)} for _ in range(s.layers)]
        self.norm, self.head = gain(model), mat(model, s.vocab)
        self.cos, self.sin = lm.rope_tables(s.longest, s.dim, device=device)


class Cache:
    """A paged cache for all layers: planes 2 l and 2 l + 1 hold the keys and values of layer l."""

    def __init__(self, sizes: Sizes, slots: int, pages: int, device="cuda"):
        s = sizes
        # pages are read only as far as sequences reach, so they need no initial values
        self.pool = torch.empty(2 * s.layers, pages, s.page, s.heads_kv, s.dim, device=device)
        self.table = torch.full((slots, s.longest // s.page), -1, device=device, dtype=torch.int32)
        self.lens = torch.zeros(slots, device=device, dtype=torch.int32)
        self.refs = torch.zeros(pages, device=device, dtype=torch.int32)


def forward(model: Decoder, cache: Cache, tokens, slots, positions, prefix, granted):
    """Logits [sequences, queries, vocab] of the newest tokens [sequences, queries] of the slots, whose places in the
    cache are reserved where granted [sequences] is not 0."""
    s = model.s
    n, q = tokens.shape
    x = model.embedding[tokens].view(n * q, -1)
    rows = cache.table[slots.long()].contiguous()
    lens = cache.lens[slots.long()].contiguous()
    hq, hkv, d = s.heads_q, s.heads_kv, s.dim
    for i, w in enumerate(model.layers):
        qkv = ops.matmul(ops.rms_norm(x, w["norm"]), w["qkv"])
        queries, keys = lm.qk_norm_rope(qkv[:, : hq * d].view(-1, hq, d), qkv[:, hq * d: (hq + hkv) * d].view(-1, hkv, d),
                                        w["q_norm"], w["k_norm"], model.cos, model.sin, positions)
        values = qkv[:, (hq + hkv) * d:].view(n, q, hkv, d)
        k_pages, v_pages = cache.pool[2 * i], cache.pool[2 * i + 1]
        lm.cache_append(keys.view(n, q, hkv, d), values, k_pages, v_pages, cache.table, cache.lens, slots, granted)
        o, _ = lm.shared_prefix_attention(queries.view(n, q, hq, d), k_pages, v_pages, prefix, rows, lens)
        x = x + ops.matmul(o.view(n * q, hq * d), w["out"])
        x = x + ops.matmul(ops.gelu_tanh(ops.matmul(ops.rms_norm(x, w["norm2"]), w["up"])), w["down"])
    return ops.matmul(ops.rms_norm(x, model.norm), model.head).view(n, q, s.vocab)


def generate(model: Decoder, prompt, samples: int, steps: int, seed: int = 0, repetition: float = 1.1,
             frequency: float = 0.1, end_token: int | None = None, pages: int | None = None):
    """`samples` continuations [samples, steps] of the prompt [length] (-1 after an end token, or where the cache of
    `pages` pages, enough for all unless given, had no more room), and the logits of every step as the model gave them
    [samples, steps, vocab]."""
    s, dev = model.s, prompt.device
    length = prompt.shape[0]
    per_sample = -(-(length % s.page + steps) // s.page) + 1
    cache = Cache(s, samples + 1, -(-length // s.page) + samples * per_sample if pages is None else pages, dev)
    root = torch.zeros(1, device=dev, dtype=torch.int32)
    none = torch.empty(0, device=dev, dtype=torch.int32)

    # the prompt, once
    granted = lm.cache_reserve(cache.table, cache.lens, cache.refs, root, length, s.page)
    logits = forward(model, cache, prompt[None], root, torch.arange(length, device=dev), none, granted)[:, -1].expand(samples, -1)
    # its slot for every sample; full pages are shared
    slots = torch.arange(1, samples + 1, device=dev, dtype=torch.int32)
    forked = lm.cache_fork(cache.pool, cache.table, cache.lens, cache.refs, root.expand(samples).contiguous(), slots)
    if not (granted.all() and forked.all()):  # the one look from the host, before the first step
        raise RuntimeError(f"the prompt's {length} tokens and {samples} copies of it do not fit the cache")
    prefix = cache.table[0, : length // s.page].contiguous()

    g = torch.Generator(device=dev).manual_seed(seed)
    made = torch.full((samples, steps), -1, device=dev, dtype=torch.int64)
    history = prompt[None].expand(samples, -1).contiguous()
    rep, freq = (torch.full((samples,), v, device=dev) for v in (repetition, frequency))
    seen = []
    alive = torch.ones(samples, device=dev, dtype=torch.bool)
    for step in range(steps):
        seen.append(logits)
        p = ops.softmax(lm.penalize_logits(logits.contiguous(), prompt=history, output=made, repetition=rep, frequency=freq))
        u = torch.rand(samples, 1, device=dev, generator=g)
        token = (ops.cumsum(p, 1) < u).sum(1).clamp_(max=s.vocab - 1)
        token = torch.where(alive, token, -1)
        made[:, step] = token
        if step + 1 == steps:
            break
        if end_token is not None:
            alive &= token != end_token
        # samples that have ended give their pages back and ask for nothing: slot -1 is passed over
        lm.cache_free(cache.table, cache.lens, cache.refs, torch.where(alive, -1, slots))
        granted = lm.cache_reserve(cache.table, cache.lens, cache.refs, torch.where(alive, slots, -1), 1, s.page)
        alive = granted != 0
        positions = torch.full((samples,), length + step, device=dev)
        logits = forward(model, cache, token.clamp(min=0)[:, None], slots, positions, prefix, granted)[:, 0]
    lm.cache_compact(cache.pool, cache.table, cache.refs)
    return made, torch.stack(seen, 1)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=100, help="tokens of the (random) prompt")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    model = Decoder(Sizes())
    prompt = torch.randint(0, model.s.vocab, (a.prompt,), device="cuda", generator=torch.Generator("cuda").manual_seed(a.seed))
    tokens, _ = generate(model, prompt, a.samples, a.steps, a.seed)
    for i, row in enumerate(tokens.tolist()):
        print(f"sample {i}: {' '.join(map(str, row))}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
