"""A long-context serving loop over PagedCache: prompts read in chunks, then decode steps that keep each
sequence within a budget of cache rows a head, by evicting the rows that drew the least attention (of
sliding layers, those behind the window).

    python examples/long_context.py [--seqs 8] [--prompt 3000] [--steps 400] [--budget 1024] [--check]

The layers are random (a gpt-oss-like stack: every other one attends to a sliding window behind a few first
tokens that stay visible, with sink logits; the others to everything their cache holds). Each layer has two
caches over one pool of pages and its eviction copies from one into the other, whose pages then hold the
sequence; the old ones are free again. --check runs the same tokens without evictions and prints how far
the outputs move.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from hwnpu_b200 import PagedCache

HEADS, KV, DIM, PAGE, FIRST, RECENT = 16, 4, 64, 32, 4, 64


def rope(x, pos):
    """Rotates x [rows][heads][DIM] by the rows' positions."""
    inv = 10000.0 ** (-torch.arange(0, DIM, 2, device=x.device) / DIM)
    a = pos.view(-1, 1, 1) * inv
    x1, x2 = x.float().chunk(2, -1)
    return torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1).to(x.dtype)


class Layer:
    def __init__(self, seqs, capacity, kept, window, gen, dtype):
        dev = "cuda"
        self.window, hidden = window, HEADS * DIM
        rand = lambda *s: torch.randn(s, device=dev, generator=gen)  # noqa: E731
        self.qkv = (rand((HEADS + 2 * KV) * DIM, hidden) / hidden ** 0.5).to(dtype)
        self.out = (rand(hidden, hidden) / hidden ** 0.5).to(dtype)
        self.sinks = rand(HEADS) if window else None
        # one pool, two block tables: the rows live in one of them, an eviction moves them into the other
        pages = -(-capacity // PAGE)
        k, v = (torch.zeros((2 * seqs * pages, KV, PAGE, DIM), device=dev, dtype=dtype) for _ in range(2))
        ids = torch.randperm(2 * seqs * pages, device=dev, generator=gen).to(torch.int32).view(2, seqs, pages)
        self.caches = [PagedCache(k, v, ids[n].contiguous(), torch.zeros(seqs, dtype=torch.int32, device=dev),
                                  weights=torch.zeros((seqs, KV, pages * PAGE), device=dev)) for n in range(2)]
        c = self.caches[0]
        need = [c.decode_scratch(HEADS, window=window, first=FIRST, accumulate=True),
                c.prompt_scratch(HEADS, seqs * 512, 512, window=window, first=FIRST), c.evict_scratch(kept)]
        self.scratch = torch.empty(max(16, *need), dtype=torch.uint8, device=dev)

    def __call__(self, x, seq, pos, slot, lengths, starts, rows):
        """x [rows][hidden]: one row a sequence (starts None), or up to `rows` of each."""
        cache = self.caches[0]
        y = (x @ self.qkv.T).view(x.shape[0], HEADS + 2 * KV, DIM)
        q, k = rope(y[:, :HEADS], pos), rope(y[:, HEADS : HEADS + KV], pos)
        cache.append(k, y[:, HEADS + KV :], seq, slot)
        cache.lengths.copy_(lengths)
        o = torch.empty_like(q)
        if starts is None:
            # a sliding layer's newest slots are neighbours still, so its window counts slots
            cache.decode(q, o, DIM ** -0.5, window=self.window, first=FIRST, sinks=self.sinks,
                         accumulate=self.window == 0, scratch=self.scratch)
        else:
            cache.prompt(q, o, starts, rows, DIM ** -0.5, window=self.window, first=FIRST, sinks=self.sinks,
                         scratch=self.scratch)
        x = x + o.view_as(x) @ self.out.T
        return x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)

    def evict(self, keep):
        # a sliding layer sees its newest rows and the first ones, so it keeps those; the others choose by weight
        recent = keep - FIRST if self.window else RECENT
        self.caches[0].evict(self.caches[1], keep, first=FIRST, recent=recent, scratch=self.scratch)
        self.caches.reverse()


def run(seqs, prompt, steps, budget, layers=4, window=128, chunk=512, evicting=True, seed=0, dtype=torch.bfloat16):
    """Returns (the last step's hidden rows, rows a head at the end, device milliseconds a decode step)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    keep = budget * 3 // 4  # what an eviction leaves, so that it is not due every step
    if evicting and keep < FIRST + max(window, RECENT):
        raise ValueError(f"a budget of {budget} leaves {keep} rows, fewer than the first {FIRST} and a window of {window}")
    stack = [Layer(seqs, prompt + steps, max(keep, 1), window if n % 2 == 0 else 0, gen, dtype) for n in range(layers)]
    x_all = torch.randn((seqs, prompt, HEADS * DIM), device="cuda", generator=gen).to(dtype)
    ids = torch.arange(seqs, dtype=torch.int32, device="cuda")
    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        x = x_all[:, at : at + n].reshape(seqs * n, -1)
        pos = (at + torch.arange(n, device="cuda")).repeat(seqs)
        starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * n
        lengths = torch.full((seqs,), at + n, dtype=torch.int32, device="cuda")
        for layer in stack:
            x = layer(x, ids.repeat_interleave(n), pos, pos.to(torch.int32), lengths, starts, n)
    x, held = x.view(seqs, n, -1)[:, -1].contiguous(), prompt
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    for step in range(steps):
        if evicting and held >= budget and step > 0:  # the first step gathers the weights the choice is made by
            for layer in stack:
                layer.evict(keep)
            held = min(held, keep)
        pos = torch.full((seqs,), prompt + step, device="cuda")
        slot = torch.full((seqs,), held, dtype=torch.int32, device="cuda")
        held += 1
        lengths = slot + 1
        for layer in stack:
            x = layer(x, ids, pos, slot, lengths, None, 1)
    t1.record()
    torch.cuda.synchronize()
    return x, held, t0.elapsed_time(t1) / max(1, steps)


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--seqs", type=int, default=8)
    p.add_argument("--prompt", type=int, default=3000)
    p.add_argument("--steps", type=int, default=400)
    p.add_argument("--budget", type=int, default=1024)
    p.add_argument("--check", action="store_true")
    a = p.parse_args()
    x, held, ms = run(a.seqs, a.prompt, a.steps, a.budget)
    print(f"{a.seqs} sequences, {a.prompt} + {a.steps} tokens: {held} rows a head held, {ms:.3f} ms a step")
    if a.check:
        y, full, ms = run(a.seqs, a.prompt, a.steps, a.budget, evicting=False)
        cos = torch.nn.functional.cosine_similarity(x.float(), y.float()).min()
        print(f"without evictions: {full} rows a head held, {ms:.3f} ms a step, cosine of the outputs {cos:.4f}")


if __name__ == "__main__":
    main()
