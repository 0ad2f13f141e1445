"""A small int4 decoder with a paged key/value cache: what a layer does between its
projections, put together.

    python examples/cached_decode.py [--cache int8|fp16|bf16] [--steps 16]

Prompts of different lengths go through in one ragged chunk, then every request decodes token
by token.  Per step the page tables and slot maps are built on the GPU (assignPages); per layer
the projections run on packed int4 weights, new keys and values are written to the cache
(storeKV) and the queries attend to it (pagedAttention).  Weights are random.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import nim_lowprec_b200 as L  # noqa: E402

GROUP = 32


class Linear:
    """Packed int4 weights with fp32 group scales (calibrateSymmetric + quantizeI4Packed)."""

    def __init__(self, rows, cols, gen):
        w = torch.randn(rows * cols, generator=gen, device="cuda") * cols ** -0.5
        self.rows, self.cols = rows, cols
        self.scales = torch.empty(rows * cols // GROUP, device="cuda")
        self.packed = torch.empty(rows * cols // 2, dtype=torch.uint8, device="cuda")
        L.calibrateSymmetric(w, GROUP, 7.0, self.scales)
        L.quantizeI4Packed(w, self.scales, GROUP, self.packed)

    def __call__(self, x):
        """fp32 [tokens, cols] -> fp32 [tokens, rows]; activations go through Q8_0."""
        t = x.shape[0]
        if t == 1:
            y = torch.empty(1, self.rows, device="cuda")
            L.quantizeDequantGemvI4Q8(self.packed, self.scales, GROUP, x.reshape(-1), y.view(-1))
            return y
        xq = torch.empty(t * self.cols, dtype=torch.int8, device="cuda")
        xs = torch.empty(t * self.cols // GROUP, device="cuda")
        L.quantizeQ8_0Split(x.reshape(-1), xq, xs)
        y = torch.empty(self.rows * t, device="cuda")
        L.dequantGemmI4Q8(self.packed, self.scales, GROUP, xq, xs, t, y)
        return y.view(self.rows, t).t().contiguous()


class Decoder:
    def __init__(self, layers=2, heads=8, kvHeads=2, dim=64, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.heads, self.kvHeads, self.dim = heads, kvHeads, dim
        self.width = heads * dim
        qkv = (heads + 2 * kvHeads) * dim
        self.layers = [(Linear(qkv, self.width, gen), Linear(self.width, self.width, gen))
                       for _ in range(layers)]

    def new_caches(self, pages, pageSize, dtype):
        return [L.KVCache.allocate(pages, pageSize, self.kvHeads, self.dim, dtype)
                for _ in self.layers]

    def forward(self, x, caches, step, window=0, sinks=0):
        """x [tokens, width]: the new tokens' hidden states, request after request."""
        t, h, g = x.shape[0], self.heads, self.kvHeads
        for (proj, outp), cache in zip(self.layers, caches):
            norm = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
            rows = proj(norm).view(t, h + 2 * g, self.dim)
            L.storeKV(cache, rows[:, h:h + g], rows[:, h + g:], step.slots)
            out = torch.empty(t, h, self.dim, device="cuda")
            L.pagedAttention(cache, step.tables, step.qStart, step.seqLens, rows[:, :h], out,
                             window=window, sinks=sinks)
            x = x + outp(out.view(t, self.width))
        return x


class Step:
    """What the layers read of a step."""

    def __init__(self, batch):
        self.tables, self.qStart, self.seqLens = batch.tables, batch.qStart, batch.seqLens
        self.slots, self.positions = batch.slots, batch.positions


class Batch:
    """Requests, their page tables and the free list, all on the GPU."""

    def __init__(self, requests, pages, pageSize, pagesPerRequest):
        i32 = dict(dtype=torch.int32, device="cuda")
        self.pageSize = pageSize
        self.free = torch.arange(pages, **i32)
        self.head, self.headNext = torch.zeros(1, **i32), torch.zeros(1, **i32)
        self.tables = torch.full((requests, pagesPerRequest), -1, **i32)
        self.ctx = torch.zeros(requests, **i32)
        self.qStart = torch.zeros(requests + 1, **i32)
        self.seqLens = torch.zeros(requests, **i32)

    def advance(self, newLens, tokens):
        """Room for newLens tokens per request (`tokens` in all)."""
        self.slots = torch.empty(tokens, dtype=torch.int64, device="cuda")
        self.positions = torch.empty(tokens, dtype=torch.int32, device="cuda")
        L.assignPages(self.ctx, newLens, self.pageSize, self.free, self.head, self.tables,
                      self.qStart, self.seqLens, self.slots, self.positions, self.headNext)
        self.head, self.headNext = self.headNext, self.head
        # the lengths after this step are the cached ones of the next
        self.step, self.ctx, self.seqLens = Step(self), self.seqLens, torch.empty_like(self.ctx)
        return self.step


def run(cache="int8", steps=16, lens=(37, 5, 120), window=0, sinks=0, seed=0, one_chunk=False):
    """Hidden states of the prompts and the decoded tokens, [requests][tokens, width].  The next
    token's hidden state is the last one's, normed.  one_chunk: all tokens again as one chunk
    (the decoded ones given), which must give the same states."""
    dtype = {"int8": torch.int8, "fp16": torch.float16, "bf16": torch.bfloat16}[cache]
    model, page = Decoder(seed=seed), 16
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + 1)
    prompts = [torch.randn(n, model.width, generator=gen, device="cuda") for n in lens]
    per = -(-(max(lens) + steps) // page)
    pages = per * len(lens)

    def feed(inputs, batch, caches):
        new = torch.tensor([x.shape[0] for x in inputs], dtype=torch.int32, device="cuda")
        x = torch.cat(inputs)
        y = model.forward(x, caches, batch.advance(new, x.shape[0]), window, sinks)
        return list(y.split([i.shape[0] for i in inputs]))

    def new_token(states):
        last = states[-1:]
        return last * torch.rsqrt(last.square().mean(-1, keepdim=True) + 1e-6)

    batch, caches = Batch(len(lens), pages, page, per), model.new_caches(pages, page, dtype)
    states = feed(prompts, batch, caches)
    inputs = list(prompts)
    for _ in range(steps):
        tokens = [new_token(s) for s in states]
        inputs = [torch.cat(p) for p in zip(inputs, tokens)]
        states = [torch.cat(p) for p in zip(states, feed(tokens, batch, caches))]
    if not one_chunk:
        return states
    batch, caches = Batch(len(lens), pages, page, per), model.new_caches(pages, page, dtype)
    return states, feed(inputs, batch, caches)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--cache", choices=("int8", "fp16", "bf16"), default="int8")
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    step_by_step, at_once = run(a.cache, a.steps, one_chunk=True)
    for i, (s, c) in enumerate(zip(step_by_step, at_once)):
        off = ((s - c).norm() / c.norm()).item()
        print(f"request {i}: {s.shape[0]} tokens, decoded against one chunk: {off:.1e} apart")
