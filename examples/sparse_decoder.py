"""A decoder whose layers end in a sparse feed-forward: attention over a paged cache, then norm,
router and experts over 8-bit rows, put together.

    python examples/sparse_decoder.py [--weights mx4|mx8] [--steps 16]

Prompts of different lengths go through in one ragged chunk, then every request decodes token by
token.  Per layer: the int4 projections and the attention of cached_decode.py, then addRmsNorm (the
residual stream, and its norm as MXFP8 rows), routeExperts, expertGemmGated, expertGemm and
combineExperts, which adds the experts' sum back to the stream.  Weights are random.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import cached_decode as base  # noqa: E402
import nim_lowprec_b200 as L  # noqa: E402


def encode(w, kind):
    """Experts' weights [experts, rows, columns] in fp32, by the library's own encoders."""
    e, m, k = w.shape
    if kind == "mx4":
        scales = torch.empty(e * m * k // 32, device="cuda")
        packed = torch.empty(e * m * k // 2, dtype=torch.uint8, device="cuda")
        L.calibrateMX(w.reshape(-1), 32, 2, scales)
        L.quantizeF4Packed(w.reshape(-1), scales, 32, packed)
        return packed.view(e, m, k // 2), scales.view(e, m, k // 32)
    codes = torch.empty(e * m, k, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(e * m, k // 32, dtype=torch.uint8, device="cuda")
    L.quantizeRows(w.view(e * m, k), codes, scales)
    return codes.view(e, m, k), scales.view(e, m, k // 32)


class SparseLayer:
    """x -> x + sum over the chosen experts of down(silu(gate(n)) * up(n)), n the norm of x."""

    def __init__(self, width, inner, experts, k, kind, gen):
        def matrix(rows, cols):
            return torch.randn(experts, rows, cols, generator=gen, device="cuda") * cols ** -0.5
        self.width, self.inner, self.experts, self.k = width, inner, experts, k
        self.norm = 1.0 + 0.1 * torch.randn(width, generator=gen, device="cuda")
        self.router = torch.randn(width, experts, generator=gen, device="cuda") * width ** -0.5
        self.up = L.ExpertWeights(*encode(matrix(2 * inner, width), kind), gated=True)
        self.down = L.ExpertWeights(*encode(matrix(width, inner), kind))

    def __call__(self, x, delta):
        """x + delta is the stream: both [tokens, width] in fp32; returns the new stream."""
        t, k = x.shape[0], self.k

        def rows8(n, cols):
            return (torch.empty(n, cols, dtype=torch.float8_e4m3fn, device="cuda"),
                    torch.empty(n, cols // 32, dtype=torch.uint8, device="cuda"))
        i32 = dict(dtype=torch.int32, device="cuda")
        stream, n = torch.empty_like(x), torch.empty_like(x)
        rows = rows8(t, self.width)
        L.addRmsNorm(delta, x, self.norm, 1e-6, total=stream, y=n, codes=rows[0], scales=rows[1])
        weights, chosen = torch.empty(t, k, device="cuda"), torch.empty(t, k, **i32)
        offsets, rowToken = torch.empty(self.experts + 1, **i32), torch.empty(t * k, **i32)
        places = torch.empty(t, k, **i32)
        L.routeExperts(n @ self.router, weights, chosen, offsets, rowToken, places)
        hidden = rows8(t * k, self.inner)
        L.expertGemmGated(self.up, *rows, offsets, *hidden, rowToken=rowToken)
        out = torch.empty(t * k, self.width, device="cuda")
        L.expertGemm(self.down, *hidden, offsets, out)
        L.combineExperts(out, weights, places, stream, residual=stream)
        return stream


class SparseDecoder(base.Decoder):
    def __init__(self, layers=2, heads=8, kvHeads=2, dim=64, seed=0, inner=256, experts=8, k=2, kind="mx4"):
        super().__init__(layers, heads, kvHeads, dim, seed)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed + 2)
        self.sparse = [SparseLayer(self.width, inner, experts, k, kind, gen) for _ in range(layers)]

    def after(self, layer, x, delta):
        return self.sparse[layer](x, delta)


def run(kind="mx4", **kw):
    """cached_decode.run with the sparse decoder."""
    return base.run(model=SparseDecoder(seed=kw.get("seed", 0), kind=kind), **kw)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--weights", choices=("mx4", "mx8"), default="mx4")
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    for i, s in enumerate(run(a.weights, steps=a.steps)):
        print(f"request {i}: {s.shape[0]} tokens, last state's norm {s[-1].norm().item():.3f}")
