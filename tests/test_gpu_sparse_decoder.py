"""The operators of a sparse feed-forward layer together: one layer against its formulas in 64 bits,
captured into a graph, and the example that decodes with it."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from conftest import ROOT  # noqa: E402
import nim_lowprec_b200 as L  # noqa: E402
from nim_lowprec_b200 import _native as N  # noqa: E402
import experts_refs as R  # noqa: E402

spec = importlib.util.spec_from_file_location("sparse_decoder", os.path.join(ROOT, "examples", "sparse_decoder.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


@pytest.mark.parametrize("kind", ["mx4", "mx8"])
@pytest.mark.parametrize("t", [1, 7, 200])
def test_a_layer_against_64_bits(kind, t):
    """Each call on what the call before it wrote, so that every rounding in between is the layer's
    own and each step keeps its bound."""
    g, width, inner, experts, k = R.gen(t), 256, 192, 6, 2
    cu, su, vu = R.weights(g, experts, 2 * inner, width, kind)
    cd, sd, vd = R.weights(g, experts, width, inner, kind)
    up, down = L.ExpertWeights(cu, su, gated=True), L.ExpertWeights(cd, sd)
    x, res, norm = R.randn(g, t, width), R.randn(g, t, width), 1.0 + 0.1 * R.randn(g, width)
    logits = R.randn(g, t, experts)
    if t > 2:
        logits[2] = -torch.inf  # a padded token
    total, n = torch.empty_like(x), torch.empty_like(x)
    rows, hidden = R.empty_rows8(t, width), R.empty_rows8(t * k, inner)
    i32 = dict(dtype=torch.int32, device="cuda")
    w, e = torch.empty(t, k, device="cuda"), torch.empty(t, k, **i32)
    off, tok, pl = torch.empty(experts + 1, **i32), torch.full((t * k,), -9, **i32), torch.empty(t, k, **i32)
    y, out = torch.zeros(t * k, width, device="cuda"), torch.empty(t, width, dtype=torch.bfloat16, device="cuda")
    ws = L.expertsWorkspace(None, t * k, width)

    def layer():
        L.addRmsNorm(x, res, norm, 1e-6, total=total, y=n, codes=rows[0], scales=rows[1])
        L.routeExperts(logits, w, e, off, tok, pl, workspace=ws)
        L.expertGemmGated(up, *rows, off, *hidden, rowToken=tok, workspace=ws)
        L.expertGemm(down, *hidden, off, y, workspace=ws)
        L.combineExperts(y, w, pl, out)

    def check():
        assert N.device_error() == 0
        assert torch.equal(total, x + res)
        want, scales = R.rows8(n)
        assert torch.equal(R.bits(rows[0]), R.bits(want)) and torch.equal(rows[1], scales)
        chosen, _, offsets, token, places = R.route(logits, k, True)
        assert e.tolist() == chosen and off.tolist() == offsets and pl.tolist() == places
        assert tok[:len(token)].tolist() == token
        yy, a = R.product(vu, R.values(*rows), off, tok)
        R.check_rows8(*hidden, *R.gate(yy, a, width))
        yy, a = R.product(vd, torch.nan_to_num(R.values(*hidden)), off)
        R.check_product(y, yy, a, inner)
        there = pl >= 0
        terms = torch.where(there[..., None], y[pl.clamp(min=0).long()].double(), 0.0) * w.double()[..., None]
        tol = terms.abs().sum(1) * (k + 1) * 2.0 ** -24 + terms.sum(1).abs() * 2.0 ** -8 * (1 + 2.0 ** -7) + 2.0 ** -134
        assert bool(((out.double() - terms.sum(1)).abs() <= tol).all())

    layer()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for seed in (1, 2):  # other inputs through the captured layer, another choice of experts
        x.copy_(R.randn(R.gen(100 + seed), t, width))
        logits.copy_(R.randn(R.gen(200 + seed), t, experts))
        tok.fill_(-9)
        graph.replay()
        torch.cuda.synchronize()
        check()


@pytest.mark.parametrize("kind", ["mx4", "mx8"])
def test_the_example_decodes(kind):
    """It runs, and gives every request its states.  (Token by token and one chunk may choose other
    experts where logits are near, so they are not compared.)"""
    steps, lens = 4, (37, 5, 120)
    a = example.run(kind, steps=steps, lens=lens, cache="fp16")
    for n, s in zip(lens, a):
        assert s.shape == (n + steps, 512) and bool(torch.isfinite(s).all())
