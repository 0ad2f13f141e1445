"""routeExperts against choices made token by token."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

import nim_lowprec_b200 as L  # noqa: E402
import experts_refs as R  # noqa: E402


def tensors(t, k, n):
    i32 = dict(dtype=torch.int32, device="cuda")
    return (torch.full((t, k), 9.0, device="cuda"), torch.full((t, k), 77, **i32),
            torch.full((n + 1,), 77, **i32), torch.full((t * k,), 77, **i32), torch.full((t, k), 77, **i32))


def check(l, k, renormalize=True, **kw):
    t, n = l.shape
    out = tensors(t, k, n)
    L.routeExperts(l, *out, renormalize=renormalize, **kw)
    compare(l, k, renormalize, out)
    return out


def compare(l, k, renormalize, out):
    weights, experts, offsets, row_token, places = out
    e, w, off, tok, pl = R.route(l, k, renormalize)
    assert experts.tolist() == e and offsets.tolist() == off and places.tolist() == pl
    assert row_token[:len(tok)].tolist() == tok
    assert bool((row_token[len(tok):] == 77).all())  # behind the last row nothing is written
    # differences round once, of up to 100; the exponential is off by an ulp or two, sums of up to 32
    # and 5 terms and the quotient by theirs
    w = torch.tensor(w, dtype=torch.float64).reshape(weights.shape)
    assert bool(((weights.cpu().double() - w).abs() <= w * (100 + 64) * 2.0 ** -24 + 2.0 ** -140).all())


@pytest.mark.parametrize("n,k", [(1, 1), (8, 2), (8, 8), (31, 3), (33, 5), (64, 6), (100, 8), (128, 32),
                                 (257, 4), (1024, 9)])
@pytest.mark.parametrize("t", [1, 13, 64, 65, 200])
@pytest.mark.parametrize("renormalize", [True, False])
def test_choices(n, k, t, renormalize):
    check(2.0 * R.randn(R.gen(n * t), t, n), k, renormalize)


@pytest.mark.parametrize("x", ["fp16", "bf16"])
def test_types_strides_and_ties(x):
    """Few different logits, so that the lower expert has to win; rows of a wider matrix."""
    l = torch.randint(-2, 3, (90, 50), generator=R.gen(3), device="cuda").to(R.DT[x])
    check(l[:, 7:47], 6)
    zeros = torch.zeros(3, 16, device="cuda", dtype=R.DT[x])
    zeros[1, 3] = -0.0
    check(zeros, 4, False)


@pytest.mark.parametrize("t", [5, 300])
def test_masked_experts_and_padded_tokens(t):
    """-inf, the lowest value, NaN and +inf; tokens that see fewer than k experts, or none."""
    l = R.randn(R.gen(4), t, 24)
    l[0] = -torch.inf
    l[1, 2:] = -torch.inf
    l[2, ::2] = torch.nan
    l[3, 5:] = torch.finfo(torch.float32).min
    l[4, 9] = torch.inf
    l[-1] = torch.nan
    check(l, 4)
    check(l, 4, False)
    check(torch.full((t, 24), -torch.inf, device="cuda"), 3)


def test_one_expert_takes_all():
    l = torch.zeros(3000, 40, device="cuda")
    l[:, 17] = 5.0
    check(l, 2)


def test_no_tokens():
    out = tensors(0, 2, 6)
    L.routeExperts(torch.empty(0, 6, device="cuda"), *out)
    assert out[2].tolist() == [0] * 7


def test_many_tokens():
    """Counts over all CTAs; checked by what they have to fulfil."""
    t, n, k = 40000, 96, 4
    l = R.randn(R.gen(6), t, n)
    w, e, off, tok, pl = tensors(t, k, n)
    L.routeExperts(l, w, e, off, tok, pl)
    want = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :k].int()
    assert torch.equal(e, want)
    order = torch.sort(e.reshape(-1), stable=True)
    assert torch.equal(tok.long(), order.indices // k)
    assert torch.equal(off[1:].long(), torch.bincount(e.reshape(-1), minlength=n).cumsum(0))
    assert torch.equal(pl.reshape(-1)[order.indices].long(), torch.arange(t * k, device="cuda"))


def test_captured_and_replayed_with_its_own_workspace():
    l, k = R.randn(R.gen(7), 300, 32), 4
    out, ws = tensors(300, k, 32), L.expertsWorkspace()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        L.routeExperts(l, *out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError):
            L.routeExperts(l, *out)
        L.routeExperts(l, *out, workspace=ws)
    for seed in (8, 9):
        l.copy_(R.randn(R.gen(seed), 300, 32))
        out[3].fill_(77)
        g.replay()
        torch.cuda.synchronize()
        compare(l, k, True, out)
