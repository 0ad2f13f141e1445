"""Experts' products against 64 bits: types, ragged segments, odd sizes, gathered rows, the gated
form, cut tiles, rows that belong to nobody."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

import nim_lowprec_b200 as L  # noqa: E402
from nim_lowprec_b200 import _native as N  # noqa: E402
import experts_refs as R  # noqa: E402


def rows_of(g, t, k):
    """(codes, scales, values) of x, blocks of different magnitudes."""
    x = R.randn(g, t, k) * torch.exp2(torch.randint(-6, 7, (t, k // 32), generator=g, device="cuda")
                                      .float()).repeat_interleave(32, -1)
    c, s = R.rows8(x)
    return c, s, R.values(c, s)


def run(seed, counts, experts, rows, cols, kind="mx4", out="fp32", gather=None, gated=False, extra=0, **kw):
    g = R.gen(seed)
    wc, ws, wv = R.weights(g, experts, rows, cols, kind)
    w = L.ExpertWeights(wc, ws, gated=gated)
    del wc, ws
    off = R.segments(list(counts), experts)
    r = int(off[-1]) + extra
    token = None
    if gather:
        token = torch.randint(0, gather, (r,), generator=g, device="cuda").to(torch.int32)
        if r > 2:
            token[1] = -1  # rows of zeros
            token[2] = gather
    c, s, x = rows_of(g, gather or r, cols)
    y, a = R.product(wv, x, off, token)
    if gated:
        oc, os_ = R.empty_rows8(r, rows // 2, fill=0x55)
        L.expertGemmGated(w, c, s, off, oc, os_, rowToken=token, **kw)
        assert N.device_error() == 0
        h, e = R.gate(y, a, cols)
        R.check_rows8(oc, os_, h, e)
        behind = slice(int(off[-1]), None)
        assert bool((R.bits(oc)[behind] == 0x55).all()) and bool((os_[behind] == 0x55).all())
    else:
        o = torch.full((r, rows), 7.0, dtype=R.DT[out], device="cuda")
        L.expertGemm(w, c, s, off, o, rowToken=token, **kw)
        assert N.device_error() == 0
        R.check_product(o, y, a, cols)
        assert bool((o[int(off[-1]):] == 7).all())  # rows of no expert


RAGGED = [5, 0, 1, 17, 0, 33, 16]


@pytest.mark.parametrize("kind", ["mx4", "mx8"])
@pytest.mark.parametrize("out", list(R.DT))
@pytest.mark.parametrize("gather", [None, 20])
def test_types(kind, out, gather):
    run(1, RAGGED, 8, 160, 256, kind, out, gather, extra=3)


@pytest.mark.parametrize("cols", [32, 64, 96, 128, 160, 416, 1024, 4064])
@pytest.mark.parametrize("gather", [None, 9])
def test_inner_sizes(cols, gather):
    """One chunk of K and less, chunks that end early, scales that are no whole words."""
    run(2, RAGGED, 8, 130, cols, "mx4", "fp32", gather)
    run(2, RAGGED, 8, 130, cols, "mx8", "fp32", gather)


@pytest.mark.parametrize("rows", [1, 5, 127, 128, 129, 257, 1003])
def test_features(rows):
    run(3, RAGGED, 7, rows, 192, "mx4", "bf16")


@pytest.mark.parametrize("counts", [
    [1], [16], [0, 0, 31], [64, 64], [65, 3], [100] * 3, [128, 129, 240, 241], [250, 700, 1], [1500],
    [3000, 0, 5], [480] * 4, [33] * 40])
@pytest.mark.parametrize("kind", ["mx4", "mx8"])
def test_segments(counts, kind):
    """From one row to several tiles of rows, through every way in which tiles are cut."""
    run(4, counts, len(counts), 300, 352, kind, "fp32")
    run(4, counts, len(counts), 384, 352, kind, gated=True)
    run(5, counts, len(counts) + 2, 256, 352, kind, "bf16", gather=max(counts))


@pytest.mark.parametrize("counts", [[700], [500, 0, 300]])
@pytest.mark.parametrize("tokens", [1, 20, 60, 100])
def test_a_token_many_times(counts, tokens):
    """More rows than tokens: the same few rows of x, again and again, for one expert."""
    run(17, counts, len(counts), 300, 1024, "mx4", "fp32", gather=tokens)
    run(17, counts, len(counts), 256, 1024, "mx8", gated=True, gather=tokens)


@pytest.mark.parametrize("experts", [1, 31, 32, 33, 100, 1024])
def test_experts(experts):
    counts = [(i * 7) % 5 if i % 3 else 0 for i in range(experts)]
    counts[-1] = 2
    run(6, counts, experts, 64, 64, "mx4", "fp32")


@pytest.mark.parametrize("counts", [[1], [1, 1, 0, 1], [3, 0, 20], [40] * 4])
@pytest.mark.parametrize("cols", [2048, 8192])
def test_few_rows_over_a_long_axis(counts, cols):
    """Tiles cut along K, by two CTAs and by many, and joined."""
    run(7, counts, len(counts), 200, cols, "mx4", "fp32")
    run(7, counts, len(counts), 256, cols, "mx8", gated=True, gather=50)


@pytest.mark.parametrize("inner", [32, 64, 96, 480, 1440])
@pytest.mark.parametrize("kind", ["mx4", "mx8"])
@pytest.mark.parametrize("gather", [None, 30])
def test_gated(inner, kind, gather):
    run(8, RAGGED, 8, 2 * inner, 288, kind, gated=True, gather=gather, extra=2)
    run(8, [300, 20, 290], 3, 2 * inner, 288, kind, gated=True, gather=gather and 400)


def test_sums_do_not_depend_on_the_rows_beside():
    """A row alone, and among others of the same call: the same bits (no sum follows an order that
    other CTAs decide)."""
    g = R.gen(9)
    wc, ws, _ = R.weights(g, 2, 384, 4096, "mx4")
    w = L.ExpertWeights(wc, ws)
    c, s, _ = rows_of(g, 30, 4096)
    off = R.segments([13, 17], 2)
    a, b = (torch.empty(30, 384, device="cuda") for _ in range(2))
    for _ in range(5):
        L.expertGemm(w, c, s, off, a)
        L.expertGemm(w, c, s, off, b)
        assert torch.equal(a, b)


def test_long_sums_of_one_sign():
    """16384 products of one sign: a cut at every step would add up (the bound is derived in
    experts_refs.sum_error; results are much nearer)."""
    k = 16384
    codes = torch.full((1, 128, k // 2), 0x77, dtype=torch.uint8, device="cuda")
    w = L.ExpertWeights(codes, torch.ones(1, 128, k // 32, device="cuda"))
    x = 1.0 + torch.rand(40, k, generator=R.gen(10), device="cuda")
    c, s = R.rows8(x)
    o = torch.empty(40, 128, device="cuda")
    L.expertGemm(w, c, s, R.segments([40], 1), o)
    want = 6.0 * R.values(c, s).sum(-1, keepdim=True)
    assert float(((o.double() - want) / want).abs().max()) <= R.sum_error(k)


def test_infinities_and_nans_stay_in_their_rows():
    g = R.gen(11)
    wc, ws, wv = R.weights(g, 2, 200, 256, "mx4")
    w = L.ExpertWeights(wc, ws)
    c, s, x = rows_of(g, 40, 256)
    R.bits(c)  # (a view: the codes below change in place)
    c.view(torch.uint8)[3, 9] = 0x7f  # NaN
    s[20, 2] = 255  # a NaN scale
    off = R.segments([21, 19], 2)
    o = torch.empty(40, 200, device="cuda")
    L.expertGemm(w, c, s, off, o)
    y, a = R.product(wv, torch.nan_to_num(x), off)
    bad = torch.isnan(o).any(-1)
    assert bool(torch.isnan(o[3]).all()) and bool(torch.isnan(o[20]).all()) and int(bad.sum()) == 2
    keep = ~bad
    R.check_product(o[keep], y[keep], a[keep], 256)


def test_strides():
    """Rows, scales and results that are views of wider tensors."""
    g, k, m = R.gen(12), 320, 70
    wc, ws, wv = R.weights(g, 3, m, k, "mx8")
    w = L.ExpertWeights(wc, ws)
    c, s, x = rows_of(g, 33, k)
    wide_c = torch.zeros(33, k + 48, dtype=torch.uint8, device="cuda")
    wide_c[:, 16:16 + k] = c.view(torch.uint8)
    wide_s = torch.zeros(33, k // 32 + 5, dtype=torch.uint8, device="cuda")
    wide_s[:, 3:3 + k // 32] = s
    off = R.segments([10, 3, 20], 3)
    wide_o = torch.full((33, m + 9), 3.0, dtype=torch.bfloat16, device="cuda")
    y, a = R.product(wv, x, off)
    L.expertGemm(w, wide_c[:, 16:16 + k].view(torch.float8_e4m3fn), wide_s[:, 3:3 + k // 32], off, wide_o[:, 1:1 + m])
    R.check_product(wide_o[:, 1:1 + m], y, a, k)
    assert bool((wide_o[:, 0] == 3).all()) and bool((wide_o[:, 1 + m:] == 3).all())


def test_offsets_are_clamped():
    """Offsets that lead out of the rows, or back: nothing outside is touched."""
    g = R.gen(13)
    wc, ws, _ = R.weights(g, 4, 128, 128, "mx4")
    w = L.ExpertWeights(wc, ws)
    c, s, _ = rows_of(g, 8, 128)
    o = torch.full((24, 128), 7.0, device="cuda")
    for off in ([-5, 3, 1000, 2, 2 ** 31 - 1], [2 ** 31 - 1, 0, -2 ** 31, 5, 4], [0, 0, 0, 0, 0]):
        L.expertGemm(w, c, s, torch.tensor(off, dtype=torch.int32, device="cuda"), o[8:16])
        assert N.device_error() == 0
        assert bool((o[:8] == 7).all()) and bool((o[16:] == 7).all())


def test_weights_of_the_library_s_encoders():
    """calibrateMX + quantizeF4Packed, and quantizeRows, as weights; one expert is a projection."""
    g, m, k, t = R.gen(14), 96, 256, 5
    v = R.randn(g, m, k)
    scales, packed = torch.empty(m * k // 32, device="cuda"), torch.empty(m * k // 2, dtype=torch.uint8, device="cuda")
    L.calibrateMX(v.reshape(-1), 32, 2, scales)
    L.quantizeF4Packed(v.reshape(-1), scales, 32, packed)
    c, s, x = rows_of(g, t, k)
    off = R.segments([t], 1)
    n = torch.stack((packed & 15, packed >> 4), -1).reshape(m, k).long()
    wv = R.E2M1.cuda()[n & 7].double() * torch.where(n >= 8, -1.0, 1.0) * scales.view(m, -1).double().repeat_interleave(32, -1)
    o = torch.empty(t, m, device="cuda")
    L.expertGemm(L.ExpertWeights(packed.view(1, m, -1), scales.view(1, m, -1)), c, s, off, o)
    R.check_product(o, x @ wv.T, x.abs() @ wv.abs().T, k)
    wc, wsc = R.empty_rows8(m, k)
    L.quantizeRows(v, wc, wsc)
    wv = R.values(wc, wsc)
    L.expertGemm(L.ExpertWeights(wc[None], wsc[None].view(torch.float8_e8m0fnu)), c, s.view(torch.float8_e8m0fnu), off, o)
    R.check_product(o, x @ wv.T, x.abs() @ wv.abs().T, k)


def test_streams_and_captured_graphs():
    """Calls of two streams at once, and two captured graphs with a workspace each."""
    g, k, m = R.gen(15), 2048, 256
    wc, ws, wv = R.weights(g, 2, m, k, "mx4")
    w = L.ExpertWeights(wc, ws)
    c, s, x = rows_of(g, 6, k)
    off = R.segments([4, 5], 2)
    token = torch.tensor([0, 1, 2, 3, 5, 4, 3, 2, 1], dtype=torch.int32, device="cuda")
    y, a = R.product(wv, x, off, token)
    outs = [torch.zeros(9, m, device="cuda") for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                L.expertGemm(w, c, s, off, o, rowToken=token)
    torch.cuda.synchronize()
    graphs = []
    for o in outs[2:]:
        ws_ = L.expertsWorkspace(None, 9, k)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            L.expertGemm(w, c, s, off, o, rowToken=token, workspace=ws_)
        graphs.append((gr, ws_))
    for _ in range(5):
        for (gr, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert N.device_error() == 0
    for o in outs:
        R.check_product(o, y, a, k)


def test_refusals_on_the_device():
    g = R.gen(16)
    wc, ws, _ = R.weights(g, 2, 64, 64, "mx4")
    w, wg = L.ExpertWeights(wc, ws), L.ExpertWeights(wc, ws, gated=True)
    c, s = R.empty_rows8(4, 64)
    off, o = R.segments([2, 2], 2), torch.empty(4, 64, device="cuda")
    L.expertGemm(w, c, s, off, o)
    bad = [(AssertionError, lambda: L.expertGemm(w, c, s, off[:2], o)),
           (AssertionError, lambda: L.expertGemm(w, c, s, off, o[:3])),
           (AssertionError, lambda: L.expertGemm(w, c, s, off, o[:, :63])),
           (AssertionError, lambda: L.expertGemm(w, *R.empty_rows8(4, 96), off, o)),
           (AssertionError, lambda: L.expertGemm(w, c, s[:, :1], off, o)),
           (TypeError, lambda: L.expertGemm(w, *R.empty_rows8(4, 64, "int8"), off, o)),
           (TypeError, lambda: L.expertGemm(w, c, s.float(), off, o)),
           (TypeError, lambda: L.expertGemm(w, c, s, off.long(), o)),
           (TypeError, lambda: L.expertGemm(w, c, s, off, o.double())),
           (TypeError, lambda: L.expertGemm(w, c.cpu(), s, off, o)),
           (ValueError, lambda: L.expertGemm(w, c, s, off, o.t())),
           (N.NativeError, lambda: L.expertGemm(wg, c, s, off, o)),
           (N.NativeError, lambda: L.expertGemmGated(w, c, s, off, *R.empty_rows8(4, 32))),
           (AssertionError, lambda: L.expertGemm(w, c, s, off, o, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))),
           (N.NativeError, lambda: L.expertGemm(w, R.bits(R.empty_rows8(4, 160)[0])[:, 8:72].view(torch.float8_e4m3fn), s, off, o)),
           (AssertionError, lambda: L.ExpertWeights(wc, ws[:, :, :1])),
           (AssertionError, lambda: L.ExpertWeights(wc[:, :32].contiguous(), ws[:, :32].contiguous(), gated=True)),
           (ValueError, lambda: L.ExpertWeights(wc[:, :, ::2], ws[:, :, :1])),
           (TypeError, lambda: L.ExpertWeights(wc.float(), ws)),
           (AssertionError, lambda: L.quantizeRows(o, *R.empty_rows8(4, 96))),
           (TypeError, lambda: L.addRmsNorm(o, None, o[0], 1e-5, codes=c)),
           (N.NativeError, lambda: L.addRmsNorm(o, None, o[0], 1e-5)),
           (N.NativeError, lambda: L.addRmsNorm(o, o.half(), o[0], 1e-5, y=o)),
           (AssertionError, lambda: L.addRmsNorm(o, None, o[0, :63], 1e-5, y=o))]
    for i, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"case {i}")
