"""8-bit rows, the norm that makes them and the sum of experts' rows, against their formulas."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

import nim_lowprec_b200 as L  # noqa: E402
import experts_refs as R  # noqa: E402

KINDS = [("mx8", 32), ("int8", 32), ("int8", 64), ("int8", 128), ("int8", 256)]


def hard(g, t, k, dtype):
    """Rows of every magnitude: zeros, subnormals, ties of the codes, values over 448 scales."""
    x = R.randn(g, t, k) * torch.exp2(torch.randint(-30, 30, (t, k // 32), generator=g, device="cuda")
                                      .float()).repeat_interleave(32, -1)
    x[:, :32] = 0.0
    if k >= 128:
        x[0, 32:64] = torch.arange(32, device="cuda") * 1.0625  # ties between e4m3 values
        x[0, 64:96] = 0.9999 * 2.0 ** 9
        x[0, 96] = 2.0 ** -130 if dtype == torch.float32 else 2.0 ** -20
    return x.to(dtype)


@pytest.mark.parametrize("kind,group", KINDS)
@pytest.mark.parametrize("x", list(R.DT))
@pytest.mark.parametrize("t,k", [(1, 256), (3, 1024), (37, 2816), (700, 512)])
def test_codec(kind, group, x, t, k):
    g = R.gen(t + k)
    v = hard(g, t, k, R.DT[x])
    codes, scales = R.empty_rows8(t, k, kind, group, 3)
    L.quantizeRows(v, codes, scales)
    want, ws = R.rows8(v, kind, group)
    assert torch.equal(R.bits(scales), R.bits(ws)) and torch.equal(R.bits(codes), R.bits(want))
    for dt in R.DT.values():
        out = torch.empty(t, k, dtype=dt, device="cuda")
        L.dequantizeRows(codes, scales, out)
        assert R.same(out, R.values(codes, scales).float().to(dt))


@pytest.mark.parametrize("kind,group", KINDS[:3])
@pytest.mark.parametrize("x", list(R.DT))
def test_codec_strides_and_alignment(kind, group, x):
    """Views that start anywhere, with rows further apart than they are long."""
    g, t, k = R.gen(5), 19, 192
    big = R.randn(g, t, k + 11, dtype=R.DT[x])
    v = big[:, 3:3 + k]
    codes, scales = R.empty_rows8(t, 8 * k, kind, group)
    codes, scales = codes.view(torch.uint8)[:, 5:5 + k].view(codes.dtype), scales[:, 1:1 + k // group]
    L.quantizeRows(v, codes, scales)
    want, ws = R.rows8(v, kind, group)
    assert torch.equal(R.bits(scales), R.bits(ws)) and torch.equal(R.bits(codes), R.bits(want))
    out = torch.full((t, k + 9), 7.0, device="cuda")
    L.dequantizeRows(codes, scales, out[:, 1:1 + k])
    assert torch.equal(out[:, 1:1 + k], R.values(codes, scales).float())
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 1 + k:] == 7).all())


def test_int8_rows_are_the_bytes_of_calibrate_and_quantize():
    g = R.gen(6)
    x = R.randn(g, 9, 640)
    for group in (32, 64, 128):
        codes, scales = R.empty_rows8(9, 640, "int8", group)
        L.quantizeRows(x, codes, scales)
        s, q = torch.empty(9 * 640 // group, device="cuda"), torch.empty(9 * 640, dtype=torch.int8, device="cuda")
        L.calibrateSymmetric(x.reshape(-1), group, 127.0, s)
        L.quantizeBatch(x.reshape(-1), s, group, q)
        assert torch.equal(scales.reshape(-1), s) and torch.equal(codes.reshape(-1), q)


def test_mxfp8_scales_are_those_of_calibrate_mx():
    x = R.randn(R.gen(7), 9, 640) * 1e-3
    codes, scales = R.empty_rows8(9, 640)
    L.quantizeRows(x, codes, scales)
    s = torch.empty(9 * 20, device="cuda")
    L.calibrateMX(x.reshape(-1), 32, 8, s)
    assert torch.equal(torch.exp2(scales.float() - 127).reshape(-1), s)


def test_infinities_and_nans_stay_in_their_block():
    x = R.randn(R.gen(8), 2, 128)
    x[0, 5], x[0, 40], x[1, 70] = torch.inf, torch.nan, -torch.inf
    clean = x.clone()
    clean[0, 5] = clean[0, 40] = clean[1, 70] = 0.0
    (a, sa), (b, sb) = R.empty_rows8(2, 128), R.empty_rows8(2, 128)
    L.quantizeRows(x, a, sa)
    L.quantizeRows(clean, b, sb)
    out = torch.empty(2, 128, device="cuda")
    L.dequantizeRows(a, sa, out)
    assert out[0, 5] == torch.inf and torch.isnan(out[0, 40]) and out[1, 70] == -torch.inf
    for r, blocks in ((0, (2, 3)), (1, (0, 1, 3))):
        for i in blocks:
            assert torch.equal(R.bits(a)[r, 32 * i:32 * i + 32], R.bits(b)[r, 32 * i:32 * i + 32])
    keep = R.bits(a)[0, 32:64] == R.bits(b)[0, 32:64]  # the NaN does not count for the scale
    assert int((~keep).sum()) == 1 and sa[0, 1] == sb[0, 1]


def check_norm(x, res, w, eps, total, y):
    r = x if res is None else (x.float() + res.float()).to(res.dtype)
    if total is not None:
        assert torch.equal(total, r)
    d = r.double()
    n = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w.double()
    # squares sum up over at most 32 + 10 roundings, halved by the root; mean, eps, root, quotient and
    # two products round once each
    tol = n.abs() * (HALF(y) + 32 * 2.0 ** -24) + R.TINY[y.dtype]
    assert bool(((y.double() - n).abs() <= tol).all())


def HALF(y):
    return R.HALF_ULP[y.dtype]


@pytest.mark.parametrize("x", list(R.DT))
@pytest.mark.parametrize("t,k", [(1, 32), (1, 4096), (5, 2880), (200, 64), (301, 1000), (2, 32768), (150, 8192),
                                 (3, 7)])
def test_norm(x, t, k):
    g = R.gen(k)
    a, b = R.randn(g, t, k, dtype=R.DT[x]), 3.0 * R.randn(g, t, k)
    b = b.to(R.DT[x])
    w = (1.0 + 0.1 * R.randn(g, k)).to(R.DT[x])
    total, y = torch.empty_like(a), torch.empty_like(a)
    L.addRmsNorm(a, b, w, 1e-5, total=total, y=y)
    check_norm(a, b, w, 1e-5, total, y)
    L.addRmsNorm(a, None, w, 1e-5, y=y)
    check_norm(a, None, w, 1e-5, None, y)


@pytest.mark.parametrize("kind,group", KINDS)
@pytest.mark.parametrize("x,stream", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32"), ("bf16", "fp32")])
@pytest.mark.parametrize("t,k", [(3, 256), (160, 4096), (2, 1280)])
def test_norm_in_8_bits_is_the_codec_of_the_norm(kind, group, x, stream, t, k):
    """Rows, norm and stream from one call: the codes are those of the norm in fp32."""
    g = R.gen(11)
    a, b = R.randn(g, t, k, dtype=R.DT[x]), R.randn(g, t, k, dtype=R.DT[stream])
    b0, w = b.clone(), 1.0 + 0.1 * R.randn(g, k)
    y = torch.empty(t, k, device="cuda")
    codes, scales = R.empty_rows8(t, k, kind, group)
    L.addRmsNorm(a, b, w, 1e-6, total=b, y=y, codes=codes, scales=scales)  # the stream in place
    check_norm(a, b0, w, 1e-6, b, y)
    c2, s2 = R.empty_rows8(t, k, kind, group)
    L.quantizeRows(y, c2, s2)
    assert torch.equal(R.bits(codes), R.bits(c2)) and torch.equal(R.bits(scales), R.bits(s2))


def test_norm_of_views_and_in_place():
    g = R.gen(12)
    big = R.randn(g, 9, 2, 100, dtype=torch.bfloat16)
    x, res = big[:, 0, 1:97], big[:, 1, 3:99].clone()
    w = R.randn(g, 96)
    y = torch.empty(9, 96, dtype=torch.float16, device="cuda")
    keep = x.clone()
    L.addRmsNorm(x, res, w, 1e-5, total=x, y=y)
    check_norm(keep, res, w, 1e-5, x, y)
    keep = x.clone()
    L.addRmsNorm(x, None, w, 1e-5, y=x)
    check_norm(keep, None, w, 1e-5, None, x)


def test_rows_of_zeros_and_empty_calls():
    z = torch.zeros(2, 64, device="cuda")
    codes, scales = R.empty_rows8(2, 64, fill=5)
    y = torch.ones_like(z)
    L.addRmsNorm(z, z, torch.ones(64, device="cuda"), 1e-5, y=y, codes=codes, scales=scales)
    assert not bool(y.any()) and not bool(R.bits(codes).any()) and bool((scales == 127).all())
    e = torch.empty(0, 64, device="cuda")
    L.addRmsNorm(e, None, torch.ones(64, device="cuda"), 1e-5, y=e)
    L.quantizeRows(e, *R.empty_rows8(0, 64))
    L.dequantizeRows(*R.empty_rows8(0, 64), e)


def test_int8_rows_feed_the_int8_product():
    """The norm's int8 rows are xq and xScales of dequantGemmQ8."""
    g, t, k, m = R.gen(13), 6, 256, 64
    x, w = R.randn(g, t, k), R.randn(g, m * k)
    codes, scales = R.empty_rows8(t, k, "int8", 32)
    L.addRmsNorm(x, None, torch.ones(k, device="cuda"), 1e-6, codes=codes, scales=scales)
    ws, wq = torch.empty(m * k // 32, device="cuda"), torch.empty(m * k, dtype=torch.int8, device="cuda")
    L.calibrateSymmetric(w, 32, 127.0, ws)
    L.quantizeBatch(w, ws, 32, wq)
    y = torch.empty(m * t, device="cuda")
    L.dequantGemmQ8(wq, ws, 32, codes.reshape(-1), scales.reshape(-1), t, y)
    wv = R.values(wq.view(m, k), ws.view(m, -1))
    want, a = wv @ R.values(codes, scales).T, wv.abs() @ R.values(codes, scales).abs().T
    # 8 groups: exact dots, two products and a sum round once each
    assert bool(((y.view(m, t).double() - want).abs() <= a * 12 * 2.0 ** -24).all())


def test_rows_may_be_the_next_product_s_weights():
    """A GEMV reads its weights before it waits for the kernel before it, so that kernel must not let
    it begin early: each call's product is that of the weights just written."""
    g, m, k = R.gen(14), 8192, 2048
    codes, scales = R.empty_rows8(m, k, "int8", 32)
    xq = torch.randint(-127, 128, (k,), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(k // 32, generator=g, device="cuda")
    a, b = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    for _ in range(6):
        w = R.randn(g, m, k)
        torch.cuda.synchronize()
        L.quantizeRows(w, codes, scales)
        L.dequantGemvQ8(codes.reshape(-1), scales.reshape(-1), 32, xq, xs, a)
        torch.cuda.synchronize()
        L.dequantGemvQ8(codes.reshape(-1), scales.reshape(-1), 32, xq, xs, b)
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", list(R.DT))
@pytest.mark.parametrize("out", list(R.DT))
@pytest.mark.parametrize("t,k,cols", [(1, 8, 4096), (37, 3, 96), (300, 1, 1000), (5, 9, 33)])
def test_combine(rows, out, t, k, cols):
    g = R.gen(t + cols)
    y = R.randn(g, t * k + 3, cols, dtype=R.DT[rows])
    w = torch.rand(t, k, generator=g, device="cuda")
    places = torch.randperm(t * k, generator=g, device="cuda").to(torch.int32).view(t, k)
    places[0, 0] = -1
    if t > 1:
        places[1] = t * k + 3  # no rows at all
    there = (places >= 0) & (places < y.shape[0])
    terms = torch.where(there[..., None], y[places.clamp(0, y.shape[0] - 1).long()].double(), 0.0) * w.double()[..., None]
    for res in (None, R.randn(g, t, cols, dtype=R.DT[out])):
        o = torch.empty(t, cols, dtype=R.DT[out], device="cuda")
        L.combineExperts(y, w, places, o, residual=res)
        want, a = terms.sum(1), terms.abs().sum(1)
        if res is not None:
            want, a = want + res.double(), a + res.double().abs()
        tol = a * (k + 1) * 2.0 ** -24 + want.abs() * HALF(o) * (1 + 2.0 ** -7) + R.TINY[o.dtype]
        assert bool(((o.double() - want).abs() <= tol).all())
    keep = o.clone()
    L.combineExperts(y, w, places, o, residual=o)  # in place
    want = terms.sum(1) + keep.double()
    # (one rounding of the result itself: half an ulp of |terms + keep|, which |terms + residual| + |keep|
    # does not bound, as -2.3 + 2.0 and -2.3 - 0.3 show)
    tol = (a + keep.double().abs()) * (k + 1) * 2.0 ** -24 + want.abs() * HALF(o) * (1 + 2.0 ** -7) + R.TINY[o.dtype]
    assert bool(((o.double() - want).abs() <= tol).all())


def test_a_row_of_infinities_touches_its_token_alone():
    y = torch.ones(4, 64, device="cuda")
    y[2] = torch.inf
    o = torch.empty(2, 64, device="cuda")
    places = torch.tensor([[0, 1], [3, -1]], dtype=torch.int32, device="cuda")
    L.combineExperts(y, torch.ones(2, 2, device="cuda"), places, o)
    assert torch.equal(o, torch.tensor([[2.0], [1.0]], device="cuda").expand(2, 64))
