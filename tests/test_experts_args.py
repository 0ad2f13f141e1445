"""What the entry points of 8-bit rows, the router and the experts refuse, without a GPU: statuses of
the C ABI before any device work, and the Python layer's checks of types."""
import ctypes

import numpy as np
import pytest

from nim_lowprec_b200 import _native as N

torch = pytest.importorskip("torch")

import nim_lowprec_b200 as L  # noqa: E402
from nim_lowprec_b200.experts import _WeightsStruct  # noqa: E402


def P(i=1):
    return ctypes.c_void_p(i << 24)  # a pointer that is only looked at


class Matrix(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("stride", ctypes.c_int64), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class Rows8(ctypes.Structure):
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("rows", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("code_stride", ctypes.c_int64), ("scale_stride", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("group", ctypes.c_int32)]


def make(cls, defaults, kw):
    s = cls()
    for k, v in {**defaults, **kw}.items():
        setattr(s, k, v)
    return s


def matrix(**kw):
    return make(Matrix, dict(data=1 << 24, rows=4, cols=64, stride=64, dtype=N.LP_F32, reserved=0), kw)


def rows8(**kw):
    return make(Rows8, dict(codes=1 << 24, scales=2 << 24, rows=4, cols=64, code_stride=64, scale_stride=2,
                            dtype=N.LP_E4M3, group=32), kw)


def weights(**kw):
    return make(_WeightsStruct, dict(tiles=3 << 24, scales=4 << 24, experts=2, rows=64, cols=64, dtype=N.LP_E2M1,
                                     gated=0), kw)


ref = ctypes.byref
MATRICES = [(dict(dtype=N.LP_I8), N.LP_ERR_ARG), (dict(data=None), N.LP_ERR_ARG), (dict(rows=-1), N.LP_ERR_SHAPE),
            (dict(stride=-1), N.LP_ERR_SHAPE), (dict(stride=1 << 31), N.LP_ERR_SHAPE), (dict(rows=5), N.LP_ERR_SHAPE),
            (dict(cols=96), N.LP_ERR_SHAPE)]
ROWS8 = [(dict(dtype=N.LP_F32), N.LP_ERR_ARG), (dict(codes=None), N.LP_ERR_ARG), (dict(scales=None), N.LP_ERR_ARG),
         (dict(group=64), N.LP_ERR_SHAPE), (dict(group=0), N.LP_ERR_SHAPE), (dict(rows=-1), N.LP_ERR_SHAPE),
         (dict(cols=63), N.LP_ERR_SHAPE), (dict(code_stride=-64), N.LP_ERR_SHAPE),
         (dict(scale_stride=1 << 32), N.LP_ERR_SHAPE), (dict(rows=5), N.LP_ERR_SHAPE)]


@pytest.mark.parametrize("change,status", MATRICES)
def test_matrices_that_are_refused(change, status):
    m, q, ok = matrix(**change), rows8(), matrix()
    lib = N.lib()
    assert lib.lp_quantize_rows(ref(m), ref(q), None) == status
    assert lib.lp_dequantize_rows(ref(q), ref(m), None) == status
    for at in range(3):
        ms = [ref(ok), ref(ok), ref(ok)]
        ms[at] = ref(m)
        assert lib.lp_add_rms_norm(ref(ok), ms[0], P(), 64, N.LP_F32, 1e-5, ms[1], ms[2], None, None) == status


@pytest.mark.parametrize("change,status", ROWS8)
def test_rows_that_are_refused(change, status):
    q, ok = rows8(**change), matrix()
    lib = N.lib()
    assert lib.lp_quantize_rows(ref(ok), ref(q), None) == status
    assert lib.lp_dequantize_rows(ref(q), ref(ok), None) == status
    assert lib.lp_add_rms_norm(ref(ok), None, P(), 64, N.LP_F32, 1e-5, None, None, ref(q), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(n=63), N.LP_ERR_SHAPE), (dict(w=None), N.LP_ERR_ARG), (dict(wt=N.LP_I8), N.LP_ERR_ARG),
    (dict(eps=float("nan")), N.LP_ERR_ARG), (dict(eps=-1e-5), N.LP_ERR_ARG), (dict(y=None), N.LP_ERR_ARG),
    (dict(res=matrix(dtype=N.LP_F16)), N.LP_ERR_ARG), (dict(total=matrix(dtype=N.LP_BF16)), N.LP_ERR_ARG)])
def test_norm_refuses(kw, status):
    a = dict(res=None, w=P(), n=64, wt=N.LP_F32, eps=1e-5, total=None, y=matrix())
    a.update(kw)
    r = [None if m is None else ref(m) for m in (a["res"], a["total"], a["y"])]
    x = matrix()
    assert N.lib().lp_add_rms_norm(ref(x), r[0], a["w"], a["n"], a["wt"], a["eps"], r[1], r[2], None, None) == status


def test_norm_refuses_long_rows():
    x = matrix(cols=32776, stride=32776)
    assert N.lib().lp_add_rms_norm(ref(x), None, P(), 32776, N.LP_F32, 1e-5, None, ref(x), None,
                                   None) == N.LP_ERR_UNSUPPORTED


def route(l=None, **kw):
    a = dict(w=P(2), wn=8, e=P(3), en=8, off=P(4), offn=65, tok=P(5), tokn=8, pl=P(6), pln=8, k=2, renorm=1,
             ws=P(7), wsn=1 << 40)
    a.update(kw)
    l = l or matrix()
    return N.lib().lp_route_experts(ref(l), *a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(wn=7), N.LP_ERR_SHAPE), (dict(en=9), N.LP_ERR_SHAPE), (dict(offn=64), N.LP_ERR_SHAPE),
    (dict(tokn=7), N.LP_ERR_SHAPE), (dict(pln=4), N.LP_ERR_SHAPE), (dict(k=0), N.LP_ERR_SHAPE),
    (dict(k=65), N.LP_ERR_SHAPE), (dict(k=33), N.LP_ERR_UNSUPPORTED), (dict(w=None), N.LP_ERR_ARG),
    (dict(e=None), N.LP_ERR_ARG), (dict(off=None), N.LP_ERR_ARG), (dict(tok=None), N.LP_ERR_ARG),
    (dict(pl=None), N.LP_ERR_ARG), (dict(renorm=2), N.LP_ERR_ARG), (dict(pl=P(3)), N.LP_ERR_ARG),
    (dict(w=P(1)), N.LP_ERR_ARG), (dict(off=ctypes.c_void_p((5 << 24) + 28)), N.LP_ERR_ARG)])
def test_router_refuses(kw, status):
    assert route(**kw) == status


def test_router_refuses_logits():
    assert route(matrix(dtype=N.LP_I8)) == N.LP_ERR_ARG
    assert route(matrix(cols=1025, stride=1025), offn=1026) == N.LP_ERR_UNSUPPORTED
    assert route(matrix(cols=0)) == N.LP_ERR_SHAPE


WEIGHTS = [(dict(dtype=N.LP_F32), N.LP_ERR_ARG), (dict(gated=2), N.LP_ERR_ARG), (dict(experts=0), N.LP_ERR_SHAPE),
           (dict(rows=0), N.LP_ERR_SHAPE), (dict(cols=48), N.LP_ERR_SHAPE), (dict(cols=0), N.LP_ERR_SHAPE),
           (dict(experts=1025), N.LP_ERR_UNSUPPORTED), (dict(gated=1, rows=96), N.LP_ERR_SHAPE),
           (dict(rows=1 << 29, cols=1 << 20), N.LP_ERR_UNSUPPORTED)]


@pytest.mark.parametrize("change,status", WEIGHTS)
def test_weights_that_are_refused(change, status):
    w = weights(**change)
    n = ctypes.c_int64()
    assert N.lib().lp_expert_weights_bytes(ref(w), ref(n), ref(n)) == status
    assert N.lib().lp_expert_weights_pack(P(), 4096, P(2), 256, N.LP_F32, ref(w), None) == status


def test_weights_sizes_and_packing():
    a, b = ctypes.c_int64(), ctypes.c_int64()
    lib = N.lib()
    w = weights(rows=130, cols=160)
    assert lib.lp_expert_weights_bytes(ref(w), ref(a), ref(b)) == N.LP_OK
    assert (a.value, b.value) == (2 * 2 * 2 * 8192, 2 * 2 * 2 * 512)
    w = weights(rows=192, gated=1, dtype=N.LP_E4M3)
    assert lib.lp_expert_weights_bytes(ref(w), ref(a), ref(b)) == N.LP_OK
    assert (a.value, b.value) == (2 * 2 * 16384, 2 * 2 * 512)
    assert lib.lp_expert_weights_bytes(ref(w), None, ref(b)) == N.LP_ERR_ARG
    w = weights()
    for args, status in [((P(), 4095, P(2), 256, N.LP_F32), N.LP_ERR_SHAPE),
                         ((P(), 4096, P(2), 255, N.LP_F32), N.LP_ERR_SHAPE),
                         ((P(), 4096, P(2), 256, N.LP_I8), N.LP_ERR_ARG),
                         ((None, 4096, P(2), 256, N.LP_E8M0), N.LP_ERR_ARG)]:
        assert lib.lp_expert_weights_pack(*args, ref(w), None) == status


def gemm(w=None, x=None, out=None, gated=False, **kw):
    a = dict(off=P(5), offn=3, tok=None, tokn=0)
    a.update(kw)
    w, x = w or weights(gated=int(gated)), x or rows8()
    out = out or (rows8(cols=32, code_stride=32, scale_stride=1) if gated else matrix())
    f = N.lib().lp_expert_gemm_gated if gated else N.lib().lp_expert_gemm
    return f(ref(w), ref(x), *a.values(), ref(out), P(9), a.pop("wsn", 0), None)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(offn=2), N.LP_ERR_SHAPE), (dict(off=None), N.LP_ERR_ARG), (dict(tokn=3), N.LP_ERR_SHAPE),
    (dict(tok=P(6), tokn=-1), N.LP_ERR_SHAPE), (dict(tok=P(6), tokn=5), N.LP_ERR_SHAPE),
    (dict(x=rows8(cols=96, code_stride=96, scale_stride=3)), N.LP_ERR_SHAPE),
    (dict(x=rows8(dtype=N.LP_I8)), N.LP_ERR_ARG), (dict(x=rows8(code_stride=72)), N.LP_ERR_UNSUPPORTED),
    (dict(x=rows8(codes=(1 << 24) + 8)), N.LP_ERR_UNSUPPORTED), (dict(), N.LP_ERR_SHAPE)])  # (no workspace)
def test_products_refuse(gated, kw, status):
    assert gemm(gated=gated, **kw) == status


def test_products_refuse_weights_and_results():
    assert gemm(weights(gated=1)) == N.LP_ERR_ARG
    assert gemm(weights(), gated=True, out=rows8()) == N.LP_ERR_ARG
    assert gemm(weights(tiles=None)) == N.LP_ERR_ARG
    assert gemm(weights(tiles=(3 << 24) + 16)) == N.LP_ERR_ARG
    assert gemm(out=matrix(cols=65, stride=65)) == N.LP_ERR_SHAPE
    assert gemm(out=matrix(dtype=N.LP_I8)) == N.LP_ERR_ARG
    assert gemm(gated=True, out=rows8(dtype=N.LP_I8, cols=32)) == N.LP_ERR_ARG
    assert gemm(gated=True, out=rows8(cols=32, code_stride=40)) == N.LP_ERR_UNSUPPORTED


def combine(rows=None, res=None, out=None, **kw):
    a = dict(w=P(2), wn=8, pl=P(3), pln=8)
    a.update(kw)
    rows, out = rows or matrix(rows=9), out or matrix()
    return N.lib().lp_combine_experts(ref(rows), *a.values(), None if res is None else ref(res), ref(out), None)


@pytest.mark.parametrize("kw,status", [
    (dict(wn=7), N.LP_ERR_SHAPE), (dict(wn=9, pln=9), N.LP_ERR_SHAPE), (dict(w=None), N.LP_ERR_ARG),
    (dict(pl=None), N.LP_ERR_ARG), (dict(rows=matrix(cols=32)), N.LP_ERR_SHAPE),
    (dict(res=matrix(rows=3)), N.LP_ERR_SHAPE), (dict(res=matrix(dtype=N.LP_F16)), N.LP_ERR_ARG),
    (dict(out=matrix(dtype=N.LP_E4M3)), N.LP_ERR_ARG)])
def test_combine_refuses(kw, status):
    assert combine(**kw) == status


def test_workspace_sizes():
    assert N.lib().lp_experts_workspace(0, 0, None) == N.LP_ERR_ARG
    n = ctypes.c_int64()
    assert N.lib().lp_experts_workspace(-1, 0, ref(n)) == N.LP_ERR_SHAPE


def test_empty_calls_need_nothing():
    none8, none = rows8(rows=0, codes=None, scales=None), matrix(rows=0, data=None)
    lib = N.lib()
    assert lib.lp_quantize_rows(ref(none), ref(none8), None) == N.LP_OK
    assert lib.lp_dequantize_rows(ref(none8), ref(none), None) == N.LP_OK
    assert lib.lp_add_rms_norm(ref(none), None, P(), 64, N.LP_F32, 1e-5, None, ref(none), None, None) == N.LP_OK
    assert combine(out=none, w=None, wn=0, pl=None, pln=0) == N.LP_OK


def test_python_refuses_what_is_no_cuda_tensor():
    x, i = torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.int32)
    c, s = torch.zeros(2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8)
    for f in (lambda: L.quantizeRows(x, c, s), lambda: L.dequantizeRows(c, s, x),
              lambda: L.addRmsNorm(x, None, x[0], 1e-5, y=x), lambda: L.ExpertWeights(c[None], s[None]),
              lambda: L.quantizeRows(np.zeros((2, 64), np.float32), c, s),
              lambda: L.routeExperts(x, x, i, i, i, i), lambda: L.combineExperts(x, x, i, x)):
        with pytest.raises(TypeError):
            f()
