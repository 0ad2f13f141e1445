"""What the paged cache's entry points refuse, without a GPU: statuses of the C ABI before any
device work, and the Python layer's checks of types."""
import ctypes

import numpy as np
import pytest

from nim_lowprec_b200 import _native as N

torch = pytest.importorskip("torch")

import nim_lowprec_b200 as L  # noqa: E402
from nim_lowprec_b200.attention import _CacheStruct  # noqa: E402

P = ctypes.c_void_p(1 << 20)  # a pointer that is only looked at


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("tokens", ctypes.c_int64), ("heads", ctypes.c_int64),
                ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def cache(**kw):
    c = _CacheStruct()
    c.k = c.v = c.k_scales = c.v_scales = 1 << 20
    c.pages, c.page_size, c.kv_heads, c.head_dim, c.dtype = 8, 16, 2, 64, N.LP_F16
    c.k_strides[:] = c.v_strides[:] = [16 * 2 * 64, 2 * 64, 64]
    c.k_scale_strides[:] = c.v_scale_strides[:] = [32, 2, 1]
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


def rows(**kw):
    r = Rows(1 << 20, 4, 2, 128, 64, N.LP_F32, 0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def store(c=None, k=None, v=None, slots=P, n=4):
    c, k, v = c or cache(), k or rows(), v or rows()
    return N.lib().lp_store_kv(ctypes.byref(c), ctypes.byref(k), ctypes.byref(v), slots, n, None)


CACHES = [
    (dict(dtype=N.LP_F32), N.LP_ERR_ARG), (dict(dtype=9), N.LP_ERR_ARG),
    (dict(k=None), N.LP_ERR_ARG), (dict(v=None), N.LP_ERR_ARG),
    (dict(dtype=N.LP_I8, k_scales=None), N.LP_ERR_ARG),
    (dict(page_size=0), N.LP_ERR_SHAPE), (dict(kv_heads=0), N.LP_ERR_SHAPE),
    (dict(pages=-1), N.LP_ERR_SHAPE), (dict(head_dim=60), N.LP_ERR_SHAPE),
    (dict(head_dim=272), N.LP_ERR_UNSUPPORTED),
    (dict(k=(1 << 20) + 8), N.LP_ERR_UNSUPPORTED),
    (dict(v_strides=[2048, 124, 64]), N.LP_ERR_UNSUPPORTED),
    (dict(k_strides=[-2048, 128, 64]), N.LP_ERR_SHAPE),
    (dict(k_strides=[1 << 36, 128, 64]), N.LP_ERR_SHAPE),
]


@pytest.mark.parametrize("change,status", CACHES)
def test_caches_that_are_refused(change, status):
    c = cache(**change)
    assert store(c) == status
    q = rows()
    assert N.lib().lp_load_kv(ctypes.byref(c), P, 4, ctypes.byref(q), ctypes.byref(q),
                              None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.LP_I8), N.LP_ERR_ARG), (dict(data=None), N.LP_ERR_ARG),
    (dict(tokens=-1), N.LP_ERR_SHAPE), (dict(tokens=5), N.LP_ERR_SHAPE),
    (dict(heads=3), N.LP_ERR_SHAPE), (dict(token_stride=-128), N.LP_ERR_SHAPE),
    (dict(head_stride=1 << 33), N.LP_ERR_SHAPE), (dict(dtype=N.LP_F16), N.LP_ERR_ARG),
])
def test_rows_that_are_refused(change, status):
    assert store(k=rows(**change)) == status
    assert store(v=rows(**change)) == status


def test_slots_that_are_refused():
    assert store(n=3) == N.LP_ERR_SHAPE
    assert store(slots=None) == N.LP_ERR_ARG
    none = rows(tokens=0, data=None)
    assert store(k=none, v=none, slots=None, n=0) == N.LP_OK


def assign(**kw):
    a = dict(ctx=P, ctx_n=3, new=P, new_n=3, ps=16, free=P, free_n=9, head=P, tables=P, width=4,
             stride=4, qs=P, qs_n=4, seq=P, seq_n=3, slots=P, slots_n=7, pos=P, pos_n=7,
             out=ctypes.c_void_p(2 << 20))
    a.update(kw)
    return N.lib().lp_assign_pages(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(new_n=2), N.LP_ERR_SHAPE), (dict(seq_n=4), N.LP_ERR_SHAPE),
    (dict(qs_n=3), N.LP_ERR_SHAPE), (dict(ps=0), N.LP_ERR_SHAPE), (dict(ps=-4), N.LP_ERR_SHAPE),
    (dict(stride=3), N.LP_ERR_SHAPE), (dict(width=-1), N.LP_ERR_SHAPE),
    (dict(pos_n=6), N.LP_ERR_SHAPE), (dict(slots_n=-1), N.LP_ERR_SHAPE),
    (dict(free_n=-1), N.LP_ERR_SHAPE),
    (dict(ctx=None), N.LP_ERR_ARG), (dict(new=None), N.LP_ERR_ARG), (dict(qs=None), N.LP_ERR_ARG),
    (dict(seq=None), N.LP_ERR_ARG), (dict(slots=None), N.LP_ERR_ARG),
    (dict(tables=None), N.LP_ERR_ARG), (dict(free=None), N.LP_ERR_ARG),
    (dict(head=None), N.LP_ERR_ARG), (dict(out=None), N.LP_ERR_ARG),
    (dict(out=P), N.LP_ERR_ARG),  # the free head is read by every block while one writes the next
])
def test_page_assignments_that_are_refused(change, status):
    assert assign(**change) == status


INPUTS = dict(ctx=3, new=3, free=9, head=1)  # and their lengths
OUTPUTS = dict(qs=4, seq=3, slots=7, pos=7, out=1)


def apart(**kw):
    """assign() with every array in a place of its own."""
    a = {name: ctypes.c_void_p((16 + i) << 20)
         for i, name in enumerate([*INPUTS, *OUTPUTS, "tables"])}
    a.update(kw)
    return a


def test_page_assignments_refuse_outputs_on_other_arrays():
    """Blocks read the lengths and the free list while others write: an output on an input, as
    in lengths updated in place, would be a race."""
    at = apart()
    for o, n in OUTPUTS.items():
        size = 8 if o == "slots" else 4
        for other, length in (*INPUTS.items(), *OUTPUTS.items()):
            if other == o:
                continue
            p, bytes_ = at[other].value, length * (8 if other == "slots" else 4)
            assert assign(**apart(**{o: at[other]})) == N.LP_ERR_ARG, (o, other)
            # and by one byte at either end
            for q in (p + bytes_ - 1, p - n * size + 1):
                assert assign(**apart(**{o: ctypes.c_void_p(q)})) == N.LP_ERR_ARG, (o, other)


def test_page_assignments_refuse_tables_on_other_arrays():
    """Three rows of four entries, ten apart: what lies between the rows is not theirs."""
    base = apart()["tables"].value
    for name, n in (*INPUTS.items(), *OUTPUTS.items()):
        size = 4 * n * (2 if name == "slots" else 1)
        for row in range(3):
            for q in (base + 40 * row, base + 40 * row + 15, base + 40 * row - size + 1):
                a = apart(**{name: ctypes.c_void_p(q)})
                assert assign(**a, stride=10) == N.LP_ERR_ARG, (name, row)


def attend(c=None, q=None, out=None, **kw):
    c, q, out = c or cache(), q or rows(heads=4, token_stride=256), out or rows(heads=4)
    a = dict(tables=P, width=4, stride=4, qs=P, qs_n=4, seq=P, seq_n=3, q=ctypes.byref(q),
             out=ctypes.byref(out), scale=0.125, window=0, sinks=0, lse=None, lse_n=0, ws=P,
             ws_n=1 << 40)
    a.update(kw)
    return N.lib().lp_paged_attention(ctypes.byref(c), *a.values(), None)


@pytest.mark.parametrize("change,status", CACHES + [
    (dict(head_dim=32), N.LP_ERR_UNSUPPORTED), (dict(head_dim=256), N.LP_ERR_UNSUPPORTED)])
def test_attention_refuses_caches(change, status):
    assert attend(cache(**change)) == status


@pytest.mark.parametrize("change,status", [
    (dict(qs_n=3), N.LP_ERR_SHAPE), (dict(seq_n=2), N.LP_ERR_SHAPE),
    (dict(window=-1), N.LP_ERR_SHAPE), (dict(sinks=-1), N.LP_ERR_SHAPE),
    (dict(stride=2), N.LP_ERR_SHAPE), (dict(lse=P, lse_n=15), N.LP_ERR_SHAPE),
    (dict(scale=float("nan")), N.LP_ERR_ARG), (dict(scale=float("inf")), N.LP_ERR_ARG),
    (dict(tables=None), N.LP_ERR_ARG), (dict(qs=None), N.LP_ERR_ARG), (dict(seq=None), N.LP_ERR_ARG),
])
def test_attention_refuses_arguments(change, status):
    assert attend(**change) == status


def test_attention_refuses_rows():
    assert attend(q=rows(heads=3)) == N.LP_ERR_SHAPE  # out has 4 heads
    odd = rows(heads=3)
    assert attend(q=odd, out=odd) == N.LP_ERR_SHAPE  # 3 heads over 2 key heads
    assert attend(out=rows(heads=4, dtype=N.LP_F16)) == N.LP_ERR_ARG
    assert attend(out=rows(heads=4, tokens=5)) == N.LP_ERR_SHAPE
    assert attend(out=rows(heads=4, data=None)) == N.LP_ERR_ARG
    none = rows(heads=4, tokens=0, data=None)
    assert attend(q=none, out=none, ws=None, ws_n=0) == N.LP_OK


def test_workspace_size_needs_a_place():
    assert N.lib().lp_paged_attention_workspace(None) == N.LP_ERR_ARG


def test_python_refuses_what_is_no_cuda_tensor():
    h = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        L.KVCache(h, h)
    with pytest.raises(TypeError):
        L.KVCache(np.zeros((2, 16, 1, 64), np.float16), h)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError):
        L.assignPages(i, i, 16, i, i[:1], i.view(3, 1), torch.zeros(4, dtype=torch.int32), i,
                      i.long(), i, i[:1])
    with pytest.raises(TypeError):
        L.assignPages(np.zeros(3, np.int32), i, 16, i, i, i, i, i, i, i, i)
