"""A paged key/value cache and the attention that reads it, over the CUDA library.

What a decoder layer does between its projections (``dequant``'s GEMVs and GEMMs) and its
output projection; the reference ends at the products, so these have no counterpart proc.
Like the rest of the package the functions write into the tensors that they are given, on
``torch.cuda.current_stream()``.  Torch CUDA tensors only.  A wrong shape raises
``AssertionError``, a wrong type ``TypeError``, what the kernels do not take ``NativeError``.
"""
from __future__ import annotations

import ctypes

from . import _native as N

try:  # as in dequant: importing the package needs no torch
    import torch
except Exception:  # pragma: no cover
    torch = None

_ROW_TYPES, _CACHE_TYPES = {}, {}
if torch is not None:
    _ROW_TYPES = {torch.float32: N.LP_F32, torch.float16: N.LP_F16, torch.bfloat16: N.LP_BF16}
    _CACHE_TYPES = {torch.float16: N.LP_F16, torch.bfloat16: N.LP_BF16, torch.int8: N.LP_I8}

_I3 = ctypes.c_int64 * 3


class _CacheStruct(ctypes.Structure):  # lp_kv_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("page_size", ctypes.c_int64),
                ("kv_heads", ctypes.c_int64), ("k_strides", _I3), ("v_strides", _I3),
                ("k_scale_strides", _I3), ("v_scale_strides", _I3),
                ("dtype", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


class _RowsStruct(ctypes.Structure):  # lp_rows
    _fields_ = [("data", ctypes.c_void_p), ("tokens", ctypes.c_int64), ("heads", ctypes.c_int64),
                ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def _cuda(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name}: expected a torch CUDA tensor")
    return t


class KVCache:
    """Pages of keys and values, [pages, pageSize, kvHeads, headDim] each, in fp16, bf16 or
    int8.  The head dimension is contiguous; the other strides are free (a cache that keeps
    heads outside of tokens is passed as ``t.transpose(1, 2)``), rows start on 16-byte
    boundaries.  int8 pages come with fp32 scales [pages, pageSize, kvHeads], one per (token,
    head).  The tensors stay the caller's; the cache keeps references to them."""

    def __init__(self, k, v, kScales=None, vScales=None):
        _cuda(k, "k"), _cuda(v, "v")
        if k.dtype not in _CACHE_TYPES or v.dtype != k.dtype:
            raise TypeError(f"pages are fp16, bf16 or int8, k and v alike: {k.dtype}, {v.dtype}")
        int8 = k.dtype == torch.int8
        if int8 != (kScales is not None) or int8 != (vScales is not None):
            raise TypeError("int8 pages need both scales, others take none")
        if k.dim() != 4 or v.shape != k.shape:
            raise AssertionError(f"pages [pages, pageSize, kvHeads, headDim]: {tuple(k.shape)}, "
                                 f"{tuple(v.shape)}")
        if k.numel() and (k.stride(3) != 1 or v.stride(3) != 1):
            raise ValueError("the head dimension must be contiguous")
        if v.device != k.device:
            raise ValueError("pages on different devices")
        s = _CacheStruct()
        s.k, s.v = k.data_ptr(), v.data_ptr()
        s.pages, s.page_size, s.kv_heads, s.head_dim = k.shape
        s.k_strides, s.v_strides = _I3(*k.stride()[:3]), _I3(*v.stride()[:3])
        s.dtype = _CACHE_TYPES[k.dtype]
        if int8:
            for t, name in ((kScales, "kScales"), (vScales, "vScales")):
                if _cuda(t, name).dtype != torch.float32:
                    raise TypeError(f"{name}: expected fp32, got {t.dtype}")
                if t.shape != k.shape[:3]:
                    raise AssertionError(f"{name}: {tuple(t.shape)} for pages {tuple(k.shape)}")
                if t.device != k.device:
                    raise ValueError("scales on another device than the pages")
            s.k_scales, s.v_scales = kScales.data_ptr(), vScales.data_ptr()
            s.k_scale_strides = _I3(*kScales.stride())
            s.v_scale_strides = _I3(*vScales.stride())
        self.k, self.v, self.kScales, self.vScales = k, v, kScales, vScales
        self.device = k.device
        self._index = k.device.index
        self._struct = s
        self._ref = ctypes.addressof(s)

    @classmethod
    def allocate(cls, pages, pageSize, kvHeads, headDim, dtype, device="cuda"):
        """A new cache, zeroed."""
        def new(*shape, dt):
            return torch.zeros(*shape, dtype=dt, device=device)
        k, v = (new(pages, pageSize, kvHeads, headDim, dt=dtype) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        # scales with tokens innermost: an attention step reads a head's run of them
        ks, vs = (new(pages, kvHeads, pageSize, dt=torch.float32).transpose(1, 2)
                  for _ in range(2))
        return cls(k, v, ks, vs)

    pages = property(lambda s: s._struct.pages)
    pageSize = property(lambda s: s._struct.page_size)
    kvHeads = property(lambda s: s._struct.kv_heads)
    headDim = property(lambda s: s._struct.head_dim)


def _rows(t, name, dim, device):
    """lp_rows of a [tokens, heads, dim] tensor; the last dimension contiguous."""
    if not isinstance(t, torch.Tensor) or t.device != device:
        raise TypeError(f"{name}: expected a tensor on {device}")
    dt = _ROW_TYPES.get(t.dtype)
    if dt is None:
        raise TypeError(f"{name}: expected fp32, fp16 or bf16, got {t.dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim:
        raise AssertionError(f"{name}: [tokens, heads, {dim}] expected, got {tuple(shape)}")
    st = t.stride()
    if st[2] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return _RowsStruct(t.data_ptr(), shape[0], shape[1], st[0], st[1], dt, 0)


def _ints(t, name, dtype, device):
    """Pointer and length of a contiguous vector of whole numbers."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        raise TypeError(f"{name}: expected {dtype} on {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensors must be contiguous")
    return t.data_ptr(), t.numel()


def _table(t, requests, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device:
        raise TypeError(f"blockTables: expected int32 on {device}")
    shape, st = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != requests:
        raise AssertionError(f"blockTables: [{requests}, pages] expected, got {tuple(shape)}")
    if shape[1] > 1 and st[1] != 1:
        raise ValueError("blockTables: rows must be contiguous")
    # (torch gives a one-row or empty tensor any stride)
    return t.data_ptr(), shape[1], st[0] if requests > 1 else shape[1]


def _launch(index, name, *args):
    """The call on the current stream of the tensors' device."""
    if index == torch.cuda.current_device():
        st = getattr(N.lib(), name)(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(index):
            st = getattr(N.lib(), name)(*args, torch.cuda.current_stream().cuda_stream)
    if st:
        N.check(st, name[3:])


def assignPages(ctxLens, newLens, pageSize, freePages, freeHead, blockTables, qStart, seqLens,
                slots, positions, freeHeadOut):
    """Page tables and slot maps from request lengths, on the GPU (lp_assign_pages).

    Request b has ctxLens[b] tokens cached and gets newLens[b] more.  The pages it lacks are
    taken, in request order, from freePages[freeHead[0]:] and written into blockTables[b]
    (-1 once the list has run out).  Written: qStart [requests + 1], seqLens, and per flat
    token its slot (int64) and position; -1 past the last token and where there is no page.
    freeHeadOut[0] is the next free entry; it must be another tensor than freeHead.
    positions may be None.  Whole numbers are int32, slots int64."""
    dev = _cuda(ctxLens, "ctxLens").device
    i32 = torch.int32
    ctx, n = _ints(ctxLens, "ctxLens", i32, dev)
    for t, name in ((freeHead, "freeHead"), (freeHeadOut, "freeHeadOut")):
        if _ints(t, name, i32, dev)[1] != 1:
            raise AssertionError(f"{name}: one element expected")
    pos = (None, 0) if positions is None else _ints(positions, "positions", i32, dev)
    _launch(dev.index, "lp_assign_pages", ctx, n, *_ints(newLens, "newLens", i32, dev),
            int(pageSize), *_ints(freePages, "freePages", i32, dev), freeHead.data_ptr(),
            *_table(blockTables, n, dev), *_ints(qStart, "qStart", i32, dev),
            *_ints(seqLens, "seqLens", i32, dev), *_ints(slots, "slots", torch.int64, dev),
            *pos, freeHeadOut.data_ptr())


def storeKV(cache, k, v, slots):
    """Write k and v [tokens, kvHeads, headDim] (fp32, fp16, bf16; any strides but the last) to
    their slots (lp_store_kv).  A token whose slot is outside the cache is skipped.  int8 pages
    take the codes and scales of calibrateSymmetric and quantizeBatch over each row."""
    dev, dim = cache.device, cache._struct.head_dim
    kr, vr = _rows(k, "k", dim, dev), _rows(v, "v", dim, dev)
    _launch(cache._index, "lp_store_kv", cache._ref, ctypes.addressof(kr), ctypes.addressof(vr),
            *_ints(slots, "slots", torch.int64, dev))


def loadKV(cache, slots, k, v):
    """Read the rows at `slots` back into k and v (lp_load_kv); zeros where a slot is outside
    the cache."""
    dev, dim = cache.device, cache._struct.head_dim
    kr, vr = _rows(k, "k", dim, dev), _rows(v, "v", dim, dev)
    _launch(cache._index, "lp_load_kv", cache._ref,
            *_ints(slots, "slots", torch.int64, dev), ctypes.addressof(kr), ctypes.addressof(vr))


def attentionWorkspace(device=None):
    """A workspace for pagedAttention, zeroed.  Calls that may run at the same time (on several
    streams, in several captured graphs) need one each."""
    with torch.cuda.device(device):
        size = ctypes.c_int64()
        N.check(N.lib().lp_paged_attention_workspace(ctypes.byref(size)), "attentionWorkspace")
        return torch.zeros(size.value, dtype=torch.uint8, device="cuda")


_workspaces = {}  # (device, stream) -> the workspace of calls that bring none


def pagedAttention(cache, blockTables, qStart, seqLens, q, out, scale=None, window=0, sinks=0,
                   lse=None, workspace=None):
    """Attention of each request's new tokens over its cached keys (lp_paged_attention).

    q and out [tokens, heads, headDim] (fp32, fp16 or bf16, alike); request b's rows are
    qStart[b]:qStart[b + 1], the last of them at position seqLens[b] - 1, its keys those that
    blockTables[b] holds.  A token at position p sees key j if j <= p and, with a window,
    j > p - window or j < sinks.  heads is a multiple of the cache's kvHeads.  `scale`
    defaults to headDim ** -0.5.  lse (fp32 [tokens, heads] or None) receives the logarithm of
    each row's sum of exponentials.  A row that sees no key gives zeros (lse -inf).

    Without `workspace` one is kept per device and stream; pass your own
    (attentionWorkspace()) to graphs that may be replayed on other streams."""
    dev, index, dim = cache.device, cache._index, cache._struct.head_dim
    qr, orr = _rows(q, "q", dim, dev), _rows(out, "out", dim, dev)
    seq, n = _ints(seqLens, "seqLens", torch.int32, dev)
    if lse is None:
        lp, ln = None, 0
    else:
        if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.device != dev:
            raise TypeError(f"lse: expected fp32 on {dev}")
        if not lse.is_contiguous():
            raise ValueError("lse: tensors must be contiguous")
        lp, ln = lse.data_ptr(), lse.numel()
    if workspace is None:
        key = (index, torch.cuda.current_stream(dev).cuda_stream)
        workspace = _workspaces.get(key)
        if workspace is None:
            workspace = _workspaces[key] = attentionWorkspace(dev)
    elif not isinstance(workspace, torch.Tensor) or workspace.device != dev or \
            workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise TypeError(f"workspace: expected attentionWorkspace() of {dev}")
    _launch(index, "lp_paged_attention", cache._ref, *_table(blockTables, n, dev),
            *_ints(qStart, "qStart", torch.int32, dev), seq, n, ctypes.addressof(qr),
            ctypes.addressof(orr), dim ** -0.5 if scale is None else float(scale), int(window),
            int(sinks), lp, ln, workspace.data_ptr(), workspace.numel())
