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

_CACHE_TYPES = {}
if torch is not None:
    _CACHE_TYPES = {torch.float16: N.LP_F16, torch.bfloat16: N.LP_BF16, torch.int8: N.LP_I8}

_I3 = ctypes.c_int64 * 3


class _CacheStruct(ctypes.Structure):  # lp_kv_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("page_size", ctypes.c_int64),
                ("kv_heads", ctypes.c_int64), ("k_strides", _I3), ("v_strides", _I3),
                ("k_scale_strides", _I3), ("v_scale_strides", _I3),
                ("dtype", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


_binding = None


def _fast():
    """The compiled argument checks and calls (csrc/torch_binding.cpp)."""
    global _binding
    if _binding is None:
        try:
            from . import _torch_binding
        except ImportError as e:
            raise ImportError("nim_lowprec_b200/_torch_binding.so is missing or was built for another "
                              "torch: build it with `python nim_lowprec_b200/build.py`") from e
        _binding = _torch_binding
    return _binding


def _cuda(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name}: expected a torch CUDA tensor")
    return t


def _strides(t):
    """Of pages, tokens and heads; a dimension of one may have any, and needs none."""
    return _I3(*(st if n > 1 else 0 for n, st in zip(t.shape[:3], t.stride())))


class KVCache:
    """Pages of keys and values, [pages, pageSize, kvHeads, headDim] each, in fp16, bf16 or
    int8.  The head dimension is contiguous; the other strides are free (a cache that keeps
    heads outside of tokens is passed as ``t.transpose(1, 2)``), rows start on 16-byte
    boundaries.  headDim: storeKV and loadKV take multiples of 16 up to 256, pagedAttention
    64, 96 and 128 alone.  int8 pages come with fp32 scales [pages, pageSize, kvHeads], one per (token,
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
        s.k_strides, s.v_strides = _strides(k), _strides(v)
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
            s.k_scale_strides, s.v_scale_strides = _strides(kScales), _strides(vScales)
        self.k, self.v, self.kScales, self.vScales = k, v, kScales, vScales
        self.device = k.device
        self._index = k.device.index
        self._struct = s
        self._ref = ctypes.addressof(s)
        self._dim = s.head_dim
        self._scale = s.head_dim ** -0.5 if s.head_dim else 1.0

    @classmethod
    def allocate(cls, pages, pageSize, kvHeads, headDim, dtype, device="cuda"):
        """A new cache, zeroed.  (headDim: see above; pagedAttention takes 64, 96 and 128.)"""
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


def assignPages(ctxLens, newLens, pageSize, freePages, freeHead, blockTables, qStart, seqLens,
                slots, positions, freeHeadOut):
    """Page tables and slot maps from request lengths, on the GPU (lp_assign_pages).

    Request b has ctxLens[b] tokens cached and gets newLens[b] more.  The pages it lacks are
    taken, in request order, from freePages[freeHead[0]:] and written into blockTables[b]
    (-1 once the list has run out).  Written: qStart [requests + 1], seqLens, and per flat
    token its slot (int64) and position; -1 past the last token and where there is no page.
    freeHeadOut[0] is the next free entry, at most the list's length.  No output may share
    memory with an input or another output (``NativeError``): seqLens and freeHeadOut are other
    tensors than ctxLens and freeHead, and take turns with them from step to step.  positions
    may be None.  Whole numbers are int32, slots int64."""
    status = _fast().assign_pages(ctxLens, newLens, pageSize, freePages, freeHead, blockTables, qStart,
                                  seqLens, slots, positions, freeHeadOut)
    if status:
        N.check(status, "assignPages")


def storeKV(cache, k, v, slots):
    """Write k and v [tokens, kvHeads, headDim] (fp32, fp16, bf16; any strides but the last) to
    their slots (lp_store_kv).  A token whose slot is outside the cache is skipped.  int8 pages
    take the codes and scales of calibrateSymmetric and quantizeBatch over each row."""
    status = _fast().store_kv(cache._ref, cache._index, cache._dim, k, v, slots)
    if status:
        N.check(status, "storeKV")


def loadKV(cache, slots, k, v):
    """Read the rows at `slots` back into k and v (lp_load_kv); zeros where a slot is outside
    the cache."""
    status = _fast().load_kv(cache._ref, cache._index, cache._dim, k, v, slots)
    if status:
        N.check(status, "loadKV")


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
    defaults to headDim ** -0.5.  out must not share memory with q.  lse (fp32 [tokens, heads] or None) receives the logarithm of
    each row's sum of exponentials.  A row that sees no key gives zeros (lse -inf).  fp32
    results are fp32 throughout; 16-bit ones round each weight once to 16 bits in calls of
    chunks (include/lowprec_cuda.h says which).

    Without `workspace` one is kept per device and stream.  A call that is captured into a graph
    must bring its own (attentionWorkspace(), made before the capture; ``RuntimeError``): the
    graph may be replayed on any stream, beside calls and graphs that use the kept one."""
    fast, index = _fast(), cache._index
    if workspace is None:
        if fast.capturing(index):
            raise RuntimeError("pagedAttention: a captured call needs a workspace of its own "
                               "(attentionWorkspace(), made before the capture)")
        key = (index, fast.current_stream(index))
        workspace = _workspaces.get(key)
        if workspace is None:
            workspace = _workspaces[key] = attentionWorkspace(cache.device)
    status = fast.paged_attention(cache._ref, index, cache._dim, blockTables, qStart, seqLens, q, out,
                                  cache._scale if scale is None else scale, window, sinks, lse, workspace)
    if status:
        N.check(status, "pagedAttention")
