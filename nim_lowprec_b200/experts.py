"""The sparse feed-forward layer over 8-bit rows: norm, router, experts' products, their sum.

What stands between two attentions (``attention``); the reference ends at the products, so these
have no counterpart proc.  Like the rest of the package the functions write into the tensors that
they are given, on ``torch.cuda.current_stream()``.  Torch CUDA tensors only.  A wrong shape raises
``AssertionError``, a wrong type ``TypeError``, a layout that is not taken ``ValueError``, what the
kernels do not take ``NativeError``.  Outputs must not share memory with inputs or each other, except
where it says so.

8-bit rows are a pair of tensors, ``codes`` [rows, columns] and ``scales`` [rows, columns / group]:

* MXFP8: codes ``float8_e4m3fn``, scales E8M0 bytes (``uint8`` or ``float8_e8m0fnu``), groups of 32;
  what the experts' products take.
* int8: codes ``int8``, scales fp32, groups of 32, 64, 128 or 256; flat and contiguous, they are the
  xq and xScales of dequantGemmQ8, dequantGemmI4Q8 and the GEMVs over int8 activations.
"""
from __future__ import annotations

import ctypes

from . import _native as N
from .attention import _cuda, _fast

try:  # as in dequant: importing the package needs no torch
    import torch
except Exception:  # pragma: no cover
    torch = None


class _WeightsStruct(ctypes.Structure):  # lp_expert_weights
    _fields_ = [("tiles", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("experts", ctypes.c_int64), ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("gated", ctypes.c_int32)]


def quantizeRows(x, codes, scales):
    """x [rows, columns] (fp32, fp16, bf16) as 8-bit rows (lp_quantize_rows): MXFP8 or int8, as the
    tensors' types say, the group as their shapes say."""
    status = _fast().quantize_rows(x, codes, scales)
    if status:
        N.check(status, "quantizeRows")


def dequantizeRows(codes, scales, dst):
    """The values of 8-bit rows, rounded once to dst's type (lp_dequantize_rows).  bf16 holds every
    finite value of an MXFP8 row."""
    status = _fast().dequantize_rows(codes, scales, dst)
    if status:
        N.check(status, "dequantizeRows")


def addRmsNorm(x, residual, weight, eps, total=None, y=None, codes=None, scales=None):
    """r = x + residual, and n = r / sqrt(mean(r ** 2) + eps) * weight over each row
    (lp_add_rms_norm).  Written, each if given: total = r, y = n, codes and scales = n as 8-bit rows.

    x, residual, total, y [rows, columns], columns at most 32768.  residual may be None; it, and
    total, have x's type or fp32, and r is rounded to that type before it is normed.  weight
    [columns] and y may have any of fp32, fp16 and bf16.  total may be x or residual itself, y may
    be x."""
    if (codes is None) != (scales is None):
        raise TypeError("addRmsNorm: codes and scales come together")
    status = _fast().add_rms_norm(x, residual, weight, eps, total, y, codes, scales)
    if status:
        N.check(status, "addRmsNorm")


def expertsWorkspace(device=None, rows=0, columns=0):
    """A workspace for routeExperts, expertGemm and expertGemmGated, zeroed; rows and columns are
    those of the largest product with a rowToken.  Calls that may run at the same time (on several
    streams, in several captured graphs) need one each."""
    with torch.cuda.device(device):
        return torch.zeros(_workspace_bytes(rows, columns), dtype=torch.uint8, device="cuda")


def _workspace_bytes(rows, columns):
    size = ctypes.c_int64()
    N.check(N.lib().lp_experts_workspace(rows, columns, ctypes.byref(size)), "expertsWorkspace")
    return size.value


_workspaces = {}  # (device, stream) -> the workspace of calls that bring none


def _workspace(t, name, gather=None):
    fast, index = _fast(), _cuda(t, name).device.index
    if fast.capturing(index):
        raise RuntimeError(f"{name}: a captured call needs a workspace of its own "
                           "(expertsWorkspace(), made before the capture)")
    key = (index, fast.current_stream(index))
    workspace = _workspaces.get(key)
    rows, columns = (gather.numel(), t.shape[-1]) if gather is not None else (0, 0)
    if workspace is None or (rows and workspace.numel() < _workspace_bytes(rows, columns)):
        workspace = _workspaces[key] = expertsWorkspace(t.device, rows, columns)
    return workspace


def routeExperts(logits, weights, experts, offsets, rowToken, places, renormalize=True,
                 workspace=None):
    """Each token's k largest logits and the order of their rows (lp_route_experts).

    logits [tokens, n] (fp32, fp16, bf16), n at most 1024.  Written: experts (int32) and weights
    (fp32) [tokens, k], k at most 32, the largest first, of equal ones the lower expert; weights are
    exp(l - max) over their sum over the chosen, or over all experts with renormalize=False.  Rows,
    one for each token and choice, are sorted by expert, then by token: expert e has rows
    offsets[e]:offsets[e + 1] (int32 [n + 1]), rowToken (int32 [tokens * k]) is each row's token,
    places (int32 [tokens, k]) each choice's row.  A logit of -inf or NaN is never chosen: a token
    with fewer than k others has expert and place -1 and weight 0 in the rest, and rowToken is left
    alone from offsets[n] on.

    Without `workspace` one is kept per device and stream.  A call that is captured into a graph
    must bring its own (expertsWorkspace(), made before the capture; ``RuntimeError``)."""
    if workspace is None:
        workspace = _workspace(logits, "routeExperts")
    status = _fast().route_experts(logits, weights, experts, offsets, rowToken, places,
                                   int(bool(renormalize)), workspace)
    if status:
        N.check(status, "routeExperts")


class ExpertWeights:
    """Experts' weights, laid out once for the products: y = W[e] x.

    MXFP4: codes uint8 [experts, rows, columns / 2], two to a byte as quantizeF4Packed packs them,
    and scales [experts, rows, columns / 32] in fp32, powers of two as calibrateMX writes them, or
    as E8M0 bytes.  MXFP8: codes float8_e4m3fn [experts, rows, columns] and the same scales
    (quantizeRows's).  One expert makes a plain projection.  columns are a multiple of 32.

    gated=True: the first half of the rows are the gate's, the second half the up projection's
    (rows a multiple of 64), for expertGemmGated.  The laid-out copy is the object's own (`tiles`,
    `scales`; 0.53 or 1.03 bytes an element, M in multiples of 128 and columns of 128); codes and
    scales may be dropped."""

    def __init__(self, codes, scales, gated=False):
        _cuda(codes, "codes"), _cuda(scales, "scales")
        if codes.dtype not in (torch.uint8, torch.float8_e4m3fn):
            raise TypeError(f"codes: expected packed uint8 or float8_e4m3fn, got {codes.dtype}")
        if scales.dtype not in (torch.float32, torch.uint8, torch.float8_e8m0fnu):
            raise TypeError(f"scales: expected fp32 or E8M0 bytes, got {scales.dtype}")
        if codes.dim() != 3 or scales.dim() != 3:
            raise AssertionError("codes [experts, rows, columns] and scales [experts, rows, "
                                 f"columns / 32]: {tuple(codes.shape)}, {tuple(scales.shape)}")
        fp4 = codes.dtype == torch.uint8
        s = _WeightsStruct()
        s.experts, s.rows, s.cols = codes.shape
        s.cols *= 2 if fp4 else 1
        if tuple(scales.shape) != (s.experts, s.rows, s.cols // 32):
            raise AssertionError(f"scales: {tuple(scales.shape)} for codes {tuple(codes.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        if scales.device != codes.device:
            raise TypeError("codes and scales on different devices")
        s.dtype = N.LP_E2M1 if fp4 else N.LP_E4M3
        s.gated = int(bool(gated))
        sizes = ctypes.c_int64(), ctypes.c_int64()
        lib = N.lib()
        N.check(lib.lp_expert_weights_bytes(ctypes.addressof(s), *map(ctypes.byref, sizes)),
                "ExpertWeights")
        self.tiles, self.scales = (torch.empty(n.value, dtype=torch.uint8, device=codes.device)
                                   for n in sizes)
        s.tiles, s.scales = self.tiles.data_ptr(), self.scales.data_ptr()
        with torch.cuda.device(codes.device):
            N.check(lib.lp_expert_weights_pack(
                codes.data_ptr(), codes.numel(), scales.data_ptr(), scales.numel(),
                N.LP_F32 if scales.dtype == torch.float32 else N.LP_E8M0, ctypes.addressof(s),
                torch.cuda.current_stream().cuda_stream), "ExpertWeights")
        self.device = codes.device
        self._index = codes.device.index
        self._struct = s
        self._ref = ctypes.addressof(s)

    experts = property(lambda s: s._struct.experts)
    rows = property(lambda s: s._struct.rows)
    columns = property(lambda s: s._struct.cols)
    gated = property(lambda s: bool(s._struct.gated))


def expertGemm(w, codes, scales, offsets, out, rowToken=None, workspace=None):
    """out[r] = W[e] x[t] for each expert's rows r in offsets[e]:offsets[e + 1] (lp_expert_gemm).

    codes and scales: MXFP8 rows x [tokens, columns]; t = rowToken[r] (int32, one for each row of
    out), or r without it (rows in the experts' order).  out [rows, w.rows] in fp32, fp16 or bf16;
    rows of no expert are left alone.  Products are exact, sums fp32, results rounded once.
    Workspace as in routeExperts."""
    if workspace is None:
        workspace = _workspace(codes, "expertGemm", rowToken)
    status = _fast().expert_gemm(w._ref, w._index, codes, scales, offsets, rowToken, out, workspace)
    if status:
        N.check(status, "expertGemm")


def expertGemmGated(w, codes, scales, offsets, outCodes, outScales, rowToken=None, workspace=None):
    """g / (1 + exp(-g)) * u as MXFP8 rows [rows, w.rows / 2], where g and u are the halves of
    expertGemm's rows (lp_expert_gemm_gated): the rows of the down projection's expertGemm.
    `w` is laid out with gated=True."""
    if workspace is None:
        workspace = _workspace(codes, "expertGemmGated", rowToken)
    status = _fast().expert_gemm_gated(w._ref, w._index, codes, scales, offsets, rowToken, outCodes,
                                       outScales, workspace)
    if status:
        N.check(status, "expertGemmGated")


def combineExperts(rows, weights, places, out, residual=None):
    """out[t] = residual[t] + sum_j weights[t, j] * rows[places[t, j]], in fp32 in the order of j,
    rounded once (lp_combine_experts).  A place outside rows adds nothing.  residual has out's type,
    and may be out itself."""
    status = _fast().combine_experts(rows, weights, places, residual, out)
    if status:
        N.check(status, "combineExperts")
