// torch_binding.cpp -- the entry points of the paged cache and of the experts for
// torch tensors, as a CPython module: argument checks and one call of the C ABI.  A decode step
// calls these once per layer; through ctypes a call with eleven tensors costs
// 13 us, about four times its kernel.
//
// Functions take their arguments by position; attention.py and experts.py have the public
// signatures and their documentation.  A wrong shape raises AssertionError, a
// wrong type TypeError, a layout that is not taken ValueError; other statuses
// of the library come back as whole numbers for _native.check.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>

#include "lowprec_cuda.h"

namespace {

struct Error {};  // a Python exception has been set

[[noreturn]] void fail(PyObject* type, const char* format, ...) {
  char text[256];
  va_list ap;
  va_start(ap, format);
  vsnprintf(text, sizeof(text), format, ap);
  va_end(ap);
  PyErr_SetString(type, text);
  throw Error{};
}

const at::Tensor& tensor(PyObject* o, const char* name, int device) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, "%s: expected a torch CUDA tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) fail(PyExc_TypeError, "%s: expected a torch CUDA tensor", name);
  if (device >= 0 && t.get_device() != device)
    fail(PyExc_TypeError, "%s: expected a tensor on cuda:%d, got cuda:%d", name, device,
         static_cast<int>(t.get_device()));
  return t;
}

// A contiguous vector of whole numbers.
struct Ints {
  void* p;
  int64_t n;
};
Ints ints(PyObject* o, const char* name, at::ScalarType type, int device) {
  const at::Tensor& t = tensor(o, name, device);
  if (t.scalar_type() != type)
    fail(PyExc_TypeError, "%s: expected %s, got %s", name, at::toString(type),
         at::toString(t.scalar_type()));
  if (!t.is_contiguous()) fail(PyExc_ValueError, "%s: tensors must be contiguous", name);
  return {t.data_ptr(), t.numel()};
}
int32_t* i32(const Ints& v) { return static_cast<int32_t*>(v.p); }

struct Table {
  int32_t* p;
  int64_t width, stride;
};
Table table(PyObject* o, int64_t requests, int device) {
  const at::Tensor& t = tensor(o, "blockTables", device);
  if (t.scalar_type() != at::kInt)
    fail(PyExc_TypeError, "blockTables: expected int32, got %s", at::toString(t.scalar_type()));
  if (t.dim() != 2 || t.size(0) != requests)
    fail(PyExc_AssertionError, "blockTables: [%lld, pages] expected", static_cast<long long>(requests));
  if (t.size(1) > 1 && t.stride(1) != 1) fail(PyExc_ValueError, "blockTables: rows must be contiguous");
  // (a tensor of one row may have any stride)
  return {static_cast<int32_t*>(t.data_ptr()), t.size(1), requests > 1 ? t.stride(0) : t.size(1)};
}

// [tokens, heads, dim] rows; the last dimension contiguous.
lp_rows rows(PyObject* o, const char* name, int64_t dim, int device) {
  const at::Tensor& t = tensor(o, name, device);
  lp_rows r;
  switch (t.scalar_type()) {
    case at::kFloat: r.dtype = LP_F32; break;
    case at::kHalf: r.dtype = LP_F16; break;
    case at::kBFloat16: r.dtype = LP_BF16; break;
    default:
      fail(PyExc_TypeError, "%s: expected fp32, fp16 or bf16, got %s", name,
           at::toString(t.scalar_type()));
  }
  if (t.dim() != 3 || t.size(2) != dim)
    fail(PyExc_AssertionError, "%s: [tokens, heads, %lld] expected", name, static_cast<long long>(dim));
  if (t.stride(2) != 1) fail(PyExc_ValueError, "%s: the last dimension must be contiguous", name);
  r.data = t.data_ptr();
  r.tokens = t.size(0);
  r.heads = t.size(1);
  r.token_stride = r.tokens > 1 ? t.stride(0) : 0;  // (a dimension of one may have any)
  r.head_stride = r.heads > 1 ? t.stride(1) : 0;
  r.reserved = 0;
  return r;
}

int64_t number(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Error{};
  return v;
}
const lp_kv_cache* cache_of(PyObject* o) { return reinterpret_cast<const lp_kv_cache*>(number(o)); }

// Runs f(stream) with the tensors' device current.
template <class F>
PyObject* on_device(int device, F f) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != device) guard.set_index(device);
  const int status = f(static_cast<lp_stream_t>(c10::cuda::getCurrentCUDAStream(device).stream()));
  return PyLong_FromLong(status);
}

// An exception never leaves a C entry.
template <class F>
PyObject* entry(Py_ssize_t n, Py_ssize_t want, F f) {
  try {
    if (n != want)
      fail(PyExc_TypeError, "%d arguments expected, got %d", static_cast<int>(want), static_cast<int>(n));
    return f();
  } catch (const Error&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (ctxLens, newLens, pageSize, freePages, freeHead, blockTables, qStart, seqLens, slots,
//  positions, freeHeadOut)
PyObject* assign_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 11, [&] {
    const int dev = static_cast<int>(tensor(a[0], "ctxLens", -1).get_device());
    const Ints ctx = ints(a[0], "ctxLens", at::kInt, dev), add = ints(a[1], "newLens", at::kInt, dev);
    const int64_t page_size = number(a[2]);
    const Ints free = ints(a[3], "freePages", at::kInt, dev);
    const Ints head = ints(a[4], "freeHead", at::kInt, dev);
    const Table tab = table(a[5], ctx.n, dev);
    const Ints qs = ints(a[6], "qStart", at::kInt, dev), seq = ints(a[7], "seqLens", at::kInt, dev);
    const Ints slots = ints(a[8], "slots", at::kLong, dev);
    const Ints pos = a[9] == Py_None ? Ints{nullptr, 0} : ints(a[9], "positions", at::kInt, dev);
    const Ints out = ints(a[10], "freeHeadOut", at::kInt, dev);
    if (head.n != 1 || out.n != 1)
      fail(PyExc_AssertionError, "freeHead, freeHeadOut: one element expected");
    if (a[9] != Py_None && pos.n != slots.n)
      fail(PyExc_AssertionError, "positions: %lld elements expected", static_cast<long long>(slots.n));
    return on_device(dev, [&](lp_stream_t st) {
      return lp_assign_pages(i32(ctx), ctx.n, i32(add), add.n, page_size, i32(free), free.n, i32(head),
                             tab.p, tab.width, tab.stride, i32(qs), qs.n, i32(seq), seq.n,
                             static_cast<int64_t*>(slots.p), slots.n, i32(pos), pos.n, i32(out), st);
    });
  });
}

// (cache, device, headDim, k, v, slots)
template <bool STORE>
PyObject* move_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 6, [&] {
    const lp_kv_cache* c = cache_of(a[0]);
    const int dev = static_cast<int>(number(a[1]));
    const int64_t dim = number(a[2]);
    const lp_rows k = rows(a[3], "k", dim, dev), v = rows(a[4], "v", dim, dev);
    const Ints slots = ints(a[5], "slots", at::kLong, dev);
    const int64_t* s = static_cast<int64_t*>(slots.p);
    return on_device(dev, [&](lp_stream_t st) {
      return STORE ? lp_store_kv(c, &k, &v, s, slots.n, st) : lp_load_kv(c, s, slots.n, &k, &v, st);
    });
  });
}

// (cache, device, headDim, blockTables, qStart, seqLens, q, out, scale, window, sinks, lse,
//  workspace)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 13, [&] {
    const lp_kv_cache* c = cache_of(a[0]);
    const int dev = static_cast<int>(number(a[1]));
    const int64_t dim = number(a[2]);
    const Ints seq = ints(a[5], "seqLens", at::kInt, dev), qs = ints(a[4], "qStart", at::kInt, dev);
    const Table tab = table(a[3], seq.n, dev);
    const lp_rows q = rows(a[6], "q", dim, dev), out = rows(a[7], "out", dim, dev);
    const double scale = PyFloat_AsDouble(a[8]);
    if (scale == -1.0 && PyErr_Occurred()) throw Error{};
    const int64_t window = number(a[9]), sinks = number(a[10]);
    float* lse = nullptr;
    int64_t lse_n = 0;
    if (a[11] != Py_None) {
      const Ints l = ints(a[11], "lse", at::kFloat, dev);
      lse = static_cast<float*>(l.p);
      lse_n = l.n;
      if (lse_n != q.tokens * q.heads)
        fail(PyExc_AssertionError, "lse: [%lld, %lld] expected", static_cast<long long>(q.tokens),
             static_cast<long long>(q.heads));
    }
    const Ints ws = ints(a[12], "workspace", at::kByte, dev);
    return on_device(dev, [&](lp_stream_t st) {
      return lp_paged_attention(c, tab.p, tab.width, tab.stride, i32(qs), qs.n, i32(seq), seq.n, &q,
                                &out, static_cast<float>(scale), window, sinks, lse, lse_n, ws.p,
                                ws.n, st);
    });
  });
}

// ------------------------------------------- 8-bit rows, router, experts

int32_t type_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return LP_F32;
    case at::kHalf: return LP_F16;
    case at::kBFloat16: return LP_BF16;
    default:
      fail(PyExc_TypeError, "%s: expected fp32, fp16 or bf16, got %s", name, at::toString(t.scalar_type()));
  }
}

// [rows, columns], the last dimension contiguous.
void two_dims(const at::Tensor& t, const char* name) {
  if (t.dim() != 2) fail(PyExc_AssertionError, "%s: [rows, columns] expected", name);
  if (t.size(1) > 1 && t.stride(1) != 1)
    fail(PyExc_ValueError, "%s: the last dimension must be contiguous", name);
}
lp_matrix matrix(PyObject* o, const char* name, int device) {
  const at::Tensor& t = tensor(o, name, device);
  lp_matrix m;
  m.dtype = type_of(t, name);
  two_dims(t, name);
  m.data = t.data_ptr();
  m.rows = t.size(0);
  m.cols = t.size(1);
  m.stride = m.rows > 1 ? t.stride(0) : m.cols;  // (a dimension of one may have any)
  m.reserved = 0;
  return m;
}

// codes [rows, columns] and scales [rows, columns / group]
lp_rows8 rows8(PyObject* co, PyObject* so, const char* cname, const char* sname, int device) {
  const at::Tensor& c = tensor(co, cname, device);
  const at::Tensor& s = tensor(so, sname, device);
  lp_rows8 r;
  if (c.scalar_type() == at::kChar) {
    r.dtype = LP_I8;
    if (s.scalar_type() != at::kFloat)
      fail(PyExc_TypeError, "%s: expected fp32 for int8 codes, got %s", sname, at::toString(s.scalar_type()));
  } else if (c.scalar_type() == at::kFloat8_e4m3fn) {
    r.dtype = LP_E4M3;
    if (s.scalar_type() != at::kByte && s.scalar_type() != at::kFloat8_e8m0fnu)
      fail(PyExc_TypeError, "%s: expected E8M0 bytes for e4m3 codes, got %s", sname,
           at::toString(s.scalar_type()));
  } else {
    fail(PyExc_TypeError, "%s: expected int8 or float8_e4m3fn, got %s", cname, at::toString(c.scalar_type()));
  }
  two_dims(c, cname);
  two_dims(s, sname);
  r.codes = c.data_ptr();
  r.scales = s.data_ptr();
  r.rows = c.size(0);
  r.cols = c.size(1);
  const int64_t n = s.size(1);
  if (s.size(0) != r.rows || (n ? r.cols % n || r.cols / n > 256 : r.cols > 0))
    fail(PyExc_AssertionError, "%s: [%lld, %lld] for codes [%lld, %lld]", sname,
         static_cast<long long>(s.size(0)), static_cast<long long>(n), static_cast<long long>(r.rows),
         static_cast<long long>(r.cols));
  r.group = n ? static_cast<int32_t>(r.cols / n) : 32;
  r.code_stride = r.rows > 1 ? c.stride(0) : r.cols;
  r.scale_stride = r.rows > 1 ? s.stride(0) : n;
  return r;
}

int device_of(PyObject* o, const char* name) { return static_cast<int>(tensor(o, name, -1).get_device()); }

// (x, codes, scales)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 3, [&] {
    const int dev = device_of(a[0], "x");
    const lp_matrix x = matrix(a[0], "x", dev);
    const lp_rows8 q = rows8(a[1], a[2], "codes", "scales", dev);
    return on_device(dev, [&](lp_stream_t st) { return lp_quantize_rows(&x, &q, st); });
  });
}

// (codes, scales, dst)
PyObject* dequantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 3, [&] {
    const int dev = device_of(a[0], "codes");
    const lp_rows8 q = rows8(a[0], a[1], "codes", "scales", dev);
    const lp_matrix x = matrix(a[2], "dst", dev);
    return on_device(dev, [&](lp_stream_t st) { return lp_dequantize_rows(&q, &x, st); });
  });
}

// (x, residual, weight, eps, total, y, codes, scales)
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 8, [&] {
    const int dev = device_of(a[0], "x");
    const lp_matrix x = matrix(a[0], "x", dev);
    lp_matrix residual, total, y;
    lp_rows8 q;
    if (a[1] != Py_None) residual = matrix(a[1], "residual", dev);
    const at::Tensor& w = tensor(a[2], "weight", dev);
    const int32_t wtype = type_of(w, "weight");
    if (!w.is_contiguous()) fail(PyExc_ValueError, "weight: tensors must be contiguous");
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw Error{};
    if (a[4] != Py_None) total = matrix(a[4], "total", dev);
    if (a[5] != Py_None) y = matrix(a[5], "y", dev);
    if (a[6] != Py_None) q = rows8(a[6], a[7], "codes", "scales", dev);
    return on_device(dev, [&](lp_stream_t st) {
      return lp_add_rms_norm(&x, a[1] != Py_None ? &residual : nullptr, w.data_ptr(), w.numel(), wtype,
                             static_cast<float>(eps), a[4] != Py_None ? &total : nullptr,
                             a[5] != Py_None ? &y : nullptr, a[6] != Py_None ? &q : nullptr, st);
    });
  });
}

// [tokens, k], contiguous
Ints pairs(PyObject* o, const char* name, at::ScalarType type, int64_t tokens, int64_t* k, int device) {
  const Ints v = ints(o, name, type, device);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != 2 || (tokens >= 0 && t.size(0) != tokens) || (*k >= 0 && t.size(1) != *k))
    fail(PyExc_AssertionError, "%s: [tokens, k] expected", name);
  *k = t.size(1);
  return v;
}

// (logits, weights, experts, offsets, rowToken, places, renormalize, workspace)
PyObject* route_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 8, [&] {
    const int dev = device_of(a[0], "logits");
    const lp_matrix l = matrix(a[0], "logits", dev);
    int64_t k = -1;
    const Ints w = pairs(a[1], "weights", at::kFloat, l.rows, &k, dev);
    const Ints ids = pairs(a[2], "experts", at::kInt, l.rows, &k, dev);
    const Ints off = ints(a[3], "offsets", at::kInt, dev), rt = ints(a[4], "rowToken", at::kInt, dev);
    const Ints pl = pairs(a[5], "places", at::kInt, l.rows, &k, dev);
    const int32_t renorm = static_cast<int32_t>(number(a[6]));
    const Ints ws = ints(a[7], "workspace", at::kByte, dev);
    return on_device(dev, [&](lp_stream_t st) {
      return lp_route_experts(&l, static_cast<float*>(w.p), w.n, i32(ids), ids.n, i32(off), off.n, i32(rt), rt.n,
                              i32(pl), pl.n, k, renorm, ws.p, ws.n, st);
    });
  });
}

const lp_expert_weights* weights_of(PyObject* o) {
  return reinterpret_cast<const lp_expert_weights*>(number(o));
}

// (weights, device, codes, scales, offsets, rowToken, out, workspace), gated:
// (weights, device, codes, scales, offsets, rowToken, outCodes, outScales, workspace)
template <bool GATED>
PyObject* expert_gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, GATED ? 9 : 8, [&] {
    const lp_expert_weights* w = weights_of(a[0]);
    const int dev = static_cast<int>(number(a[1]));
    const lp_rows8 x = rows8(a[2], a[3], "codes", "scales", dev);
    if (x.dtype != LP_E4M3) fail(PyExc_TypeError, "codes: expected float8_e4m3fn");
    const Ints off = ints(a[4], "offsets", at::kInt, dev);
    const bool gather = a[5] != Py_None;
    const Ints rt = gather ? ints(a[5], "rowToken", at::kInt, dev) : Ints{nullptr, 0};
    const Ints ws = ints(a[GATED ? 8 : 7], "workspace", at::kByte, dev);
    if (gather && rt.n == 0) return PyLong_FromLong(LP_OK);  // (no rows; an empty tensor has no address)
    if constexpr (GATED) {
      const lp_rows8 out = rows8(a[6], a[7], "outCodes", "outScales", dev);
      if (out.dtype != LP_E4M3) fail(PyExc_TypeError, "outCodes: expected float8_e4m3fn");
      return on_device(dev, [&](lp_stream_t st) {
        return lp_expert_gemm_gated(w, &x, i32(off), off.n, i32(rt), rt.n, &out, ws.p, ws.n, st);
      });
    } else {
      const lp_matrix out = matrix(a[6], "out", dev);
      return on_device(dev, [&](lp_stream_t st) {
        return lp_expert_gemm(w, &x, i32(off), off.n, i32(rt), rt.n, &out, ws.p, ws.n, st);
      });
    }
  });
}

// (rows, weights, places, residual, out)
PyObject* combine_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 5, [&] {
    const int dev = device_of(a[0], "rows");
    const lp_matrix r = matrix(a[0], "rows", dev), out = matrix(a[4], "out", dev);
    int64_t k = -1;
    const Ints w = pairs(a[1], "weights", at::kFloat, out.rows, &k, dev);
    const Ints pl = pairs(a[2], "places", at::kInt, out.rows, &k, dev);
    lp_matrix residual;
    if (a[3] != Py_None) residual = matrix(a[3], "residual", dev);
    return on_device(dev, [&](lp_stream_t st) {
      return lp_combine_experts(&r, static_cast<float*>(w.p), w.n, i32(pl), pl.n,
                                a[3] != Py_None ? &residual : nullptr, &out, st);
    });
  });
}

// The current stream of a device, as a whole number.
PyObject* current_stream(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 1, [&] {
    const int dev = static_cast<int>(number(a[0]));
    return PyLong_FromVoidPtr(c10::cuda::getCurrentCUDAStream(dev).stream());
  });
}

// Whether a device's current stream is being captured into a graph.
PyObject* capturing(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 1, [&] {
    const int dev = static_cast<int>(number(a[0]));
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(dev).stream(), &status) != cudaSuccess)
      (void)cudaGetLastError();  // (a launch would say the same)
    return PyBool_FromLong(status != cudaStreamCaptureStatusNone);
  });
}

#define LP_METHOD(name, f) \
  { name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {
    LP_METHOD("assign_pages", assign_pages),
    LP_METHOD("store_kv", (move_kv<true>)),
    LP_METHOD("load_kv", (move_kv<false>)),
    LP_METHOD("paged_attention", paged_attention),
    LP_METHOD("quantize_rows", quantize_rows),
    LP_METHOD("dequantize_rows", dequantize_rows),
    LP_METHOD("add_rms_norm", add_rms_norm),
    LP_METHOD("route_experts", route_experts),
    LP_METHOD("expert_gemm", expert_gemm<false>),
    LP_METHOD("expert_gemm_gated", expert_gemm<true>),
    LP_METHOD("combine_experts", combine_experts),
    LP_METHOD("current_stream", current_stream),
    LP_METHOD("capturing", capturing),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&module); }
