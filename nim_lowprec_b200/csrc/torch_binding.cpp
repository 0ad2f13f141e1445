// torch_binding.cpp -- the paged cache's entry points for torch tensors, as a
// CPython module: argument checks and one call of the C ABI.  A decode step
// calls these once per layer; through ctypes a call with eleven tensors costs
// 13 us, about four times its kernel.
//
// Functions take their arguments by position; attention.py has the public
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
    LP_METHOD("current_stream", current_stream),
    LP_METHOD("capturing", capturing),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&module); }
