// The calls of PagedKv on torch tensors: checks, results and scratch, then the C ABI.
//
// A CPython module rather than ctypes, because these calls are a handful a layer and last microseconds on the
// GPU: checking the tensors in Python and converting 17 arguments took 9.0 us a decode call, 4.4 us of it the
// C ABI's through ctypes.  Errors found here are ValueErrors; a status of the C ABI is returned as an int for the
// caller to raise.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <new>
#include <optional>
#include <stdexcept>
#include <string>

#include "bfvgpu.h"

namespace {

constexpr const char* kName = "bfvgpu.kv";
constexpr const char* kWhere = " on the cache's device";

struct Cache {
  bfvgpu_kv kv;
  int device;
  double scale;
  at::Tensor k, v;  // the pages, where open was given them
  at::ScalarType type() const { return kv.dtype == BFVGPU_KV_BF16 ? at::kBFloat16 : at::kHalf; }
};

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const std::string& what) { throw Refused(what); }

// ---- arguments ----
const Cache& cache_of(PyObject* o) {
  auto* c = static_cast<Cache*>(PyCapsule_GetPointer(o, kName));
  if (!c) throw python_error();
  return *c;
}
bfvgpu_ctx* context_of(PyObject* o) {
  if (o == Py_None) return nullptr;
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw python_error();
  return static_cast<bfvgpu_ctx*>(p);
}
int32_t int_of(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  if (v != (int32_t)v) {
    PyErr_SetString(PyExc_OverflowError, "a 32-bit number is wanted");
    throw python_error();
  }
  return (int32_t)v;
}
const at::Tensor& tensor_of(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: a tensor is wanted", name);
    throw python_error();
  }
  return THPVariable_Unpack(o);
}
bool there(const at::Tensor& t, const Cache& c) { return t.is_cuda() && t.get_device() == c.device; }

struct Table {
  int32_t* at = nullptr;
  uint64_t rows = 0, width = 0;
};
Table table_of(PyObject* o, const Cache& c) {
  const at::Tensor& t = tensor_of(o, "table");
  if (t.scalar_type() != at::kInt || !there(t, c) || t.dim() != 2 || !t.is_contiguous())
    refuse(std::string("E_KV_SHAPE: the table is a dense int32 tensor [rows][width]") + kWhere);
  return {static_cast<int32_t*>(t.data_ptr()), (uint64_t)t.size(0), (uint64_t)t.size(1)};
}
int32_t* ints_of(PyObject* o, const char* name, uint64_t count, const Cache& c) {
  const at::Tensor& t = tensor_of(o, name);
  if (t.scalar_type() != at::kInt || !there(t, c) || t.dim() != 1 || (uint64_t)t.size(0) != count || !t.is_contiguous())
    refuse(std::string("E_KV_SHAPE: ") + name + " is a dense int32 tensor [" + std::to_string(count) + "]" + kWhere);
  return static_cast<int32_t*>(t.data_ptr());
}
uint64_t count_of(PyObject* o, const char* name) {
  const at::Tensor& t = tensor_of(o, name);
  return t.dim() == 1 ? (uint64_t)t.size(0) : 0;
}
// [tokens][heads][dim], dim contiguous
const at::Tensor& rows_of(PyObject* o, const char* name, const Cache& c) {
  const at::Tensor& t = tensor_of(o, name);
  if (!there(t, c) || t.dim() != 3 || t.size(2) != c.kv.dim || t.stride(2) != 1)
    refuse(std::string("E_KV_SHAPE: ") + name + " is [tokens][heads][" + std::to_string(c.kv.dim) + "], dim contiguous," + kWhere);
  return t;
}

// The stream of a call: the given handle, or torch's current one (whose null handle is the legacy stream: the C
// ABI reads a null stream as the context's).  What is allocated meanwhile belongs to it, and a given one is recorded
// with the tensors it uses, so that memory which the caller lets go is not given out again before the call's work is done.
struct Stream {
  std::optional<c10::cuda::CUDAStreamGuard> guard;
  void* handle = nullptr;
  Stream(PyObject* o, const Cache& c) {
    if (o != Py_None) {
      handle = PyLong_AsVoidPtr(o);
      if (!handle && PyErr_Occurred()) throw python_error();
    }
    if (handle)
      guard.emplace(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(handle), (c10::DeviceIndex)c.device));
    else
      handle = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)c.device).stream();
    if (!handle) handle = cudaStreamLegacy;
  }
  void uses(const at::Tensor& t) const {
    if (guard && t.defined()) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), guard->current_stream());
  }
  void uses(const Cache& c, std::initializer_list<PyObject*> tensors) const {
    if (!guard) return;
    uses(c.k);
    uses(c.v);
    for (PyObject* o : tensors)
      if (o && o != Py_None) uses(THPVariable_Unpack(o));
  }
};

template <class F>
PyObject* answered(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
bool wants(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
  return false;
}

// ---- calls ----
// open(address of a bfvgpu_kv, device[, k, v]) -> cache, which keeps the pages k and v
PyObject* open_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4 && !wants(n, 2)) return nullptr;
  return answered([&]() -> PyObject* {
    const void* from = PyLong_AsVoidPtr(a[0]);
    if (!from) {
      if (PyErr_Occurred()) throw python_error();
      refuse("E_KV_ARGUMENT");
    }
    at::Tensor k, v;
    if (n == 4) k = tensor_of(a[2], "k"), v = tensor_of(a[3], "v");
    auto* c = new Cache{*static_cast<const bfvgpu_kv*>(from), int_of(a[1]), 0.0, k, v};
    c->scale = 1.0 / std::sqrt((double)c->kv.dim);
    PyObject* o = PyCapsule_New(c, kName, [](PyObject* o) { delete static_cast<Cache*>(PyCapsule_GetPointer(o, kName)); });
    if (!o) delete c;
    return o;
  });
}

// append(cache, ctx, k_new, v_new, starts | None, table, lengths, layer, stream | None) -> status
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!wants(n, 9)) return nullptr;
  return answered([&]() -> PyObject* {
    const Cache& c = cache_of(a[0]);
    const at::Tensor &k = rows_of(a[2], "k_new", c), &v = tensor_of(a[3], "v_new");
    const bool wide = k.scalar_type() == at::kFloat;
    if (k.size(1) != c.kv.heads || !(wide || k.scalar_type() == c.type()))
      refuse("E_KV_SHAPE: k_new has the cache's heads, and its type or float32");
    if (v.sizes() != k.sizes() || v.strides() != k.strides() || v.scalar_type() != k.scalar_type() || !there(v, c))
      refuse("E_KV_SHAPE: k_new and v_new need one shape, type and layout");
    const Table t = table_of(a[5], c);
    const int32_t* starts = a[4] == Py_None ? nullptr : ints_of(a[4], "starts", t.rows + 1, c);
    const int32_t* lengths = ints_of(a[6], "lengths", t.rows, c);
    const Stream s(a[8], c);
    s.uses(c, {a[2], a[3], a[4], a[5], a[6]});
    return PyLong_FromLong(bfvgpu_kv_append_device(context_of(a[1]), &c.kv, int_of(a[7]), k.data_ptr(), v.data_ptr(),
                                                   wide ? BFVGPU_KV_F32 : c.kv.dtype, k.stride(0), k.stride(1),
                                                   (uint64_t)k.size(0), starts, t.at, t.width, lengths, t.rows, s.handle));
  });
}

// fork(cache, ctx, parents, children, fresh, table, lengths, stream | None) -> status
PyObject* fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!wants(n, 8)) return nullptr;
  return answered([&]() -> PyObject* {
    const Cache& c = cache_of(a[0]);
    const Table t = table_of(a[5], c);
    const uint64_t count = count_of(a[2], "parents");
    const int32_t *parents = ints_of(a[2], "parents", count, c), *children = ints_of(a[3], "children", count, c),
                  *fresh = ints_of(a[4], "fresh", count, c);
    int32_t* lengths = ints_of(a[6], "lengths", t.rows, c);
    const Stream s(a[7], c);
    s.uses(c, {a[2], a[3], a[4], a[5], a[6]});
    return PyLong_FromLong(bfvgpu_kv_fork_device(context_of(a[1]), &c.kv, parents, children, fresh, count, t.at, t.rows,
                                                 t.width, lengths, s.handle));
  });
}

// move(cache, ctx, src, dst, table | None, stream | None) -> status
PyObject* move(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!wants(n, 6)) return nullptr;
  return answered([&]() -> PyObject* {
    const Cache& c = cache_of(a[0]);
    const Table t = a[4] == Py_None ? Table{} : table_of(a[4], c);
    const uint64_t count = count_of(a[2], "src");
    const int32_t *src = ints_of(a[2], "src", count, c), *dst = ints_of(a[3], "dst", count, c);
    const Stream s(a[5], c);
    s.uses(c, {a[2], a[3], a[4]});
    return PyLong_FromLong(
        bfvgpu_kv_move_device(context_of(a[1]), &c.kv, src, dst, count, t.at, t.rows, t.width, s.handle));
  });
}

// The attention of q: of single tokens where starts is null.
PyObject* attend(PyObject* const* a, PyObject* of_starts, PyObject* const* rest) {
  // a: cache, ctx, q; rest: table, lengths, layer, window, sinks, scale | None, out | None, stream | None
  return answered([&]() -> PyObject* {
    const Cache& c = cache_of(a[0]);
    bfvgpu_ctx* ctx = context_of(a[1]);
    const at::Tensor& q = rows_of(a[2], "q", c);
    const uint64_t tokens = (uint64_t)q.size(0), heads = (uint64_t)q.size(1);
    const Table t = table_of(rest[0], c);
    if (!of_starts && tokens != t.rows) refuse("E_KV_SHAPE: one query per row of the table");
    const int32_t* starts = of_starts ? ints_of(of_starts, "starts", t.rows + 1, c) : nullptr;
    const int32_t* lengths = ints_of(rest[1], "lengths", t.rows, c);
    const int32_t layer = int_of(rest[2]), window = int_of(rest[3]), sinks = int_of(rest[4]);
    double scale = c.scale;
    if (rest[5] != Py_None) {
      scale = PyFloat_AsDouble(rest[5]);
      if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    }
    if (q.scalar_type() != c.type()) refuse("E_KV_DTYPE: q has the cache's type");
    const Stream s(rest[7], c);
    at::Tensor made;
    if (rest[6] == Py_None) {
      made = at::empty(q.sizes(), q.options());
    } else {
      const at::Tensor& given = tensor_of(rest[6], "out");
      if (given.sizes() != q.sizes() || given.scalar_type() != q.scalar_type() || !there(given, c) || !given.is_contiguous())
        refuse("E_KV_SHAPE: out is dense, of q's shape and type");
    }
    s.uses(c, {a[2], of_starts, rest[0], rest[1], rest[6]});
    const at::Tensor& out = made.defined() ? made : THPVariable_Unpack(rest[6]);
    const uint64_t words =
        of_starts ? bfvgpu_kv_prompt_scratch_words(ctx, &c.kv, heads, tokens, t.rows, t.width, window, sinks)
                  : bfvgpu_kv_decode_scratch_words(ctx, &c.kv, heads, t.rows, t.width, window, sinks);
    at::Tensor scratch;
    if (words) scratch = at::empty({(int64_t)words}, q.options().dtype(at::kLong));
    auto* space = words ? static_cast<uint64_t*>(scratch.data_ptr()) : nullptr;
    const int32_t rc =
        of_starts ? bfvgpu_kv_prompt_device(ctx, &c.kv, layer, q.data_ptr(), q.stride(0), q.stride(1), heads, tokens, starts,
                                            t.at, t.width, lengths, t.rows, window, sinks, (float)scale, space,
                                            out.data_ptr(), s.handle)
                  : bfvgpu_kv_decode_device(ctx, &c.kv, layer, q.data_ptr(), q.stride(0), q.stride(1), heads, t.at, t.width,
                                            lengths, t.rows, window, sinks, (float)scale, space, out.data_ptr(), s.handle);
    if (rc) return PyLong_FromLong(rc);
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(rest[6]);
    return rest[6];
  });
}
// decode(cache, ctx, q, table, lengths, layer, window, sinks, scale | None, out | None, stream | None) -> out | status
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) { return wants(n, 11) ? attend(a, nullptr, a + 3) : nullptr; }
// prompt(cache, ctx, q, starts, table, ...) -> out | status
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) { return wants(n, 12) ? attend(a, a[3], a + 4) : nullptr; }

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F)), METH_FASTCALL, nullptr};
}

}  // namespace

PyMODINIT_FUNC PyInit_bfvgpu_kv_calls() {
  static PyMethodDef methods[] = {method<open_cache>("open"), method<append>("append"), method<fork>("fork"), method<move>("move"),
                                  method<decode>("decode"),   method<prompt>("prompt"), {nullptr, nullptr, 0, nullptr}};
  static PyModuleDef module = {PyModuleDef_HEAD_INIT, "bfvgpu_kv_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
  return PyModule_Create(&module);
}
