// The Python calls of the 8-bit KV cache (rapidtinyrec_b200/kv_cache.py): argument checks,
// outputs and workspace from torch's allocator, and one call into the C ABI, in C++.  A
// call that checks six tensors and passes fourteen arguments through ctypes costs 9 - 12 us of
// the host, longer than the smallest kernels run; here a write 2.5, an attention 3.6, a read with
// its two outputs 4.2.
//
// The module links against torch only; setup() hands it the C entry points' addresses.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdarg>
#include <cstdio>

#include "rtr_b200.h"

namespace {

decltype(&rtr_kv_write) kv_write;
decltype(&rtr_kv_read) kv_read;
decltype(&rtr_kv_attention) kv_attention;
decltype(&rtr_kv_attention_workspace) kv_workspace;
decltype(&rtr_last_error) last_error;
PyObject* native_error;  // _native.NativeError(code, message)

// Thrown where a Python exception is set already.
struct Raised {};

[[noreturn]] void refuse(const char* format, ...) {
  char text[256];
  va_list args;
  va_start(args, format);
  vsnprintf(text, sizeof text, format, args);
  va_end(args);
  PyErr_SetString(PyExc_ValueError, text);
  throw Raised{};
}

void check(int code) {
  if (code == RTR_OK) return;
  if (PyObject* e = PyObject_CallFunction(native_error, "is", code, last_error(nullptr))) {
    PyErr_SetObject(native_error, e);
    Py_DECREF(e);
  }
  throw Raised{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

// The cache a call works on: its C struct (kept by KvCache8) and device.
struct Cache {
  const rtr_kv_cache* c;
  int index;
  Cache(PyObject* at, PyObject* device)
      : c(static_cast<const rtr_kv_cache*>(PyLong_AsVoidPtr(at))), index((int)PyLong_AsLong(device)) {
    if (PyErr_Occurred()) throw Raised{};
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }
  bool here(const at::Tensor& t) const { return t.is_cuda() && t.get_device() == index; }
};

rtr_kv_batch batch_of(const Cache& cache, int64_t rows, PyObject* table_, PyObject* lens_, PyObject* starts_) {
  const at::Tensor &table = tensor(table_, "table"), &lens = tensor(lens_, "lens");
  if (table.scalar_type() != at::kInt || lens.scalar_type() != at::kInt || table.dim() != 2 || lens.dim() != 1 ||
      lens.size(0) != table.size(0))
    refuse("table must be int32 [seqs, width] and lens int32 [seqs]");
  const int64_t seqs = table.size(0), width = table.size(1);
  if ((width > 1 && table.stride(1) != 1) || (seqs > 1 && lens.stride(0) != 1))
    refuse("the rows of table and lens must be contiguous");
  if (!cache.here(table) || !cache.here(lens)) refuse("table and lens must lie on the cache's device");
  if (rows > INT32_MAX || seqs > INT32_MAX || width > INT32_MAX) refuse("rows, seqs and width must fit 32 bits");
  rtr_kv_batch b = {};
  b.table = static_cast<const int32_t*>(table.data_ptr());
  b.lens = static_cast<const int32_t*>(lens.data_ptr());
  b.table_stride = seqs > 1 ? table.stride(0) : width;
  b.table_width = (int32_t)width;
  b.seqs = (int32_t)seqs;
  b.rows = (int32_t)rows;
  if (starts_ == Py_None) {
    if (seqs ? rows % seqs : rows) refuse("without starts the rows must be a multiple of the sequences");
  } else {
    const at::Tensor& starts = tensor(starts_, "starts");
    if (starts.scalar_type() != at::kInt || starts.dim() != 1 || starts.size(0) != seqs + 1 || !starts.is_contiguous())
      refuse("starts must be int32 [seqs + 1], contiguous");
    if (!cache.here(starts)) refuse("starts must lie on the cache's device");
    b.starts = static_cast<const int32_t*>(starts.data_ptr());
  }
  return b;
}

// Rows must be [rows, heads, head_dim] of one of the two types; false where the kernels
// cannot take them as they lie (dimensions contiguous, 16-byte steps).
bool dense(const Cache& cache, const at::Tensor& x, int64_t heads, const char* name, bool heads_contiguous) {
  const int64_t dim = cache.c->head_dim;
  if (x.dim() != 3 || x.size(1) != heads || x.size(2) != dim || !cache.here(x))
    refuse("%s must be [rows, %lld, %lld] on the cache's device", name, (long long)heads, (long long)dim);
  if (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16) refuse("%s must be float32 or bfloat16", name);
  const int64_t step = 16 / x.element_size();
  return x.stride(2) == 1 && x.stride(0) % step == 0 && x.stride(1) % step == 0 &&
         (!heads_contiguous || heads == 1 || x.stride(1) == dim) &&
         reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}

// Whether out, contiguous, shares memory with q [rows, row], rows `step` apart, without being q itself.
// (A block has read its rows before any of them is written; other blocks' rows it must not touch.)
bool overlaps(const at::Tensor& out, const at::Tensor& q) {
  const int64_t size = q.element_size(), rows = q.size(0), row = q.size(1) * q.size(2) * size, step = q.stride(0) * size;
  const int64_t from = static_cast<const char*>(out.data_ptr()) - static_cast<const char*>(q.data_ptr());
  if (!rows || from >= (rows - 1) * step + row || from + rows * row <= 0) return false;
  if (from == 0 && (rows == 1 || step == row)) return false;
  return !(step > row && from > 0 && from % step >= row && from % step + rows * row <= step);  // between two rows
}

int32_t type_of(const at::Tensor& x) { return x.scalar_type() == at::kFloat ? RTR_DTYPE_F32 : RTR_DTYPE_BF16; }

// A new tensor on the cache's device, by its allocator without a pass through the dispatcher.
at::Tensor room_for(const Cache& cache, at::IntArrayRef size, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(size, type, at::Device(at::kCUDA, (c10::DeviceIndex)cache.index), std::nullopt));
}

at::Tensor copied(const at::Tensor& x) { return x.clone(at::MemoryFormat::Contiguous); }

template <typename F> PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& body) {
  HANDLE_TH_ERRORS  // torch's own exceptions as torch raises them (OutOfMemoryError, say)
  try {
    if (given != wanted) refuse("%d arguments expected", (int)wanted);
    return body();
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// write(cache, device, k, v, table, lens, starts)
PyObject* call_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Cache cache(a[0], a[1]);
    at::Tensor k = tensor(a[2], "k"), v = tensor(a[3], "v");
    if (k.scalar_type() != v.scalar_type() || k.sizes() != v.sizes()) refuse("k and v must have one type and shape");
    if (!dense(cache, k, cache.c->kv_heads, "k", false)) k = copied(k);
    if (!dense(cache, v, cache.c->kv_heads, "v", false)) v = copied(v);
    const rtr_kv_batch b = batch_of(cache, k.size(0), a[4], a[5], a[6]);
    check(kv_write(cache.c, &b, k.data_ptr(), v.data_ptr(), type_of(k), k.stride(0), k.stride(1), v.stride(0),
                   v.stride(1), cache.index, cache.stream()));
    Py_RETURN_NONE;
  });
}

// read(cache, device, rows, table, lens, starts, dtype (0 float32, 1 bfloat16), out or None)
PyObject* call_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Cache cache(a[0], a[1]);
    const int64_t rows = PyLong_AsLongLong(a[2]), dtype = PyLong_AsLongLong(a[6]);
    if (PyErr_Occurred()) throw Raised{};
    const int64_t heads = cache.c->kv_heads, dim = cache.c->head_dim;
    if (rows < 0) refuse("negative row count");
    at::Tensor k, v;
    if (a[7] == Py_None) {
      const at::ScalarType type = dtype ? at::kBFloat16 : at::kFloat;
      k = room_for(cache, {rows, heads, dim}, type);
      v = room_for(cache, {rows, heads, dim}, type);
    } else {
      if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 2) refuse("out must be a pair of tensors");
      k = tensor(PyTuple_GET_ITEM(a[7], 0), "out");
      v = tensor(PyTuple_GET_ITEM(a[7], 1), "out");
      if (k.scalar_type() != v.scalar_type()) refuse("out must be two tensors of one type");
      if (rows && k.data_ptr() == v.data_ptr()) refuse("out must be two tensors, not one twice");
      for (const at::Tensor* x : {&k, &v}) {
        bool own = dense(cache, *x, heads, "out", false) && x->size(0) == rows;
        for (int d = 0; d < 2; ++d) own = own && (x->size(d) < 2 || x->stride(d) != 0);
        if (!own) refuse("out must have %lld rows of their own, contiguous dimensions, at multiples of 16 bytes", (long long)rows);
      }
    }
    const rtr_kv_batch b = batch_of(cache, rows, a[3], a[4], a[5]);
    check(kv_read(cache.c, &b, k.data_ptr(), v.data_ptr(), type_of(k), k.stride(0), k.stride(1), v.stride(0),
                  v.stride(1), cache.index, cache.stream()));
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw Raised{};
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(k));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(v));
    return pair;
  });
}

// attention(cache, device, q, table, lens, starts, causal, scale, return_lse, out or None)
PyObject* call_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    const Cache cache(a[0], a[1]);
    at::Tensor q = tensor(a[2], "q");
    const int64_t kv = cache.c->kv_heads, dim = cache.c->head_dim;
    if (q.dim() != 3 || q.size(1) < 1 || q.size(1) % kv)
      refuse("q must be [rows, heads, %lld], heads a multiple of %lld", (long long)dim, (long long)kv);
    const int64_t rows = q.size(0), heads = q.size(1);
    if (!dense(cache, q, heads, "q", true)) q = copied(q);
    const rtr_kv_batch b = batch_of(cache, rows, a[3], a[4], a[5]);
    const int causal = PyObject_IsTrue(a[6]), with_lse = PyObject_IsTrue(a[8]);
    const double scale = PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred()) throw Raised{};
    at::Tensor out, lse, work;
    if (a[9] == Py_None) {
      out = room_for(cache, {rows, heads, dim}, q.scalar_type());
    } else {
      out = tensor(a[9], "out");
      if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !cache.here(out) || !out.is_contiguous() ||
          reinterpret_cast<uintptr_t>(out.data_ptr()) % 16)
        refuse("out must be contiguous and like q");
      if (overlaps(out, q)) refuse("out must be q itself or lie apart from it");
    }
    int64_t room = 0;
    check(kv_workspace(cache.c, &b, type_of(q), (int32_t)heads, cache.index, &room));
    if (with_lse) lse = room_for(cache, {rows, heads}, at::kFloat);
    if (room) work = room_for(cache, {room}, at::kByte);
    check(kv_attention(cache.c, &b, q.data_ptr(), type_of(q), (int32_t)heads, q.stride(0), causal, (float)scale,
                       out.data_ptr(), with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr,
                       room ? work.data_ptr() : nullptr, room, cache.index, cache.stream()));
    if (!with_lse) return THPVariable_Wrap(out);
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw Raised{};
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(lse));
    return pair;
  });
}

// setup(write, read, attention, workspace, last_error addresses, NativeError)
PyObject* call_setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    void* at[5];
    for (int i = 0; i < 5; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) throw Raised{};
    kv_write = reinterpret_cast<decltype(kv_write)>(at[0]);
    kv_read = reinterpret_cast<decltype(kv_read)>(at[1]);
    kv_attention = reinterpret_cast<decltype(kv_attention)>(at[2]);
    kv_workspace = reinterpret_cast<decltype(kv_workspace)>(at[3]);
    last_error = reinterpret_cast<decltype(last_error)>(at[4]);
    Py_INCREF(a[5]);
    Py_XSETREF(native_error, a[5]);
    Py_RETURN_NONE;
  });
}

#define CALL(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"setup", CALL(call_setup)},
                         {"write", CALL(call_write)},
                         {"read", CALL(call_read)},
                         {"attention", CALL(call_attention)},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_call() { return PyModule_Create(&module); }
