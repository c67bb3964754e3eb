// What the Python call modules share: refusals, errors of the C ABI, and the frame that turns
// both, and torch's own exceptions, into Python ones.  Each module links against torch only;
// its setup() hands it the C entry points' addresses.
#pragma once

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdarg>
#include <cstdio>

#include "rtr_b200.h"

namespace {

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

#define CALL(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr

}  // namespace
