// What the compiled bindings share: reading arguments, checking tensors, and the call on the
// tensors' own device and its current stream. Included by one source file per module.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../../include/pkv.h"

namespace {

using at::Tensor;

struct Refused : std::runtime_error {  // ValueError
  using std::runtime_error::runtime_error;
};

const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw torch::TypeError(std::string("expected a tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
int32_t integer32(PyObject* o) {
  const int64_t v = integer(o);
  if (v != (int32_t)v) throw Refused("a count is past 32 bits");
  return (int32_t)v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
template <typename T>
T* handle(PyObject* o) {  // the address of a ctypes structure
  return reinterpret_cast<T*>(integer(o));
}
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }

// A new contiguous tensor of t's type and device, without the dispatcher's part of the call.
Tensor fresh(at::IntArrayRef sizes, const Tensor& t) {
  return Tensor(at::detail::empty_cuda(sizes, t.scalar_type(), t.device(), std::nullopt));
}

int cuda_index(const Tensor& t) {
  if (!t.is_cuda()) throw std::runtime_error("the paged-KV kernels need CUDA tensors (there is no CPU path)");
  return t.get_device();
}

// The device and what is asked of flat arguments on it.
struct Call {
  const char* name;
  int device;
  c10::cuda::CUDAGuard guard;
  pkv_stream_t stream;

  Call(const char* n, const Tensor& t)
      : name(n), device(cuda_index(t)), guard((c10::DeviceIndex)device),
        stream(reinterpret_cast<pkv_stream_t>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream())) {}

  [[noreturn]] void refuse(const std::string& why) const { throw Refused(std::string(name) + ": " + why); }
  void here(const Tensor& t) const {
    if (!t.is_cuda() || t.get_device() != device) refuse("every tensor must be on cuda:" + std::to_string(device));
  }
  const Tensor& flat(PyObject* o, at::ScalarType type, const char* what) const {
    const Tensor& t = tensor(o);
    if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != device || !t.is_contiguous())
      refuse(std::string(what) + " must be a contiguous " + at::toString(type) + " tensor on cuda:" + std::to_string(device));
    return t;
  }
  int32_t* i32(PyObject* o, const char* what, int64_t least) const {
    const Tensor& t = flat(o, at::kInt, what);
    if (t.numel() < least) refuse(std::string(what) + " is too short");
    return t.data_ptr<int32_t>();
  }
  int64_t* i64(PyObject* o, const char* what, int64_t count) const {
    const Tensor& t = flat(o, at::kLong, what);
    if (t.numel() != count) refuse(std::string(what) + " must have " + std::to_string(count) + " entries");
    return t.data_ptr<int64_t>();
  }
  int32_t* status(PyObject* o) const { return given(o) ? i32(o, "status", 1) : nullptr; }
};

at::ScalarType pool_type(const pkv_pool& pool) { return pool.dtype == PKV_F16 ? at::kHalf : at::kBFloat16; }

void check_pool_type(const Call& call, const pkv_pool& pool, const Tensor& t) {
  if (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16) {
    PyErr_Format(PyExc_NotImplementedError, "the sm_100a kernels take float16 or bfloat16 KV caches, not %s",
                 at::toString(t.scalar_type()));
    throw python_error();
  }
  if (t.scalar_type() != pool_type(pool)) call.refuse("the tensors and the pool must share one dtype");
}

PyObject* status_or_none(int status) { return status == PKV_OK ? Py_NewRef(Py_None) : PyLong_FromLong(status); }

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t), int N>
PyObject* exactly(PyObject* self, PyObject* const* args, Py_ssize_t count) {
  if (count == N) return F(self, args, count);
  PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, count);
  return nullptr;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(exactly<F, N>)), METH_FASTCALL, nullptr};
}

}  // namespace
