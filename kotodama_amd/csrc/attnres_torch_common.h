// What the sources of the native call path share (attnres_torch.cpp: routing,
// lm_torch.cpp: the language-model operators).
#ifndef KOTODAMA_AMD_ATTNRES_TORCH_COMMON_H
#define KOTODAMA_AMD_ATTNRES_TORCH_COMMON_H

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>
#include <vector>

#include "attnres.h"

namespace attnres_torch {

using at::Tensor;
using c10::DispatchKey;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------ plain calls --

// Dispatch keys whose tensors are not plain device memory (subclasses, functorch
// wrappers, lazy conjugation and the like).
constexpr c10::DispatchKeySet kOddKeys({DispatchKey::Python, DispatchKey::PythonTLSSnapshot, DispatchKey::Functionalize,
                                        DispatchKey::FuncTorchBatched, DispatchKey::BatchedNestedTensor,
                                        DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched,
                                        DispatchKey::Conjugate, DispatchKey::Negative, DispatchKey::ZeroTensor,
                                        DispatchKey::Tracer});

inline bool dtype_ok(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }
inline int code(at::ScalarType t) { return t == at::kBFloat16 ? ATTNRES_DTYPE_BF16 : ATTNRES_DTYPE_F32; }

inline bool dense(const Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided && !t.key_set().has_any(kOddKeys); }
inline bool plain(const Tensor& t) { return dense(t) && dtype_ok(t.scalar_type()) && t.is_contiguous(); }

// Nothing is watching the calls of this thread: no dispatch mode, no function
// mode, no functorch transform, no tracer.
inline bool unwatched() {
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled()) return false;
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  if (tls.included_.has(DispatchKey::FuncTorchDynamicLayerFrontMode) ||
      tls.included_.has(DispatchKey::FuncTorchDynamicLayerBackMode) || tls.included_.has(DispatchKey::Functionalize) ||
      tls.included_.has(DispatchKey::Python) || tls.included_.has(DispatchKey::FuncTorchVmapMode))
    return false;
  return !torch::jit::tracer::isTracing();
}

// Makes the tensors' device current for the C-ABI call; `stream` is its current stream.
struct OnDevice {
  c10::OptionalDeviceGuard guard;
  void* stream;
  explicit OnDevice(const Tensor& t) {
    const c10::Device dev = t.device();
    if (c10::hip::current_device() != dev.index()) guard.reset_device(dev);
    stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
  }
};

inline Tensor empty(at::IntArrayRef size, at::ScalarType dtype, c10::Device device) {
  return Tensor(at::detail::empty_cuda(size, dtype, device, std::nullopt));
}

using Dims = c10::SmallVector<int64_t, 6>;

inline const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
template <typename T>
T* out_ptr(const Tensor& t) {
  return t.defined() && t.numel() ? static_cast<T*>(t.mutable_data_ptr()) : nullptr;
}

// A profiler's event of a launch that does not pass the dispatcher, under the op's name.
#define ATTNRES_RECORD(name) RECORD_FUNCTION(name, c10::ArrayRef<const c10::IValue>{})

inline Tensor workspace(int64_t bytes, c10::Device dev) {
  return empty({std::max<int64_t>(1, (bytes + 3) / 4)}, at::kFloat, dev);
}

// The registered op, called through the dispatcher (the cases the direct
// launches leave out, and backward passes that are themselves recorded).
template <typename... Args>
std::vector<c10::IValue> call_op(const char* name, Args&&... args) {
  const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "");
  std::vector<c10::IValue> stack{c10::IValue(std::forward<Args>(args))...};
  op.callBoxed(&stack);
  return stack;
}
inline std::optional<Tensor> opt(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// ------------------------------------------------------- Python arguments --

// The tensor behind an argument of exactly type Tensor or Parameter; undefined
// for None; false for anything else.
inline bool take(PyObject* o, bool none_ok, Tensor* t) {
  if (o == Py_None) {
    *t = Tensor();
    return none_ok;
  }
  if (!THPVariable_CheckExact(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}
inline bool take(PyObject* o, double* v) {
  *v = PyFloat_AsDouble(o);
  if (*v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
inline bool take(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}
// exactly True or False (another truthy value is left to Python)
inline bool take(PyObject* o, bool* v) {
  *v = o == Py_True;
  return PyBool_Check(o);
}
inline bool take_list(PyObject* o, std::vector<Tensor>* v) {
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(o);
  PyObject** items = PySequence_Fast_ITEMS(o);
  v->reserve((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    Tensor t;
    if (!take(items[i], false, &t)) return false;
    v->push_back(std::move(t));
  }
  return true;
}

// Whether autograd would record a call on these tensors.
inline bool recorded(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
inline bool recorded(const std::vector<Tensor>& ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.requires_grad()) return true;
  return false;
}
// No tensor carries a forward-mode tangent (the autograd functions here have no forward-mode rule: the op reports it).
inline bool no_tangent(const Tensor& t) { return !t.defined() || !t._fw_grad(0).defined(); }

inline PyObject* none() { Py_RETURN_NONE; }
inline PyObject* wrap(const Tensor& t) {
  if (!t.defined()) return none();
  return THPVariable_Wrap(t);
}
// The entries of lm_torch.cpp.
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* py_embedding(PyObject*, PyObject* const* a, Py_ssize_t n);

}  // namespace attnres_torch

#endif  // KOTODAMA_AMD_ATTNRES_TORCH_COMMON_H
