// What the operators' host sides that build autograd nodes share: checks of arguments, where a call runs, what nodes save and get back.
#pragma once
#include <torch/csrc/python_headers.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <mutex>
#include <string>

#include "gact_hip.h"
#include "torch_layers.h"

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GACT_F32;
    case at::kHalf: return GACT_F16;
    case at::kBFloat16: return GACT_BF16;
    default: return -1;
  }
}

inline void check_status(int rc) { TORCH_CHECK(rc == GACT_OK, "gact: ", gact_strerror(rc)); }

inline c10::DispatchKeySet wrapped_keys() {
  return c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor,
                              c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper});
}
inline bool plain(const at::Tensor& t) { return t.layout() == at::kStrided && t.has_storage() && !t.key_set().has_any(wrapped_keys()); }
// a tensor (or parameter) itself, no subclass and no wrapper, dense on the GPU
inline const at::Tensor& tensor_of(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA tensor!");
  TORCH_CHECK(plain(t), name, " must be a plain dense tensor");
  TORCH_CHECK(dtype_code(t.scalar_type()) >= 0, "The type of ", name, " is not correct!");
  return t;
}
inline std::optional<at::Tensor> tensor_or_none(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor_of(o, name);
}
// The type that autocast runs an operator in; its arguments may then be of others
using Autocast = std::optional<at::ScalarType>;
inline void check_like(const at::Tensor& t, const at::Tensor& like, const char* name, const Autocast& autocast) {
  TORCH_CHECK(autocast || t.scalar_type() == like.scalar_type(), "The type of ", name, " is not correct!");
  TORCH_CHECK(t.device() == like.device(), name, " is on another device");
}
// the argument as autocast's operators take it, differentiably
inline at::Tensor cast(const at::Tensor& t, const Autocast& autocast) { return autocast ? t.to(*autocast) : t; }
inline std::optional<at::Tensor> cast(const std::optional<at::Tensor>& t, const Autocast& autocast) {
  return t && autocast ? std::optional<at::Tensor>(t->to(*autocast)) : t;
}

// Everything a call needs to know about where it runs
struct Place {
  c10::Device device;
  c10::DeviceGuard guard;
  void* stream;
  bool ordinary;
  explicit Place(const at::Tensor& t)
      : device(t.device()), guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()), ordinary(gact_torch_ordinary()) {}
  at::Tensor empty(c10::IntArrayRef shape, at::ScalarType dtype) const {
    if (ordinary) return gact_torch_empty(shape, dtype, device);
    return at::empty(shape, at::TensorOptions().dtype(dtype).device(device));
  }
  at::Tensor bytes(int64_t size) const { return size ? empty({size}, at::kByte) : at::Tensor(); }
  at::Tensor zeros(c10::IntArrayRef shape, at::ScalarType dtype) const {
    return at::zeros(shape, at::TensorOptions().dtype(dtype).device(device));
  }
};
inline const void* in(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
inline void* out(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
inline bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

inline at::Tensor dense_of(const at::Tensor& t) { return t.is_contiguous() && !t.is_neg() ? t : t.resolve_neg().contiguous(); }
inline void no_tangent(const std::optional<at::Tensor>& t, const char* operation) {
  TORCH_CHECK(!t.has_value() || !torch::autograd::isFwGradDefined(*t), operation, " has no forward-mode derivative");
}

// A leaf whose gradient's accumulator was made on the default stream - an eager graph of it is still alive - cannot be differentiated in a
// pass that is being captured: autograd would make the default stream wait for the capture, which the runtime answers by ending it, and
// torch by ending the process.
inline void refuse_stale_leaves(std::initializer_list<const at::Tensor*> tensors, const at::Tensor& like) {
  const c10::hip::HIPStream current = c10::hip::getCurrentHIPStream(like.device().index());
  hipStreamCaptureStatus status;
  if (current.stream() == nullptr || hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  for (const at::Tensor* t : tensors) {
    if (!t || !t->requires_grad() || !t->is_leaf()) continue;
    const std::shared_ptr<Node> accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!accumulator) continue;
    const std::optional<c10::Stream> stream = accumulator->stream();
    TORCH_CHECK(!stream || stream->id() != 0,
                "a training pass is captured while an eager graph of one of its leaves, made on the default stream, is alive: drop it first");
  }
}
inline const at::Tensor* held(const std::optional<at::Tensor>& t) { return t ? &*t : nullptr; }

// results of a backward pass that is itself being differentiated: an error once somebody goes through them
inline variable_list once(variable_list grads, const char* name) {
  if (!c10::GradMode::is_enabled()) return grads;
  const auto stop = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice a function that was marked with @once_differentiable: ") + name, (int64_t)grads.size());
  for (at::Tensor& g : grads)      // the error's node hangs on tensors that need a gradient, which the result does through what was saved
    if (g.defined()) g = g.detach().set_requires_grad(true);
  return (*stop)(std::move(grads));
}
inline void give_up(SavedVariable& v) { v.reset_data(); }
// What was saved, as it was saved: hooks for saved tensors may give back anything, and the kernels would read it as if it were the same
inline at::Tensor again(SavedVariable& v, at::ScalarType dtype, c10::IntArrayRef shape, const at::Tensor& grad, bool dense = true) {
  const at::Tensor t = v.unpack();
  TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.scalar_type() == dtype && t.device() == grad.device() && t.sizes() == shape &&
                  (!dense || (t.is_contiguous() && !t.is_neg())),
              "the hooks for saved tensors gave back another tensor than they were given");
  return dense && !aligned(in(t)) ? t.clone() : t;      // a place in a larger buffer, say
}
// a gradient that the kernels can read: no batch of them, no subclass
inline void check_grad(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda() && plain(t), "the gradient must be a plain dense tensor");
}

// the operator itself: its allocations and launches may wait for the GPU, and other threads of Python's go on meanwhile
template <typename F>
auto without_gil(const F& call) {
  const WithoutGil released;
  return call();
}
inline double number_of(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
inline int64_t integer_of(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
// How many there are, and that no trace is being recorded: of these operators it would hold the results' allocations and nothing that fills them
inline void arguments(Py_ssize_t n, Py_ssize_t wanted, const char* what = "the layers on 8-bit checkpoints") {
  TORCH_CHECK_TYPE(n == wanted, "expected ", wanted, " arguments, got ", n);
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer), what, " cannot be traced");
}

inline Autocast autocast_of(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  TORCH_CHECK_TYPE(THPDtype_Check(o), "a type is expected");
  const at::ScalarType t = ((THPDtype*)o)->scalar_type;
  TORCH_CHECK(dtype_code(t) >= 0, "autocast's type is not correct");
  return t;
}

}  // namespace

#define FASTCALL(name, f) {name, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
