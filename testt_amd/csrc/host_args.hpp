// Arguments, errors and nodes of the native operators that may be asked for a gradient: what
// host_autograd.cpp and host_generate.cpp share.
#pragma once

#include <optional>
#include <utility>

#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>

#include "host_common.hpp"

namespace soupk_host {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// The interpreter lock for a scope, on a thread that may or may not hold it.
struct Gil {
  PyGILState_STATE state = PyGILState_Ensure();
  ~Gil() { PyGILState_Release(state); }
};

// Raises SoupkError for a status, on any thread.
inline void check(const char* name, int rc) {
  if (rc == 0) return;
  const char* text = p_status_string ? p_status_string(rc) : nullptr;
  const Gil gil;
  PyErr_Format(g_error ? g_error : PyExc_RuntimeError, "%s failed with status %d: %s", name, rc,
               text ? text : "?");
  python_error err;
  err.persist();
  throw std::move(err);
}

// Backwards are differentiable once: under create_graph a gradient of theirs that is differentiated again
// raises when it is (also where only the saved inputs carry gradients, which
// torch.autograd.function.once_differentiable does not see).
struct Twice : Function<Twice> {
  static Tensor forward(AutogradContext*, Tensor x) { return x; }
  static variable_list backward(AutogradContext*, variable_list) {
    throw std::runtime_error(
        "trying to differentiate twice an operator that is differentiable once");
  }
};

template <class F>
variable_list once(F&& f) {
  const bool again = at::GradMode::is_enabled();
  variable_list out;
  {
    at::AutoGradMode off(false);
    out = f();
  }
  if (again)
    for (Tensor& o : out)
      if (o.defined()) o = Twice::apply(o.detach().requires_grad_(true));
  return out;
}

// (A tensor with a tangent goes through the node too, whatever the grad mode: it raises there, as no
// forward-mode derivative is given.)
inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
  const bool grads = at::GradMode::is_enabled();
  for (const Tensor* t : ts)
    if (t && t->defined() && ((grads && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}

inline int32_t code_of(at::ScalarType t) {
  return t == at::kHalf ? SOUPK_DTYPE_F16
                        : t == at::kBFloat16 ? SOUPK_DTYPE_BF16
                                             : t == at::kFloat ? SOUPK_DTYPE_F32 : -1;
}

// A tensor argument, subclasses included (the Python caller has asked their __torch_function__); null for
// anything else and for a subclass with a __torch_dispatch__, whose memory (if it has any) is not its values.
inline const Tensor* tensor(PyObject* o) {
  if (!THPVariable_Check(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.unsafeGetTensorImpl()->is_python_dispatch() ? nullptr : &t;
}
inline bool maybe(PyObject* o, Tensor& t) {
  if (o == Py_None) return true;
  const Tensor* p = tensor(o);
  if (p != nullptr) t = *p;
  return p != nullptr;
}
inline bool on(const Tensor& t, const at::Device& dev) {
  return t.is_cuda() && t.device() == dev && t.layout() == at::kStrided;
}
inline void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <class T>
T* address(const Tensor& t) {
  return static_cast<T*>(address(t));
}

// A Python int of 0 .. 2^64 - 1 (not a bool); false (no Python error) for anything else.
inline bool word(PyObject* o, uint64_t& v) {
  if (!PyLong_Check(o) || PyBool_Check(o)) return false;
  v = PyLong_AsUnsignedLongLong(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
inline bool integer(PyObject* o, int64_t& v) {
  if (!PyLong_Check(o) || PyBool_Check(o)) return false;
  v = PyLong_AsLongLong(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}
// A number, or a tensor of one that wants no gradient (none would be given; the Python caller says so).
inline bool number(PyObject* o, double& v) {
  if (THPVariable_Check(o) && at::GradMode::is_enabled() && THPVariable_Unpack(o).requires_grad())
    return false;
  v = PyFloat_AsDouble(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

inline std::optional<Tensor> given(const Tensor& t) {
  return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

}  // namespace soupk_host
