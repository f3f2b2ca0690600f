// What the sources of the host extension share: the library's entry points, bound once under the
// import of the library, and the argument, allocation and launch helpers of the native operators.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>

#include "../../include/soupk.h"

namespace soupk_host {

using at::Tensor;

// ---- entry points ------------------------------------------------------------------------------

#define SOUPK_ENTRIES(X)                                                                          \
  X(soupk_nf4_unpack) X(soupk_nf4_unpack_multi) X(soupk_nf4_unpack_multi_lora)                    \
  X(soupk_index_inverse) X(soupk_sum_partials) X(soupk_rmsnorm_fwd) X(soupk_rmsnorm_bwd)          \
  X(soupk_rope_pack_fwd) X(soupk_rope_pack_bwd) X(soupk_rope_pack_tokens) X(soupk_swiglu_fwd)     \
  X(soupk_swiglu_bwd_inplace) X(soupk_head_stats_grad) X(soupk_head_stats_grad_rows)              \
  X(soupk_head_plan) X(soupk_head_stats_grad_planned) X(soupk_head_finish) X(soupk_head_dh)       \
  X(soupk_attention_fwd) X(soupk_attention_bwd) X(soupk_attention_varlen_fwd)                     \
  X(soupk_attention_varlen_bwd) X(soupk_lora_stage) X(soupk_lora_fwd) X(soupk_lora_rope_fwd)      \
  X(soupk_lora_bwd_rows) X(soupk_lora_bwd_params) X(soupk_lora_bwd_params_noalloc)                \
  X(soupk_gemm_tn) X(soupk_gemm_nn_nf4) X(soupk_gemm_tn_nf4) X(soupk_gemm_tn_nf4_split)           \
  X(soupk_gemm_nn_nf4_split) X(soupk_gemm_lt) X(soupk_gemm_nn) X(soupk_gemm_nn_workspace)         \
  X(soupk_token_logprobs_fwd) X(soupk_token_logprobs_bwd) X(soupk_token_logprobs_workspace)      \
  X(soupk_qk_norm_rope_fwd) X(soupk_qk_norm_rope_bwd) X(soupk_dropout) X(soupk_embedding_fwd)     \
  X(soupk_embedding_bwd) X(soupk_embedding_bwd_workspace) X(soupk_layer_fwd) X(soupk_layer_bwd)    \
  X(soupk_rotary_tables) X(soupk_rotary) X(soupk_rope_append) X(soupk_paged_attention)            \
  X(soupk_paged_attention_workspace) X(soupk_verify_drafts) X(soupk_verify_drafts_workspace)

#define X(name) inline decltype(&name) p_##name = nullptr;
SOUPK_ENTRIES(X)
#undef X

// The tensor behind a plain torch.Tensor or Parameter (no subclass: those keep the Python path).
inline const Tensor* plain(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// An optional tensor argument: false when it is something else than None or a plain tensor.
inline bool optional(PyObject* o, const Tensor*& t) {
  t = nullptr;
  if (o == Py_None) return true;
  t = plain(o);
  return t != nullptr;
}

inline bool is(const Tensor& t, at::ScalarType dt, int64_t dims, const at::Device& dev) {
  return t.scalar_type() == dt && t.dim() == dims && t.is_cuda() && t.device() == dev &&
         t.layout() == at::kStrided && t.is_contiguous();
}

inline bool shape2(const Tensor& t, int64_t r, int64_t c) { return t.size(0) == r && t.size(1) == c; }

inline void* ptr(const Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }
template <class T>
T* ptr(const Tensor* t) {
  return static_cast<T*>(ptr(t));
}
template <class T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

inline void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline Tensor empty(at::IntArrayRef size, at::ScalarType dt, const at::Device& dev) {
  return at::empty(size, at::TensorOptions().dtype(dt).device(dev));
}

inline PyObject* g_error = nullptr;        // testt_amd._ext.SoupkError
inline const char* (*p_status_string)(int) = nullptr;

// The GIL given up for a scope, taken back also when an exception leaves it: a tensor without a
// storage (a functorch wrapper, for one) throws from data_ptr, and HANDLE_TH_ERRORS sets the Python
// error from it.
class NoGil {
 public:
  NoGil() : state_(PyEval_SaveThread()) {}
  ~NoGil() { PyEval_RestoreThread(state_); }
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;

 private:
  PyThreadState* state_;
};

// The launch's status as the Python layer reports it; true when it succeeded.
template <class F>
bool launched(const char* name, F&& f) {
  const int rc = [&] {
    const NoGil released;
    return f();
  }();
  if (rc == 0) return true;
  const char* text = p_status_string ? p_status_string(rc) : nullptr;
  PyErr_Format(g_error ? g_error : PyExc_RuntimeError, "%s failed with status %d: %s", name, rc,
               text ? text : "?");
  return false;
}

inline PyObject* pack(std::initializer_list<Tensor> ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

}  // namespace soupk_host

#define OP(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)
#define ARGS(count) \
  if (n != (count)) return PyErr_Format(PyExc_TypeError, "%d arguments are expected", (count))
#define ELSE_PYTHON Py_RETURN_NONE
#define NUM(i) PyLong_AsLongLong(a[i])
