// The operators whose autograd node is native too (host_autograd.cpp), as the extension's table lists
// them.
#pragma once

#include <Python.h>

namespace soupk_host {

PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n);

}  // namespace soupk_host
