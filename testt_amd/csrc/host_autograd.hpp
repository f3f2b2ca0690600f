// The operators around the layer (host_autograd.cpp, with native autograd nodes) and those of a generating
// program (host_generate.cpp), as the extension's table lists them.
#pragma once

#include <Python.h>

namespace soupk_host {

PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* rotary_tables(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n);

}  // namespace soupk_host
