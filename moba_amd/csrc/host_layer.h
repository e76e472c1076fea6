// Functions of the extension module that host_layer.cpp and host_serving.cpp hold.
#pragma once
#include <Python.h>

PyObject* py_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_check_leaves(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_bind_layer(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_block_attention(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_key_sums(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_select_blocks(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_reserve(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_release(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_bind_serving(PyObject*, PyObject* const* args, Py_ssize_t n);
