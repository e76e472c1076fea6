// Functions of the extension module that host_layer.cpp holds.
#pragma once
#include <Python.h>

PyObject* py_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_check_leaves(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* py_bind_layer(PyObject*, PyObject* const* args, Py_ssize_t n);
