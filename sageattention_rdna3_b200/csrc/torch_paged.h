// What torch_ops.cpp (the module `_C`) and torch_paged_ops.cpp share.
#pragma once

#include <Python.h>

#include <cstdint>

// The status word of a registered device and its mirror in pinned host memory (null if that is switched off); false if the
// device is not registered yet.
bool sage_device_status(int index, int** status, const volatile int32_t** mirror);

// Short ways into the operators around a growing cache (METH_FASTCALL): None where the call is not a plain one.
PyObject* sage_rotary_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* sage_paged_append_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* sage_paged_attn_plain(PyObject*, PyObject* const* args, Py_ssize_t nargs);
