// What the sources of _d3d_host.so share.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>

#include "../../../include/deploy3d_b200.h"

extern PyObject* g_check;  // check(function name, status): raises

int dtype_of(const at::Tensor& t);  // d3d_dtype, or -1

extern PyMethodDef sequence_methods[];  // sequence.cpp; ends with an empty entry
