// The operators of tensorcalls.cpp as methods of the module that pycalls.cpp makes (built where torch's headers are).
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

extern PyMethodDef spd_tensor_methods[];
// takes the addresses that it calls from {name: (address, ctypes function)}
void spd_tensor_bind(PyObject* functions);
