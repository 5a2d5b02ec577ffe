// what tensors.cpp (module vc3d._tensors) takes from autograd.cpp
#pragma once
#include <Python.h>

PyObject* vc_bind(PyObject*, PyObject* args);
PyObject* vc_gated_scan_py(PyObject*, PyObject* args);
PyObject* vc_gated_scan_step_py(PyObject*, PyObject* args);
PyObject* vc_linear_cross_entropy_py(PyObject*, PyObject* args);
