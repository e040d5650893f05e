// What the native sides of paperkiln_amd.ops and paperkiln_amd.blockops on torch tensors share: arguments as Python passes them (by position),
// refusals as Python exceptions, the current stream.
#pragma once
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/python_numbers.h>

#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "paperkiln_amd.h"

namespace pk_torch {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline PyObject* g_error = nullptr;  // paperkiln_amd._lib.PkError

// A refused C ABI call as the package's own exception, on any thread (the autograd engine's included).
inline void check(int rc) {
    if (rc == PK_OK) return;
    const std::string msg = pk_last_error();
    pybind11::gil_scoped_acquire gil;
    if (PyObject* e = PyObject_CallFunction(g_error, "is", rc, msg.c_str())) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw python_error();
}

inline int dtype_code(at::ScalarType t) {
    if (t == at::kFloat) return PK_F32;
    if (t == at::kBFloat16) return PK_BF16;
    throw std::runtime_error("dtype must be float32 or bfloat16");
}

inline void* stream() { return at::hip::getCurrentHIPStream().stream(); }

inline Tensor empty_of(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) {
    return at::empty(sizes, like.options().dtype(t).memory_format(c10::nullopt));
}

inline const Tensor& tensor_arg(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) throw torch::TypeError(std::string(what) + " must be a tensor, not " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
inline int int_arg(PyObject* o) {  // what Python's int() takes, inside 32 bits
    PyObject* i = PyNumber_Long(o);
    if (!i) throw python_error();
    const long x = PyLong_AsLong(i);
    Py_DECREF(i);
    if (x == -1 && PyErr_Occurred()) throw python_error();
    return static_cast<int>(x);
}
inline double float_arg(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw python_error();
    return x;
}
inline bool bool_arg(PyObject* o) {
    const int x = PyObject_IsTrue(o);
    if (x < 0) throw python_error();
    return x != 0;
}
inline void expect(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) throw torch::TypeError("expected " + std::to_string(want) + " arguments, got " + std::to_string(n));
}

PyMethodDef* post_methods();  // post_ops.cpp

}  // namespace pk_torch
