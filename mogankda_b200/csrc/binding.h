// What the Python entry points of the layer (binding.cpp) and of the operators around it (block.cpp) share.
#pragma once
#include <Python.h>

#include "layer.h"

#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/mkda_block.h"

namespace mkda_host {

// An error of the library is a mogankda_b200._lib.MkdaError, in the forward call and out of the autograd engine.  Called without the GIL.
template <typename F>
auto library_call(F f) {
    try {
        return f();
    } catch (const LibraryError& e) {
        pybind11::gil_scoped_acquire gil;
        PyObject* mod = PyImport_ImportModule("mogankda_b200._lib");
        PyObject* type = mod ? PyObject_GetAttrString(mod, "MkdaError") : nullptr;
        if (type) PyErr_SetString(type, e.what());
        Py_XDECREF(type);
        Py_XDECREF(mod);
        python_error err;
        err.persist();
        throw err;
    }
}

inline PyObject* fail(PyObject* type, const std::string& msg) {
    PyErr_SetString(type, msg.c_str());
    return nullptr;
}
#define REQUIRE(cond, msg) do { if (!(cond)) return fail(PyExc_AssertionError, msg); } while (0)

inline bool tensor_arg(PyObject* o, Tensor& t) {
    if (o == Py_None) return true;
    if (!THPVariable_Check(o)) { PyErr_Format(PyExc_TypeError, "expected a tensor, got %s", Py_TYPE(o)->tp_name); return false; }
    t = THPVariable_Unpack(o);
    return true;
}
inline constexpr char NEED_CUDA[] = "mogankda_b200 kernels need CUDA tensors (there is no CPU fallback)";

extern PyMethodDef block_methods[];        // block.cpp

}  // namespace mkda_host
