// What the Python entry points of the layer (binding.cpp) and of the operators around it (block.cpp) share.
#pragma once
#include <Python.h>

#include "layer.h"

#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/edge.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <memory>
#include <string>
#include <vector>

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

// Gradients of these gradients are not provided: where a node runs under create_graph, using a gradient that is a function of something that wants one has to fail, not
// to lose a term.  It is a function of the incoming gradients, and of the inputs whose bits depends[i] has.  The error has edges to all that it stands for: the engine only
// runs what leads to an argument that was asked for.
inline void refuse_second(const torch::autograd::Node& node, const std::string& what, const torch::autograd::variable_list& grads, const std::vector<uint32_t>& depends,
                          torch::autograd::variable_list& out) {
    if (!c10::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges;
    uint32_t want = 0;
    for (uint32_t j = 0; j < node.num_outputs(); ++j)
        if (node.next_edge(j).is_valid()) {
            want |= 1u << j;
            edges.push_back(node.next_edge(j));
        }
    bool up = false;
    for (const Tensor& g : grads)
        if (g.defined() && g.requires_grad()) {
            up = true;
            edges.push_back(torch::autograd::impl::gradient_edge(g));
        }
    const auto err = std::make_shared<torch::autograd::Error>(what + ": double backward is not supported", std::move(edges));
    for (size_t i = 0; i < out.size(); ++i)
        if (out[i].defined() && (up || (want & depends[i]))) torch::autograd::set_history(out[i], err);
}

extern PyMethodDef block_methods[];        // block.cpp

}  // namespace mkda_host
