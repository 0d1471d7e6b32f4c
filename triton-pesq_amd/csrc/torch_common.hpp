// What the translation units of the PyTorch extension module share.
#pragma once

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>

#include "pesq_hip.h"

// Adds the operators of torch_network.cpp to the module.
void bind_network(pybind11::module_ &m);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[maybe_unused]] inline void check(int status, const char *what) {
    if (status != PESQ_OK) {
        throw std::runtime_error(std::string(what) + ": " + pesq_last_error() + " (status " +
                                 std::to_string(status) + ")");
    }
}

[[maybe_unused]] inline hipStream_t current_stream(const at::Tensor &t) {
    return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

template <class T>
T *data_or_null(const at::Tensor &t) {
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

// Identity whose derivative raises: attached to the gradients when a double
// backward would need the derivative of the pipeline's backward, as Python's
// @once_differentiable does.
struct OnceDifferentiable : public torch::autograd::Function<OnceDifferentiable> {
    static at::Tensor forward(AutogradContext *, const at::Tensor &x) { return x.clone(); }
    static variable_list backward(AutogradContext *, variable_list) {
        throw std::runtime_error(
            "trying to differentiate twice a function that was marked with @once_differentiable");
    }
};

}  // namespace
