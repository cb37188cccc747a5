// Shared by the translation units of _native.so: which tensors the native calls take, and what they allocate.
#pragma once

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>

#include "../../include/wkv6_b200.h"

namespace wkv6_native {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The losses and the optimizer step (wkv6_torch_training.cpp): their entry points from the loaded library (the name of one that it
// lacks, or nullptr), and their rows of the module's method table.
const char *bind_training(void *library);
PyObject *py_token_log_probs(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *py_policy_loss(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *py_preference_loss(PyObject *, PyObject *const *args, Py_ssize_t n);
PyObject *py_adamw_step(PyObject *, PyObject *const *args, Py_ssize_t n);

inline int dtype_code(at::ScalarType t) {
    switch (t) {
        case at::kBFloat16: return WKV6_BF16;
        case at::kHalf: return WKV6_F16;
        case at::kFloat: return WKV6_F32;
        default: return -1;
    }
}

// No tracing, no dispatch or function mode: a call is what it says.
inline bool plain_mode() {
    return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() &&
           !torch::jit::tracer::isTracing();
}

// A strided CUDA tensor that is what its memory holds: not wrapped by a transform, no lazy negation.
inline bool plain_storage(const Tensor &t) {
    constexpr c10::DispatchKeySet odd({c10::DispatchKey::Python, c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched,
                                       c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                       c10::DispatchKey::Conjugate, c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
    return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && (t.key_set() & odd).empty();
}

// ... and of the exact class Tensor (or Parameter).
inline bool plain_tensor(PyObject *o) { return THPVariable_CheckExact(o) && plain_storage(THPVariable_Unpack(o)); }

inline Tensor bytes(size_t n, const Tensor &r) { return at::detail::empty_cuda({(int64_t)n}, at::kByte, r.device(), std::nullopt); }

inline void *stream_of(const Tensor &r) { return c10::cuda::getCurrentCUDAStream(r.device().index()).stream(); }

inline PyObject *none() { Py_RETURN_NONE; }

}  // namespace wkv6_native
