// What the operators' host side in C++ shares: which tensors and calls it takes, and small parts of autograd nodes.
#pragma once
#include <torch/extension.h>
#include <torch/version.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include "../../../include/vrwkv_hip.h"


namespace host {
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using torch::autograd::Variable;

inline int code(at::ScalarType t) { return t == at::kFloat ? VRWKV_F32 : t == at::kBFloat16 ? VRWKV_BF16 : t == at::kHalf ? VRWKV_F16 : -1; }

inline void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;

// Tracing, functorch levels, dispatch and function modes are to see the operators' Python classes.
inline bool transformed() {
    return torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
           at::impl::PythonTorchFunctionTLS::stack_len() > 0;
}

// Forward-mode tangents are refused by the Python classes.
inline bool tangent(const at::Tensor& t) { return t._fw_grad(0).defined(); }

inline at::Tensor bytes(size_t n, const at::Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)); }

// An exact Tensor or Parameter on a GPU whose memory the kernels may read at its strides, channels side by side (`t` outlives the call: the caller holds it).
inline const at::Tensor* strided(py::handle o) {
    if (!THPVariable_CheckExact(o.ptr())) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o.ptr());
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg()) return nullptr;
    const auto keys = t.key_set();
    if (keys.has(c10::DispatchKey::FuncTorchBatched) || keys.has(c10::DispatchKey::Batched) || keys.has(c10::DispatchKey::Python) ||
        keys.has(c10::DispatchKey::FuncTorchGradWrapper) || keys.has(c10::DispatchKey::Functionalize))
        return nullptr;
    return &t;
}
inline bool index_fits(const at::Tensor& t, const at::Tensor& q) {
    return t.dim() == 1 && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.is_contiguous() && t.numel() > 0 && t.device() == q.device();
}

inline bool pages_fit(const at::Tensor& pool) {
    int64_t want = 1;
    for (int64_t i = pool.dim() - 1; i > 0; --i) {
        if (pool.size(i) != 1 && pool.stride(i) != want) return false;
        want *= pool.size(i);
    }
    return pool.size(0) == 1 || pool.stride(0) >= want;
}

// create_graph: differentiating these gradients once more raises
inline void only_once(tensor_list& out) {
    tensor_list some;
    for (auto& t : out)
        if (t.defined()) some.push_back(t.detach().set_requires_grad(true));
    const auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)some.size());
    some = (*error)(std::move(some));
    size_t i = 0;
    for (auto& t : out)
        if (t.defined()) t = some[i++];
}

inline py::object wrapped(const at::Tensor& t) { return t.defined() ? py::reinterpret_steal<py::object>(THPVariable_Wrap(t)) : py::none(); }
}  // namespace host
