// calls.hpp -- what the operators' host sides on torch tensors share.
#pragma once

#include <c10/hip/HIPStream.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <stdexcept>

#include "neural_shift_hip.h"

namespace nsh_calls {


using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

template <typename T = void>
T* address(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
inline Tensor given(const Maybe& t) { return t ? *t : Tensor(); }

inline void strides(int64_t (&to)[3], const Tensor& t) {
    for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

inline int32_t code(const Tensor& t, const char* op) {
    switch (t.scalar_type()) {
        case at::kHalf: return NSH_DTYPE_FLOAT16;
        case at::kBFloat16: return NSH_DTYPE_BFLOAT16;
        case at::kFloat: return NSH_DTYPE_FLOAT32;
        default:
            throw std::runtime_error(std::string("\"") + op + "\" not implemented for '" +
                                     c10::toString(t.scalar_type()) + "'");
    }
}

inline void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

inline void done(int rc) {
    if (rc != NSH_OK) throw std::runtime_error(nsh_last_error());
}

inline Tensor scratch(const Tensor& t, int64_t bytes) {
    return bytes > 0 ? at::empty({bytes}, t.options().dtype(at::kByte)) : Tensor();
}

// Gradients of gradients are refused where they are asked for.
inline variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a token operator, whose gradients are not differentiable",
        static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

// A tangent would be dropped without a word: what the kernels write has none.
inline void no_tangents(const char* op, std::initializer_list<const Tensor*> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), op,
                                    ": forward-mode derivatives are not implemented");
}

inline bool graph(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ---------------------------------------------------------------------------
// What calls that need no conversion are looked over for
// ---------------------------------------------------------------------------

// In memory with its own sign (the imaginary part of a conjugate, say, is not).
inline bool as_it_lies(const Tensor& t) { return !t.is_neg(); }

inline bool served(const Tensor& t) {
    const auto type = t.scalar_type();
    return (type == at::kHalf || type == at::kBFloat16 || type == at::kFloat) && as_it_lies(t);
}

inline bool alike(const Tensor& t, const Tensor& q) {
    return t.scalar_type() == q.scalar_type() && t.device() == q.device() && as_it_lies(t);
}

// Not given, or contiguous in `type` and of this shape.
inline bool plain(const Maybe& t, const Tensor& q, at::ScalarType type, at::IntArrayRef shape) {
    return !t || (t->scalar_type() == type && t->device() == q.device() && t->sizes() == shape && t->is_contiguous() &&
                  as_it_lies(*t));
}

}  // namespace nsh_calls
