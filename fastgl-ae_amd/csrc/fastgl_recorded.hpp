// What the host halves of the recorded operators share (fastgl_autograd.cpp, fastgl_layers.cpp).
#pragma once

#include "fastgl_autograd.h"

#include <ATen/autocast_mode.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <string>
#include <tuple>

#include "fastgl_hip.h"

namespace fastgl {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = c10::optional<Tensor>;

inline void ok(int rc) { TORCH_CHECK(rc == FGL_OK, "fastgl: ", fgl_last_error(), " (error ", rc, ")"); }

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

inline int type_of(const Tensor& t) { return t.scalar_type() == torch::kFloat32 ? FGL_F32 : FGL_BF16; }

inline bool is_feature(const Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16; }

// Scratch of the call's own, from torch's allocator (in stream order, also under capture)
inline Tensor bytes_like(const Tensor& t, size_t n)
{
    return torch::empty({(int64_t)(n < 256 ? 256 : n)}, t.options().dtype(torch::kUInt8).requires_grad(false));
}

inline void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Whether t only looks like a tensor of its sizes and has no memory of its own: a gradient that torch.autograd.grad(is_grads_batched=True) and
// jacobian(vectorize=True) hand to a backward pass, many at once
inline bool is_wrapped(const Tensor& t)
{
    return t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper}));
}

// In a backward pass: where a graph of the gradients is being built, and they have none, who asks for them is told so.  By a node that leads on to what
// they would be of, so that it is met also where only some tensor's gradients are asked for.  `like`: a plain tensor of the gradients' type.
inline void refuse_gradients_of(std::initializer_list<Tensor*> made, const Tensor& grad, const at::TensorOptions& like, const char* message)
{
    if (!torch::GradMode::is_enabled()) return;
    torch::autograd::edge_list of;
    for (const auto& edge : torch::autograd::get_current_node()->next_edges())
        if (edge.is_valid()) of.push_back(edge);
    const bool wrapped = is_wrapped(grad);
    if (!wrapped && grad.requires_grad()) of.push_back(torch::autograd::impl::gradient_edge(grad));
    const auto node = std::make_shared<torch::autograd::Error>(message, std::move(of));
    Tensor zero;  // wrapped tensors get no node: one is added that has it
    if (wrapped) {
        zero = torch::full({}, -0.0, like);
        torch::autograd::set_history(zero, node);
    }
    for (Tensor* t : made) {
        if (!t->defined()) continue;
        if (wrapped) *t = *t + zero;
        else torch::autograd::set_history(*t, node);
    }
}

}  // namespace fastgl
