// Host half of the operators that are recorded for a backward pass (fastgl/dropouts.py, fastgl/losses.py): their checks, outputs
// and autograd nodes.
//
// A training step calls them once a layer, on rows that take the GPU tens of microseconds; recorded by a Python function, forward and
// backward cost 90 us (dropout) and 130 us (the loss) of the host's time, here 46 and 73, on a host where torch's relu takes 42 (27, 45 and 24 on
// a faster one).
#include "fastgl_autograd.h"

#include <ATen/autocast_mode.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <string>
#include <tuple>

#include "fastgl_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = c10::optional<Tensor>;

void ok(int rc) { TORCH_CHECK(rc == FGL_OK, "fastgl: ", fgl_last_error(), " (error ", rc, ")"); }

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int type_of(const Tensor& t) { return t.scalar_type() == torch::kFloat32 ? FGL_F32 : FGL_BF16; }

bool is_feature(const Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16; }

// Scratch of the call's own, from torch's allocator (in stream order, also under capture)
Tensor bytes_like(const Tensor& t, size_t n)
{
    return torch::empty({(int64_t)(n < 256 ? 256 : n)}, t.options().dtype(torch::kUInt8).requires_grad(false));
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// Whether t only looks like a tensor of its sizes and has no memory of its own: a gradient that torch.autograd.grad(is_grads_batched=True) and
// jacobian(vectorize=True) hand to a backward pass, many at once
bool is_wrapped(const Tensor& t)
{
    return t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper}));
}

// ---- dropout -------------------------------------------------------------------------------------------------------
bool gaps_in_rows_only(const Tensor& x) { return x.is_contiguous() || (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= x.size(1)); }

Tensor drop(const Tensor& x, double p, uint64_t seed, uint32_t stream, bool relu, const Tensor& offset)
{
    c10::hip::HIPGuard guard(x.get_device());
    Tensor out = torch::empty(x.sizes(), x.options().requires_grad(false));
    if (out.numel() == 0) return out;
    const bool whole = x.is_contiguous();
    ok(fgl_dropout(x.data_ptr(), whole ? x.numel() : x.stride(0), whole ? 1 : x.size(0), whole ? x.numel() : x.size(1), type_of(x), p, seed, stream,
                   static_cast<const int32_t*>(address(offset)), relu, out.data_ptr(), stream_of(x)));
    return out;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, uint64_t seed, uint32_t stream, bool relu, const Maybe& offset)
    {
        Tensor out = drop(x, p, seed, stream, relu, offset.value_or(Tensor()));
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = (int64_t)seed;
        ctx->saved_data["stream"] = (int64_t)stream;
        ctx->saved_data["relu"] = relu;
        // (the mask is made again from the same offset: one that was changed meanwhile is an error)
        ctx->save_for_backward({relu ? out : Tensor(), offset.value_or(Tensor())});
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        Tensor d_out = grads[0];
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &out = saved[0], &offset = saved[1];
        const double p = ctx->saved_data["p"].toDouble();
        const uint64_t seed = (uint64_t)ctx->saved_data["seed"].toInt();
        const uint32_t stream = (uint32_t)ctx->saved_data["stream"].toInt();
        Tensor d_x;
        if (!d_out.defined()) return {d_x, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        const bool recorded = torch::GradMode::is_enabled();  // (a graph of the gradients is being built; they are linear in d_out)
        const bool wrapped = is_wrapped(d_out);
        const double scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
        if (ctx->saved_data["relu"].toBool()) {
            if (recorded || wrapped) {
                d_x = torch::where(out <= 0, torch::zeros({}, d_out.options()), d_out * scale);
            } else {
                c10::hip::HIPGuard guard(out.get_device());
                d_out = d_out.contiguous();
                d_x = torch::empty(out.sizes(), out.options().requires_grad(false));
                if (d_x.numel() > 0)
                    ok(fgl_dropout_relu_backward(d_out.data_ptr(), out.data_ptr(), out.numel(), type_of(out), p, d_x.data_ptr(), stream_of(out)));
            }
        } else if (wrapped) {
            const auto like = at::TensorOptions().dtype(d_out.scalar_type()).device(d_out.device());
            const Tensor kept = drop(torch::ones(d_out.sizes(), like), p, seed, stream, false, offset);
            d_x = torch::where(kept == 0, torch::zeros({}, like), d_out * scale);
        } else {
            if (!gaps_in_rows_only(d_out)) d_out = d_out.contiguous();
            if (recorded) d_x = DropoutNode::apply(d_out, p, seed, stream, false, offset.defined() ? Maybe(offset) : Maybe());
            else d_x = drop(d_out, p, seed, stream, false, offset);
        }
        return {d_x, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, uint32_t stream, bool relu, const Maybe& offset)
{
    TORCH_CHECK(is_feature(x), "x must have dtype in ['torch.float32', 'torch.bfloat16'], got ", x.scalar_type());
    TORCH_CHECK(gaps_in_rows_only(x), "x must be contiguous, or a matrix with unit column stride");
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "p (", p, ") is no probability");
    if (offset.has_value()) {
        TORCH_CHECK(offset->scalar_type() == torch::kInt32 && offset->numel() == 1, "stream_offset must hold one int32");
        TORCH_CHECK(offset->device() == x.device(), "all tensors must live on the same device");
    }
    if (!(torch::GradMode::is_enabled() && x.requires_grad())) return drop(x, p, seed, stream, relu, offset.value_or(Tensor()));
    return DropoutNode::apply(x, p, seed, stream, relu, offset);
}

// ---- the loss of a last layer --------------------------------------------------------------------------------------
struct LossSizes {
    int64_t n, classes;
    int dim, dtype, reduction, want;
};

Tensor no_rows_loss(const Tensor& x, int reduction)
{
    const auto of = x.options().dtype(torch::kFloat32).requires_grad(false);
    if (reduction == FGL_REDUCE_NONE) return torch::empty({0}, of);
    return torch::full({}, reduction == FGL_REDUCE_MEAN ? std::numeric_limits<double>::quiet_NaN() : 0.0, of);
}

// (loss, state)
std::tuple<Tensor, Tensor> form_loss(const Tensor& x, const Tensor& w, const Maybe& bias, const Tensor& labels, int64_t ignore, const LossSizes& z)
{
    c10::hip::HIPGuard guard(x.get_device());
    Tensor state = bytes_like(x, fgl_linear_cross_entropy_state_bytes(z.n, z.classes, z.dim, z.dtype, z.want));
    if (z.n == 0) return {no_rows_loss(x, z.reduction), state};
    const auto of = x.options().dtype(torch::kFloat32).requires_grad(false);
    Tensor loss = z.reduction == FGL_REDUCE_NONE ? torch::empty({z.n}, of) : torch::empty({}, of);
    Tensor ws = bytes_like(x, fgl_linear_cross_entropy_workspace_bytes(z.n, z.classes, z.dim, z.dtype, z.want, 0));
    ok(fgl_linear_cross_entropy(x.data_ptr(), x.stride(0), x.stride(1), w.data_ptr(), w.stride(0), w.stride(1), bias.has_value() ? bias->data_ptr() : nullptr,
                                labels.data_ptr(), labels.scalar_type() == torch::kInt64, ignore, z.n, z.classes, z.dim, z.dtype, z.reduction, z.want,
                                loss.data_ptr<float>(), state.data_ptr(), (size_t)state.numel(), ws.data_ptr(), (size_t)ws.numel(), stream_of(x)));
    return {loss, state};
}

// What the forward pass left in `state` -> the gradients that are asked for
std::tuple<Tensor, Tensor, Tensor> loss_gradients(const Tensor& d_loss_of, const Tensor& state, int64_t n, int64_t classes, int64_t dim, int64_t reduction, int64_t want,
                                                  at::ScalarType type, bool need_x, bool need_w, bool need_b)
{
    torch::NoGradGuard no_grad;
    c10::hip::HIPGuard guard(state.get_device());
    const auto of = state.options().dtype(type);
    const int dtype = type == torch::kFloat32 ? FGL_F32 : FGL_BF16;
    auto make = [&](at::IntArrayRef size) { return n > 0 ? torch::empty(size, of) : torch::zeros(size, of); };
    Tensor d_x, d_w, d_b;
    if (need_x) d_x = make({n, dim});
    if (need_w || need_b) d_w = make({classes, dim});
    if (need_b) d_b = make({classes});
    if (n > 0 && (need_x || need_w || need_b)) {
        const Tensor d_loss = d_loss_of.contiguous();
        const size_t ws_bytes = fgl_linear_cross_entropy_workspace_bytes(n, classes, (int)dim, dtype, (int)want, 1);
        Tensor ws;
        if (ws_bytes > 0) ws = bytes_like(state, ws_bytes);
        ok(fgl_linear_cross_entropy_backward(d_loss.data_ptr<float>(), n, classes, (int)dim, dtype, (int)reduction, (int)want, state.data_ptr(), (size_t)state.numel(),
                                             address(d_x), address(d_w), address(d_b), address(ws), ws_bytes, stream_of(state)));
    }
    return {d_x, need_w ? d_w : Tensor(), d_b};
}

// The same as an operator of torch's, whose loop takes gradients of the loss that are many at once apart; it wants a tensor in each place.
std::tuple<Tensor, Tensor, Tensor> loss_gradients_operator(const Tensor& d_loss, const Tensor& state, int64_t n, int64_t classes, int64_t dim, int64_t reduction, int64_t want,
                                                           at::ScalarType type, bool need_x, bool need_w, bool need_b)
{
    auto made = loss_gradients(d_loss, state, n, classes, dim, reduction, want, type, need_x, need_w, need_b);
    const auto some = [&](const Tensor& t) { return t.defined() ? t : torch::empty({0}, state.options().dtype(type)); };
    return {some(std::get<0>(made)), some(std::get<1>(made)), some(std::get<2>(made))};
}

TORCH_LIBRARY_FRAGMENT(fastgl, m)
{
    m.def("linear_cross_entropy_gradients(Tensor d_loss, Tensor state, int n, int classes, int dim, int reduction, int want, ScalarType type, bool need_x, bool need_w, "
          "bool need_b) -> (Tensor, Tensor, Tensor)",
          torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, TORCH_FN(loss_gradients_operator)));
}

struct LossNode : torch::autograd::Function<LossNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias, const Tensor& labels, int64_t ignore, LossSizes z)
    {
        auto [loss, state] = form_loss(x, w, bias, labels, ignore, z);
        ctx->saved_data["n"] = z.n;
        ctx->saved_data["classes"] = z.classes;
        ctx->saved_data["dim"] = (int64_t)z.dim;
        ctx->saved_data["reduction"] = (int64_t)z.reduction;
        ctx->saved_data["want"] = (int64_t)z.want;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["type"] = x.scalar_type();
        ctx->save_for_backward({state});  // (no tensor of the caller's: nothing of it can be changed in between)
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const Tensor state = ctx->get_saved_variables()[0];
        const bool with_bias = ctx->saved_data["bias"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = with_bias && ctx->needs_input_grad(2);
        const auto sizes = [&](const char* name) { return ctx->saved_data[name].toInt(); };
        const auto form = [&](auto&& gradients) {
            return gradients(grads[0], state, sizes("n"), sizes("classes"), sizes("dim"), sizes("reduction"), sizes("want"), ctx->saved_data["type"].toScalarType(), need_x,
                             need_w, need_b);
        };
        Tensor d_x, d_w, d_b;
        if (is_wrapped(grads[0])) {
            static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fastgl::linear_cross_entropy_gradients", "").typed<decltype(loss_gradients)>();
            std::tie(d_x, d_w, d_b) = form([](auto&&... a) { return op.call(a...); });
            if (!need_x) d_x = Tensor();
            if (!need_w) d_w = Tensor();
            if (!need_b) d_b = Tensor();
        } else {
            std::tie(d_x, d_w, d_b) = form(loss_gradients);
        }
        if (torch::GradMode::is_enabled()) {
            // A graph of the gradients is being built, and they have none: who asks for them is told so.  By a node that leads on to what they would be of, so
            // that it is met also where only some tensor's gradients are asked for.
            torch::autograd::edge_list of;
            for (const auto& edge : torch::autograd::get_current_node()->next_edges())
                if (edge.is_valid()) of.push_back(edge);
            const bool wrapped = is_wrapped(grads[0]);
            if (!wrapped && grads[0].requires_grad()) of.push_back(torch::autograd::impl::gradient_edge(grads[0]));
            const auto node = std::make_shared<torch::autograd::Error>("linear_cross_entropy has no gradients of its gradients", std::move(of));
            Tensor zero;  // wrapped tensors get no node: one is added that has it
            if (wrapped) {
                zero = torch::full({}, -0.0, state.options().dtype(ctx->saved_data["type"].toScalarType()));
                torch::autograd::set_history(zero, node);
            }
            for (Tensor* t : {&d_x, &d_w, &d_b}) {
                if (!t->defined()) continue;
                if (wrapped) *t = *t + zero;
                else torch::autograd::set_history(*t, node);
            }
        }
        out[0] = d_x;
        out[1] = d_w;
        out[2] = d_b;
        return out;
    }
};

Tensor linear_cross_entropy(Tensor x, Tensor w, const Tensor& labels, Maybe bias, int64_t ignore, int reduction, int64_t max_dim)
{
    if (at::autocast::is_autocast_enabled(at::kCUDA)) {
        const auto to = at::autocast::get_autocast_dtype(at::kCUDA);
        x = x.to(to);
        w = w.to(to);
        if (bias.has_value()) bias = bias->to(to);
    }
    TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && w.size(0) >= 1 && x.size(1) >= 1 && x.size(1) <= max_dim, "x ", x.sizes(), " and weight ",
                w.sizes(), " must be [n, d] and [classes, d] with 1 <= d <= ", max_dim);
    TORCH_CHECK(is_feature(x) && w.scalar_type() == x.scalar_type() && (!bias.has_value() || bias->scalar_type() == x.scalar_type()),
                "x, weight and bias must all be of one type in ['torch.float32', 'torch.bfloat16']");
    TORCH_CHECK(!bias.has_value() || (bias->dim() == 1 && bias->size(0) == w.size(0) && bias->is_contiguous()), "bias must be contiguous and hold a value for each class");
    TORCH_CHECK(labels.dim() == 1 && labels.size(0) == x.size(0) && (labels.scalar_type() == torch::kInt64 || labels.scalar_type() == torch::kInt32) && labels.is_contiguous(),
                "labels must be contiguous int32 or int64, one for each row of x");
    TORCH_CHECK(w.device() == x.device() && labels.device() == x.device() && (!bias.has_value() || bias->device() == x.device()),
                "all tensors must live on the same device");
    LossSizes z{x.size(0), w.size(0), (int)x.size(1), type_of(x), reduction, 0};
    if (torch::GradMode::is_enabled())
        z.want = (x.requires_grad() ? FGL_XENT_ROWS : 0) | (w.requires_grad() || (bias.has_value() && bias->requires_grad()) ? FGL_XENT_WEIGHTS : 0);
    if (z.want == 0) return std::get<0>(form_loss(x, w, bias, labels, ignore, z));
    return LossNode::apply(x, w, bias, labels, ignore, z);
}

}  // namespace

void bind_recorded_operators(py::module& m)
{
    m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
    m.def("linear_cross_entropy", &linear_cross_entropy, py::call_guard<py::gil_scoped_release>());
}
