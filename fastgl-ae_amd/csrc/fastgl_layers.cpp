// Host half of the operators between the aggregations (fastgl/layers.py): their checks, outputs and autograd nodes, as fastgl_autograd.cpp
// has them for dropout and the loss.
#include "fastgl_recorded.hpp"

namespace {

using namespace fastgl;

// The rows of x, any number of leading dimensions, as a matrix whose rows are whole: x itself, a view, or a copy.  `even`: rows start on four bytes.
Tensor as_rows(const Tensor& x, bool even)
{
    const int64_t d = x.size(-1);
    Tensor m = x.dim() == 2 ? x : x.reshape({-1, d});
    if (m.size(0) == 0 || d == 0) return m;
    if ((d > 1 && m.stride(1) != 1) || (m.size(0) > 1 && (m.stride(0) < d || m.stride(0) >= 1 << 24))) m = m.contiguous();
    if (even && ((m.size(0) > 1 && m.stride(0) % 2 != 0) || (reinterpret_cast<uintptr_t>(m.data_ptr()) & 3) != 0)) {
        Tensor wider = torch::empty({m.size(0), (d + 1) / 2 * 2}, m.options().requires_grad(false));
        Tensor copy = wider.narrow(1, 0, d);
        copy.copy_(m);
        m = copy;
    }
    return m;
}

int64_t row_stride(const Tensor& m, int64_t d) { return m.size(0) > 1 ? m.stride(0) : (d + 1) / 2 * 2; }

Tensor like_rows(const Tensor& x, int64_t columns)
{
    auto size = x.sizes().vec();
    size.back() = columns;
    return torch::empty(size, x.options().requires_grad(false).memory_format(c10::MemoryFormat::Contiguous));
}

// ---- norm of the rows ----------------------------------------------------------------------------------------------
// (y, state)
std::tuple<Tensor, Tensor> form_norm(const Tensor& x, const Tensor& rows, const Tensor& w, const Tensor& b, double eps, bool relu, bool keep8, bool keep)
{
    c10::hip::HIPGuard guard(x.get_device());
    const int64_t d = x.size(-1), n = rows.size(0);
    Tensor y = like_rows(x, d), state;
    if (keep) state = bytes_like(x, fgl_layer_norm_state_bytes(n, (int)d, relu, keep8));
    ok(fgl_layer_norm(rows.data_ptr(), row_stride(rows, d), address(w), address(b), n, (int)d, type_of(x), eps, relu, keep8, y.data_ptr(), address(state),
                      keep ? (size_t)state.numel() : 0, stream_of(x)));
    return {y, state};
}

std::tuple<Tensor, Tensor, Tensor> norm_gradients(const Tensor& d_y, const Tensor& rows, const Tensor& w, const Tensor& state, bool relu, bool keep8, bool need_x,
                                                  bool need_w, bool need_b)
{
    torch::NoGradGuard no_grad;
    c10::hip::HIPGuard guard(state.get_device());
    const int64_t d = d_y.size(-1);
    const auto of = d_y.options().requires_grad(false);
    const Tensor g = as_rows(d_y, false);
    const int64_t n = g.size(0);
    Tensor d_x, d_w, d_b;
    if (need_x) d_x = torch::empty(d_y.sizes(), of.memory_format(c10::MemoryFormat::Contiguous));
    auto sums = [&] { return n > 0 ? torch::empty({d}, of) : torch::zeros({d}, of); };
    if (need_w) d_w = sums();
    if (need_b) d_b = sums();
    if (n > 0 && (need_x || need_w || need_b)) {
        const size_t ws_bytes = need_w || need_b ? fgl_layer_norm_workspace_bytes(n, (int)d, type_of(g)) : 0;
        Tensor ws;
        if (ws_bytes > 0) ws = bytes_like(state, ws_bytes);
        ok(fgl_layer_norm_backward(g.data_ptr(), row_stride(g, d), keep8 ? nullptr : rows.data_ptr(), keep8 ? d : row_stride(rows, d), address(w), n, (int)d, type_of(g),
                                   relu, keep8, state.data_ptr(), (size_t)state.numel(), address(d_x), address(d_w), address(d_b), address(ws), ws_bytes,
                                   stream_of(state)));
    }
    return {d_x, d_w, d_b};
}

// The same as an operator of torch's, whose loop takes gradients that are many at once apart; it wants a tensor in each place.
std::tuple<Tensor, Tensor, Tensor> norm_gradients_operator(const Tensor& d_y, const Maybe& rows, const Maybe& w, const Tensor& state, bool relu, bool keep8, bool need_x,
                                                           bool need_w, bool need_b)
{
    auto made = norm_gradients(d_y, rows.value_or(Tensor()), w.value_or(Tensor()), state, relu, keep8, need_x, need_w, need_b);
    const auto some = [&](const Tensor& t) { return t.defined() ? t : torch::empty({0}, d_y.options()); };
    return {some(std::get<0>(made)), some(std::get<1>(made)), some(std::get<2>(made))};
}

TORCH_LIBRARY_FRAGMENT(fastgl, m)
{
    m.def("layer_norm_gradients(Tensor d_y, Tensor? rows, Tensor? weight, Tensor state, bool relu, bool keep8, bool need_x, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)",
          torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, TORCH_FN(norm_gradients_operator)));
}

Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

struct NormNode : torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& w, const Maybe& b, double eps, bool relu, bool keep8)
    {
        const Tensor rows = as_rows(x, false);
        auto [y, state] = form_norm(x, rows, w.value_or(Tensor()), b.value_or(Tensor()), eps, relu, keep8, true);
        ctx->saved_data["relu"] = relu;
        ctx->saved_data["keep8"] = keep8;
        ctx->saved_data["weight"] = w.has_value();
        ctx->saved_data["bias"] = b.has_value();
        ctx->save_for_backward({keep8 ? Tensor() : x, w.value_or(Tensor()), state});
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(6);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &state = saved[2];
        const bool relu = ctx->saved_data["relu"].toBool(), keep8 = ctx->saved_data["keep8"].toBool();
        // (inputs that were not given are not counted)
        const bool with_w = ctx->saved_data["weight"].toBool(), with_b = ctx->saved_data["bias"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = with_w && ctx->needs_input_grad(1), need_b = with_b && ctx->needs_input_grad(with_w ? 2 : 1);
        Tensor rows;
        if (!keep8) {
            torch::NoGradGuard no_grad;
            rows = as_rows(x, false);
        }
        Tensor d_x, d_w, d_b;
        if (is_wrapped(grads[0])) {
            static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fastgl::layer_norm_gradients", "").typed<decltype(norm_gradients_operator)>();
            std::tie(d_x, d_w, d_b) = op.call(grads[0], maybe(rows), maybe(w), state, relu, keep8, need_x, need_w, need_b);
            if (!need_x) d_x = Tensor();
            if (!need_w) d_w = Tensor();
            if (!need_b) d_b = Tensor();
        } else {
            std::tie(d_x, d_w, d_b) = norm_gradients(grads[0], rows, w, state, relu, keep8, need_x, need_w, need_b);
        }
        refuse_gradients_of({&d_x, &d_w, &d_b}, grads[0], state.options().dtype(grads[0].scalar_type()), "layer_norm has no gradients of its gradients");
        out[0] = d_x;
        out[1] = d_w;
        out[2] = d_b;
        return out;
    }
};

bool records(const Tensor& t) { return t.requires_grad(); }
bool records(const Maybe& t) { return t.has_value() && t->requires_grad(); }

Tensor layer_norm(Tensor x, Maybe w, Maybe b, double eps, bool relu, bool keep8, int64_t most_columns)
{
    if (at::autocast::is_autocast_enabled(at::kCUDA)) {  // (as torch's, which takes fp32 there)
        x = x.to(torch::kFloat32);
        if (w.has_value()) w = w->to(torch::kFloat32);
        if (b.has_value()) b = b->to(torch::kFloat32);
    }
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= most_columns, "x ", x.sizes(), " must have rows of 1 to ", most_columns, " columns");
    TORCH_CHECK(is_feature(x), "x must have dtype in ['torch.float32', 'torch.bfloat16'], got ", x.scalar_type());
    for (Maybe* t : {&w, &b}) {
        if (!t->has_value()) continue;
        TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == x.size(-1) && (*t)->scalar_type() == x.scalar_type(), "weight and bias must hold a value of x's type for each column");
        TORCH_CHECK((*t)->device() == x.device(), "all tensors must live on the same device");
        *t = (*t)->contiguous();
    }
    TORCH_CHECK(eps >= 0.0 && eps < 1e300, "eps (", eps, ") must not be negative");
    if (!(torch::GradMode::is_enabled() && (records(x) || records(w) || records(b)))) {
        const Tensor rows = as_rows(x, false);
        return std::get<0>(form_norm(x, rows, w.value_or(Tensor()), b.value_or(Tensor()), eps, relu, false, false));
    }
    return NormNode::apply(x, w, b, eps, relu, keep8);
}

// ---- dense layer ---------------------------------------------------------------------------------------------------
struct LinearSizes {
    int64_t n;
    int dim, out, dtype, act;
    bool keep8;
};

// (y, state)
std::tuple<Tensor, Tensor> form_linear(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, const LinearSizes& z, bool keep)
{
    c10::hip::HIPGuard guard(x.get_device());
    const bool even = z.dtype == FGL_BF16;
    const Tensor rows = as_rows(x, even), weights = as_rows(w, even);
    Tensor y = like_rows(x, z.out), more, state;
    if (residual.defined()) more = as_rows(residual, false);
    if (keep) state = bytes_like(x, fgl_linear_state_bytes(z.n, z.dim, z.out, z.dtype, z.act, z.keep8));
    ok(fgl_linear(rows.data_ptr(), row_stride(rows, z.dim), weights.data_ptr(), row_stride(weights, z.dim), address(bias), address(more),
                  more.defined() ? row_stride(more, z.out) : 0, z.n, z.dim, z.out, z.dtype, z.act, z.keep8, y.data_ptr(), z.out, address(state),
                  keep ? (size_t)state.numel() : 0, stream_of(x)));
    return {y, state};
}

std::tuple<Tensor, Tensor, Tensor> linear_gradients(const Tensor& d_y, const Tensor& x, const Tensor& w, const Tensor& state, int64_t dim, int64_t act, bool keep8,
                                                    bool need_x, bool need_w, bool need_b)
{
    torch::NoGradGuard no_grad;
    c10::hip::HIPGuard guard(w.get_device());
    const auto of = w.options().requires_grad(false);
    const bool even = w.scalar_type() == torch::kBFloat16;
    const int64_t out = w.size(0);
    const Tensor g = as_rows(d_y, even && act == 0);
    const int64_t n = g.size(0);
    auto make = [&](at::IntArrayRef size) { return n > 0 ? torch::empty(size, of) : torch::zeros(size, of); };
    Tensor d_x, d_w, d_b;
    if (need_x) {
        auto size = d_y.sizes().vec();
        size.back() = dim;
        d_x = make(size);
    }
    if (need_w) d_w = make({out, dim});
    if (need_b) d_b = make({out});
    if (n > 0 && (need_x || need_w || need_b)) {
        const int dtype = type_of(w);
        const Tensor weights = as_rows(w, false);
        Tensor rows, ws;
        if (x.defined() && need_w) rows = as_rows(x, even);
        const size_t ws_bytes = fgl_linear_workspace_bytes(n, (int)dim, (int)out, dtype, (int)act, keep8, need_w, need_b);
        if (ws_bytes > 0) ws = bytes_like(w, ws_bytes);
        ok(fgl_linear_backward(g.data_ptr(), row_stride(g, out), address(rows), rows.defined() ? row_stride(rows, dim) : 0, weights.data_ptr(), row_stride(weights, dim), n,
                               (int)dim, (int)out, dtype, (int)act, keep8, address(state), state.defined() ? (size_t)state.numel() : 0, address(d_x), dim, address(d_w),
                               address(d_b), address(ws), ws_bytes, stream_of(w)));
    }
    return {d_x, d_w, d_b};
}

std::tuple<Tensor, Tensor, Tensor> linear_gradients_operator(const Tensor& d_y, const Maybe& x, const Tensor& w, const Maybe& state, int64_t dim, int64_t act, bool keep8,
                                                             bool need_x, bool need_w, bool need_b)
{
    auto made = linear_gradients(d_y, x.value_or(Tensor()), w, state.value_or(Tensor()), dim, act, keep8, need_x, need_w, need_b);
    const auto some = [&](const Tensor& t) { return t.defined() ? t : torch::empty({0}, d_y.options()); };
    return {some(std::get<0>(made)), some(std::get<1>(made)), some(std::get<2>(made))};
}

TORCH_LIBRARY_FRAGMENT(fastgl, m)
{
    m.def("linear_gradients(Tensor d_y, Tensor? x, Tensor weight, Tensor? state, int dim, int act, bool keep8, bool need_x, bool need_w, bool need_b) -> "
          "(Tensor, Tensor, Tensor)",
          torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, TORCH_FN(linear_gradients_operator)));
}

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& bias, const Maybe& residual, LinearSizes z)
    {
        const bool keep8 = z.keep8, sums = w.requires_grad();  // (nothing but the weight's gradient reads x)
        z.keep8 = keep8 && sums;
        const bool kept = z.keep8 || (z.act != 0 && (x.requires_grad() || sums || (bias.has_value() && bias->requires_grad())));  // (the residual's gradient is the output's)
        auto [y, state] = form_linear(x, w, bias.value_or(Tensor()), residual.value_or(Tensor()), z, kept);
        ctx->saved_data["dim"] = (int64_t)z.dim;
        ctx->saved_data["act"] = (int64_t)z.act;
        ctx->saved_data["keep8"] = keep8;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        ctx->save_for_backward({sums && !keep8 ? x : Tensor(), w, state});
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &state = saved[2];
        const int64_t dim = ctx->saved_data["dim"].toInt(), act = ctx->saved_data["act"].toInt();
        const bool keep8 = ctx->saved_data["keep8"].toBool();
        // (inputs that were not given are not counted)
        const bool with_b = ctx->saved_data["bias"].toBool(), with_r = ctx->saved_data["residual"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = with_b && ctx->needs_input_grad(2);
        const bool need_r = with_r && ctx->needs_input_grad(with_b ? 3 : 2);
        Tensor d_x, d_w, d_b;
        if (is_wrapped(grads[0])) {
            static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fastgl::linear_gradients", "").typed<decltype(linear_gradients_operator)>();
            std::tie(d_x, d_w, d_b) = op.call(grads[0], maybe(x), w, maybe(state), dim, act, keep8, need_x, need_w, need_b);
            if (!need_x) d_x = Tensor();
            if (!need_w) d_w = Tensor();
            if (!need_b) d_b = Tensor();
        } else {
            std::tie(d_x, d_w, d_b) = linear_gradients(grads[0], x, w, state, dim, act, keep8, need_x, need_w, need_b);
        }
        refuse_gradients_of({&d_x, &d_w, &d_b}, grads[0], w.options(), "linear has no gradients of its gradients");
        out[0] = d_x;
        out[1] = d_w;
        out[2] = d_b;
        if (need_r) out[3] = grads[0];
        return out;
    }
};

Tensor linear(Tensor x, Tensor w, Maybe bias, int act, Maybe residual, bool keep8, int64_t most_columns)
{
    if (at::autocast::is_autocast_enabled(at::kCUDA)) {
        const auto to = at::autocast::get_autocast_dtype(at::kCUDA);
        x = x.to(to);
        w = w.to(to);
        if (bias.has_value()) bias = bias->to(to);
        if (residual.has_value()) residual = residual->to(to);
    }
    TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.size(0) >= 1 && w.size(1) >= 1 && w.size(0) <= most_columns && w.size(1) <= most_columns, "x ",
                x.sizes(), " and weight ", w.sizes(), " must be [.., d] and [out, d] with 1 <= d, out <= ", most_columns);
    TORCH_CHECK(is_feature(x) && w.scalar_type() == x.scalar_type() && (!bias.has_value() || bias->scalar_type() == x.scalar_type()) &&
                    (!residual.has_value() || residual->scalar_type() == x.scalar_type()),
                "x, weight, bias and residual must all be of one type in ['torch.float32', 'torch.bfloat16']");
    TORCH_CHECK(!bias.has_value() || (bias->dim() == 1 && bias->size(0) == w.size(0)), "bias must hold a value for each row of weight");
    if (residual.has_value()) {
        auto size = x.sizes().vec();
        size.back() = w.size(0);
        TORCH_CHECK(residual->sizes() == at::IntArrayRef(size), "residual ", residual->sizes(), " must be of the output's sizes ", at::IntArrayRef(size));
    }
    TORCH_CHECK(w.device() == x.device() && (!bias.has_value() || bias->device() == x.device()) && (!residual.has_value() || residual->device() == x.device()),
                "all tensors must live on the same device");
    if (bias.has_value()) bias = bias->contiguous();
    const LinearSizes z{x.numel() / x.size(-1), (int)w.size(1), (int)w.size(0), type_of(x), act, keep8};
    if (!(torch::GradMode::is_enabled() && (records(x) || records(w) || records(bias) || records(residual))))
        return std::get<0>(form_linear(x, w, bias.value_or(Tensor()), residual.value_or(Tensor()), z, false));
    return LinearNode::apply(x, w, bias, residual, z);
}

}  // namespace

void bind_layers(py::module& m)
{
    m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
    m.def("linear", &linear, py::call_guard<py::gil_scoped_release>());
}
