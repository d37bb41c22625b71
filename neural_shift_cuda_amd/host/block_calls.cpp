// block_calls.cpp -- layer norm and the gated projections on torch tensors:
// outputs and workspaces from torch's allocator, the C ABI's argument structs,
// and the autograd nodes.  feedforward.py has checked shapes and types by then;
// rows are whatever dimensions stand before the last one.
#include "calls.hpp"

namespace {

using namespace nsh_calls;

// Rows with a unit last stride and one step from each to the next, where the tensor
// lies so; a copy otherwise.
Tensor rows_of(const Tensor& t0) {
    const Tensor t = t0.resolve_neg();  // (a conjugate's imaginary part)
    const int64_t dim = t.dim(), n = t.size(dim - 1);
    if (dim == 2 && (t.stride(1) == 1 || n == 1)) return t;
    bool whole = t.stride(dim - 1) == 1 || n == 1;
    int64_t rows = 1, step = n, next = -1;  // next: where the dimension in front has to step
    for (int64_t d = dim - 2; d >= 0 && whole; --d) {
        if (t.size(d) != 1) {
            if (next >= 0 && t.stride(d) != next) whole = false;
            if (next < 0) step = t.stride(d);
            next = t.stride(d) * t.size(d);
        }
        rows *= t.size(d);
    }
    if (whole && t.numel()) return t.as_strided({rows, n}, {step, 1});
    return t.contiguous().view({n ? t.numel() / n : 0, n});
}

int64_t step(const Tensor& rows) { return rows.stride(0); }

// ---------------------------------------------------------------------------
// Layer norm
// ---------------------------------------------------------------------------

// y, s (with a residual), stats (with `keep`)
variable_list layer_norm_forward(const Tensor& x0, const Tensor& residual0, const Tensor& weight, const Tensor& bias,
                                 double eps, bool keep) {
    const Tensor x = rows_of(x0);
    variable_list out = {at::empty(x0.sizes(), x0.options()), Tensor(), Tensor()};
    if (residual0.defined()) out[1] = at::empty(x0.sizes(), x0.options());
    if (keep) out[2] = at::empty({x.size(0), 2}, x0.options().dtype(at::kFloat));
    nsh_layer_norm_args a{};
    a.dtype = code(x, "layer_norm");
    if (!x.numel()) return out;
    a.x = address(x), a.weight = address(weight), a.bias = address(bias);
    a.rows = x.size(0), a.n = x.size(1), a.x_stride = step(x), a.eps = eps;
    Tensor residual;
    if (residual0.defined()) {
        residual = rows_of(residual0);
        a.residual = address(residual), a.residual_stride = step(residual), a.s = address(out[1]);
    }
    a.y = address(out[0]), a.stats = address<float>(out[2]);
    done(nsh_layer_norm_forward(&a, stream(x)));
    return out;
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, const Maybe& weight0,
                                 const Maybe& bias, double eps) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor weight = given(weight0);
        variable_list out = layer_norm_forward(x, given(residual), weight, given(bias), eps, true);
        ctx->save_for_backward({residual ? out[1] : x, weight, out[2]});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["given"] = (residual ? 1 : 0) + (weight0 ? 2 : 0) + (bias ? 4 : 0);
        ctx->set_materialize_grads(false);
        if (residual) return {out[0], out[1]};
        return {out[0]};
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &normed = saved[0], &weight = saved[1], &stats = saved[2];
        c10::DeviceGuard on(normed.device());
        variable_list grads(5);
        {
            at::NoGradGuard none;
            const int64_t have = ctx->saved_data["given"].toInt();
            // an input's place among those that may have a gradient
            int place = 0;
            const bool want_x = ctx->needs_input_grad(place++);
            const bool want_residual = (have & 1) && ctx->needs_input_grad(place++);
            const bool want_weight = (have & 2) && ctx->needs_input_grad(place++);
            const bool want_bias = (have & 4) && ctx->needs_input_grad(place++);
            const Tensor x = rows_of(normed);
            const Tensor gy = rows_of(upstream[0].defined() ? upstream[0] : at::zeros(normed.sizes(), normed.options()));
            Tensor gs, gx;
            if (upstream.size() > 1 && upstream[1].defined()) gs = rows_of(upstream[1]);
            if (want_x || want_residual) gx = at::empty(normed.sizes(), normed.options());
            if (want_weight) grads[2] = at::empty({x.size(1)}, x.options());
            if (want_bias) grads[3] = at::empty({x.size(1)}, x.options());
            if (!x.numel()) {
                for (int i = 2; i < 4; ++i)
                    if (grads[i].defined()) grads[i].zero_();
            } else if (gx.defined() || want_weight || want_bias) {
                nsh_layer_norm_args a{};
                a.x = address(x), a.weight = address(weight), a.rows = x.size(0), a.n = x.size(1);
                a.x_stride = step(x), a.eps = ctx->saved_data["eps"].toDouble(), a.dtype = code(x, "layer_norm");
                a.stats = address<float>(stats);
                a.grad_y = address(gy), a.gy_stride = step(gy);
                if (gs.defined()) a.grad_s = address(gs), a.gs_stride = step(gs);
                a.grad_x = address(gx), a.grad_weight = address(grads[2]), a.grad_bias = address(grads[3]);
                Tensor ws;
                if (want_weight || want_bias) {
                    a.workspace_bytes = nsh_layer_norm_workspace_bytes(&a);
                    ws = scratch(x, a.workspace_bytes);
                    a.workspace = address(ws);
                }
                done(nsh_layer_norm_backward(&a, stream(x)));
            }
            if (want_x) grads[0] = gx;
            if (want_residual) grads[1] = gx;
        }
        return once(std::move(grads));
    }
};

std::tuple<Tensor, Maybe> layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, const Maybe& residual,
                                     double eps) {
    c10::DeviceGuard on(x.device());
    const Tensor w = given(weight), b = given(bias), r = given(residual);
    no_tangents("layer_norm", {&x, &w, &b, &r});
    const variable_list out = graph({&x, &w, &b, &r}) ? LayerNormNode::apply(x, residual, weight, bias, eps)
                                                      : layer_norm_forward(x, r, w, b, eps, false);
    return {out[0], residual ? Maybe(out[1]) : Maybe()};
}

// ---------------------------------------------------------------------------
// Gated projections
// ---------------------------------------------------------------------------

nsh_gated_linear_args gated_args(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation) {
    nsh_gated_linear_args a{};
    a.x = address(x), a.gate_weight = address(gate), a.up_weight = address(up);
    a.rows = x.size(0), a.K = x.size(1), a.F = gate.size(0);
    a.x_stride = step(x), a.gate_stride = step(gate), a.up_stride = step(up);
    a.dtype = code(x, "gated_linear"), a.activation = static_cast<int32_t>(activation);
    return a;
}

// h, kept (with `keep`)
std::tuple<Tensor, Tensor> gated_forward(const Tensor& x0, const Tensor& gate0, const Tensor& up0, int64_t activation,
                                         bool keep) {
    const Tensor x = rows_of(x0), gate = rows_of(gate0), up = rows_of(up0);
    auto shape = x0.sizes().vec();
    shape.back() = gate0.size(0);  // (a copy of weights without a width has lost its rows)
    const Tensor h = at::empty(shape, x0.options());
    nsh_gated_linear_args a = gated_args(x, gate, up, activation);
    Tensor kept;
    if (!h.numel()) return {h, kept};
    if (!x.size(1)) return {h.zero_(), kept};  // act(0) * 0
    if (keep) kept = scratch(x, nsh_gated_linear_kept_bytes(&a));
    a.h = address(h), a.kept = address(kept);
    a.workspace_bytes = nsh_gated_linear_workspace_bytes(&a, 0);
    const Tensor ws = scratch(x, a.workspace_bytes);
    a.workspace = address(ws);
    done(nsh_gated_linear_forward(&a, stream(x)));
    return {h, kept};
}

struct GatedNode : torch::autograd::Function<GatedNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation) {
        at::AutoDispatchBelowADInplaceOrView below;
        auto [h, kept] = gated_forward(x, gate, up, activation, true);
        ctx->save_for_backward({x, gate, up, kept});
        ctx->saved_data["activation"] = activation;
        return h;
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &kept = saved[3];
        c10::DeviceGuard on(saved[0].device());
        variable_list grads(4);
        {
            at::NoGradGuard none;
            const Tensor x = rows_of(saved[0]), gate = rows_of(saved[1]), up = rows_of(saved[2]);
            const Tensor gh = rows_of(upstream[0]);
            for (int i = 0; i < 3; ++i)
                if (ctx->needs_input_grad(i)) grads[i] = at::empty(saved[i].sizes(), saved[i].options());
            if (!kept.defined()) {
                for (auto& g : grads)
                    if (g.defined()) g.zero_();
            } else if (grads[0].defined() || grads[1].defined() || grads[2].defined()) {
                nsh_gated_linear_args a = gated_args(x, gate, up, ctx->saved_data["activation"].toInt());
                a.kept = address(kept);
                a.grad_h = address(gh), a.gh_stride = step(gh);
                a.grad_x = address(grads[0]), a.grad_gate = address(grads[1]), a.grad_up = address(grads[2]);
                a.workspace_bytes = nsh_gated_linear_workspace_bytes(&a, 1);
                const Tensor ws = scratch(x, a.workspace_bytes);
                a.workspace = address(ws);
                done(nsh_gated_linear_backward(&a, stream(x)));
            }
        }
        return once(std::move(grads));
    }
};

Tensor gated_linear(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation) {
    c10::DeviceGuard on(x.device());
    no_tangents("gated_linear", {&x, &gate, &up});
    if (graph({&x, &gate, &up})) return GatedNode::apply(x, gate, up, activation);
    return std::get<0>(gated_forward(x, gate, up, activation, false));
}

// ---------------------------------------------------------------------------
// Calls as a program's loop makes them: looked over here, and None for anything
// else, wrong or only to be converted, whose checks are feedforward.py's.  So does a
// call under torch.jit.trace, which would record the allocations and no kernel.
// ---------------------------------------------------------------------------

std::optional<std::tuple<Tensor, Maybe>> layer_norm_as_is(const Tensor& x, const Maybe& weight, const Maybe& bias,
                                                          const Maybe& residual, double eps) {
    if (torch::jit::tracer::isTracing()) return {};
    if (x.dim() < 1 || !served(x) || !(eps >= 0) || std::isinf(eps)) return {};
    const int64_t n = x.size(-1);
    if (!plain(weight, x, x.scalar_type(), {n}) || !plain(bias, x, x.scalar_type(), {n})) return {};
    if (residual && (!alike(*residual, x) || residual->sizes() != x.sizes())) return {};
    return layer_norm(x, weight, bias, residual, eps);
}

Maybe gated_linear_as_is(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation) {
    if (torch::jit::tracer::isTracing()) return {};
    if (x.dim() < 1 || gate.dim() != 2 || !served(x) || !alike(gate, x) || !alike(up, x)) return {};
    if (gate.sizes() != up.sizes() || gate.size(1) != x.size(-1)) return {};
    return gated_linear(x, gate, up, activation);
}

}  // namespace

void block_calls(pybind11::module_& m) {
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("layer_norm", &layer_norm, release());
    m.def("gated_linear", &gated_linear, release());
    m.def("layer_norm_as_is", &layer_norm_as_is, release());
    m.def("gated_linear_as_is", &gated_linear_as_is, release());
}
