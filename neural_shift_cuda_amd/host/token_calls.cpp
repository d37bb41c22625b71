// token_calls.cpp -- the token operators' host side on torch tensors: outputs
// and workspaces from torch's allocator, the C ABI's argument structs, and the
// autograd nodes.  attention.py has checked shapes and types and laid out what
// the entries want by then.
//
// A small call is all host time.  With these steps in Python a training pass of
// the norm (3 x 12 heads, 1025 tokens, 28 us of kernels) took 175 us, 50 of them
// for the backward in the autograd thread, whose caches are cold for the
// interpreter; here 96.  One token over a short cache: 17 us, here 10.
#include <c10/hip/HIPStream.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <stdexcept>

#include "neural_shift_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

template <typename T = void>
T* address(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor given(const Maybe& t) { return t ? *t : Tensor(); }

void strides(int64_t (&to)[3], const Tensor& t) {
    for (int i = 0; i < 3; ++i) to[i] = t.stride(i);
}

int32_t code(const Tensor& t, const char* op) {
    switch (t.scalar_type()) {
        case at::kHalf: return NSH_DTYPE_FLOAT16;
        case at::kBFloat16: return NSH_DTYPE_BFLOAT16;
        case at::kFloat: return NSH_DTYPE_FLOAT32;
        default:
            throw std::runtime_error(std::string("\"") + op + "\" not implemented for '" +
                                     c10::toString(t.scalar_type()) + "'");
    }
}

void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void done(int rc) {
    if (rc != NSH_OK) throw std::runtime_error(nsh_last_error());
}

// A new tensor that keeps t's order of heads and tokens in memory.
Tensor like(const Tensor& t) {
    if (!t.is_contiguous() && t.stride(1) < t.stride(2))
        return at::empty({t.size(0), t.size(2), t.size(1), t.size(3)}, t.options()).transpose(1, 2);
    return at::empty(t.sizes(), t.options());
}

Tensor scratch(const Tensor& t, int64_t bytes) {
    return bytes > 0 ? at::empty({bytes}, t.options().dtype(at::kByte)) : Tensor();
}

// Rows with a unit last stride, in whole (`rows16`) 16-byte pieces.
Tensor unit(const Tensor& t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); }
Tensor rows16(const Tensor& t) {
    const int64_t e = t.element_size(), all = t.stride(0) | t.stride(1) | t.stride(2);
    if (t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && all * e % 16 == 0 &&
        t.stride(2) * e <= int64_t(1) << 24)
        return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

// Gradients of gradients are refused where they are asked for.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a token operator, whose gradients are not differentiable",
        static_cast<int64_t>(grads.size()));
    return (*error)(std::move(grads));
}

// A tangent would be dropped without a word: what the kernels write has none.
void no_tangents(const char* op, std::initializer_list<const Tensor*> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), op,
                                    ": forward-mode derivatives are not implemented");
}

bool graph(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// ---------------------------------------------------------------------------
// Norm and rotation
// ---------------------------------------------------------------------------

struct NormRules {
    double eps;
    bool interleaved;
};

nsh_norm_rotary_args norm_args(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                               const Tensor& cos, const Tensor& sin, const Tensor& positions, NormRules r) {
    nsh_norm_rotary_args a{};
    a.q = address(q), a.k = address(k), a.q_weight = address(wq), a.k_weight = address(wk);
    a.cos = address<float>(cos), a.sin = address<float>(sin), a.positions = address<int32_t>(positions);
    a.position_stride = positions.defined() && positions.dim() == 2 ? q.size(2) : 0;
    a.B = q.size(0), a.Hq = q.size(1), a.Hk = k.size(1), a.L = q.size(2), a.D = q.size(3);
    a.half = cos.size(1), a.rows = cos.size(0);
    strides(a.q_stride, q), strides(a.k_stride, k);
    a.eps = r.eps, a.dtype = code(q, "norm_rotary"), a.interleaved = r.interleaved;
    return a;
}

variable_list norm_forward(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk,
                           const Tensor& cos, const Tensor& sin, const Tensor& positions, NormRules r) {
    nsh_norm_rotary_args a = norm_args(q, k, wq, wk, cos, sin, positions, r);
    variable_list out = {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
    if (q.numel() || k.numel()) {
        a.q_out = address(out[0]), a.k_out = address(out[1]);
        done(nsh_norm_rotary_forward(&a, stream(q)));
    }
    return out;
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Maybe& wq0,
                                 const Maybe& wk0, const Tensor& cos, const Tensor& sin, const Maybe& at,
                                 NormRules r) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor q = unit(q0), k = unit(k0), wq = given(wq0), wk = given(wk0), positions = given(at);
        ctx->save_for_backward({q, k, wq, wk, cos, sin, positions});
        ctx->saved_data["eps"] = r.eps;
        ctx->saved_data["interleaved"] = r.interleaved;
        ctx->saved_data["given"] = (wq.defined() ? 1 : 0) + (wk.defined() ? 2 : 0);
        return norm_forward(q, k, wq, wk, cos, sin, positions, r);
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &wq = s[2], &wk = s[3];
        c10::DeviceGuard on(q.device());
        variable_list grads(8);
        {
            at::NoGradGuard none;
            const Tensor gq = unit(upstream[0]), gk = unit(upstream[1]);
            nsh_norm_rotary_args a = norm_args(q, k, wq, wk, s[4], s[5], s[6],
                                               {ctx->saved_data["eps"].toDouble(),
                                                ctx->saved_data["interleaved"].toBool()});
            grads[0] = at::empty(q.sizes(), q.options()), grads[1] = at::empty(k.sizes(), k.options());
            // an input's place among those that may have a gradient
            const int64_t have = ctx->saved_data["given"].toInt();
            if ((have & 1) && ctx->needs_input_grad(2)) grads[2] = at::empty_like(wq);
            if ((have & 2) && ctx->needs_input_grad(have & 1 ? 3 : 2)) grads[3] = at::empty_like(wk);
            if (!q.numel() && !k.numel()) {
                for (int i = 2; i < 4; ++i)
                    if (grads[i].defined()) grads[i].zero_();
            } else {
                a.grad_q_out = address(gq), a.grad_k_out = address(gk);
                strides(a.gq_stride, gq), strides(a.gk_stride, gk);
                a.grad_q = address(grads[0]), a.grad_k = address(grads[1]);
                a.grad_q_weight = address(grads[2]), a.grad_k_weight = address(grads[3]);
                Tensor ws;
                if (grads[2].defined() || grads[3].defined()) {
                    a.workspace_bytes = nsh_norm_rotary_workspace_bytes(&a);
                    ws = scratch(q, a.workspace_bytes);
                    a.workspace = address(ws);
                }
                done(nsh_norm_rotary_backward(&a, stream(q)));
            }
        }
        return once(std::move(grads));
    }
};

std::tuple<Tensor, Tensor> norm_rotary(const Tensor& q, const Tensor& k, const Maybe& wq, const Maybe& wk,
                                       const Tensor& cos, const Tensor& sin, const Maybe& positions,
                                       double eps, bool interleaved) {
    c10::DeviceGuard on(q.device());
    const Tensor w0 = given(wq), w1 = given(wk);
    no_tangents("norm_rotary", {&q, &k, &w0, &w1, &cos, &sin});
    const variable_list out =
        graph({&q, &k, &w0, &w1})
            ? NormNode::apply(q, k, wq, wk, cos, sin, positions, NormRules{eps, interleaved})
            : norm_forward(unit(q), unit(k), w0, w1, cos, sin, given(positions), {eps, interleaved});
    return {out[0], out[1]};
}

// ---------------------------------------------------------------------------
// Position bias
// ---------------------------------------------------------------------------

Tensor bias_forward(const Tensor& table, const Tensor& buckets, int64_t Lq, int64_t Lk) {
    const int32_t dtype = code(table, "position_bias");
    const Tensor out = at::empty({table.size(1), Lq, Lk}, table.options());
    if (out.numel())
        done(nsh_position_bias_forward(address(table), address<int32_t>(buckets), table.size(1), Lq, Lk, table.size(0),
                                       (buckets.numel() - 1) / 2, dtype, address(out), stream(table)));
    return out;
}

struct BiasNode : torch::autograd::Function<BiasNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& buckets, int64_t Lq, int64_t Lk) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({buckets});
        ctx->saved_data["rows"] = table.size(0);
        return bias_forward(table.contiguous(), buckets, Lq, Lk);
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const Tensor buckets = ctx->get_saved_variables()[0];
        c10::DeviceGuard on(buckets.device());
        variable_list grads(4);
        {
            at::NoGradGuard none;
            const Tensor g = upstream[0].contiguous();
            const int64_t rows = ctx->saved_data["rows"].toInt(), reach = (buckets.numel() - 1) / 2;
            grads[0] = at::empty({rows, g.size(0)}, g.options());
            if (!g.numel()) {
                grads[0].zero_();
            } else {
                const int64_t n = nsh_position_bias_workspace_bytes(g.size(0), g.size(1), g.size(2), reach);
                const Tensor ws = scratch(g, n);
                done(nsh_position_bias_backward(address(g), address<int32_t>(buckets), g.size(0), g.size(1),
                                                g.size(2), rows, reach, code(g, "position_bias"), address(grads[0]),
                                                address(ws), n, stream(g)));
            }
        }
        return once(std::move(grads));
    }
};

Tensor position_bias(const Tensor& table, const Tensor& buckets, int64_t Lq, int64_t Lk) {
    c10::DeviceGuard on(table.device());
    no_tangents("position_bias", {&table});
    return graph({&table}) ? BiasNode::apply(table, buckets, Lq, Lk)
                           : bias_forward(table.contiguous(), buckets, Lq, Lk);
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

struct Masks {
    Tensor lengths, prefix, documents, slopes, buckets;
};
struct Rules {
    double scale, cap;
    bool causal, degree;
};

// kept: out_rest (16-bit types), then row_stats.
nsh_attention_args attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                                  const Tensor& out, const Tensor& kept, const Masks& m, Rules r) {
    nsh_attention_args a{};
    a.q = address(q), a.k = address(k), a.v = address(v), a.out = address(out);
    a.B = q.size(0), a.Hq = q.size(1), a.Hk = k.size(1), a.Lq = q.size(2), a.Lk = k.size(2), a.D = q.size(3);
    strides(a.q_stride, q), strides(a.k_stride, k), strides(a.v_stride, v), strides(a.out_stride, out);
    a.lengths = address<int32_t>(m.lengths), a.prefix = address<int32_t>(m.prefix);
    a.documents = address<int32_t>(m.documents), a.slopes = address<float>(m.slopes);
    if (table.defined()) {
        a.bias_table = address(table), a.buckets = address<int32_t>(m.buckets);
        a.num_buckets = table.size(0), a.reach = (m.buckets.numel() - 1) / 2;
    }
    a.scale = r.scale, a.cap = r.cap, a.causal = r.causal, a.dtype = code(q, "attention");
    if (kept.defined()) {
        char* p = address<char>(kept);
        if (q.element_size() == 2) a.out_rest = p, p += 2 * out.numel();
        a.row_stats = reinterpret_cast<float*>(p);
    }
    return a;
}

// out, log_degree (or undefined), kept (with `keep`, else undefined)
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                     const Tensor& table, const Masks& m, Rules r, bool keep) {
    const int64_t rows = q.size(0) * q.size(1) * q.size(2);
    Tensor out = like(q), degree, kept;
    if (r.degree) degree = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    if (keep)
        kept = at::empty({rows * (2 + (q.element_size() == 2 ? q.size(3) / 2 : 0))}, q.options().dtype(at::kFloat));
    if (!out.numel()) return {out, degree, kept};
    if (!k.numel()) {
        out.zero_();
        if (r.degree) degree.fill_(-INFINITY);
        return {out, degree, kept};
    }
    nsh_attention_args a = attention_args(q, k, v, table, out, kept, m, r);
    a.log_degree = address<float>(degree);
    a.workspace_bytes = nsh_attention_workspace_bytes(&a, 0);
    const Tensor ws = scratch(q, a.workspace_bytes);
    a.workspace = address(ws);
    done(nsh_attention_forward(&a, stream(q)));
    return {out, degree, kept};
}

struct AttentionNode : torch::autograd::Function<AttentionNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Maybe& bias_table, const Masks& m, Rules r) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor table = bias_table ? bias_table->contiguous() : Tensor();
        auto [out, degree, kept] = attention_forward(q, k, v, table, m, r, true);
        ctx->save_for_backward({q, k, v, table, out, kept, m.lengths, m.prefix, m.documents, m.slopes, m.buckets});
        ctx->saved_data["scale"] = r.scale;
        ctx->saved_data["cap"] = r.cap;
        ctx->saved_data["causal"] = r.causal;
        ctx->set_materialize_grads(false);
        if (r.degree) return {out, degree};
        return {out};
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &table = s[3], &out = s[4], &kept = s[5];
        c10::DeviceGuard on(q.device());
        variable_list grads(6);
        {
            at::NoGradGuard none;
            const Tensor go = upstream[0].defined() ? rows16(upstream[0]) : at::zeros_like(out);
            const Tensor gdegree = upstream.size() > 1 && upstream[1].defined() ? upstream[1].contiguous() : Tensor();
            grads[0] = like(q), grads[1] = like(k), grads[2] = like(v);
            if (table.defined() && ctx->needs_input_grad(3)) grads[3] = at::empty_like(table);
            if (!q.numel() || !k.numel()) {
                for (auto& g : grads)
                    if (g.defined()) g.zero_();
            } else {
                nsh_attention_args a = attention_args(
                    q, k, v, table, out, kept, {s[6], s[7], s[8], s[9], s[10]},
                    {ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(),
                     ctx->saved_data["causal"].toBool(), false});
                a.grad_out = address(go), a.grad_log_degree = address<float>(gdegree);
                strides(a.go_stride, go);
                a.grad_q = address(grads[0]), a.grad_k = address(grads[1]), a.grad_v = address(grads[2]);
                strides(a.gq_stride, grads[0]), strides(a.gk_stride, grads[1]), strides(a.gv_stride, grads[2]);
                a.grad_bias_table = address(grads[3]);
                a.workspace_bytes = nsh_attention_workspace_bytes(&a, 1);
                const Tensor ws = scratch(q, a.workspace_bytes);
                a.workspace = address(ws);
                done(nsh_attention_backward(&a, stream(q)));
            }
        }
        return once(std::move(grads));
    }
};

std::tuple<Tensor, Maybe> attention(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Maybe& table,
                                    const Maybe& lengths, const Maybe& prefix, const Maybe& documents,
                                    const Maybe& slopes, const Maybe& buckets, double scale, double cap, bool causal,
                                    bool degree) {
    c10::DeviceGuard on(q0.device());
    const Tensor q = rows16(q0), k = rows16(k0), v = rows16(v0), t = given(table);
    const Masks m{given(lengths), given(prefix), given(documents), given(slopes), given(buckets)};
    no_tangents("attention", {&q, &k, &v, &t, &m.slopes});
    const Rules r{scale, cap, causal, degree};
    if (graph({&q, &k, &v, &t})) {
        const variable_list out = AttentionNode::apply(q, k, v, table, m, r);
        return {out[0], degree ? Maybe(out[1]) : Maybe()};
    }
    auto [out, log_degree, kept] =
        attention_forward(q, k, v, t.defined() ? t.contiguous() : t, m, r, false);
    return {out, degree ? Maybe(log_degree) : Maybe()};
}

// ---------------------------------------------------------------------------
// Calls as a program's loop makes them: every tensor already in the type and
// layout that the entries take.  These look that over and run; anything else,
// wrong or only to be converted, gives None, and attention.py's own checks say
// what it is.  So does a call under torch.jit.trace, which would record the
// allocations here and no kernel.  (They take 4 to 9 us in Python, as long as the rest of a call.)
// ---------------------------------------------------------------------------

bool served(const Tensor& t) {
    const auto type = t.scalar_type();
    return type == at::kHalf || type == at::kBFloat16 || type == at::kFloat;
}

bool alike(const Tensor& t, const Tensor& q) { return t.scalar_type() == q.scalar_type() && t.device() == q.device(); }

// Not given, or contiguous in `type` and of this shape.
bool plain(const Maybe& t, const Tensor& q, at::ScalarType type, at::IntArrayRef shape) {
    return !t || (t->scalar_type() == type && t->device() == q.device() && t->sizes() == shape && t->is_contiguous());
}

bool map_of_buckets(const Tensor& table, const Maybe& buckets) {
    return table.dim() == 2 && table.size(0) >= 1 && table.size(0) <= 4097 && buckets && buckets->dim() == 1 &&
           buckets->size(0) % 2 == 1 && buckets->size(0) <= 4097 &&
           plain(buckets, table, at::kInt, buckets->sizes());
}

std::optional<std::tuple<Tensor, Tensor>> norm_rotary_as_is(const Tensor& q, const Tensor& k, const Maybe& wq,
                                                            const Maybe& wk, const Tensor& cos, const Tensor& sin,
                                                            const Maybe& positions, double eps, bool interleaved) {
    if (torch::jit::tracer::isTracing()) return {};
    if (q.dim() != 4 || k.dim() != 4 || !served(q) || !alike(k, q)) return {};
    const int64_t B = q.size(0), L = q.size(2), D = q.size(3);
    if (k.size(0) != B || k.size(2) != L || k.size(3) != D || D > 512) return {};
    if (!plain(wq, q, q.scalar_type(), {D}) || !plain(wk, q, q.scalar_type(), {D})) return {};
    if (cos.dim() != 2 || 2 * cos.size(1) > D || cos.requires_grad() || sin.requires_grad()) return {};
    if (!plain(cos, q, at::kFloat, cos.sizes()) || !plain(sin, q, at::kFloat, cos.sizes())) return {};
    if (positions ? !plain(positions, q, at::kInt, {L}) && !plain(positions, q, at::kInt, {B, L}) : L > cos.size(0))
        return {};
    return norm_rotary(q, k, wq, wk, cos, sin, positions, eps, interleaved);
}

Maybe position_bias_as_is(const Tensor& table, const Maybe& buckets, int64_t Lq, int64_t Lk) {
    if (torch::jit::tracer::isTracing()) return {};
    if (Lq < 0 || Lk < 0 || !served(table) || !map_of_buckets(table, buckets)) return {};
    return position_bias(table, *buckets, Lq, Lk);
}

std::optional<std::tuple<Tensor, Maybe>> attention_as_is(
    const Tensor& q, const Tensor& k, const Tensor& v, std::optional<double> scale, std::optional<double> cap,
    bool causal, const Maybe& prefix, const Maybe& documents, const Maybe& lengths, const Maybe& slopes,
    const Maybe& table, const Maybe& buckets, bool degree) {
    if (torch::jit::tracer::isTracing()) return {};
    if (q.dim() != 4 || k.dim() != 4 || !served(q) || !alike(k, q) || !alike(v, q) || k.sizes() != v.sizes()) return {};
    const int64_t B = q.size(0), Hq = q.size(1), D = q.size(3), Hk = k.size(1), Lk = k.size(2);
    if (k.size(0) != B || k.size(3) != D || D < 8 || D > 128 || D % 8 || Hk < 1 || Hq % Hk) return {};
    const double by = scale ? *scale : std::pow(static_cast<double>(D), -0.5), top = cap ? *cap : 0.0;
    if (!std::isfinite(by) || !std::isfinite(top) || top < 0 || (prefix && !causal)) return {};
    if (!plain(prefix, q, at::kInt, {B}) || !plain(lengths, q, at::kInt, {B}) ||
        !plain(documents, q, at::kInt, {B, Lk}) || !plain(slopes, q, at::kFloat, {Hq}) ||
        (slopes && slopes->requires_grad()))
        return {};
    if (table ? !alike(*table, q) || !map_of_buckets(*table, buckets) || table->size(1) != Hq : buckets.has_value())
        return {};
    return attention(q, k, v, table, lengths, prefix, documents, slopes, buckets, by, top, causal, degree);
}

std::tuple<Tensor, Maybe, Maybe> attention_plain(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& table,
                                                 const Maybe& lengths, const Maybe& prefix, const Maybe& documents,
                                                 const Maybe& slopes, const Maybe& buckets, double scale, double cap,
                                                 bool causal, bool degree, bool keep) {
    c10::DeviceGuard on(q.device());
    auto [out, log_degree, kept] = attention_forward(
        q, k, v, given(table), {given(lengths), given(prefix), given(documents), given(slopes), given(buckets)},
        {scale, cap, causal, degree}, keep);
    return {out, degree ? Maybe(log_degree) : Maybe(), keep ? Maybe(kept) : Maybe()};
}

}  // namespace

PYBIND11_MODULE(_token_calls, m) {
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("norm_rotary", &norm_rotary, release());
    m.def("position_bias", &position_bias, release());
    m.def("attention", &attention, release());
    m.def("norm_rotary_as_is", &norm_rotary_as_is, release());
    m.def("position_bias_as_is", &position_bias_as_is, release());
    m.def("attention_as_is", &attention_as_is, release());
    m.def("attention_forward", &attention_plain, release());
}
