// torch_layer.cpp -- the operators of layer_ops.py as torch calls them: allocation, autograd nodes and the
// C entry points of libdynamis_graph.so, without the interpreter.
//
// A training step's backward pass runs on a thread of the autograd engine, where each of the
// interpreter's instructions costs twice.  Host time of a call and of a training step, in Python and here:
// rotate_heads 15.3 and 7.5 us, 157 and 50; route_rows 20.7 and 10.3, 102 and 33; dispatch_rows 8.8 and 5.0, 89 and
// 44; combine_rows 10.2 and 6.0, 105 and 57; grouped_linear with an activation 10.3 and 7.6, 128 and 72 (the engine's
// hand-over to its thread alone takes some 35).  Arguments have been checked by the caller.  The entry
// points come as addresses of the library that the caller has loaded.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstring>
#include <map>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/dynamis_graph.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entries {
    decltype(&dg_last_error) last_error;
    decltype(&dg_rotate_forward) rotate_forward;
    decltype(&dg_rotate_workspace_size) rotate_workspace_size;
    decltype(&dg_rotate_backward) rotate_backward;
    decltype(&dg_route_workspace_size) route_workspace_size;
    decltype(&dg_route_forward) route_forward;
    decltype(&dg_route_backward) route_backward;
    decltype(&dg_exchange_dispatch) exchange_dispatch;
    decltype(&dg_exchange_combine) exchange_combine;
    decltype(&dg_exchange_combine_backward) exchange_combine_backward;
    decltype(&dg_grouped_apply) grouped_apply;
    decltype(&dg_grouped_apply_workspace_size) grouped_apply_workspace_size;
    decltype(&dg_grouped_apply_gradients) grouped_apply_gradients;
    decltype(&dg_grouped_workspace_size) grouped_workspace_size;
} dg;

void load(const std::map<std::string, uintptr_t>& at)
{
    auto get = [&](auto& f, const char* name) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at.at(name)); };
    get(dg.last_error, "dg_last_error");
    get(dg.rotate_forward, "dg_rotate_forward");
    get(dg.rotate_workspace_size, "dg_rotate_workspace_size");
    get(dg.rotate_backward, "dg_rotate_backward");
    get(dg.route_workspace_size, "dg_route_workspace_size");
    get(dg.route_forward, "dg_route_forward");
    get(dg.route_backward, "dg_route_backward");
    get(dg.exchange_dispatch, "dg_exchange_dispatch");
    get(dg.exchange_combine, "dg_exchange_combine");
    get(dg.exchange_combine_backward, "dg_exchange_combine_backward");
    get(dg.grouped_apply, "dg_grouped_apply");
    get(dg.grouped_apply_workspace_size, "dg_grouped_apply_workspace_size");
    get(dg.grouped_apply_gradients, "dg_grouped_apply_gradients");
    get(dg.grouped_workspace_size, "dg_grouped_workspace_size");
}

void check(dg_status status, const char* what)
{
    if (status != DG_OK) throw std::runtime_error(std::string(what) + ": " + dg.last_error());
}

int32_t type_of(const Tensor& t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return DG_F32;
        case at::kDouble: return DG_F64;
        case at::kLong: return DG_I64;
        case at::kBFloat16: return DG_BF16;
        default: throw std::runtime_error("unexpected dtype");
    }
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor plain(const Tensor& like) { return at::empty(like.sizes(), like.options()); }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
Tensor value(const OptTensor& t) { return t ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }

// t [n, heads, dim] as it is if its rows are whole, start at 16 bytes and lie a multiple of 16 bytes apart; else a copy.
Tensor rows_16(const Tensor& t)
{
    const int64_t step = 16 / t.element_size();
    if (t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2)) && t.stride(0) % step == 0 &&
        (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0)
        return t;
    return t.clone(at::MemoryFormat::Contiguous);
}

// t [rows, width] as it is if its rows are whole; else a copy.
Tensor whole_rows(const Tensor& t)
{
    return (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= 0 && t.stride(0) <= 1ll << 31 ? t : t.contiguous();
}

// Gradients that may not be differentiated again: where a graph of them is asked for, doing so raises.
variable_list once(variable_list grads, const char* what)
{
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate twice ") + what + ", which is differentiable once", (int64_t)grads.size());
    // (the node that raises is made where something requires a gradient)
    variable_list in;
    for (auto& g : grads) {
        if (g.defined()) {
            g = g.detach();
            g.requires_grad_(true);
        }
        in.push_back(g);
    }
    return (*error)(std::move(in));
}

// A saved tensor as it comes back from a hook, which may have laid it out anew but is held to its shape, type and device.
const Tensor& same(const Tensor& t, at::IntArrayRef sizes, int32_t type, at::Device device, const char* what)
{
    const bool typed = t.defined() && (type == DG_I32 ? t.scalar_type() == at::kInt : t.scalar_type() != at::kInt && type_of(t) == type);
    if (!typed || t.sizes() != sizes || t.device() != device)
        throw std::runtime_error(std::string(what) + ": a saved tensor came back with another shape, dtype or device");
    return t;
}

std::string text(const void* d, size_t n) { return std::string((const char*)d, n); }

// ---------------------------------------------------------------- rotate_heads

std::tuple<Tensor, Tensor> rotate_forward(dg_rotate_desc& d, const Tensor& q, const Tensor& k, const Tensor& positions,
                                          const Tensor& frequencies, const Tensor& q_weight, const Tensor& k_weight)
{
    Tensor q_out = plain(q), k_out = plain(k);
    d.ld_q = q.stride(0);
    d.ld_k = k.stride(0);
    check(dg.rotate_forward(&d, q.data_ptr(), k.data_ptr(), positions.data_ptr(), (const float*)frequencies.data_ptr(), ptr(q_weight),
                            ptr(k_weight), q_out.data_ptr(), k_out.data_ptr(), stream_of(q)), "rotate_heads");
    return {q_out, k_out};
}

struct Rotate : torch::autograd::Function<Rotate> {
    static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& frequencies,
                                 const OptTensor& q_weight_, const OptTensor& k_weight_, std::string desc)
    {
        const Tensor q_weight = value(q_weight_), k_weight = value(k_weight_);
        dg_rotate_desc d;
        memcpy(&d, desc.data(), sizeof d);
        Tensor qr = rows_16(q), kr = rows_16(k);
        auto [q_out, k_out] = rotate_forward(d, qr, kr, positions, frequencies, q_weight, k_weight);
        ctx->save_for_backward({qr, kr, positions, frequencies, q_weight, k_weight});
        ctx->saved_data["desc"] = text(&d, sizeof d);
        return {q_out, k_out};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const at::Device dev = grads[0].device();
        c10::OptionalDeviceGuard guard(dev);
        dg_rotate_desc d;
        memcpy(&d, ctx->saved_data["desc"].toStringRef().data(), sizeof d);
        const char* const what = "rotate_heads";
        int64_t pairs = 0;
        for (int i = 0; i < d.axes; ++i) pairs += d.sections[i];
        const Tensor q = rows_16(same(s[0], {d.n_targets, d.heads, d.dim}, d.dtype, dev, what));
        const Tensor k = rows_16(same(s[1], {d.n_nodes, d.kv_heads, d.dim}, d.dtype, dev, what));
        const Tensor positions = same(s[2], {d.n_nodes, d.axes}, d.pos_dtype, dev, what).contiguous();
        const Tensor frequencies = same(s[3], {pairs}, DG_F32, dev, what).contiguous();
        Tensor q_weight, k_weight;
        if (s[4].defined()) q_weight = same(s[4], {d.dim}, d.weight_dtype, dev, what).contiguous();
        if (s[5].defined()) k_weight = same(s[5], {d.dim}, d.weight_dtype, dev, what).contiguous();
        const Tensor gq = rows_16(grads[0]), gk = rows_16(grads[1]);
        d.ld_q = q.stride(0);
        d.ld_k = k.stride(0);
        d.ld_gq = gq.stride(0);
        d.ld_gk = gk.stride(0);
        Tensor dq = plain(q), dk = plain(k), dpos, dqw, dkw, ws;
        if (ctx->needs_input_grad(2)) dpos = plain(positions);
        // (inputs count where they are given)
        if (q_weight.defined() && ctx->needs_input_grad(4)) dqw = plain(q_weight);
        if (k_weight.defined() && ctx->needs_input_grad(q_weight.defined() ? 5 : 4)) dkw = plain(k_weight);
        size_t n = 0;
        if (dqw.defined() || dkw.defined()) ws = bytes(n = dg.rotate_workspace_size(&d), q);
        check(dg.rotate_backward(&d, q.data_ptr(), k.data_ptr(), positions.data_ptr(), (const float*)frequencies.data_ptr(), ptr(q_weight),
                                 ptr(k_weight), gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), ptr(dpos), ptr(dqw), ptr(dkw),
                                 ptr(ws), n, stream_of(q)), "rotate_heads");
        return once({dq, dk, dpos, Tensor(), dqw, dkw, Tensor()}, "rotate_heads");
    }
};

std::tuple<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& frequencies,
                                  const OptTensor& q_weight_, const OptTensor& k_weight_, const std::vector<int32_t>& sections, double eps,
                                  bool norm, bool interleaved)
{
    c10::OptionalDeviceGuard guard(q.device());
    const Tensor at = positions.contiguous(), f = frequencies.contiguous();
    Tensor qw = value(q_weight_), kw = value(k_weight_);
    if (qw.defined()) qw = qw.contiguous();
    if (kw.defined()) kw = kw.contiguous();
    dg_rotate_desc d = {};
    d.n_targets = q.size(0);
    d.n_nodes = k.size(0);
    d.heads = (int32_t)q.size(1);
    d.kv_heads = (int32_t)k.size(1);
    d.dim = (int32_t)q.size(2);
    d.axes = (int32_t)at.size(1);
    for (size_t i = 0; i < sections.size() && i < 8; ++i) d.sections[i] = sections[i];
    d.dtype = type_of(q);
    d.weight_dtype = qw.defined() ? type_of(qw) : kw.defined() ? type_of(kw) : d.dtype;
    d.pos_dtype = type_of(at);
    d.norm = norm;
    d.interleaved = interleaved;
    d.eps = (float)eps;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || at.requires_grad() || wanted(qw) || wanted(kw))) {
        auto out = Rotate::apply(q, k, at, f, maybe(qw), maybe(kw), text(&d, sizeof d));
        return {out[0], out[1]};
    }
    return rotate_forward(d, rows_16(q), rows_16(k), at, f, qw, kw);
}

// ---------------------------------------------------------------- route_rows

variable_list route_forward(const dg_route_desc& d, const Tensor& logits, const Tensor& bias)
{
    const auto o = logits.options();
    Tensor weights = at::empty({d.n_rows, d.k}, o.dtype(at::kFloat)), experts = at::empty({d.n_rows, d.k}, o.dtype(at::kInt));
    Tensor places = at::empty({d.n_rows, d.k}, o.dtype(at::kInt)), sizes = at::empty({d.n_experts}, o.dtype(at::kLong));
    const size_t n = dg.route_workspace_size(&d);
    Tensor ws = bytes(n, logits);
    check(dg.route_forward(&d, logits.data_ptr(), (const float*)ptr(bias), (float*)weights.data_ptr(), (int32_t*)experts.data_ptr(),
                           (int64_t*)sizes.data_ptr(), (int32_t*)places.data_ptr(), ws.data_ptr(), n, stream_of(logits)), "route_rows");
    return {weights, experts, sizes, places};
}

struct Route : torch::autograd::Function<Route> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& bias, std::string desc)
    {
        dg_route_desc d;
        memcpy(&d, desc.data(), sizeof d);
        auto out = route_forward(d, logits, value(bias));
        ctx->save_for_backward({logits, out[1]});
        ctx->saved_data["desc"] = desc;
        ctx->mark_non_differentiable({out[1], out[2], out[3]});
        ctx->set_materialize_grads(false);  // (zeros for the outputs without one are three launches)
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const auto s = ctx->get_saved_variables();
        const at::Device dev = grads[0].device();
        c10::OptionalDeviceGuard guard(dev);
        dg_route_desc d;
        memcpy(&d, ctx->saved_data["desc"].toStringRef().data(), sizeof d);
        const Tensor logits = whole_rows(same(s[0], {d.n_rows, d.n_experts}, d.dtype, dev, "route_rows"));
        const Tensor experts = same(s[1], {d.n_rows, d.k}, DG_I32, dev, "route_rows").contiguous();
        d.ld = logits.stride(0);
        Tensor g = grads[0].contiguous(), dlogits = plain(logits);
        check(dg.route_backward(&d, logits.data_ptr(), (const int32_t*)experts.data_ptr(), (const float*)g.data_ptr(), dlogits.data_ptr(),
                                stream_of(g)), "route_rows");
        return once({dlogits, Tensor(), Tensor()}, "route_rows");
    }
};

variable_list route(const Tensor& logits_, const OptTensor& bias_, int k, bool sigmoid, int groups, int top_groups, int group_best,
                    bool renormalize, double scale)
{
    c10::OptionalDeviceGuard guard(logits_.device());
    const Tensor logits = whole_rows(logits_);
    Tensor bias = value(bias_);
    if (bias.defined()) bias = bias.detach().to(at::kFloat).contiguous();
    dg_route_desc d = {};
    d.n_rows = logits.size(0);
    d.ld = logits.stride(0);
    d.n_experts = (int32_t)logits.size(1);
    d.k = k;
    d.groups = groups;
    d.top_groups = top_groups;
    d.group_best = group_best;
    d.sigmoid = sigmoid;
    d.renormalize = renormalize;
    d.dtype = type_of(logits);
    d.scale = (float)scale;
    if (at::GradMode::is_enabled() && logits.requires_grad()) return Route::apply(logits, maybe(bias), text(&d, sizeof d));
    return route_forward(d, logits, bias);
}

// ---------------------------------------------------------------- dispatch_rows, combine_rows

dg_exchange_desc exchange_of(const Tensor& places, int64_t ld, int64_t width, const Tensor& t)
{
    dg_exchange_desc d = {};
    d.n_rows = places.size(0);
    d.k = (int32_t)places.size(1);
    d.ld = ld;
    d.width = (int32_t)width;
    d.dtype = type_of(t);
    return d;
}

Tensor dispatch_forward(const Tensor& x, const Tensor& places)
{
    Tensor out = at::empty({places.size(0) * places.size(1), x.size(1)}, x.options());
    const auto d = exchange_of(places, x.stride(0), x.size(1), x);
    check(dg.exchange_dispatch(&d, x.data_ptr(), (const int32_t*)places.data_ptr(), out.data_ptr(), stream_of(x)), "dispatch_rows");
    return out;
}

Tensor combine_forward(const Tensor& y, const Tensor& places, const Tensor& weights, const Tensor& residual, const char* what)
{
    Tensor out = at::empty({places.size(0), y.size(1)}, y.options());
    const auto d = exchange_of(places, residual.defined() ? residual.stride(0) : 0, y.size(1), y);
    check(dg.exchange_combine(&d, y.data_ptr(), (const int32_t*)places.data_ptr(), (const float*)ptr(weights), ptr(residual), out.data_ptr(),
                              stream_of(y)), what);
    return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& places)
    {
        ctx->save_for_backward({places});
        ctx->saved_data["rows"] = places.size(0);
        return dispatch_forward(x, places);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const at::Device dev = grads[0].device();
        c10::OptionalDeviceGuard guard(dev);
        const auto s = ctx->get_saved_variables();
        const int64_t rows = ctx->saved_data["rows"].toInt(), k = rows ? grads[0].size(0) / rows : s[0].size(1);
        const Tensor places = same(s[0], {rows, k}, DG_I32, dev, "dispatch_rows").contiguous();
        return once({combine_forward(grads[0].contiguous(), places, Tensor(), Tensor(), "dispatch_rows"), Tensor()}, "dispatch_rows");
    }
};

Tensor dispatch(const Tensor& x_, const Tensor& places)
{
    c10::OptionalDeviceGuard guard(x_.device());
    const Tensor x = whole_rows(x_), p = places.contiguous();
    return at::GradMode::is_enabled() && x.requires_grad() ? Dispatch::apply(x, p) : dispatch_forward(x, p);
}

struct Combine : torch::autograd::Function<Combine> {
    static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& weights, const Tensor& places,
                          const OptTensor& residual)
    {
        ctx->save_for_backward({y, weights, places});
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["k"] = places.size(1);
        return combine_forward(y, places, weights, value(residual), "combine_rows");
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const at::Device dev = grads[0].device();
        c10::OptionalDeviceGuard guard(dev);
        const char* const what = "combine_rows";
        const int64_t rows = grads[0].size(0), k = ctx->saved_data["k"].toInt();
        const Tensor y = same(s[0], {rows * k, grads[0].size(1)}, type_of(grads[0]), dev, what).contiguous();
        const Tensor weights = same(s[1], {rows, k}, DG_F32, dev, what).contiguous();
        const Tensor places = same(s[2], {rows, k}, DG_I32, dev, what).contiguous();
        Tensor dy, dw, dr;
        if (ctx->needs_input_grad(0)) dy = plain(y);
        if (ctx->needs_input_grad(1)) dw = plain(weights);
        const Tensor g = whole_rows(grads[0]);
        const auto d = exchange_of(places, g.stride(0), y.size(1), y);
        check(dg.exchange_combine_backward(&d, y.data_ptr(), (const int32_t*)places.data_ptr(), (const float*)weights.data_ptr(),
                                           g.data_ptr(), ptr(dy), (float*)ptr(dw), stream_of(y)), "combine_rows");
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(3)) dr = grads[0];
        return once({dy, dw, Tensor(), dr}, "combine_rows");
    }
};

Tensor combine(const Tensor& y_, const Tensor& weights_, const OptTensor& residual_, const Tensor& places)
{
    c10::OptionalDeviceGuard guard(y_.device());
    const Tensor y = y_.contiguous(), weights = weights_.contiguous(), p = places.contiguous();
    Tensor residual = value(residual_);
    if (residual.defined()) residual = whole_rows(residual);
    if (at::GradMode::is_enabled() && (y.requires_grad() || weights.requires_grad() || wanted(residual)))
        return Combine::apply(y, weights, p, maybe(residual));
    return combine_forward(y, p, weights, residual, "combine_rows");
}

// ---------------------------------------------------------------- grouped_linear with an activation or a residual

dg_grouped_desc grouped_of(const Tensor& x, const Tensor& weight)
{
    dg_grouped_desc d = {};
    d.n_rows = x.size(0);
    d.n_groups = weight.size(0);
    d.k = (int32_t)weight.size(2);
    d.n = (int32_t)weight.size(1);
    d.dtype = type_of(x);
    return d;
}

Tensor grouped_forward(const Tensor& x, const Tensor& weight, const Tensor& sizes, const Tensor& bias, int act, const Tensor& residual)
{
    Tensor y = at::empty({x.size(0), weight.size(1)}, x.options());
    const auto d = grouped_of(x, weight);
    check(dg.grouped_apply(&d, act, x.data_ptr(), weight.data_ptr(), (const int64_t*)sizes.data_ptr(), ptr(bias), ptr(residual), y.data_ptr(),
                           stream_of(x)), "grouped_linear");
    return y;
}

struct Grouped : torch::autograd::Function<Grouped> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& sizes, const OptTensor& bias_,
                          int64_t act, const OptTensor& residual)
    {
        const Tensor bias = value(bias_);
        // (the backward pass makes z again)
        ctx->save_for_backward({x, weight, sizes, bias});
        ctx->saved_data["act"] = act;
        ctx->saved_data["groups"] = weight.size(0);
        ctx->saved_data["k"] = weight.size(2);
        ctx->saved_data["residual"] = residual.has_value();
        return grouped_forward(x, weight, sizes, bias, (int)act, value(residual));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const auto s = ctx->get_saved_variables();
        const at::Device dev = grads[0].device();
        c10::OptionalDeviceGuard guard(dev);
        const char* const what = "grouped_linear";
        const int64_t rows = grads[0].size(0), n = grads[0].size(1);
        const int64_t groups = ctx->saved_data["groups"].toInt(), depth = ctx->saved_data["k"].toInt();
        const int32_t type = type_of(grads[0]);
        const Tensor x = same(s[0], {rows, depth}, type, dev, what).contiguous();
        const Tensor weight = same(s[1], {groups, n, depth}, type, dev, what).contiguous();
        const Tensor sizes = same(s[2], {groups}, DG_I64, dev, what).contiguous();
        Tensor bias;
        if (s[3].defined()) bias = same(s[3], {groups, n}, type, dev, what).contiguous();
        const int act = (int)ctx->saved_data["act"].toInt();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = bias.defined() && ctx->needs_input_grad(3);
        Tensor dx, dw, db, ws, dr;
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(bias.defined() ? 4 : 3)) dr = grads[0];
        if (need_x || need_w || need_b) {
            const auto d = grouped_of(x, weight);
            const Tensor g = grads[0].contiguous();
            if (need_x) dx = plain(x);
            if (need_w || need_b) dw = plain(weight);
            if (need_b) db = plain(bias);
            // (dz, and what the sums of the weight's gradient need)
            const size_t sums = dg.grouped_workspace_size(&d);
            const size_t size = (act == DG_ACT_NONE ? sums : dg.grouped_apply_workspace_size(&d)) - (need_w || need_b ? 0 : sums);
            if (size) ws = bytes(size, x);
            check(dg.grouped_apply_gradients(&d, act, x.data_ptr(), weight.data_ptr(), (const int64_t*)sizes.data_ptr(), ptr(bias),
                                             g.data_ptr(), ptr(dx), ptr(dw), ptr(db), ptr(ws), size, stream_of(x)),
                  "grouped_linear");
        }
        return once({dx, need_w ? dw : Tensor(), Tensor(), db, Tensor(), dr}, "grouped_linear");
    }
};

Tensor grouped_apply(const Tensor& x_, const Tensor& weight_, const Tensor& sizes_, const OptTensor& bias_, int act, const OptTensor& residual_)
{
    c10::OptionalDeviceGuard guard(x_.device());
    const Tensor x = x_.contiguous(), weight = weight_.contiguous(), sizes = sizes_.contiguous();
    Tensor bias = value(bias_), residual = value(residual_);
    if (bias.defined()) bias = bias.contiguous();
    if (residual.defined()) residual = residual.contiguous();
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wanted(bias) || wanted(residual)))
        return Grouped::apply(x, weight, sizes, maybe(bias), (int64_t)act, maybe(residual));
    return grouped_forward(x, weight, sizes, bias, act, residual);
}

}  // namespace

PYBIND11_MODULE(_torch_layer, m)
{
    m.def("load", &load);
    // (the interpreter's lock is not needed: other threads may go on while kernels are enqueued)
    const auto free = py::call_guard<py::gil_scoped_release>();
    m.def("rotate", &rotate, free);
    m.def("route", &route, free);
    m.def("dispatch", &dispatch, free);
    m.def("combine", &combine, free);
    m.def("grouped_apply", &grouped_apply, free);
}
