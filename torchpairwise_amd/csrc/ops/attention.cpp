// Attention and rotary positions: argument checks, the public composites, the CPU forms in
// elementary ATen operations, the GPU forms on the C ABI, and the autograd functions.
//   attention        -> _attention -> _attention_backward (probabilities formed again)
//   rotary_embedding -> _rotary    -> _rotary (turned back)
#include <torch/autograd.h>

#include <cmath>
#include <limits>

#include "tpw_attention.h"

namespace tpw_ext {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

using Results = std::tuple<at::Tensor, at::Tensor, at::Tensor>;

constexpr int64_t kMaxFeatures = 256;

at::Tensor like_dims(const at::Tensor &x4, const at::Tensor &ref) {
    return ref.dim() == 2 ? x4.squeeze(0).squeeze(0) : ref.dim() == 3 ? x4.squeeze(1) : x4;
}

Operands check_attention(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value,
                         const OptTensor &mask, const OptTensor &lengths) {
    const char *name = "attention";
    TORCH_CHECK(query.dim() >= 2 && query.dim() <= 4, name, ": expected 2-D, 3-D or 4-D tensors, got query of ",
                query.dim(), " dimensions");
    TORCH_CHECK(key.dim() == query.dim() && value.dim() == query.dim(), name,
                ": query, key and value must have the same number of dimensions");
    TORCH_CHECK(key.device() == query.device() && value.device() == query.device(), name,
                ": query, key and value are on different devices");
    TORCH_CHECK(key.scalar_type() == query.scalar_type() && value.scalar_type() == query.scalar_type(), name,
                ": query, key and value dtypes differ");
    const auto t = query.scalar_type();
    TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || (query.is_cpu() && t == at::kDouble), name,
                ": supports float32 and bfloat16", query.is_cpu() ? " and float64" : " on the GPU", ", got ", t);
    Operands o;
    o.q = as4(query);
    o.k = as4(key);
    o.v = as4(value);
    o.batch = o.q.size(0), o.heads = o.q.size(1), o.n = o.q.size(2), o.d = o.q.size(3);
    o.key_heads = o.k.size(1), o.m = o.k.size(2), o.dv = o.v.size(3);
    TORCH_CHECK(o.k.size(0) == o.batch && o.v.size(0) == o.batch, name,
                ": batch_size of query, key and value do not match.");
    TORCH_CHECK(o.k.size(3) == o.d, name, ": feature dimension of query and key do not match.");
    TORCH_CHECK(o.v.size(2) == o.m, name, ": number of keys and values do not match.");
    TORCH_CHECK(o.v.size(1) == o.key_heads, name, ": heads of key and value do not match.");
    TORCH_CHECK(o.key_heads >= 1 && o.heads % o.key_heads == 0, name,
                ": the number of query heads must be a multiple of the number of key heads, got ", o.heads, " and ",
                o.key_heads);
    TORCH_CHECK(o.d >= 1 && o.d <= kMaxFeatures && o.dv >= 1 && o.dv <= kMaxFeatures, name,
                ": rows must have 1 to ", kMaxFeatures, " features, got ", o.d, " and ", o.dv);
    check_mask_and_lengths(name, o, query, mask, lengths);
    return o;
}

// ------------------------------------------------------------------ CPU
// Additive form of what leaves keys out, in the compute type: 0 or the mask's value where a key is
// left, -inf elsewhere; undefined where every key is left.
at::Tensor additive_mask(const Operands &o, bool causal, at::ScalarType t) {
    at::Tensor add;
    const auto opts = o.q.options().dtype(t);
    const double inf = std::numeric_limits<double>::infinity();
    const auto exclude = [&](const at::Tensor &off) {
        if (!add.defined()) add = at::zeros({1, 1, 1, 1}, opts);
        add = at::where(off, at::full({}, -inf, opts), add);
    };
    if (o.mask.defined()) {
        if (o.mask.scalar_type() == at::kBool)
            exclude(o.mask.logical_not());
        else
            add = o.mask.to(t);
    }
    const auto index = o.q.options().dtype(at::kLong);
    auto j = at::arange(o.m, index);
    auto len = o.lengths.defined() ? o.lengths.clamp(0, o.m).view({o.batch, 1, 1, 1})
                                   : at::full({1, 1, 1, 1}, o.m, index);
    if (o.lengths.defined()) exclude(j >= len);
    if (causal) exclude(j - at::arange(o.n, index).unsqueeze(1) > len - o.n);
    return add;
}

// Rows of the heads that share a key head are rows of one product.
at::Tensor grouped(const at::Tensor &x, const Operands &o, at::ScalarType t) {
    return x.to(t).reshape({o.batch, o.key_heads, o.heads / o.key_heads * o.n, x.size(3)});
}
// Rows past the lengths are not read: zeros in their place.
at::Tensor live_rows(const at::Tensor &x, const Operands &o, at::ScalarType t) {
    auto y = x.to(t);
    if (!o.lengths.defined()) return y;
    auto off = at::arange(o.m, o.lengths.options()) >= o.lengths.view({o.batch, 1});
    return y.masked_fill(off.view({o.batch, 1, o.m, 1}), 0.0);
}
at::Tensor masked_scores(const at::Tensor &q, const at::Tensor &k, const Operands &o, bool causal, double scale) {
    auto s = at::matmul(q, k.transpose(-1, -2)).mul_(scale).view({o.batch, o.heads, o.n, o.m});
    auto add = additive_mask(o, causal, s.scalar_type());
    if (!add.defined()) return s;
    // a key that is left out stays out whatever its score
    return at::where(add == -std::numeric_limits<double>::infinity(), add, s + add);
}
at::ScalarType compute_type(const at::Tensor &x) { return x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

Results attention_cpu(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const OptTensor &mask,
                      const OptTensor &lengths, bool causal, double scale, bool train) {
    const Operands o = check_attention(query, key, value, mask, lengths);
    const auto t = compute_type(query);
    auto stats = at::zeros({2, o.batch, o.heads, o.n}, query.options().dtype(t));
    auto out = empty_rows({o.batch, o.heads, o.n, o.dv}, o.q);
    auto rest = at::empty({0}, out.options());
    if (train && out.scalar_type() == at::kBFloat16) rest = at::zeros_like(out);
    if (out.numel() == 0 || o.m == 0) return {like_dims(out.zero_(), query), stats, rest};
    auto s = masked_scores(grouped(o.q, o, t), live_rows(o.k, o, t), o, causal, scale);
    auto top = s.amax(-1, true);
    auto base = top.masked_fill(top == -std::numeric_limits<double>::infinity(), 0.0);
    auto p = (s - base).exp_();
    auto sum = p.sum(-1, true);
    auto acc = at::matmul(p.reshape({o.batch, o.key_heads, -1, o.m}), live_rows(o.v, o, t)).view(out.sizes());
    acc = acc / sum.masked_fill(sum == 0, 1.0);
    out.copy_(acc);
    if (rest.numel() > 0) rest.copy_(acc - out);
    stats.select(0, 0).copy_(base.squeeze(-1));
    stats.select(0, 1).copy_(sum.squeeze(-1));
    return {like_dims(out, query), stats, rest};
}

Results attention_backward_cpu(
    const at::Tensor &grad, const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const at::Tensor &out,
    const at::Tensor &stats, const at::Tensor &rest, const OptTensor &mask, const OptTensor &lengths, bool causal,
    double scale) {
    const Operands o = check_attention(query, key, value, mask, lengths);
    TORCH_CHECK(grad.sizes() == out.sizes(), "attention: gradient of shape ", grad.sizes(), " for an output of ",
                out.sizes());
    const auto t = compute_type(query);
    if (o.q.numel() == 0 || o.m == 0)
        return {at::zeros_like(query), at::zeros_like(key), at::zeros_like(value)};
    auto q = grouped(o.q, o, t), k = live_rows(o.k, o, t), v = live_rows(o.v, o, t);
    auto s = masked_scores(q, k, o, causal, scale);
    auto off = s == -std::numeric_limits<double>::infinity();
    auto base = stats.select(0, 0).unsqueeze(-1), sum = stats.select(0, 1).unsqueeze(-1);
    auto p = (s - base).exp_().div_(sum.masked_fill(sum == 0, 1.0));
    auto g4 = as4(grad).to(t);
    auto g = grouped(g4, o, t);
    auto o4 = as4(out).to(t);
    if (rest.numel() > 0) o4 = o4 + rest;
    auto delta = (g4 * o4).sum(-1, true);
    auto dp = at::matmul(g, v.transpose(-1, -2)).view(p.sizes());
    auto ds = (p * (dp - delta)).masked_fill_(off, 0.0).mul_(scale).reshape({o.batch, o.key_heads, -1, o.m});
    auto pg = p.reshape(ds.sizes());
    auto gq = at::matmul(ds, k).view({o.batch, o.heads, o.n, o.d});
    auto gk = at::matmul(ds.transpose(-1, -2), q), gv = at::matmul(pg.transpose(-1, -2), g);
    return {like_dims(gq.to(query.scalar_type()), query), like_dims(gk.to(key.scalar_type()), key),
            like_dims(gv.to(value.scalar_type()), value)};
}

at::Tensor turns_of(const at::Tensor &positions, const at::Tensor &frequencies, int64_t batch, int64_t n) {
    auto p = positions.dim() == 1 ? positions.unsqueeze(0) : positions;
    return (p.expand({batch, n}).to(at::kDouble).unsqueeze(-1) * frequencies.to(at::kDouble)).unsqueeze(1);
}

void check_rotary(const at::Tensor &x, const at::Tensor &positions, const at::Tensor &frequencies, double scale) {
    const char *name = "rotary_embedding";
    TORCH_CHECK(x.dim() >= 2 && x.dim() <= 4, name, ": expected a 2-D, 3-D or 4-D tensor, got ", x.dim(), " dimensions");
    const auto t = x.scalar_type();
    TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || (x.is_cpu() && t == at::kDouble), name,
                ": supports float32 and bfloat16", x.is_cpu() ? " and float64" : " on the GPU", ", got ", t);
    TORCH_CHECK(positions.device() == x.device() && frequencies.device() == x.device(), name,
                ": positions and frequencies must be on the device of x");
    TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, name,
                ": positions must be int64 or int32, got ", positions.scalar_type());
    const int64_t n = x.size(-2), batch = x.dim() == 2 ? 1 : x.size(0);
    TORCH_CHECK((positions.dim() == 1 && positions.size(0) == n) ||
                    (positions.dim() == 2 && positions.size(1) == n &&
                     (positions.size(0) == batch || positions.size(0) == 1)),
                name, ": positions must have shape [n] or [batch_size, n], got ", positions.sizes());
    const auto ft = frequencies.scalar_type();
    TORCH_CHECK(frequencies.dim() == 1 && (ft == at::kDouble || ft == at::kFloat),
                name, ": frequencies must be a float64 or float32 vector");
    TORCH_CHECK(2 * frequencies.size(0) <= x.size(-1), name, ": ", frequencies.size(0), " pairs do not fit rows of ",
                x.size(-1), " features");
    TORCH_CHECK(std::isfinite(scale) && std::fabs(scale) <= 3e38, name, ": scale must be finite");
}

at::Tensor rotary_cpu(const at::Tensor &x, const at::Tensor &positions, const at::Tensor &frequencies, bool interleaved,
                      double scale, bool inverse) {
    check_rotary(x, positions, frequencies, scale);
    const auto t = compute_type(x);
    auto x4 = as4(x);
    const int64_t pairs = frequencies.size(0);
    auto angle = turns_of(positions, frequencies, x4.size(0), x4.size(2));
    auto c = angle.cos().mul_(scale).to(t), s = angle.sin().mul_(inverse ? -scale : scale).to(t);
    auto r = x4.narrow(3, 0, 2 * pairs).to(t);
    at::Tensor y;
    if (interleaved) {
        auto z = r.unflatten(-1, {pairs, 2});
        auto u = z.select(-1, 0), w = z.select(-1, 1);
        y = at::stack({u * c - w * s, u * s + w * c}, -1).flatten(-2);
    } else {
        auto u = r.narrow(3, 0, pairs), w = r.narrow(3, pairs, pairs);
        y = at::cat({u * c - w * s, u * s + w * c}, -1);
    }
    auto out = empty_rows(x4.sizes(), x4);
    out.narrow(3, 0, 2 * pairs).copy_(y);
    out.narrow(3, 2 * pairs, x4.size(3) - 2 * pairs).copy_(x4.narrow(3, 2 * pairs, x4.size(3) - 2 * pairs));
    return like_dims(out, x);
}

// ------------------------------------------------------------------ GPU
tpw_attention_desc describe(const Operands &o, bool causal, double scale) {
    tpw_attention_desc a = {};
    a.dtype = o.q.scalar_type() == at::kFloat ? TPW_F32 : TPW_BF16;
    a.causal = causal;
    a.batch = o.batch, a.heads = o.heads, a.key_heads = o.key_heads;
    a.n = o.n, a.m = o.m, a.d = o.d, a.dv = o.dv;
    a.scale = scale;
    a.query = o.q.data_ptr(), a.key = o.k.data_ptr(), a.value = o.v.data_ptr();
    set_strides(a.query_strides, o.q);
    set_strides(a.key_strides, o.k);
    set_strides(a.value_strides, o.v);
    describe_mask(a, o);
    return a;
}

Results attention_cuda(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const OptTensor &mask,
                       const OptTensor &lengths, bool causal, double scale, bool train) {
    Operands o = check_attention(query, key, value, mask, lengths);
    DeviceGuard guard(query.device());
    auto out = empty_rows({o.batch, o.heads, o.n, o.dv}, o.q);
    // what only the backward reads
    at::Tensor stats = train ? at::empty({2, o.batch, o.heads, o.n}, query.options().dtype(at::kFloat))
                             : at::empty({0}, query.options().dtype(at::kFloat));
    at::Tensor rest = train && out.scalar_type() == at::kBFloat16
                          ? at::empty_strided(out.sizes(), out.strides(), out.options())
                          : at::empty({0}, out.options());
    if (out.numel() > 0) {
        o.q = dense_rows(o.q, false);
        o.k = dense_rows(o.k, true);
        o.v = dense_rows(o.v, true);
        auto a = describe(o, causal, scale);
        a.out = out.data_ptr();
        set_strides(a.out_strides, out);
        if (train) a.stats = stats.data_ptr<float>();
        if (rest.numel() > 0) a.out_rest = rest.data_ptr();
        const size_t bytes = tpw_attention_workspace_size(&a);
        at::Tensor ws;
        if (bytes > 0) ws = workspace(bytes, query);
        check_rc(tpw_attention(&a, bytes > 0 ? ws.data_ptr() : nullptr, current_stream()), "_attention");
    }
    return {like_dims(out, query), stats, rest};
}

Results attention_backward_cuda(
    const at::Tensor &grad, const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const at::Tensor &out,
    const at::Tensor &stats, const at::Tensor &rest, const OptTensor &mask, const OptTensor &lengths, bool causal,
    double scale) {
    Operands o = check_attention(query, key, value, mask, lengths);
    TORCH_CHECK(grad.sizes() == out.sizes(), "attention: gradient of shape ", grad.sizes(), " for an output of ",
                out.sizes());
    TORCH_CHECK(out.scalar_type() == query.scalar_type() && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                    stats.numel() == 2 * o.batch * o.heads * o.n && out.device() == query.device() &&
                    stats.device() == query.device() && grad.device() == query.device(),
                "_attention_backward: out and stats must be what the forward returned");
    DeviceGuard guard(query.device());
    auto gq = empty_rows(o.q.sizes(), o.q), gk = empty_rows(o.k.sizes(), o.k), gv = empty_rows(o.v.sizes(), o.v);
    if (gq.numel() + gk.numel() > 0) {
        o.q = dense_rows(o.q, true);
        o.k = dense_rows(o.k, true);
        o.v = dense_rows(o.v, true);
        auto g4 = dense_rows(as4(grad.to(query.scalar_type())), true), o4 = as4(out);
        const auto fits = [&](const at::Tensor &r) {
            bool same = r.sizes() == o4.sizes() && r.scalar_type() == out.scalar_type() && r.device() == out.device();
            for (int i = 0; same && i < 4; ++i) same = r.size(i) == 1 || r.stride(i) == o4.stride(i);
            return same;
        };
        TORCH_CHECK((rest.numel() == 0 || fits(rest)) && (o4.size(3) == 1 || o4.stride(3) == 1),
                    "_attention_backward: out and rest must be what the forward returned");
        TORCH_CHECK(o4.size(0) == o.batch && o4.size(1) == o.heads && o4.size(2) == o.n && o4.size(3) == o.dv,
                    "_attention_backward: out must be what the forward returned");
        auto a = describe(o, causal, scale);
        a.out = o4.data_ptr();
        set_strides(a.out_strides, o4);
        if (rest.numel() > 0) a.out_rest = rest.data_ptr();
        a.stats = stats.data_ptr<float>();
        a.grad_out = g4.data_ptr();
        set_strides(a.grad_out_strides, g4);
        a.grad_query = gq.data_ptr(), a.grad_key = gk.data_ptr(), a.grad_value = gv.data_ptr();
        set_strides(a.grad_query_strides, gq);
        set_strides(a.grad_key_strides, gk);
        set_strides(a.grad_value_strides, gv);
        auto ws = workspace(tpw_attention_backward_workspace_size(&a), query);
        check_rc(tpw_attention_backward(&a, ws.data_ptr(), current_stream()), "_attention_backward");
    }
    return {like_dims(gq, query), like_dims(gk, key), like_dims(gv, value)};
}

at::Tensor rotary_cuda(const at::Tensor &x, const at::Tensor &positions, const at::Tensor &frequencies, bool interleaved,
                       double scale, bool inverse) {
    check_rotary(x, positions, frequencies, scale);
    DeviceGuard guard(x.device());
    auto x4 = dense_rows(as4(x), false);
    auto out = empty_rows(x4.sizes(), x4);
    if (out.numel() > 0) {
        auto p = positions.to(at::kLong);
        auto f = frequencies.to(at::kDouble).contiguous();
        const bool shared = p.dim() == 1 || p.size(0) == 1;
        const int64_t ps[2] = {shared ? 0 : p.stride(0), p.stride(-1)};
        int64_t xs[3], os[3];
        set_strides(xs, x4);
        set_strides(os, out);
        check_rc(tpw_rotary(x4.data_ptr(), x.scalar_type() == at::kFloat ? TPW_F32 : TPW_BF16, x4.size(0), x4.size(1),
                            x4.size(2), x4.size(3), xs, p.data_ptr<int64_t>(), ps, f.data_ptr<double>(), f.size(0),
                            interleaved, inverse, scale, out.data_ptr(), os, current_stream()),
                 "_rotary");
    }
    return like_dims(out, x);
}

}  // namespace

// ------------------------------------------------------------------ dispatch
Results attention_op(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const OptTensor &mask,
                     const OptTensor &lengths, bool causal, double scale, bool train) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torchpairwise::_attention", "")
                         .typed<Results(const at::Tensor &, const at::Tensor &, const at::Tensor &, const OptTensor &,
                                        const OptTensor &, bool, double, bool)>();
    return op.call(q, k, v, mask, lengths, causal, scale, train);
}

namespace {

Results attention_backward_op(const at::Tensor &grad, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v,
                              const at::Tensor &out, const at::Tensor &stats, const at::Tensor &rest, const OptTensor &mask,
                              const OptTensor &lengths, bool causal, double scale) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torchpairwise::_attention_backward", "")
                         .typed<Results(const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                        const at::Tensor &, const at::Tensor &, const at::Tensor &, const OptTensor &,
                                        const OptTensor &, bool, double)>();
    return op.call(grad, q, k, v, out, stats, rest, mask, lengths, causal, scale);
}
at::Tensor rotary_op(const at::Tensor &x, const at::Tensor &positions, const at::Tensor &frequencies, bool interleaved,
                     double scale, bool inverse) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torchpairwise::_rotary", "")
                         .typed<at::Tensor(const at::Tensor &, const at::Tensor &, const at::Tensor &, bool, double, bool)>();
    return op.call(x, positions, frequencies, interleaved, scale, inverse);
}

at::Tensor attention(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const OptTensor &mask,
                     bool causal, c10::optional<double> scale, const OptTensor &lengths) {
    const double s = attention_scale("attention", query, scale);
    return std::get<0>(attention_op(query, key, value, mask, lengths, causal, s, false));
}

at::Tensor rotary_embedding(const at::Tensor &x, const at::Tensor &positions, const at::Tensor &frequencies,
                            bool interleaved, double scale) {
    return rotary_op(x, positions, frequencies, interleaved, scale, false);
}

// ------------------------------------------------------------------ autograd
class AttentionFunction : public torch::autograd::Function<AttentionFunction> {
   public:
    static variable_list forward(AutogradContext *ctx, const Variable &query, const Variable &key, const Variable &value,
                                 const OptTensor &mask, const OptTensor &lengths, bool causal, double scale) {
        at::AutoDispatchBelowADInplaceOrView g;
        auto r = attention_op(query, key, value, mask, lengths, causal, scale, true);
        auto out = std::get<0>(r), stats = std::get<1>(r), rest = std::get<2>(r);
        ctx->save_for_backward({query, key, value, out, stats, rest, mask.has_value() ? *mask : at::Tensor(),
                                lengths.has_value() ? *lengths : at::Tensor()});
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        ctx->mark_non_differentiable({stats, rest});
        return {out, stats, rest};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "attention: second derivatives are not implemented");
        auto s = ctx->get_saved_variables();
        const auto opt = [](const at::Tensor &x) { return x.defined() ? OptTensor(x) : OptTensor(); };
        auto grad = grads[0].defined() ? grads[0] : at::zeros_like(s[3]);
        auto g = attention_backward_op(grad, s[0], s[1], s[2], s[3], s[4], s[5], opt(s[6]), opt(s[7]),
                                       ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
        return {std::get<0>(g), std::get<1>(g), std::get<2>(g), Variable(), Variable(), Variable(), Variable()};
    }
};

class RotaryFunction : public torch::autograd::Function<RotaryFunction> {
   public:
    static Variable forward(AutogradContext *ctx, const Variable &x, const Variable &positions, const Variable &frequencies,
                            bool interleaved, double scale, bool inverse) {
        at::AutoDispatchBelowADInplaceOrView g;
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["inverse"] = inverse;
        return rotary_op(x, positions, frequencies, interleaved, scale, inverse);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        auto s = ctx->get_saved_variables();
        auto g = rotary_op(grads[0], s[0], s[1], ctx->saved_data["interleaved"].toBool(),
                           ctx->saved_data["scale"].toDouble(), !ctx->saved_data["inverse"].toBool());
        return {g, Variable(), Variable(), Variable(), Variable(), Variable()};
    }
};

// Below autograd a tangent would be lost without a word.
void refuse_tangent(const at::Tensor &x) {
    TORCH_CHECK(!x.defined() || !x._fw_grad(0).defined(), "attention: forward-mode derivatives are not implemented");
}

Results attention_autograd(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value, const OptTensor &mask,
                           const OptTensor &lengths, bool causal, double scale, bool train) {
    refuse_tangent(query);
    refuse_tangent(key);
    refuse_tangent(value);
    if (mask.has_value()) refuse_tangent(*mask);
    const bool grad = at::GradMode::is_enabled();
    TORCH_CHECK(!(grad && mask.has_value() && mask->defined() && mask->requires_grad()),
                "attention: the mask has no gradient; pass mask.detach()");
    // The operands decide, whatever a recorded call was made on.
    if (!train && !(grad && (query.requires_grad() || key.requires_grad() || value.requires_grad()))) {
        at::AutoDispatchBelowADInplaceOrView g;
        return attention_op(query, key, value, mask, lengths, causal, scale, false);
    }
    auto r = AttentionFunction::apply(query, key, value, mask, lengths, causal, scale);
    return {r[0], r[1], r[2]};
}
at::Tensor rotary_autograd(const at::Tensor &x, const at::Tensor &positions, const at::Tensor &frequencies,
                           bool interleaved, double scale, bool inverse) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && frequencies.requires_grad()),
                "rotary_embedding: frequencies have no gradient; pass frequencies.detach()");
    return RotaryFunction::apply(x, positions, frequencies, interleaved, scale, inverse);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torchpairwise, m) {
    m.def("attention(Tensor query, Tensor key, Tensor value, Tensor? mask=None, *, bool causal=False, "
          "float? scale=None, Tensor? lengths=None) -> Tensor",
          TORCH_FN(attention));
    m.def("rotary_embedding(Tensor x, Tensor positions, Tensor frequencies, *, bool interleaved=False, "
          "float scale=1.0) -> Tensor",
          TORCH_FN(rotary_embedding));
    m.def("_attention(Tensor query, Tensor key, Tensor value, Tensor? mask, Tensor? lengths, bool causal, "
          "float scale, bool train) -> (Tensor out, Tensor stats, Tensor rest)");
    m.def("_attention_backward(Tensor grad, Tensor query, Tensor key, Tensor value, Tensor out, Tensor stats, "
          "Tensor rest, Tensor? mask, Tensor? lengths, bool causal, float scale) -> (Tensor, Tensor, Tensor)");
    m.def("_rotary(Tensor x, Tensor positions, Tensor frequencies, bool interleaved, float scale, "
          "bool inverse) -> Tensor");
}

TORCH_LIBRARY_IMPL(torchpairwise, CPU, m) {
    m.impl("_attention", TORCH_FN(attention_cpu));
    m.impl("_attention_backward", TORCH_FN(attention_backward_cpu));
    m.impl("_rotary", TORCH_FN(rotary_cpu));
}

TORCH_LIBRARY_IMPL(torchpairwise, CUDA, m) {
    m.impl("_attention", TORCH_FN(attention_cuda));
    m.impl("_attention_backward", TORCH_FN(attention_backward_cuda));
    m.impl("_rotary", TORCH_FN(rotary_cuda));
}

TORCH_LIBRARY_IMPL(torchpairwise, Autograd, m) {
    m.impl("_attention", TORCH_FN(attention_autograd));
    m.impl("_rotary", TORCH_FN(rotary_autograd));
}

}  // namespace tpw_ext
