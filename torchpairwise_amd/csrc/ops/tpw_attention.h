// What the attention ops share (attention.cpp, cache.cpp): operands, their layout, the mask and the lengths.
#pragma once

#include <cmath>

#include "tpw_common.h"

namespace tpw_ext {

using OptTensor = c10::optional<at::Tensor>;

// Rows as [batch, heads, n, features]: 2-D is one batch entry of one head, 3-D one head.
inline at::Tensor as4(const at::Tensor &x) {
    return x.dim() == 2 ? x.unsqueeze(0).unsqueeze(0) : x.dim() == 3 ? x.unsqueeze(1) : x;
}
// New rows in the order of `ref` (both [batch, heads, rows, features]): rows before heads where ref
// has them so, as a transposed view of a dense tensor.
inline at::Tensor empty_rows(at::IntArrayRef sizes, const at::Tensor &ref) {
    if (ref.size(1) > 1 && ref.size(2) > 1 && ref.stride(1) < ref.stride(2))
        return at::empty({sizes[0], sizes[2], sizes[1], sizes[3]}, ref.options()).transpose(1, 2);
    return at::empty(sizes, ref.options());
}

struct Operands {
    at::Tensor q, k, v;          // 4-D
    at::Tensor mask;             // [batch, heads, n, m] (expanded) or undefined
    at::Tensor lengths;          // int64 [batch] or undefined
    int64_t batch, heads, key_heads, n, m, d, dv;
};

// Reads a call's mask and lengths into its operands, whose sizes are known.
inline void check_mask_and_lengths(const char *name, Operands &o, const at::Tensor &query, const OptTensor &mask,
                                   const OptTensor &lengths) {
    if (mask.has_value() && mask->defined()) {
        const at::Tensor &w = *mask;
        TORCH_CHECK(w.device() == query.device(), name, ": mask is on another device");
        TORCH_CHECK(w.scalar_type() == at::kBool || w.scalar_type() == at::kFloat || w.scalar_type() == at::kBFloat16 ||
                        (w.is_cpu() && w.scalar_type() == at::kDouble),
                    name, ": mask must be bool (true: kept), or float32 or bfloat16 (added), got ", w.scalar_type());
        auto want = query.sizes().vec();
        want.back() = o.m;
        TORCH_CHECK(w.dim() <= query.dim() && at::is_expandable_to(w.sizes(), want), name,
                    ": mask of shape ", w.sizes(), " does not broadcast to ", at::IntArrayRef(want));
        o.mask = as4(w.expand(want));
    }
    if (lengths.has_value() && lengths->defined()) {
        const at::Tensor &l = *lengths;
        TORCH_CHECK(l.device() == query.device(), name, ": lengths are on another device");
        TORCH_CHECK(l.dim() == 1 && l.size(0) == o.batch, name, ": lengths must have shape [batch_size], got ",
                    l.sizes());
        TORCH_CHECK(l.scalar_type() == at::kLong || l.scalar_type() == at::kInt, name,
                    ": lengths must be int64 or int32, got ", l.scalar_type());
        o.lengths = l.to(at::kLong).contiguous();
    }
}

// Features dense; with `streamed`, rows neither overlap nor lie more than the kernels' reach apart.
inline at::Tensor dense_rows(const at::Tensor &x, bool streamed) {
    const bool dense = x.size(3) == 1 || x.stride(3) == 1;
    const bool apart = !streamed || x.size(2) <= 1 ||
                       (x.stride(2) >= x.size(3) && x.stride(2) * x.element_size() <= (int64_t(1) << 23));
    return dense && apart ? x : x.contiguous();
}
inline void set_strides(int64_t (&s)[3], const at::Tensor &x) {
    for (int i = 0; i < 3; ++i) s[i] = x.stride(i);
}

inline void describe_mask(tpw_attention_desc &a, const Operands &o) {
    if (o.mask.defined()) {
        const auto t = o.mask.scalar_type();
        a.mask_type = t == at::kBool ? TPW_MASK_KEEP : t == at::kFloat ? TPW_MASK_ADD_F32 : TPW_MASK_ADD_BF16;
        a.mask = o.mask.data_ptr();
        for (int i = 0; i < 4; ++i) a.mask_strides[i] = o.mask.stride(i);
    }
    if (o.lengths.defined()) a.lengths = o.lengths.data_ptr<int64_t>();
}

// 1 / sqrt(features) where none is given.
inline double attention_scale(const char *name, const at::Tensor &query, c10::optional<double> scale) {
    const double s = scale.has_value() ? *scale
                     : query.dim() > 0 && query.size(-1) > 0 ? 1.0 / std::sqrt((double)query.size(-1))
                                                             : 1.0;
    TORCH_CHECK(std::isfinite(s) && std::fabs(s) <= 1e30, name, ": scale must be finite, got ", s);
    return s;
}

// (out, stats, rest) through the dispatcher (attention.cpp).
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_op(const at::Tensor &q, const at::Tensor &k,
                                                            const at::Tensor &v, const OptTensor &mask,
                                                            const OptTensor &lengths, bool causal, double scale,
                                                            bool train);

}  // namespace tpw_ext
