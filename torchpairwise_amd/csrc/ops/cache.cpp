// A cache of keys and values in 4 or 8 bits: argument checks, the public composites, the CPU forms in
// elementary ATen operations, and the GPU forms on the C ABI.
//   cache_attention -> _cache_attention (CPU: the cache read, then attention)
#include <ATen/MemoryOverlap.h>
#include <torch/csrc/autograd/variable.h>

#include <limits>

#include "tpw_attention.h"

namespace tpw_ext {
namespace {

constexpr int64_t kBlock = 32;  // features that share a scale

struct CacheTensors {
    at::Tensor key_codes, key_scales, value_codes, value_scales;
    at::Tensor pages;  // [batch, pages of a sequence], int32 or int64; or undefined
    int64_t bits, batch, heads, rows, capacity, key_blocks, value_blocks;
};

CacheTensors check_cache(const char *name, const at::Tensor &key_codes, const at::Tensor &key_scales,
                         const at::Tensor &value_codes, const at::Tensor &value_scales, const OptTensor &pages,
                         int64_t batch) {
    CacheTensors c{key_codes, key_scales, value_codes, value_scales, at::Tensor(), 0, batch, 0, 0, 0, 0, 0};
    const auto t = key_codes.scalar_type();
    TORCH_CHECK(t == at::kByte || t == at::kFloat8_e4m3fn, name,
                ": codes must be uint8 (4 bits) or float8_e4m3fn (8 bits), got ", t);
    c.bits = t == at::kByte ? 4 : 8;
    const int64_t bytes = kBlock * c.bits / 8;
    TORCH_CHECK(value_codes.scalar_type() == t, name, ": codes of keys and values differ in dtype");
    for (const at::Tensor *x : {&key_codes, &key_scales, &value_codes, &value_scales}) {
        TORCH_CHECK(x->dim() == 4, name, ": codes and scales must be 4-D, got ", x->dim(), " dimensions");
        TORCH_CHECK(x->device() == key_codes.device(), name, ": codes and scales are on different devices");
        TORCH_CHECK(x->stride(3) == 1 || x->size(3) <= 1, name, ": codes and scales must be dense in the last dimension");
        for (int i = 0; i < 3; ++i)
            TORCH_CHECK(x->stride(i) % 16 == 0 || x->size(i) <= 1 || x->numel() == 0, name,
                        ": codes and scales must have strides in multiples of 16, got ", x->strides());
        TORCH_CHECK(x->is_cpu() || reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0, name,
                    ": codes and scales must start at 16-byte aligned addresses");
    }
    TORCH_CHECK(key_scales.scalar_type() == at::kByte && value_scales.scalar_type() == at::kByte, name,
                ": scales must be uint8");
    c.heads = key_codes.size(1);
    c.rows = key_codes.size(2);
    TORCH_CHECK(c.heads >= 1, name, ": a cache has at least one head");
    TORCH_CHECK(c.rows % 16 == 0, name, ": rows of a cache come in multiples of 16, got ", c.rows);
    const auto side = [&](const at::Tensor &codes, const at::Tensor &scales) {
        const int64_t blocks = codes.size(3) / bytes;
        TORCH_CHECK(codes.size(3) % bytes == 0 && blocks >= 1 && blocks <= 8, name,
                    ": codes of a row must be 1 to 8 blocks of ", bytes, " bytes, got ", codes.size(3), " bytes");
        TORCH_CHECK(codes.size(0) == key_codes.size(0) && codes.size(1) == c.heads && codes.size(2) == c.rows, name,
                    ": codes of keys and values differ in shape");
        TORCH_CHECK(scales.size(0) == codes.size(0) && scales.size(1) == c.heads && scales.size(2) == blocks &&
                        scales.size(3) == c.rows,
                    name, ": scales must have shape ", at::IntArrayRef({codes.size(0), c.heads, blocks, c.rows}), ", got ",
                    scales.sizes());
        return blocks;
    };
    c.key_blocks = side(key_codes, key_scales);
    c.value_blocks = side(value_codes, value_scales);
    c.capacity = c.rows;
    if (pages.has_value() && pages->defined()) {
        const at::Tensor &p = *pages;
        TORCH_CHECK(p.device() == key_codes.device(), name, ": pages are on another device");
        TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, name,
                    ": pages must be int32 or int64, got ", p.scalar_type());
        TORCH_CHECK(p.dim() == 2 && p.size(0) == batch, name, ": pages must have shape [batch_size, pages], got ",
                    p.sizes());
        TORCH_CHECK(c.rows >= 16 && (c.rows & (c.rows - 1)) == 0 && c.rows <= (int64_t(1) << 20), name,
                    ": pages have a power of two of rows, 16 to 2^20, got ", c.rows);
        c.pages = p.size(1) <= 1 || p.stride(1) == 1 ? p : p.contiguous();
        c.capacity = p.size(1) * c.rows;
    } else {
        TORCH_CHECK(key_codes.size(0) == batch, name, ": the cache holds ", key_codes.size(0), " sequences, the call ",
                    batch);
    }
    TORCH_CHECK(c.capacity < (int64_t(1) << 31) - 1024, name, ": too many rows");
    return c;
}

at::Tensor check_index(const char *name, const char *what, const OptTensor &x, int64_t batch, const at::Tensor &like) {
    if (!x.has_value() || !x->defined()) return {};
    TORCH_CHECK(x->device() == like.device(), name, ": ", what, " are on another device");
    TORCH_CHECK(x->dim() == 1 && x->size(0) == batch, name, ": ", what, " must have shape [batch_size], got ", x->sizes());
    TORCH_CHECK(x->scalar_type() == at::kLong || x->scalar_type() == at::kInt, name, ": ", what,
                " must be int64 or int32, got ", x->scalar_type());
    return x->to(at::kLong).contiguous();
}

void check_rows_type(const char *name, at::ScalarType t) {
    TORCH_CHECK(t == at::kFloat || t == at::kBFloat16, name, ": supports float32 and bfloat16, got ", t);
}

// ------------------------------------------------------------------ CPU
// Entry of the first dimension (-1: no place) and row of rows starts + i, [batch, n] each.
std::pair<at::Tensor, at::Tensor> places(const CacheTensors &c, const at::Tensor &starts, const at::Tensor &counts,
                                         int64_t n) {
    const auto index = c.key_codes.options().dtype(at::kLong);
    auto i = at::arange(n, index).unsqueeze(0).expand({c.batch, n});
    auto j = starts.defined() ? i + starts.unsqueeze(1) : i;
    auto in = (j >= 0).logical_and(j < c.capacity);
    if (counts.defined()) in = in.logical_and(i < counts.unsqueeze(1));
    j = at::where(in, j, at::zeros({}, index));
    auto first = at::arange(c.batch, index).unsqueeze(1).expand({c.batch, n}), row = j;
    if (c.pages.defined()) {
        if (c.pages.size(1) == 0 || c.key_codes.size(0) == 0) return {at::full({c.batch, n}, -1, index), at::zeros_like(j)};
        first = c.pages.to(at::kLong).gather(1, at::floor_divide(j, c.rows));
        row = at::remainder(j, c.rows);
        in = in.logical_and(first >= 0).logical_and(first < c.key_codes.size(0));
    }
    return {at::where(in, first, at::full({}, -1, index)), row};
}

// 2^(byte - 127) for byte < 255, NaN for 255.
at::Tensor power_of(const at::Tensor &byte) {
    auto b = byte.to(at::kInt);
    auto bits = at::where(b == 0, at::full({}, 0x00400000, b.options()), at::bitwise_left_shift(b, 23));
    bits = at::where(b == 255, at::full({}, 0x7fc00000, b.options()), bits);
    return bits.view(at::kFloat);
}

// Codes [..., n, bytes] and scales [..., n, blocks] of rows x [..., n, d].
std::pair<at::Tensor, at::Tensor> quantise(const at::Tensor &x, int64_t bits, int64_t blocks) {
    auto y = at::constant_pad_nd(x.to(at::kFloat), {0, kBlock * blocks - x.size(-1)}).unflatten(-1, {blocks, kBlock});
    auto top = std::get<0>(at::bitwise_and(y.contiguous().view(at::kInt), 0x7fffffff).max(-1));
    auto e = bits == 4 ? at::bitwise_right_shift(top + 0x200000, 23) - 2 : at::bitwise_right_shift(top + 0x180000, 23) - 8;
    auto finite = top < 0x7f800000;
    auto byte = at::where(finite, e.clamp_min(0), at::full({}, 255, e.options()));
    // times 2^(127 - byte): exact but below the normal range, where every code is zero
    y = y * power_of(254 - byte.clamp_max(253)).unsqueeze(-1);
    y = at::where(finite.unsqueeze(-1), y, at::zeros({}, y.options())).flatten(-2);
    if (bits == 8) return {y.to(at::kFloat8_e4m3fn), byte.to(at::kByte)};
    auto a = y.abs();
    auto step = at::where(a < 2, at::full({}, 0.5, a.options()), at::where(a < 4, at::ones({}, a.options()),
                                                                           at::full({}, 2.0, a.options())));
    auto code = at::bucketize((a / step).round() * step, at::tensor({0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f}), true);
    code = (code + at::signbit(y).to(at::kInt) * 8).unflatten(-1, {-1, 2});
    return {(code.select(-1, 0) + code.select(-1, 1) * 16).to(at::kByte), byte.to(at::kByte)};
}

// float32 values [..., width] of codes [..., bytes] and scales [..., blocks].
at::Tensor values_of(const at::Tensor &codes, const at::Tensor &scales, int64_t bits, int64_t width) {
    at::Tensor x;
    if (bits == 8) {
        x = codes.to(at::kFloat);
    } else {
        auto table = at::tensor({0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f});
        table = at::cat({table, -table});
        auto both = at::stack({at::bitwise_and(codes, 15), at::bitwise_right_shift(codes, 4)}, -1).flatten(-2);
        x = table.index({both.to(at::kLong)});
    }
    x = x.unflatten(-1, {-1, kBlock}) * power_of(scales).unsqueeze(-1);
    return x.flatten(-2).narrow(-1, 0, width);
}

// Rows at (first, row) [batch, n] as float32 [batch, heads, n, width]; zeros where first < 0.
at::Tensor rows_at(const at::Tensor &codes, const at::Tensor &scales, int64_t bits, int64_t width, const at::Tensor &first,
                   const at::Tensor &row) {
    if (codes.size(0) == 0 || codes.size(2) == 0)
        return at::zeros({first.size(0), codes.size(1), first.size(1), width}, scales.options().dtype(at::kFloat));
    auto at_first = first.clamp_min(0);
    // float8 has no indexing of its own: bytes
    auto c = codes.view(at::kByte).transpose(1, 2).index({at_first, row}).view(codes.scalar_type());
    auto s = scales.permute({0, 3, 1, 2}).index({at_first, row});
    auto x = values_of(c, s, bits, width).transpose(1, 2);
    return x.masked_fill((first < 0).unsqueeze(1).unsqueeze(-1), 0.0);
}

int64_t batch_of(const char *name, const at::Tensor &key, const at::Tensor &value) {
    TORCH_CHECK(key.dim() == 4 && value.dim() == 4, name, ": expected 4-D key and value, got ", key.dim(), " and ",
                value.dim(), " dimensions");
    return key.size(0);
}

struct RowTensors {
    at::Tensor key, value, starts, counts;
};
RowTensors check_rows(const char *name, const CacheTensors &c, const at::Tensor &key, const at::Tensor &value,
                      const OptTensor &starts, const OptTensor &counts) {
    TORCH_CHECK(key.device() == c.key_codes.device() && value.device() == key.device(), name,
                ": key, value and the cache are on different devices");
    TORCH_CHECK(key.scalar_type() == value.scalar_type(), name, ": key and value dtypes differ");
    check_rows_type(name, key.scalar_type());
    TORCH_CHECK(key.size(1) == c.heads && value.size(1) == c.heads, name, ": the cache has ", c.heads, " heads, got ",
                key.size(1), " and ", value.size(1));
    TORCH_CHECK(value.size(0) == key.size(0) && value.size(2) == key.size(2), name,
                ": number of keys and values do not match.");
    const auto fits = [&](const at::Tensor &x, int64_t blocks) {
        return x.size(3) >= 1 && (x.size(3) + kBlock - 1) / kBlock == blocks;
    };
    TORCH_CHECK(fits(key, c.key_blocks) && fits(value, c.value_blocks), name, ": rows of ", key.size(3), " and ",
                value.size(3), " features do not fill the cache's ", c.key_blocks, " and ", c.value_blocks,
                " blocks of 32");
    return {key, value, check_index(name, "starts", starts, c.batch, key), check_index(name, "counts", counts, c.batch, key)};
}

// Rows that several others share cannot be written, nor keys where the values go, nor what is read meanwhile.
void check_written(const CacheTensors &c, const RowTensors &r) {
    const at::Tensor *all[] = {&c.key_codes, &c.key_scales, &c.value_codes, &c.value_scales};
    for (int i = 0; i < 4; ++i) {
        at::assert_no_internal_overlap(*all[i]);
        for (int j = 0; j < i; ++j) at::assert_no_overlap(*all[i], *all[j]);
        for (const at::Tensor *x : {&r.key, &r.value, &r.starts, &r.counts, &c.pages})
            if (x->defined()) at::assert_no_overlap(*all[i], *x);
    }
}

void cache_write_cpu(at::Tensor &key_codes, at::Tensor &key_scales, at::Tensor &value_codes, at::Tensor &value_scales,
                     const at::Tensor &key, const at::Tensor &value, const at::Tensor &starts, const OptTensor &counts,
                     const OptTensor &pages) {
    const char *name = "cache_write_";
    const auto c = check_cache(name, key_codes, key_scales, value_codes, value_scales, pages,
                               batch_of(name, key, value));
    const auto r = check_rows(name, c, key, value, starts, counts);
    check_written(c, r);
    auto at = places(c, r.starts, r.counts, key.size(2));
    auto live = (at.first >= 0).flatten().nonzero().flatten();
    if (live.numel() == 0) return;
    auto first = at.first.flatten().index({live}), row = at.second.flatten().index({live});
    const auto put = [&](at::Tensor codes, at::Tensor scales, const at::Tensor &x, int64_t blocks) {
        auto q = quantise(x.transpose(1, 2).flatten(0, 1).index({live}), c.bits, blocks);
        codes.view(at::kByte).transpose(1, 2).index_put_({first, row}, q.first.view(at::kByte));
        scales.permute({0, 3, 1, 2}).index_put_({first, row}, q.second);
    };
    put(key_codes, key_scales, key, c.key_blocks);
    put(value_codes, value_scales, value, c.value_blocks);
}

using Pair = std::tuple<at::Tensor, at::Tensor>;

struct ReadCall {
    CacheTensors c;
    at::Tensor starts, counts;
    int64_t n, key_width, value_width;
    at::ScalarType dtype;
};
ReadCall check_read(const at::Tensor &key_codes, const at::Tensor &key_scales, const at::Tensor &value_codes,
                    const at::Tensor &value_scales, c10::optional<int64_t> key_width, c10::optional<int64_t> value_width,
                    c10::optional<at::ScalarType> dtype, const OptTensor &starts, c10::optional<int64_t> rows, const OptTensor &counts,
                    const OptTensor &pages) {
    const char *name = "cache_read";
    const int64_t batch = pages.has_value() && pages->defined() && pages->dim() == 2 ? pages->size(0)
                          : key_codes.dim() == 4                                      ? key_codes.size(0)
                                                                                      : 0;
    ReadCall r{check_cache(name, key_codes, key_scales, value_codes, value_scales, pages, batch), {}, {}, 0, 0, 0,
               dtype.value_or(at::kBFloat16)};
    check_rows_type(name, r.dtype);
    r.starts = check_index(name, "starts", starts, batch, key_codes);
    r.counts = check_index(name, "counts", counts, batch, key_codes);
    r.n = rows.has_value() ? *rows : r.c.capacity;
    TORCH_CHECK(r.n >= 0 && r.n < (int64_t(1) << 31), name, ": invalid number of rows, ", r.n);
    const auto width = [&](c10::optional<int64_t> w, int64_t blocks) {
        const int64_t x = w.has_value() ? *w : kBlock * blocks;
        TORCH_CHECK(x >= 1 && x <= kBlock * blocks, name, ": ", x, " features of a cache of ", kBlock * blocks);
        return x;
    };
    r.key_width = width(key_width, r.c.key_blocks);
    r.value_width = width(value_width, r.c.value_blocks);
    return r;
}

Pair cache_read_cpu(const at::Tensor &key_codes, const at::Tensor &key_scales, const at::Tensor &value_codes,
                    const at::Tensor &value_scales, c10::optional<int64_t> key_width, c10::optional<int64_t> value_width,
                    c10::optional<at::ScalarType> dtype, const OptTensor &starts, c10::optional<int64_t> rows, const OptTensor &counts,
                    const OptTensor &pages) {
    const auto r = check_read(key_codes, key_scales, value_codes, value_scales, key_width, value_width, dtype, starts, rows,
                              counts, pages);
    auto at = places(r.c, r.starts, r.counts, r.n);
    return {rows_at(key_codes, key_scales, r.c.bits, r.key_width, at.first, at.second).to(r.dtype).contiguous(),
            rows_at(value_codes, value_scales, r.c.bits, r.value_width, at.first, at.second).to(r.dtype).contiguous()};
}

struct AttentionCall {
    CacheTensors c;
    Operands o;  // q, mask, lengths and sizes
};
AttentionCall check_call(const at::Tensor &query, const at::Tensor &key_codes, const at::Tensor &key_scales,
                         const at::Tensor &value_codes, const at::Tensor &value_scales, const OptTensor &mask,
                         const OptTensor &lengths, const OptTensor &pages, c10::optional<int64_t> value_width) {
    const char *name = "cache_attention";
    TORCH_CHECK(query.dim() == 4, name, ": expected a 4-D query, got ", query.dim(), " dimensions");
    AttentionCall a{check_cache(name, key_codes, key_scales, value_codes, value_scales, pages, query.size(0)), {}};
    const auto &c = a.c;
    Operands &o = a.o;
    TORCH_CHECK(query.device() == key_codes.device(), name, ": query and the cache are on different devices");
    check_rows_type(name, query.scalar_type());
    o.q = query;
    o.batch = query.size(0), o.heads = query.size(1), o.n = query.size(2), o.d = query.size(3);
    o.key_heads = c.heads, o.m = c.capacity;
    TORCH_CHECK(o.heads % o.key_heads == 0, name,
                ": the number of query heads must be a multiple of the number of key heads, got ", o.heads, " and ",
                o.key_heads);
    TORCH_CHECK(o.d >= 1 && (o.d + kBlock - 1) / kBlock == c.key_blocks, name, ": queries of ", o.d,
                " features for keys of ", c.key_blocks, " blocks of 32");
    if (value_width.has_value()) {
        o.dv = *value_width;
    } else {
        TORCH_CHECK(c.value_blocks == c.key_blocks, name, ": value_width is needed where values are not as wide as keys");
        o.dv = o.d;
    }
    TORCH_CHECK(o.dv >= 1 && (o.dv + kBlock - 1) / kBlock == c.value_blocks, name, ": value_width ", o.dv,
                " for values of ", c.value_blocks, " blocks of 32");
    check_mask_and_lengths(name, o, query, mask, lengths);
    return a;
}

at::Tensor cache_attention_cpu(const at::Tensor &query, const at::Tensor &key_codes, const at::Tensor &key_scales,
                               const at::Tensor &value_codes, const at::Tensor &value_scales, const OptTensor &mask,
                               const OptTensor &lengths, const OptTensor &pages, bool causal, double scale,
                               c10::optional<int64_t> value_width) {
    const auto a = check_call(query, key_codes, key_scales, value_codes, value_scales, mask, lengths, pages, value_width);
    const auto &c = a.c;
    auto at = places(c, {}, a.o.lengths, c.capacity);
    auto k = rows_at(key_codes, key_scales, c.bits, a.o.d, at.first, at.second).to(query.scalar_type());
    auto v = rows_at(value_codes, value_scales, c.bits, a.o.dv, at.first, at.second).to(query.scalar_type());
    OptTensor keep = mask;
    if (c.pages.defined()) {  // rows without a place are no keys
        auto there = (at.first >= 0).view({c.batch, 1, 1, c.capacity});
        if (!mask.has_value() || !mask->defined())
            keep = there;
        else if (mask->scalar_type() == at::kBool)
            keep = mask->logical_and(there);
        else
            keep = at::where(there, *mask, at::full({}, -std::numeric_limits<double>::infinity(), mask->options()));
    }
    return std::get<0>(attention_op(query, k, v, keep, lengths, causal, scale, false));
}

// ------------------------------------------------------------------ GPU
tpw_cache_desc describe(const CacheTensors &c) {
    tpw_cache_desc d = {};
    d.bits = (int32_t)c.bits;
    d.first = c.key_codes.size(0), d.heads = c.heads, d.rows = c.rows;
    d.key_blocks = c.key_blocks, d.value_blocks = c.value_blocks;
    d.key_codes = c.key_codes.data_ptr(), d.key_scales = c.key_scales.data_ptr();
    d.value_codes = c.value_codes.data_ptr(), d.value_scales = c.value_scales.data_ptr();
    const auto strides = [](int64_t (&s)[3], const at::Tensor &x) {
        for (int i = 0; i < 3; ++i) s[i] = x.size(i) <= 1 ? 0 : x.stride(i);
    };
    strides(d.key_code_strides, c.key_codes);
    strides(d.key_scale_strides, c.key_scales);
    strides(d.value_code_strides, c.value_codes);
    strides(d.value_scale_strides, c.value_scales);
    if (c.pages.defined()) {
        d.pages = c.pages.data_ptr();
        d.pages_wide = c.pages.scalar_type() == at::kLong;
        d.page_pitch = c.pages.stride(0);
        d.page_count = c.pages.size(1);
    }
    return d;
}
int type_code(const at::Tensor &x) { return x.scalar_type() == at::kFloat ? TPW_F32 : TPW_BF16; }

void cache_write_cuda(at::Tensor &key_codes, at::Tensor &key_scales, at::Tensor &value_codes, at::Tensor &value_scales,
                      const at::Tensor &key, const at::Tensor &value, const at::Tensor &starts, const OptTensor &counts,
                      const OptTensor &pages) {
    const char *name = "cache_write_";
    const auto c = check_cache(name, key_codes, key_scales, value_codes, value_scales, pages,
                               batch_of(name, key, value));
    auto r = check_rows(name, c, key, value, starts, counts);
    check_written(c, r);
    if (key.size(0) * key.size(2) == 0 || c.capacity == 0 || key_codes.size(0) == 0) return;
    DeviceGuard guard(key.device());
    r.key = dense_rows(r.key, false);
    r.value = dense_rows(r.value, false);
    const auto d = describe(c);
    int64_t ks[3], vs[3];
    set_strides(ks, r.key);
    set_strides(vs, r.value);
    check_rc(tpw_cache_write(&d, type_code(key), c.batch, key.size(2), r.key.data_ptr(), key.size(3), ks,
                             r.value.data_ptr(), value.size(3), vs, r.starts.data_ptr<int64_t>(),
                             r.counts.defined() ? r.counts.data_ptr<int64_t>() : nullptr, current_stream()),
             "cache_write_");
}

Pair cache_read_cuda(const at::Tensor &key_codes, const at::Tensor &key_scales, const at::Tensor &value_codes,
                     const at::Tensor &value_scales, c10::optional<int64_t> key_width, c10::optional<int64_t> value_width,
                     c10::optional<at::ScalarType> dtype, const OptTensor &starts, c10::optional<int64_t> rows, const OptTensor &counts,
                     const OptTensor &pages) {
    const auto r = check_read(key_codes, key_scales, value_codes, value_scales, key_width, value_width, dtype, starts, rows,
                              counts, pages);
    DeviceGuard guard(key_codes.device());
    const auto opts = key_scales.options().dtype(r.dtype);
    auto key = at::empty({r.c.batch, r.c.heads, r.n, r.key_width}, opts);
    auto value = at::empty({r.c.batch, r.c.heads, r.n, r.value_width}, opts);
    if (key.numel() == 0) return {key, value};
    if (r.c.capacity == 0 || key_codes.size(0) == 0) return {key.zero_(), value.zero_()};
    const auto d = describe(r.c);
    int64_t ks[3], vs[3];
    set_strides(ks, key);
    set_strides(vs, value);
    check_rc(tpw_cache_read(&d, type_code(key), r.c.batch, r.n, key.data_ptr(), r.key_width, ks, value.data_ptr(),
                            r.value_width, vs, r.starts.defined() ? r.starts.data_ptr<int64_t>() : nullptr,
                            r.counts.defined() ? r.counts.data_ptr<int64_t>() : nullptr, current_stream()),
             "cache_read");
    return {key, value};
}

at::Tensor cache_attention_cuda(const at::Tensor &query, const at::Tensor &key_codes, const at::Tensor &key_scales,
                                const at::Tensor &value_codes, const at::Tensor &value_scales, const OptTensor &mask,
                                const OptTensor &lengths, const OptTensor &pages, bool causal, double scale,
                                c10::optional<int64_t> value_width) {
    auto call = check_call(query, key_codes, key_scales, value_codes, value_scales, mask, lengths, pages, value_width);
    auto &o = call.o;
    DeviceGuard guard(query.device());
    auto out = empty_rows({o.batch, o.heads, o.n, o.dv}, o.q);
    if (out.numel() == 0) return out;
    if (o.m == 0 || key_codes.size(0) == 0) return out.zero_();
    o.q = dense_rows(o.q, false);
    const auto d = describe(call.c);
    tpw_attention_desc a = {};
    a.dtype = type_code(o.q);
    a.causal = causal;
    a.batch = o.batch, a.heads = o.heads, a.key_heads = o.key_heads;
    a.n = o.n, a.m = o.m, a.d = o.d, a.dv = o.dv;
    a.scale = scale;
    a.query = o.q.data_ptr();
    set_strides(a.query_strides, o.q);
    describe_mask(a, o);
    a.out = out.data_ptr();
    set_strides(a.out_strides, out);
    const size_t bytes = tpw_cache_attention_workspace_size(&a, &d);
    at::Tensor ws;
    if (bytes > 0) ws = workspace(bytes, o.q);
    check_rc(tpw_cache_attention(&a, &d, bytes > 0 ? ws.data_ptr() : nullptr, current_stream()), "_cache_attention");
    return out;
}

// ------------------------------------------------------------------ dispatch
using WriteFn = void(at::Tensor &, at::Tensor &, at::Tensor &, at::Tensor &, const at::Tensor &, const at::Tensor &,
                     const at::Tensor &, const OptTensor &, const OptTensor &);
using AttentionFn = at::Tensor(const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                               const at::Tensor &, const OptTensor &, const OptTensor &, const OptTensor &, bool, double,
                               c10::optional<int64_t>);
void write_op(at::Tensor &kc, at::Tensor &ks, at::Tensor &vc, at::Tensor &vs, const at::Tensor &key,
              const at::Tensor &value, const at::Tensor &starts, const OptTensor &counts, const OptTensor &pages) {
    static auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("torchpairwise::cache_write_", "").typed<WriteFn>();
    op.call(kc, ks, vc, vs, key, value, starts, counts, pages);
}
at::Tensor cache_attention_op(const at::Tensor &query, const at::Tensor &kc, const at::Tensor &ks, const at::Tensor &vc,
                              const at::Tensor &vs, const OptTensor &mask, const OptTensor &lengths, const OptTensor &pages,
                              bool causal, double scale, c10::optional<int64_t> value_width) {
    static auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("torchpairwise::_cache_attention", "").typed<AttentionFn>();
    return op.call(query, kc, ks, vc, vs, mask, lengths, pages, causal, scale, value_width);
}

at::Tensor cache_attention(const at::Tensor &query, const at::Tensor &kc, const at::Tensor &ks, const at::Tensor &vc,
                           const at::Tensor &vs, const OptTensor &mask, bool causal, c10::optional<double> scale,
                           const OptTensor &lengths, const OptTensor &pages, c10::optional<int64_t> value_width) {
    const double s = attention_scale("cache_attention", query, scale);
    return cache_attention_op(query, kc, ks, vc, vs, mask, lengths, pages, causal, s, value_width);
}

// ------------------------------------------------------------------ autograd
// Codes have no gradient; below autograd one would be lost without a word.
void refuse_gradient(const char *name, const at::Tensor &x) {
    if (!x.defined()) return;
    TORCH_CHECK(!(at::GradMode::is_enabled() && x.requires_grad()), name,
                ": a cache has no gradient; pass detached tensors, or call under torch.no_grad()");
    TORCH_CHECK(!x._fw_grad(0).defined(), name, ": forward-mode derivatives are not implemented");
}
void cache_write_autograd(at::Tensor &kc, at::Tensor &ks, at::Tensor &vc, at::Tensor &vs, const at::Tensor &key,
                          const at::Tensor &value, const at::Tensor &starts, const OptTensor &counts,
                          const OptTensor &pages) {
    refuse_gradient("cache_write_", key);
    refuse_gradient("cache_write_", value);
    refuse_gradient("cache_write_", kc);
    refuse_gradient("cache_write_", vc);
    {
        at::AutoDispatchBelowADInplaceOrView g;
        write_op(kc, ks, vc, vs, key, value, starts, counts, pages);
    }
    for (const at::Tensor *x : {&kc, &ks, &vc, &vs})
        if (!x->is_inference()) torch::autograd::impl::bump_version(*x);
}
Pair cache_read_autograd(const at::Tensor &kc, const at::Tensor &ks, const at::Tensor &vc, const at::Tensor &vs,
                         c10::optional<int64_t> key_width, c10::optional<int64_t> value_width,
                         c10::optional<at::ScalarType> dtype,
                         const OptTensor &starts, c10::optional<int64_t> rows, const OptTensor &counts,
                         const OptTensor &pages) {
    refuse_gradient("cache_read", kc);
    refuse_gradient("cache_read", vc);
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow("torchpairwise::cache_read", "")
                         .typed<Pair(const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                     c10::optional<int64_t>, c10::optional<int64_t>, c10::optional<at::ScalarType>,
                                     const OptTensor &,
                                     c10::optional<int64_t>, const OptTensor &, const OptTensor &)>();
    at::AutoDispatchBelowADInplaceOrView g;
    return op.call(kc, ks, vc, vs, key_width, value_width, dtype, starts, rows, counts, pages);
}
at::Tensor cache_attention_autograd(const at::Tensor &query, const at::Tensor &kc, const at::Tensor &ks,
                                    const at::Tensor &vc, const at::Tensor &vs, const OptTensor &mask,
                                    const OptTensor &lengths, const OptTensor &pages, bool causal, double scale,
                                    c10::optional<int64_t> value_width) {
    refuse_gradient("cache_attention", query);
    refuse_gradient("cache_attention", kc);
    refuse_gradient("cache_attention", vc);
    if (mask.has_value()) refuse_gradient("cache_attention", *mask);
    at::AutoDispatchBelowADInplaceOrView g;
    return cache_attention_op(query, kc, ks, vc, vs, mask, lengths, pages, causal, scale, value_width);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(torchpairwise, m) {
    m.def("cache_attention(Tensor query, Tensor key_codes, Tensor key_scales, Tensor value_codes, Tensor value_scales, "
          "Tensor? mask=None, *, bool causal=False, float? scale=None, Tensor? lengths=None, Tensor? pages=None, "
          "int? value_width=None) -> Tensor",
          TORCH_FN(cache_attention));
    m.def("cache_write_(Tensor(a!) key_codes, Tensor(b!) key_scales, Tensor(c!) value_codes, Tensor(d!) value_scales, "
          "Tensor key, Tensor value, Tensor starts, *, Tensor? counts=None, Tensor? pages=None) -> ()");
    m.def("cache_read(Tensor key_codes, Tensor key_scales, Tensor value_codes, Tensor value_scales, *, "
          "int? key_width=None, int? value_width=None, ScalarType? dtype=None, Tensor? starts=None, int? rows=None, "
          "Tensor? counts=None, Tensor? pages=None) -> (Tensor key, Tensor value)");
    m.def("_cache_attention(Tensor query, Tensor key_codes, Tensor key_scales, Tensor value_codes, Tensor value_scales, "
          "Tensor? mask, Tensor? lengths, Tensor? pages, bool causal, float scale, int? value_width) -> Tensor");
}

TORCH_LIBRARY_IMPL(torchpairwise, CPU, m) {
    m.impl("cache_write_", TORCH_FN(cache_write_cpu));
    m.impl("cache_read", TORCH_FN(cache_read_cpu));
    m.impl("_cache_attention", TORCH_FN(cache_attention_cpu));
}

TORCH_LIBRARY_IMPL(torchpairwise, CUDA, m) {
    m.impl("cache_write_", TORCH_FN(cache_write_cuda));
    m.impl("cache_read", TORCH_FN(cache_read_cuda));
    m.impl("_cache_attention", TORCH_FN(cache_attention_cuda));
}

TORCH_LIBRARY_IMPL(torchpairwise, Autograd, m) {
    m.impl("cache_write_", TORCH_FN(cache_write_autograd));
    m.impl("cache_read", TORCH_FN(cache_read_autograd));
    m.impl("_cache_attention", TORCH_FN(cache_attention_autograd));
}

}  // namespace tpw_ext
