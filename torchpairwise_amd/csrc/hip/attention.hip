// Attention forward: o_i = sum_j softmax_j(scale q_i . k_j + mask_ij) v_j in one pass over the keys
// with the running maximum and sum of every row (layouts: attention.hpp).
#include <math.h>

#include "attention.hpp"

namespace tpw {
namespace attn {

// Per-row running softmax of one wave's W rows and the loop over one key tile.
template <typename T, int W, int DP, int BN, int MM>
struct Forward {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    static constexpr int NB = BN / W, NQ = NB * M::Q, DB = DP / W, QS = DP / M::KS;

    Frag<T> q[QS];
    Acc o[DB];
    float top, sum;  // running maximum (in units of log2 e; kBias: natural) and the lane's part of the sum
    int lim, wlim_min, wlim_max;  // keys seen: this lane's row, over the wave's rows
    int64_t qh, qi;               // head and row (row -1: none)

    __device__ __forceinline__ void init(const Args &a, int64_t b, int64_t kh, int64_t row0, int64_t len, int lane) {
        const int64_t r = row0 + lane % W, rows = a.n * a.group;
        const bool live = r < rows;
        qh = kh * a.group + (live ? r / a.n : 0);
        qi = live ? r % a.n : -1;
        const int64_t l = live ? row_limit(a, len, qi) : 0;
        lim = (int)l;
        wlim_max = lim;
        wlim_min = live ? lim : 0x7fffffff;
#pragma unroll
        for (int s = 1; s < W; s <<= 1) {
            const int x = __shfl_xor(wlim_max, s, 64), y = __shfl_xor(wlim_min, s, 64);
            wlim_max = wlim_max > x ? wlim_max : x;
            wlim_min = wlim_min < y ? wlim_min : y;
        }
        wlim_max = __builtin_amdgcn_readfirstlane(wlim_max);
        wlim_min = __builtin_amdgcn_readfirstlane(wlim_min);
        const T *row = live ? reinterpret_cast<const T *>(a.q.p) + b * a.q.b + qh * a.q.h + qi * a.q.n : nullptr;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            q[s] = load_row8(row, M::KS * s + 8 * (lane / W), (int)a.d, a.vec);
            if (a.qsign != 1.0f) {
                float x[8];
                unpack8(q[s], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= a.qsign;
                q[s] = pack8(x, T{});
            }
        }
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = Acc{};
        top = -INFINITY;
        sum = 0.0f;
    }

    // keys j0 .. j0 + BN - 1 in LDS at kt (keys) and vt (values)
    __device__ __forceinline__ void tile(const Args &a, int64_t b, uint32_t kt, uint32_t vt, int j0, int lane) {
        if (j0 >= wlim_max) return;
        const int g = lane / W;
        const RowReader<T, DP, W> rr(lane);
        const ColReader<T, DP, W> cr(lane);
        Acc s[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) s[i] = Acc{};
#pragma unroll
        for (int k = 0; k < QS; ++k)
#pragma unroll
            for (int i = 0; i < NB; ++i) M::mma(s[i], rr.read(kt, i, k), q[k]);

        if constexpr (MM == kBias) {
            const void *mr = mask_row(a, b, qh, qi, a.mask_bf16 ? 2 : 4);
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int w = 0; w < M::Q; ++w) {
                    const int j = j0 + W * i + 4 * M::NG * w + 4 * g;
                    f32x4 add = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (j < lim) add = mask_bias4(a, mr, j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = s[i][4 * w + e] * a.scale + add[e];
                        s[i][4 * w + e] = add[e] == -INFINITY ? -INFINITY : x;
                    }
                }
        }
        if constexpr (MM == kKeep) {
            const uint8_t *mr = reinterpret_cast<const uint8_t *>(mask_row(a, b, qh, qi, 1));
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int w = 0; w < M::Q; ++w) {
                    const int j = j0 + W * i + 4 * M::NG * w + 4 * g;
                    uint32_t keep = 0;
                    if (j < lim) keep = mask_keep4(a, mr, j);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(keep & (0xffu << (8 * e)))) s[i][4 * w + e] = -INFINITY;
                }
        }
        if (j0 + BN > wlim_min) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int w = 0; w < M::Q; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j0 + W * i + 4 * M::NG * w + 4 * g + e >= lim) s[i][4 * w + e] = -INFINITY;
        }

        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 4 * M::Q; ++e) mx = __builtin_fmaxf(mx, s[i][e]);
        mx = over_groups_max<W>(mx);
        if constexpr (MM != kBias) mx *= a.scale;
        const float top1 = __builtin_fmaxf(top, mx);
        // a row with no key so far: exp2(-inf - 0) = 0 throughout
        const float base = top1 == -INFINITY ? 0.0f : top1;
        if (__any(top1 > top)) {
            const float f = MM == kBias ? __builtin_amdgcn_exp2f((top - base) * kLog2e) : __builtin_amdgcn_exp2f(top - base);
            sum *= f;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int e = 0; e < 4 * M::Q; ++e) o[i][e] *= f;
        }
        top = top1;
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 4 * M::Q; ++e) {
                const float x = MM == kBias ? __builtin_amdgcn_exp2f((s[i][e] - base) * kLog2e)
                                            : __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], a.scale, -base));
                s[i][e] = x;
                part += x;
            }
        sum += part;
        // The probabilities of bf16 inputs are rounded to bf16 for the matrix cores (within 2^-8 of
        // each, as the values are); their sum is not.
#pragma unroll
        for (int t = 0; t < BN / M::KS; ++t) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * u + e] = s[(2 * t + u) / M::Q][4 * ((2 * t + u) % M::Q) + e];
            const Frag<T> p = pack8(x, T{});
#pragma unroll
            for (int i = 0; i < DB; ++i) M::mma(o[i], cr.read(vt, t, i), p);
        }
    }
};

// One block: kWaves x W query rows of the rows that share a key head, over the keys of one part.
template <typename T, int W, int DP, int BN, int MM, int OCC>
__global__ __launch_bounds__(kThreads, OCC) void attention_kernel(const Args a) {
    using F = Forward<T, W, DP, BN, MM>;
    using M = typename F::M;
    constexpr uint32_t kTileBytes = BN * DP * sizeof(T);
    __shared__ uint4 smem[4 * kTileBytes / 16];  // two buffers of a key tile and a value tile
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    int64_t t = xcd_linear(blockIdx.x, gridDim.x);
    const int64_t part = t % a.splits;
    t /= a.splits;
    const int64_t tile = a.tiles - 1 - t % a.tiles;  // longest rows of a causal call first
    const int64_t bk = t / a.tiles, b = bk / a.key_heads, kh = bk % a.key_heads;
    const int64_t len = key_end(a, b), rows = a.n * a.group;
    const int64_t row0 = tile * (kWaves * W), row1 = row0 + kWaves * W < rows ? row0 + kWaves * W : rows;

    F f;
    f.init(a, b, kh, row0 + wave * W, len, lane);

    // keys that some row of the block sees
    int64_t end = len;
    if (a.causal && row0 / a.n == (row1 - 1) / a.n) end = row_limit(a, len, (row1 - 1) % a.n);
    const int nt = (int)cdiv_dev(end, BN);
    const int t0 = (int)((int64_t)nt * part / a.splits), t1 = (int)((int64_t)nt * (part + 1) / a.splits);

    const uint32_t lds = tile::lds_addr(smem);
    Stager<T, DP, BN, kWaves> sk, sv;
    sk.init(a.k.n, (int)a.d, a.vec, wave, lane);
    sv.init(a.v.n, (int)a.dv, a.vec, wave, lane);
    const T *kb = reinterpret_cast<const T *>(a.k.p) + b * a.k.b + kh * a.k.h;
    const T *vb = reinterpret_cast<const T *>(a.v.p) + b * a.v.b + kh * a.v.h;
    const auto fetch = [&](int i) {
        const int64_t j0 = (int64_t)i * BN;
        const uint32_t buf = lds + (uint32_t)((i - t0) & 1) * 2 * kTileBytes;
        sk.load(kb + j0 * a.k.n, len - j0, buf);
        sv.load(vb + j0 * a.v.n, len - j0, buf + kTileBytes);
    };
    if (t0 < t1) fetch(t0);
    for (int i = t0; i < t1; ++i) {
        tile::barrier_all();  // tile i has landed, and nobody reads the other buffer any more
        if (i + 1 < t1) fetch(i + 1);
        const uint32_t buf = lds + (uint32_t)((i - t0) & 1) * 2 * kTileBytes;
        f.tile(a, b, buf, buf + kTileBytes, i * BN, lane);
    }

    const float sum = over_groups_sum<W>(f.sum);
    if (f.qi < 0) return;
    const int g = lane / W;
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int64_t row = (b * a.heads + f.qh) * a.n + f.qi;
    if (a.splits > 1) {
        const int64_t all = a.batch * a.heads * a.n;
        float *st = a.part_stats + part * 2 * all;
        if (g == 0) {
            st[row] = f.top;
            st[all + row] = sum;
        }
        float *p = a.part + (part * all + row) * a.dv;
#pragma unroll
        for (int i = 0; i < F::DB; ++i)
#pragma unroll
            for (int w = 0; w < M::Q; ++w) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = f.o[i][4 * w + e];
                store4(p, W * i + 4 * M::NG * w + 4 * g, (int)a.dv, a.dv % 4 == 0, v);
            }
        return;
    }
    if (g == 0 && a.stats) {
        a.stats[row] = f.top;
        a.stats[a.batch * a.heads * a.n + row] = sum;
    }
    T *p = reinterpret_cast<T *>(const_cast<void *>(a.o.p)) + b * a.o.b + f.qh * a.o.h + f.qi * a.o.n;
#pragma unroll
    for (int i = 0; i < F::DB; ++i)
#pragma unroll
        for (int w = 0; w < M::Q; ++w) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = f.o[i][4 * w + e] * inv;
            store4(p, W * i + 4 * M::NG * w + 4 * g, (int)a.dv, a.vec_out, v);
        }
}

// Joins the parts of every row: m = max m_s, l = sum l_s 2^(m_s - m), o = sum o_s 2^(m_s - m) / l,
// in the order of the parts.  One thread per four features.
template <typename T, bool BIAS>
__global__ void attention_join_kernel(const Args a) {
    const int64_t rows = a.batch * a.heads * a.n, quads = (a.dv + 3) / 4;
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= rows * quads) return;
    const int64_t row = id / quads;
    const int f = (int)(id % quads) * 4;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = __builtin_fmaxf(top, a.part_stats[2 * s * rows + row]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) {
        const float d = a.part_stats[2 * s * rows + row] - base;
        const float w = __builtin_amdgcn_exp2f(BIAS ? d * kLog2e : d);
        sum += w * a.part_stats[(2 * s + 1) * rows + row];
        const float *p = a.part + (s * rows + row) * a.dv + f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e < a.dv) o[e] += w * p[e];
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    if (f == 0 && a.stats) {
        a.stats[row] = top;
        a.stats[rows + row] = sum;
    }
    const int64_t i = row % a.n, h = row / a.n % a.heads, b = row / a.n / a.heads;
    T *p = reinterpret_cast<T *>(const_cast<void *>(a.o.p)) + b * a.o.b + h * a.o.h + i * a.o.n;
    o *= inv;
    store4(p, f, (int)a.dv, a.vec_out, o);
}

namespace {

bool whole_pieces(const View &v, int64_t width, int64_t size) {
    return aligned16(v.p) && width * size % 16 == 0 && v.b * size % 16 == 0 && v.h * size % 16 == 0 && v.n * size % 16 == 0;
}
View view_of(const void *p, const int64_t *strides, int64_t rows, int64_t width) {
    return {p, strides[0], strides[1], rows == 1 ? width : strides[2]};
}

int64_t forward_parts(const Args &a, int64_t keys) { return parts_for(a.batch * a.key_heads * a.tiles, cdiv(a.m, keys)); }

// Sets tiles and splits for the element type and width.
template <typename T, int DP>
void plan(Args &a) {
    a.tiles = cdiv(a.n * a.group, (int64_t)kWaves * Tiles<T, DP>::kWidth);
    a.splits = (int)forward_parts(a, Tiles<T, DP>::kKeys);
}

}  // namespace

int read_args(const tpw_attention_desc *d, bool backward, Args &a) {
    TPW_REQUIRE(d, "null descriptor");
    TPW_REQUIRE(d->dtype == TPW_F32 || d->dtype == TPW_BF16, "attention: float32 or bfloat16 rows");
    TPW_REQUIRE(d->batch >= 0 && d->heads >= 0 && d->n >= 0 && d->m >= 0, "attention: negative size");
    TPW_REQUIRE(d->d >= 1 && d->d <= 256 && d->dv >= 1 && d->dv <= 256, "attention: rows have 1 to 256 features");
    TPW_REQUIRE(d->key_heads >= 1 && d->heads % d->key_heads == 0, "attention: heads must be a multiple of key_heads");
    TPW_REQUIRE(d->mask_type >= TPW_MASK_NONE && d->mask_type <= TPW_MASK_ADD_BF16, "attention: unknown mask type");
    TPW_REQUIRE(d->m < (int64_t(1) << 31) - 1024 && d->n < (int64_t(1) << 31) - 1024, "attention: too many rows");
    TPW_REQUIRE(d->scale == d->scale && fabs(d->scale) <= 1e30, "attention: scale must be finite");
    const int64_t size = d->dtype == TPW_F32 ? 4 : 2;
    a.batch = d->batch;
    a.heads = d->heads;
    a.key_heads = d->key_heads;
    a.group = d->heads / d->key_heads;
    a.n = d->n;
    a.m = d->m;
    a.d = d->d;
    a.dv = d->dv;
    a.causal = d->causal != 0;
    a.q = view_of(d->query, d->query_strides, d->n, d->d);
    a.k = view_of(d->key, d->key_strides, d->m, d->d);
    a.v = view_of(d->value, d->value_strides, d->m, d->dv);
    a.o = view_of(d->out, d->out_strides, d->n, d->dv);
    a.stats = d->stats;
    a.lengths = d->lengths;
    a.mask = d->mask_type == TPW_MASK_NONE ? nullptr : d->mask;
    a.mb = d->mask_strides[0];
    a.mh = d->mask_strides[1];
    a.mn = d->mask_strides[2];
    a.mm = d->mask_strides[3];
    a.mask_bf16 = d->mask_type == TPW_MASK_ADD_BF16;
    const int64_t quad = d->mask_type == TPW_MASK_KEEP ? 4 : a.mask_bf16 ? 8 : 16, unit = quad / 4;
    a.mask_vec = a.mm == 1 && reinterpret_cast<uintptr_t>(a.mask) % quad == 0 && a.mb * unit % quad == 0 &&
                 a.mh * unit % quad == 0 && a.mn * unit % quad == 0;
    const bool bias = mask_mode(d) == kBias;
    a.qsign = d->scale > 0 ? 1.0f : d->scale < 0 ? -1.0f : 0.0f;
    a.scale = d->scale == 0 ? 1.0f : (float)(fabs(d->scale) * (bias ? 1.0 : 1.4426950408889634));
    a.gscale = (float)d->scale;
    a.vec = whole_pieces(a.q, a.d, size) && whole_pieces(a.k, a.d, size) && whole_pieces(a.v, a.dv, size);
    a.vec_out = whole_pieces(a.o, a.dv, size);
    const auto streamed = [&](const View &v, int64_t rows, int64_t width) {
        return a.batch * a.heads * a.n * a.m == 0 || rows <= 1 || (v.n >= width && v.n * size <= (int64_t(1) << 23));
    };
    bool ok = streamed(a.k, d->m, d->d) && streamed(a.v, d->m, d->dv);
    if (backward) {
        a.go = view_of(d->grad_out, d->grad_out_strides, d->n, d->dv);
        a.gq = view_of(d->grad_query, d->grad_query_strides, d->n, d->d);
        a.gk = view_of(d->grad_key, d->grad_key_strides, d->m, d->d);
        a.gv = view_of(d->grad_value, d->grad_value_strides, d->m, d->dv);
        a.vec = a.vec && whole_pieces(a.go, a.dv, size) && whole_pieces(a.o, a.dv, size);
        a.vec_out = whole_pieces(a.gq, a.d, size) && whole_pieces(a.gk, a.d, size) && whole_pieces(a.gv, a.dv, size);
        ok = ok && streamed(a.q, d->n, d->d) && streamed(a.go, d->n, d->dv);
    }
    TPW_REQUIRE(ok, "attention: rows of an operand overlap or lie more than 8 MiB apart");
    return TPW_OK;
}

}  // namespace attn
}  // namespace tpw

using namespace tpw;
using namespace tpw::attn;

namespace {

size_t forward_workspace(const Args &a) {
    return a.splits > 1 ? (size_t)a.splits * a.batch * a.heads * a.n * (a.dv + 2) * 4 : 0;
}

}  // namespace

extern "C" size_t tpw_attention_workspace_size(const tpw_attention_desc *d) {
    Args a = {};
    if (read_args(d, false, a) != TPW_OK || a.batch * a.heads * a.n == 0) return 0;
    size_t bytes = 0;
    by_type(a, d->dtype, kNoMask, [&](auto t, auto dp, auto) {
        plan<decltype(t), decltype(dp)::value>(a);
        bytes = forward_workspace(a);
        return TPW_OK;
    });
    return bytes;
}

extern "C" int tpw_attention(const tpw_attention_desc *d, void *workspace, void *stream) {
    Args a = {};
    if (const int rc = read_args(d, false, a)) return rc;
    if (a.batch * a.heads * a.n == 0) return TPW_OK;
    TPW_REQUIRE(a.q.p && a.o.p && (a.m == 0 || (a.k.p && a.v.p)), "attention: null operand");
    TPW_REQUIRE(d->mask_type == TPW_MASK_NONE || a.mask || a.m == 0, "attention: null mask");
    hipStream_t s = as_stream(stream);
    return by_type(a, d->dtype, mask_mode(d), [&](auto t, auto dp, auto mode) {
        using T = decltype(t);
        constexpr int DP = decltype(dp)::value, MM = decltype(mode)::value, W = Tiles<T, DP>::kWidth;
        plan<T, DP>(a);
        const int64_t blocks = a.batch * a.key_heads * a.tiles * a.splits, rows = a.batch * a.heads * a.n;
        TPW_REQUIRE(blocks < (int64_t(1) << 31), "attention: too many rows");
        if (a.splits > 1) {
            TPW_REQUIRE(workspace && aligned16(workspace), "attention: null or unaligned workspace");
            a.part = reinterpret_cast<float *>(workspace);
            a.part_stats = a.part + a.splits * rows * a.dv;
        }
        constexpr int kOcc = sizeof(T) == 4 && DP == 256 ? 1 : 2;
        hipLaunchKernelGGL((attention_kernel<T, W, DP, Tiles<T, DP>::kKeys, MM, kOcc>), dim3((unsigned)blocks),
                           dim3(attn::kThreads), 0, s, a);
        if (const int rc = check_launch("attention_kernel")) return rc;
        if (a.splits > 1) {
            const int64_t quads = rows * cdiv(a.dv, 4);
            hipLaunchKernelGGL((attention_join_kernel<T, MM == kBias>), dim3((unsigned)cdiv(quads, 256)), dim3(256), 0, s, a);
            return check_launch("attention_join_kernel");
        }
        return TPW_OK;
    });
}
