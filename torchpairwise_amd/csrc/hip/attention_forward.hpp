// The forward's work on one tile of keys, shared by the kernels that bring tiles of keys and values into LDS
// (attention.hip: by DMA; cache_tiles.hpp: out of a cache in 4 or 8 bits), and their launch's plan.
#pragma once

#include "attention.hpp"

namespace tpw {
namespace attn {

// Per-row running softmax of one wave's W rows and the loop over one key tile.  GAPS: some of a tile's keys
// may be no keys at all.  QT: the queries' type; float over tiles of bf16 (whose values are exact) takes three products.
template <typename T, int W, int DP, int BN, int MM, bool DWORDS, bool GAPS = false, typename QT = T>
struct Forward {
    static constexpr int NP = sizeof(QT) / sizeof(T) == 2 ? 3 : 1;  // summands of a query and a probability
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    using CR = ColReader<T, DP, W>;
    static constexpr int NB = BN / W, NQ = NB * M::Q, DB = DP / W, QS = DP / M::KS;

    Frag<T> q[QS][NP];
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
        const QT *row = live ? reinterpret_cast<const QT *>(a.q.p) + b * a.q.b + qh * a.q.h + qi * a.q.n : nullptr;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            if constexpr (NP == 1) {
                q[s][0] = load_row8(row, M::KS * s + 8 * (lane / W), (int)a.d, DWORDS);
                if (a.qsign != 1.0f) {
                    float x[8];
                    unpack8(q[s][0], x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] *= a.qsign;
                    q[s][0] = pack8(x, T{});
                }
            } else {
                float x[8];
                unpack8(load_row8(row, M::KS * s + 8 * (lane / W), (int)a.d, DWORDS), x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= a.qsign;
                split3_any(x, q[s]);
            }
        }
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = Acc{};
        top = -INFINITY;
        sum = 0.0f;
    }

    // keys j0 .. j0 + BN - 1 in LDS at kt (keys) and vt (values); GAPS: key j0 + x is one where bit x is set
    __device__ __forceinline__ void tile(const Args &a, int64_t b, uint32_t kt, uint32_t vt, int j0, int lane,
                                         uint64_t present = ~uint64_t(0)) {
        if (j0 >= wlim_max) return;
        const int g = lane / W;
        const RowReader<T, DP, W> rr(lane);
        const CR cr(lane);
        // added values: where registers allow, loaded ahead of the scores' products
        constexpr bool kAhead = MM == kBias && DP <= 128;
        f32x4 add[MM == kBias ? NQ : 1];
        if constexpr (kAhead) mask_bias<NQ, 4 * M::NG>(a, mask_row(a, b, qh, qi < 0 ? 0 : qi), j0, 4 * g, BN, add);
        Acc s[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) s[i] = Acc{};
#pragma unroll
        for (int k = 0; k < QS; ++k) {
            if constexpr (sizeof(T) == 4) {  // independent products side by side
                Frag<T> f[NB];
#pragma unroll
                for (int i = 0; i < NB; ++i) f[i] = rr.read(kt, i, k);
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int i = 0; i < NB; ++i) M::mma1(s[i], f[i], q[k][0], e);
            } else {
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const Frag<T> f = rr.read(kt, i, k);
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) M::mma(s[i], f, q[k][p]);
                }
            }
        }

        if constexpr (MM == kBias) {
            if constexpr (!kAhead) mask_bias<NQ, 4 * M::NG>(a, mask_row(a, b, qh, qi < 0 ? 0 : qi), j0, 4 * g, BN, add);
#pragma unroll
            for (int x = 0; x < NQ; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = s[x / M::Q][4 * (x % M::Q) + e] * a.scale + add[x][e];
                    s[x / M::Q][4 * (x % M::Q) + e] = add[x][e] == -INFINITY ? -INFINITY : y;
                }
        }
        if constexpr (MM == kKeep) {
            const uint32_t *mr = mask_words(a, b, qh, qi) + j0 / 32;
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                const uint32_t keep = j0 + 32 * u < lim ? mr[u] >> (4 * g) : 0;
#pragma unroll
                for (int x = 0; x < 32 / (4 * M::NG); ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at = 32 * u + 4 * M::NG * x;  // of the tile's keys
                        if (!(keep & (1u << (4 * M::NG * x + e)))) s[at / W][4 * (at % W / (4 * M::NG)) + e] = -INFINITY;
                    }
            }
        }
        if (j0 + BN > wlim_min) {
            asm volatile("");  // a branch: most tiles skip this
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int w = 0; w < M::Q; ++w)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j0 + W * i + 4 * M::NG * w + 4 * g + e >= lim) s[i][4 * w + e] = -INFINITY;
        }

        if constexpr (GAPS) {
            if (~present) {
                static_assert(BN <= 64, "a bit for every key");
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w) {
                        const uint32_t four = (uint32_t)(present >> (W * i + 4 * M::NG * w + 4 * g));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(four >> e & 1)) s[i][4 * w + e] = -INFINITY;
                    }
            }
        }

        float mx = s[0][0];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 4 * M::Q; ++e) mx = __builtin_fmaxf(mx, s[i][e]);
        float top1 = top;
        bool move = true;
        if constexpr (GAPS) {  // the base follows once the maximum is 2^8 ahead: few tiles exchange and rescale
            if constexpr (MM != kBias) mx *= a.scale;
            move = __any(mx > top + (MM == kBias ? 5.0f : 8.0f));
            if (move) top1 = __builtin_fmaxf(top, over_groups_max<W>(mx));
        } else {
            mx = over_groups_max<W>(mx);
            if constexpr (MM != kBias) mx *= a.scale;
            top1 = __builtin_fmaxf(top, mx);
            move = __any(top1 > top);
        }
        // a row with no key so far: exp2(-inf - 0) = 0 throughout
        const float base = top1 == -INFINITY ? 0.0f : top1;
        if (move) {
            const float f = __builtin_amdgcn_exp2f(MM == kBias ? (top - base) * kLog2e : top - base);
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
            if constexpr (NP == 1) {
                const Frag<T> p = pack8(x, T{});
#pragma unroll
                for (int c = 0; c < CR::kPieces; ++c) CR::use(o, c, cr.read(vt, t, c), p);
            } else {
                Frag<T> p[NP];
                split3(x, p);
#pragma unroll
                for (int c = 0; c < CR::kPieces; ++c) {
                    const auto f = cr.read(vt, t, c);
#pragma unroll
                    for (int u = NP - 1; u >= 0; --u) CR::use(o, c, f, p[u]);
                }
            }
        }
    }
};

// Sets tiles and splits for the element type and width, per_cu blocks to a CU.
template <typename T, int DP>
void plan(Args &a, int64_t per_cu = Tiles<T, DP>::kPerCu, int products = 2) {
    using L = Tiles<T, DP>;
    constexpr int64_t kOwn = L::kWaves * L::kWidth;
    a.tiles = cdiv(a.n * a.group, kOwn);
    a.splits = (int)parts_for(a.batch * a.key_heads * a.tiles, cdiv(a.m, L::kKeys), per_cu, uneven(a),
                              step_us<T, DP>(kOwn, L::kKeys, products, per_cu),
                              part_us(a.batch * a.heads * a.n, quads4(a.dv)));
}

}  // namespace attn
}  // namespace tpw
