// Attention of a few query rows a key head (single tokens, drafts) over a cache in 4 or 8 bits.
#pragma once

#include <type_traits>

#include "cache_attention.hpp"

namespace tpw {
namespace attn {

using cache::Cache;
using cache::Eight;
using cache::Side;

// The codes and scales of 32 keys, as a lane (i = lane % 16, g = lane / 16) uses them.
//   Keys: first operands of 16 x 16 x 32 products.  Product t's row i is key 8 (i / 4) + 4 t + i % 4, so that
//     the scores a lane receives (rows 4 g .. + 3) are keys 8 g + 4 t .. + 3: eight consecutive ones in two
//     products.  The lane holds features F g .. + F - 1 of its key, F = 8 NB, side by side in memory: which
//     features a product sums over is free as long as the queries agree.
//   Values: lane i holds features V i .. + V - 1 (V = 2 NB) of keys 8 g .. + 7, the keys of its scores.
// Nothing passes through LDS: each code is loaded by the lane that multiplies it, in pieces of 2 to 16
// bytes, a row's 64 bytes (128 features) by 4 or 16 lanes side by side.  The values are exact in bfloat16 and go
// to its products.  (The products of codes as they lie, v_mfma_scale_f32_16x16x128_f8f6f4, would need no
// conversion, but keep only 2^-11 of the largest of their 128 terms.)
template <int BITS, int NB, int RT, int MM>
struct Codes {
    static constexpr int KS = NB > 4 ? NB / 4 : 1;                   // blocks that a lane's part of a key touches
    static constexpr int KW = NB * BITS / 4 / KS;                    // words of it in each
    static constexpr int VW = NB * BITS >= 16 ? NB * BITS / 16 : 1;  // words of a value row (4 bits, 64 features: half)
    uint32_t k[2][KS][KW], v[8][VW];
    uint2 ks[KS], vs;  // scales of the lane's granules of eight keys
    int live;          // of the 32 keys, those below this are there (16-row pages: for the lane's half of them)
    uint32_t m[RT][MM == kBias ? 8 : MM == kKeep ? 2 : 1];  // the mask's values for the lane's eight keys
};

// NP: summands in bfloat16 of a query and a probability (float32: three).  Up to 16 rows of bfloat16 have two summands of
// a probability (within 2^-17 of it), so that the output's rounding is the only one to count: single tokens over 8192 to
// 32768 are off by 1.6e-3 of their norm, where one summand makes it 2.3e-3, for 1 to 5 % of the time (16 x 16 (2) heads
// over 32768 of 128 28.7 -> 29.3 us, 16 x 32 (8) over 8192 in 8 bits 47.6 -> 48.1; 16 x 8 x 4 rows over 8192 of 64 21.9
// -> 23.0).  17 to 32 rows, and many (attention_forward.hpp), have one (within 2^-8, as the output's rounding is): two
// would cost 4 to 16 % (16 x 8 heads over 4096: 32 rows of 128 25.5 -> 27.8 us, of 256 in 8 bits 85 -> 99), in tiles 20
// to 31 (8192^2 causal 603 -> 791).
// PACK: at most 4 rows, whose summands take 4 columns of a product each: one product for all three, where 16 rows take
// three (float32, 8 x 16 (4) heads over 16000 of 90: 19.3 -> 16.9 us).
template <int BITS, int NB, int NP, int RT, int MM, bool HALVES, bool PACK, int WAVES>
struct Rows {
    static_assert(!PACK || (NP == 3 && RT == 1), "three summands of 4 rows");
    static constexpr int NM = PACK ? 1 : NP;  // products for a tile of 16 rows: of the scores,
    static constexpr int NV = PACK ? 1 : NP == 1 && RT == 1 ? 2 : NP;  // of the values
    using C = Codes<BITS, NB, RT, MM>;
    static constexpr bool BIAS = MM == kBias;
    using T = std::conditional_t<NP == 1, uint16_t, float>;
    static constexpr int KS = C::KS, F = 8 * NB, V = 2 * NB;

    Frag<uint16_t> q[RT][NB][NM];
    f32x4 o[RT][V];
    float base[RT], sum[RT];  // the row's running base, at most kSlack below its maximum; the lane's sum
    int lim[RT];              // keys that the row sees
    int64_t mrow[RT];         // bytes to its row of the mask
    int msize;                // bytes of one of its values
    uint32_t kat[KS], ksat[KS], vat, vsat;  // bytes of the lane's part: codes and scales of its key, its values

    // row0: the block's first of the rows that share the key head
    __device__ __forceinline__ void init(const Args &a, const Cache &c, int64_t b, int64_t kh, int row0, int64_t len,
                                         int lane) {
        const int i = lane & 15, g = lane >> 4;
        // Blocks past the row's are not there: block 0 in their place, against queries of zero.
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int block = F * g / 32 + s;
            const bool in = block < c.k.blocks;
            kat[s] = (uint32_t)((8 * (i >> 2) + (i & 3)) * c.k.cr + (in ? (F * g + 32 * s) * BITS / 8 : 0));
            ksat[s] = (uint32_t)((in ? block : 0) * c.k.sb + 8 * (i >> 2));
        }
        const int block = V * i / 32 < c.v.blocks ? V * i / 32 : 0;
        vat = (uint32_t)(8 * g * c.v.cr + (V * i / 32 < c.v.blocks ? V * i * BITS / 8 : 0));
        vsat = (uint32_t)(block * c.v.sb + 8 * g);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = row0 + (PACK ? i & 3 : 16 * t + i), n = (int)a.n;
            const bool in = r < n * (int)a.group;
            const int h = in ? n == 1 ? r : r / n : 0;
            const int64_t qh = kh * a.group + h, qi = in ? r - h * n : 0;
            const int64_t l = in ? row_limit(a, len, qi) : 0;
            lim[t] = (int)(l < len ? l : len);
            if constexpr (MM != kNoMask) {
                msize = MM == kKeep ? 1 : a.mask_bf16 ? 2 : 4;
                mrow[t] = (b * a.mb + qh * a.mh + qi * a.mn) * msize;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) o[t][k] = f32x4{0, 0, 0, 0};
            base[t] = -INFINITY;
            sum[t] = 0.0f;
        }
    }

    // The block's queries, times the sign of the scale, to LDS in NP summands, zeros past their width and
    // behind the last row.
    static constexpr int kRow = 64 * NB + 16;                                  // bytes of a row: 16 of them fill the banks
    static constexpr int kPlane = 16 * RT * kRow, kQueryBytes = NP * kPlane;   // of a summand; of all
    static constexpr int kPieces = RT * 16 * 4 * NB, kThreads = 64 * WAVES;    // 8 features each
    static constexpr int kOwn = (kPieces + kThreads - 1) / kThreads;           // a thread's
    struct Piece {
        T x[8];
    };
    static __device__ __forceinline__ void load_queries(const Args &a, int64_t b, int64_t kh, int row0, Piece (&y)[kOwn]) {
        const T *q = reinterpret_cast<const T *>(a.q.p) + b * a.q.b;
        const int rows = (int)(a.n * a.group), n = (int)a.n, d = (int)a.d;
#pragma unroll
        for (int x = 0; x < kOwn; ++x) {
            const int id = x * kThreads + (int)threadIdx.x, r = row0 + id / (4 * NB), f = id % (4 * NB) * 8;
            y[x] = {};
            if (id < kPieces && r < rows && f < d) {
                const int h = n == 1 ? r : r / n;
                const T *p = q + (kh * a.group + h) * a.q.h + (r - h * n) * a.q.n + f;
                if (a.whole_q) {
                    __builtin_memcpy(y[x].x, __builtin_assume_aligned(p, 16), sizeof(y[x]));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (f + e < d) y[x].x[e] = p[e];
                }
            }
        }
    }
    static __device__ __forceinline__ void form_queries(const Args &a, const Piece (&y)[kOwn], uint8_t *to) {
#pragma unroll
        for (int x = 0; x < kOwn; ++x) {
            const int id = x * kThreads + (int)threadIdx.x, r = id / (4 * NB), f = id % (4 * NB) * 8;
            if (kPieces % kThreads && id >= kPieces) break;
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = to_f32(y[x].x[e]) * a.qsign;
            Frag<uint16_t> w[NP];
            if constexpr (NP == 1)
                w[0] = pack8(z, uint16_t{});
            else
                split3_any(z, w);
#pragma unroll
            for (int p = 0; p < NP; ++p) *reinterpret_cast<uint4 *>(to + p * kPlane + r * kRow + 2 * f) = w[p].v;
        }
    }
    __device__ __forceinline__ void queries(const uint8_t *from, int lane) {
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int s = 0; s < NB; ++s)
#pragma unroll
                for (int p = 0; p < NM; ++p) {
                    // PACK: columns 12 to 15 repeat the last summand's place and are made zeros
                    const int plane = PACK ? (i >> 2 < NP ? i >> 2 : NP - 1) : p, row = PACK ? i & 3 : 16 * t + i;
                    q[t][s][p].v = *reinterpret_cast<const uint4 *>(from + plane * kPlane + row * kRow + 2 * (F * g + 8 * s));
                    if (PACK && i >= 12) q[t][s][p].v = make_uint4(0, 0, 0, 0);
                }
    }

    // The lane's own summand of its row's eight probabilities (the fourth: nothing is left for it).
    static __device__ __forceinline__ void split_own(float (&x)[8], int i, Frag<uint16_t> &f) {
        uint32_t w[8];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const float on = p < i >> 2 ? 1.0f : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = __builtin_fmaf(-on, __uint_as_float(__float_as_uint(x[e]) & 0xffff0000u), x[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(x[e]);
        f.v = make_uint4(high2(w[0], w[1]), high2(w[2], w[3]), high2(w[4], w[5]), high2(w[6], w[7]));
    }
    // The sum over a row's four columns (lanes i, i + 4, .. of 16), the same bits in every one of them: 8 apart
    // first, then 4 (the other way round the orders would differ, and with them, now and then, the columns' ideas
    // of what a probability's first summand is).
    static __device__ __forceinline__ float over_columns(float x) {
        x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true));  // row_ror:8
        return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x124, 0xf, 0xf, true));  // row_ror:4
    }

    // Rows 0 .. n - 1 from a place on: buffers whose range ends with the last of them.  The hardware counts a load's
    // scalar offset into the range without wrapping round (ranges of 0 to 4096 bytes, offsets of 0 to 8192: read is
    // exactly what ends inside), so rows from n on are neither read nor paid for, and no row where n is 0.  Were it
    // left out of the check, a load would reach at most the last row of its 8, which is there: rows come in 16s.
    struct Buffers {
        __amdgpu_buffer_rsrc_t codes, scales;
    };
    static __device__ __forceinline__ Buffers buffers(const Side &s, int64_t kh, cache::Place p, int n) {
        const uint8_t *codes = s.codes + p.first * s.cf + kh * s.ch + p.row * s.cr;
        const uint8_t *scales = s.scales + p.first * s.sf + kh * s.sh + p.row;
        // scales are read by eights: a part of one behind the range would be none of it
        const int64_t cn = n > 0 ? (n - 1) * s.cr + s.blocks * (4 * BITS) : 0;
        const int64_t sn = n > 0 ? (s.blocks - 1) * s.sb + (n + 7) / 8 * 8 : 0;
        return {__builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(codes), (short)0, (int)cn, 0x00020000),
                __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(scales), (short)0, (int)sn, 0x00020000)};
    }
    // x: buffers; HALVES: one or the other by lane, whose own bytes count from the first place's rows on.
    template <int N>
    static __device__ __forceinline__ void fetch(uint32_t *to, __amdgpu_buffer_rsrc_t x, uint32_t at, int more) {
        if constexpr (N == 1) {
            to[0] = __builtin_amdgcn_raw_buffer_load_b32(x, at, more, 0);
        } else if constexpr (N == 2) {
            const auto y = __builtin_amdgcn_raw_buffer_load_b64(x, at, more, 0);
            to[0] = y[0], to[1] = y[1];
        } else {
            const auto y = __builtin_amdgcn_raw_buffer_load_b128(x, at, more, 0);
            to[0] = y[0], to[1] = y[1], to[2] = y[2], to[3] = y[3];
        }
    }
    __device__ __forceinline__ void load_keys(const Cache &c, const Buffers &x, C &w) const {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int y = 0; y < C::KW; y += 4)
                    fetch<C::KW < 4 ? C::KW : 4>(w.k[t][s] + y, x.codes, kat[s] + 4 * y, 4 * t * (int)c.k.cr);
#pragma unroll
        for (int s = 0; s < KS; ++s) fetch<2>(&w.ks[s].x, x.scales, ksat[s], 0);
    }
    __device__ __forceinline__ void load_values(const Cache &c, const Buffers &x, C &w) const {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int at = u * (int)c.v.cr;
            if constexpr (NB * BITS < 16)
                w.v[u][0] = __builtin_amdgcn_raw_buffer_load_b16(x.codes, vat, at, 0);
            else
                fetch<C::VW>(w.v[u], x.codes, vat, at);
        }
        fetch<2>(&w.vs.x, x.scales, vsat, 0);
    }
    // The 32 keys of chunk x, which lie from `p` on (HALVES: the later 16 from `p1`), none past `end` chunks.
    // Every call reads as often, rows that are not there as zeros and without traffic: what is in flight can be
    // counted, and the loads of the chunks ahead stay there while one is worked on.
    __device__ __forceinline__ void load(const Args &a, const Cache &c, int64_t b, int64_t kh, int x, int end, int len,
                                         cache::Place p, cache::Place p1, int lane, C &w) const {
        const int left = x < end ? len - 32 * x : 0;
        const auto rows = [&](const cache::Place &q, int from, int most) {
            const int n = q.first < 0 || left < from ? 0 : left - from;
            return n < most ? n : most;
        };
        if constexpr (!HALVES) {
            w.live = rows(p, 0, 32);
            const cache::Place at = w.live ? p : cache::Place{0, 0};
            load_keys(c, buffers(c.k, kh, at, w.live), w);
            load_values(c, buffers(c.v, kh, at, w.live), w);
        } else {
            const int n0 = rows(p, 0, 16), n1 = rows(p1, 16, 16);
            const cache::Place at0 = n0 ? p : cache::Place{0, 0};
            const cache::Place at1 = n1 ? cache::Place{p1.first, p1.row - 16} : cache::Place{0, 0};
            const bool v1 = lane >= 32;
            // both halves' lanes in turn: lanes of the other half point behind the range
            by_halves(c.k, kh, at0, n0, at1, n1, (lane & 15) >= 8, [&](const Buffers &y) { load_keys(c, y, w); });
            by_halves(c.v, kh, at0, n0, at1, n1, v1, [&](const Buffers &y) { load_values(c, y, w); });
            w.live = v1 ? (n1 ? 16 + n1 : 0) : n0;
        }
        if constexpr (MM != kNoMask) {
            const int j = 32 * x + 8 * (lane >> 4);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const uint8_t *row = reinterpret_cast<const uint8_t *>(a.mask) + (int64_t)mrow[t] +
                                     (int64_t)(x < end && j < a.m ? j : 0) * msize;
                if constexpr (MM == kKeep) {
                    __builtin_memcpy(w.m[t], row, 8);
                } else {  // of bfloat16 values the first 16 bytes alone
                    __builtin_memcpy(w.m[t], row, 16);
                    __builtin_memcpy(w.m[t] + 4, row + (a.mask_bf16 ? 0 : 16), 16);
                }
            }
        }
    }
    template <typename F>
    static __device__ __forceinline__ void by_halves(const Side &s, int64_t kh, cache::Place at0, int n0, cache::Place at1,
                                                     int n1, bool second, F &&f) {
        if (second) {
            f(buffers(s, kh, at1, n1 ? 16 + n1 : 0));
        } else {
            f(buffers(s, kh, at0, n0));
            asm volatile("");  // not joined with the other branch: scalar addresses in each
        }
    }

    // What the mask makes of the scores of row t's eight keys; added values turn them into natural units.
    __device__ __forceinline__ void masked(const Args &a, const C &w, int t, float (&s)[8]) const {
        if constexpr (BIAS) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = a.mask_bf16 ? __uint_as_float(e % 2 ? w.m[t][e / 2] & 0xffff0000u : w.m[t][e / 2] << 16)
                                            : __uint_as_float(w.m[t][e]);
                s[e] = y == -INFINITY ? -INFINITY : s[e] * a.scale + y;
            }
        } else if constexpr (MM == kKeep) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = w.m[t][e / 4] >> (8 * (e % 4)) & 0xffu ? s[e] : -INFINITY;
        }
    }

    // 32 keys from j0 on.
    __device__ __forceinline__ void use(const Args &a, C &w, int j0, int lane) {
        const int i = lane & 15, g = lane >> 4, j = j0 + 8 * g;
        const int live = w.live - 8 * g;  // of the lane's eight keys, those that are there
        if (__any(live < 8)) {            // values that are not: zeros
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t there = u < live ? 0xffffffffu : 0u;
#pragma unroll
                for (int x = 0; x < C::VW; ++x) w.v[u][x] &= there;
                uint32_t &s = u < 4 ? w.vs.x : w.vs.y;
                s &= there | ~(0xffu << (8 * (u & 3)));
            }
        }
        f32x4 s[2][RT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < RT; ++r) s[t][r] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            constexpr int kSteps = NB / KS;  // products of a block
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint2 by = w.ks[k / kSteps];
                const float scale = cache::scale_of((t ? by.y : by.x) >> (8 * (i & 3)));
                Eight<BITS> e;
#pragma unroll
                for (int x = 0; x < BITS / 4; ++x) e.w[x] = w.k[t][k / kSteps][k % kSteps * (BITS / 4) + x];
                const bf16x8 f = __builtin_bit_cast(bf16x8, e.bf16(scale));
#pragma unroll
                for (int p = NM - 1; p >= 0; --p)
#pragma unroll
                    for (int r = 0; r < RT; ++r)
                        s[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, q[r][k][p].v),
                                                                          s[t][r], 0, 0, 0);
            }
        }
        Frag<uint16_t> pr[RT][NV];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = PACK ? over_columns(s[e / 4][r][e % 4]) : s[e / 4][r][e % 4];
            masked(a, w, r, x);
            // of the lane's eight keys, those the row sees
            const int end = lim[r] - j < live ? lim[r] - j : live;
            if (__any(end < 8)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = e < end ? x[e] : -INFINITY;
            }
            float top = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top = __builtin_fmaxf(top, x[e]);
            if constexpr (!BIAS) top *= a.scale;
            // the base follows the maximum once it is kSlack behind: the exchange between the row's lanes
            // and the rescaling are rare
            if (__any(top > base[r] + kSlack)) {
                const float b1 = __builtin_fmaxf(base[r], over_groups_max<16>(top));
                const float f = b1 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(unit() * (base[r] - b1));
                sum[r] *= f;
#pragma unroll
                for (int k = 0; k < V; ++k) o[r][k] *= f;
                base[r] = b1;
            }
            const float b0 = base[r] == -INFINITY ? 0.0f : base[r];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = BIAS ? __builtin_amdgcn_exp2f((x[e] - b0) * kLog2e)
                            : __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale, -b0));
                sum[r] += x[e];
            }
            if constexpr (PACK)
                split_own(x, i, pr[r][0]);
            else if constexpr (NV == 1)
                pr[r][0] = pack8(x, uint16_t{});
            else if constexpr (NV == 2)
                split2(x, pr[r]);
            else
                split3(x, pr[r]);
        }
        float vscale[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) vscale[u] = cache::scale_in(u < 4 ? w.vs.x : w.vs.y, u & 3);
        values(w, vscale, pr, std::make_integer_sequence<int, NB>{});
    }

    static __device__ __forceinline__ float unit() { return BIAS ? kLog2e : 1.0f; }
    static constexpr float kSlack = BIAS ? 5.0f : 8.0f;

    template <int... P>
    __device__ __forceinline__ void values(const C &w, const float (&scale)[8], const Frag<uint16_t> (&pr)[RT][NV],
                                           std::integer_sequence<int, P...>) {
        (pair<P>(w, scale, pr), ...);
    }
    // Features 2 P and 2 P + 1 of the lane's.
    template <int P>
    __device__ __forceinline__ void pair(const C &w, const float (&scale)[8], const Frag<uint16_t> (&pr)[RT][NV]) {
        constexpr int kWord = BITS == 4 ? P / 4 : P / 2, kPart = BITS == 4 ? P % 4 : P % 2;
        uint32_t x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = cache::bf16_pair<BITS, kPart>(w.v[u][kWord], scale[u]);
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            lo[u] = __builtin_amdgcn_perm(x[2 * u + 1], x[2 * u], 0x05040100u);
            hi[u] = __builtin_amdgcn_perm(x[2 * u + 1], x[2 * u], 0x07060302u);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int p = NV - 1; p >= 0; --p) {
                const bf16x8 f = __builtin_bit_cast(bf16x8, pr[r][p].v);
                o[r][2 * P] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3])), f, o[r][2 * P], 0, 0, 0);
                o[r][2 * P + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3])), f, o[r][2 * P + 1], 0, 0, 0);
            }
    }
};

// One block: the rows of a (sequence, key head), over the keys of one part; its waves take 32 keys in turn and
// are joined at the end, in an order that the sizes fix.  Long caches are bound by memory: 16 x 32 (8) heads over
// 8192 of 128 in 8 bits, 230 MB, 37 us one after the other (a call whose cache is in no level of cache: 47.7); in
// 4 bits, 16 x 16 (2) over 32768, lengths from a half up, 23 to 25 us for 114 MB (4.5 to 4.9 TB/s), where some 240 vector
// instructions a step (a third of them conversions) take 0.36 of the SIMDs' cycles.  Short ones by what a
// block does once: 208 blocks of one step a wave take 5.8 us, an empty kernel with these arguments 2.9.
template <int BITS, int NB, int NP, int RT, int MM, bool HALVES, bool PACK, int WAVES, int DEPTH, int OCC>
__global__ __launch_bounds__(64 * WAVES, OCC) void cache_rows_kernel(const Args a, const Cache c) {
    using R = Rows<BITS, NB, NP, RT, MM, HALVES, PACK, WAVES>;
    constexpr int V = R::V, kRows = 16 * RT, kWide = 32 * NB + 4;  // floats of a row: 16 rows fill the banks
    constexpr int kParts = WAVES * kRows * kWide * 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[kParts > R::kQueryBytes ? kParts : R::kQueryBytes];
    __shared__ float stat[2][WAVES][kRows];
    float *const mine = reinterpret_cast<float *>(smem);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    // 32 bits: divisions in 64 would take as long as several chunks
    const uint32_t all = gridDim.x, id = (all & 7) == 0 ? (blockIdx.x & 7) * (all >> 3) + (blockIdx.x >> 3) : blockIdx.x;
    const uint32_t part = id % (uint32_t)a.splits;
    uint32_t bk = id / (uint32_t)a.splits;
    int row0 = 0;
    if constexpr (in_groups(NB, NP, PACK)) {
        row0 = (int)(bk % (uint32_t)a.tiles) * kRows;
        bk /= (uint32_t)a.tiles;
    }
    const int64_t b = bk / (uint32_t)a.key_heads, kh = bk % (uint32_t)a.key_heads;
    typename R::Piece y[R::kOwn];
    R::load_queries(a, b, kh, row0, y);
    const int len = (int)key_end(a, b);
    const uint32_t chunks = (uint32_t)(len + 31) / 32;  // below 2^26, parts at most 64
    const int c0 = (int)(chunks * part / (uint32_t)a.splits), c1 = (int)(chunks * (part + 1) / (uint32_t)a.splits);

    R r;
    r.init(a, c, b, kh, row0, len, lane);
    // Codes of DEPTH chunks are in flight or worked on, the places of the next one known.
    typename R::C w[DEPTH];
    int x = c0 + wave, ahead = x;
    cache::Place p, p1;
    const auto look = [&](int y) {  // chunk y's places; those of chunk c0 in the place of one past the end
        const int j = 32 * (y < c1 ? y : c0);
        p = cache::uniform_place(c, b, j);
        if (HALVES) p1 = cache::uniform_place(c, b, j + 16 < len ? j + 16 : j);
    };
    const auto fetch = [&](typename R::C &to) {
        r.load(a, c, b, kh, ahead, c1, len, p, p1, lane, to);
        ahead += WAVES;
        look(ahead);
    };
    if (c0 < c1) {
        look(ahead);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) fetch(w[d]);
    }
    R::form_queries(a, y, smem);
    __syncthreads();
    r.queries(smem, lane);
    // No way out in the middle: a path that skips loads would make the others wait for all of them.
    for (; x + (DEPTH - 1) * WAVES < c1; x += DEPTH * WAVES) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            r.use(a, w[d], 32 * (x + d * WAVES), lane);
            fetch(w[d]);
        }
    }
#pragma unroll
    for (int d = 0; d + 1 < DEPTH; ++d)
        if (x + d * WAVES < c1) r.use(a, w[d], 32 * (x + d * WAVES), lane);

    // The waves' parts side by side in LDS; then each thread joins quads of features.
    __syncthreads();
    if constexpr (PACK) {
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[0][k][e] = R::over_columns(r.o[0][k][e]);
    }
#pragma unroll
    for (int q = 0; q < RT; ++q) {
        const float s = over_groups_sum<16>(r.sum[q]);
        if (g == 0) stat[0][wave][16 * q + i] = r.base[q];
        if (g == 0) stat[1][wave][16 * q + i] = s;
        // register e of accumulator k is feature V (4 g + e) + k
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < V; k += 4)
                *reinterpret_cast<f32x4 *>(mine + (wave * kRows + 16 * q + i) * kWide + V * (4 * g + e) + k) =
                    f32x4{r.o[q][k][e], r.o[q][k + 1][e], r.o[q][k + 2][e], r.o[q][k + 3][e]};
    }
    __syncthreads();
    const int live = (int)(a.n * a.group) - row0, quads = (int)cdiv_dev(a.dv, 4), width = (int)quads4(a.dv);
    for (int id = threadIdx.x; id < kRows * 8 * NB; id += 64 * WAVES) {
        const int q = id / (8 * NB), f = id % (8 * NB);
        if (q >= live || f >= quads) continue;
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) top = __builtin_fmaxf(top, stat[0][v][q]);
        const float base = top == -INFINITY ? 0.0f : top;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            const float w = __builtin_amdgcn_exp2f((stat[0][v][q] - base) * R::unit());
            sum += w * stat[1][v][q];
            o += *reinterpret_cast<const f32x4 *>(mine + (v * kRows + q) * kWide + 4 * f) * w;
        }
        const int n = (int)a.n, at_row = row0 + q, hi = n == 1 ? at_row : at_row / n;
        const int64_t h = kh * a.group + hi, qi = at_row - hi * n, row = (b * a.heads + h) * n + qi;
        if (a.splits > 1) {
            const int64_t all = a.batch * a.heads * n, at = part;
            if (f == 0) {
                a.part_stats[at * 2 * all + row] = top;
                a.part_stats[(at * 2 + 1) * all + row] = sum;
            }
            store4(a.part + (at * all + row) * width, 4 * f, width, o);
        } else {
            const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            store4(reinterpret_cast<typename R::T *>(const_cast<void *>(a.o.p)) + b * a.o.b + h * a.o.h + qi * a.o.n, 4 * f,
                   (int)a.dv, o * inv);
        }
    }
}

template <int BITS, int NB, int NP, int RT, bool PACK>
int launch_rows(const Args &a, const Cache &c, int mode, unsigned blocks, hipStream_t s) {
    const auto go = [&](auto mm, auto halves, auto waves) {
        constexpr int MM = decltype(mm)::value, WAVES = decltype(waves)::value;
        constexpr int kOcc = WAVES > kRowWaves ? 1 : rows_per_cu(BITS, NB, PACK ? 1 : NP, RT);
        constexpr bool HALVES = decltype(halves)::value != 0;
        hipLaunchKernelGGL((cache_rows_kernel<BITS, NB, NP, RT, MM, HALVES, PACK, WAVES, 2, kOcc>), dim3(blocks),
                           dim3(64 * WAVES), 0, s, a, c);
        return check_launch("cache_rows_kernel");
    };
    const auto by_waves = [&](auto mm, auto halves) {
        if constexpr (may_be_whole(BITS, NB, PACK ? 1 : NP, RT))
            if (a.whole_rows) return go(mm, halves, Const<kWholeWaves>{});
        return go(mm, halves, Const<kRowWaves>{});
    };
    const auto by_page = [&](auto mm) { return c.shift == 4 ? by_waves(mm, Const<1>{}) : by_waves(mm, Const<0>{}); };
    return mode == kNoMask ? by_page(Const<kNoMask>{}) : mode == kKeep ? by_page(Const<kKeep>{}) : by_page(Const<kBias>{});
}
template <int BITS, int NP, int RT, bool PACK = false>
int rows_by_blocks(const Args &a, const Cache &c, int mode, unsigned blocks, hipStream_t s) {
    const int nb = row_blocks(c.k.blocks > c.v.blocks ? c.k.blocks : c.v.blocks);
    if (nb == 2) return launch_rows<BITS, 2, NP, RT, PACK>(a, c, mode, blocks, s);
    if constexpr (NP > 1 && RT > 1)  // (wider ones: 16 a block)
        return launch_rows<BITS, 4, NP, RT, PACK>(a, c, mode, blocks, s);
    else
        return nb == 4 ? launch_rows<BITS, 4, NP, RT, PACK>(a, c, mode, blocks, s)
                       : launch_rows<BITS, 8, NP, RT, PACK>(a, c, mode, blocks, s);
}
template <int BITS>
int rows_by_type(const Args &a, const Cache &c, int dtype, int mode, hipStream_t s) {
    const int64_t blocks = a.batch * a.key_heads * a.tiles * a.splits, rows = a.n * a.group;
    TPW_REQUIRE(blocks <= cache::kMostBlocks, "attention: too many rows");
    if (dtype == TPW_BF16)
        return rows <= 16 ? rows_by_blocks<BITS, 1, 1>(a, c, mode, (unsigned)blocks, s)
                          : rows_by_blocks<BITS, 1, 2>(a, c, mode, (unsigned)blocks, s);
    return rows <= kPackedRows ? rows_by_blocks<BITS, 3, 1, true>(a, c, mode, (unsigned)blocks, s)
           : rows <= 16 || a.tiles > 1
               ? rows_by_blocks<BITS, 3, 1>(a, c, mode, (unsigned)blocks, s)
               : rows_by_blocks<BITS, 3, 2>(a, c, mode, (unsigned)blocks, s);
}

}  // namespace attn
}  // namespace tpw
