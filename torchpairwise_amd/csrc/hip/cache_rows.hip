// Attention of a few query rows a key head (single tokens, drafts) over a cache in 4 or 8 bits.
#include <type_traits>

#include "cache_attention.hpp"

namespace tpw {
namespace attn {
namespace {

using cache::Cache;
using cache::Eight;
using cache::Side;

// Loads of NW words from p (NW * 4 bytes aligned up to 16).
template <int NW>
__device__ __forceinline__ void load_words(uint32_t (&w)[NW], const uint8_t *p) {
    __builtin_memcpy(w, __builtin_assume_aligned(p, NW >= 4 ? 16 : NW * 4), sizeof(w));
}

// The codes and scales of 32 keys, as a lane (i = lane % 16, g = lane / 16) uses them.
//   Keys: first operands of 16 x 16 x 32 products.  Product t's row i is key 8 (i / 4) + 4 t + i % 4, so that
//     the scores a lane receives (rows 4 g .. + 3) are keys 8 g + 4 t .. + 3: eight consecutive ones in two
//     products.  The lane holds features F g .. + F - 1 of its key, F = 8 NB, whole words side by side: which
//     features a product sums over is free as long as the queries agree.
//   Values: lane i holds features V i .. + V - 1 (V = 2 NB) of keys 8 g .. + 7, the keys of its scores.
// Nothing passes through LDS: each code is loaded by the lane that multiplies it, in pieces of 4 to 16
// bytes, a row's 64 bytes (128 features) by 4 or 16 lanes side by side.
template <int BITS, int NB>
struct Codes {
    static constexpr int KW = NB * BITS / 4;                       // words of a key
    static constexpr int VW = NB * BITS >= 16 ? NB * BITS / 16 : 1;  // words of a value row (4 bits, 64 features: half)
    static constexpr int KS = NB > 4 ? NB / 4 : 1;                 // blocks that a lane's part of a key touches
    uint32_t k[2][KS][KW / KS], v[8][VW];
    uint2 ks[KS], vs;  // scales of the lane's granules of eight keys
    bool live;         // the values' granule lies in the cache, before the length
};

// Granules of eight keys, from sequence b's row j on: address of (entry, row), 0 where they are not to be read.
struct Granule {
    int64_t first;
    int row;
    bool live;
};
__device__ __forceinline__ Granule granule(const Cache &c, int64_t b, int j, int len) {
    if (j >= len) return {c.pages ? 0 : b, 0, false};
    const cache::Place p = cache::place(c, b, j);
    return p.first < 0 ? Granule{0, 0, false} : Granule{p.first, p.row, true};
}

template <int BITS, int NB, int NP, int RT, bool BIAS, int WAVES>
struct Rows {
    using C = Codes<BITS, NB>;
    static constexpr int F = 8 * NB, V = 2 * NB;

    Frag<uint16_t> q[RT][NB][NP];
    f32x4 o[RT][V];
    float base[RT], sum[RT];  // the row's running base, at most kSlack below its maximum; the lane's sum
    int lim[RT];              // keys that the row sees
    int64_t qh[RT], qi[RT];   // head and row (row -1: none)
    int kblock[C::KS], koff[C::KS], vblock, voff;  // blocks and bytes of a lane's part of a row

    __device__ __forceinline__ void init(const Args &a, const Cache &c, int64_t b, int64_t kh, int64_t row0, int64_t len,
                                         int lane) {
        const int i = lane & 15, g = lane >> 4;
        // blocks past the row's are not there: block 0 in their place, against queries of zero
#pragma unroll
        for (int s = 0; s < C::KS; ++s) {
            const int k = F * g / 32 + s;
            kblock[s] = k < c.k.blocks ? k : 0;
            koff[s] = k < c.k.blocks ? (F * g + 32 * s) * BITS / 8 : 0;
        }
        vblock = V * i / 32 < c.v.blocks ? V * i / 32 : 0;
        voff = V * i / 32 < c.v.blocks ? V * i * BITS / 8 : 0;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int64_t r = row0 + 16 * t + i, rows = a.n * a.group;
            const bool in = r < rows;
            qh[t] = kh * a.group + (in ? r / a.n : 0);
            qi[t] = in ? r % a.n : -1;
            const int64_t l = in ? row_limit(a, len, qi[t]) : 0;
            lim[t] = (int)(l < len ? l : len);
#pragma unroll
            for (int k = 0; k < V; ++k) o[t][k] = f32x4{0, 0, 0, 0};
            base[t] = -INFINITY;
            sum[t] = 0.0f;
        }
    }

    // The block's queries, times the sign of the scale, to LDS as float32, zeros past their width and behind the
    // last row: a thread's pieces of 8 features side by side, element by element where they do not lie so.
    static constexpr int kPitch = 32 * NB + 4;  // floats of a row: 16 rows' pieces fall on different banks
    static __device__ __forceinline__ void stage(const Args &a, int64_t b, int64_t kh, float *to) {
        using T = std::conditional_t<NP == 1, uint16_t, float>;
        const T *q = reinterpret_cast<const T *>(a.q.p) + b * a.q.b;
        const int rows = (int)(a.n * a.group), d = (int)a.d;
        const auto at = [&](int r) { return (kh * a.group + r / (int)a.n) * a.q.h + r % (int)a.n * a.q.n; };
        constexpr int kPieces = RT * 16 * 4 * NB, kThreads = 64 * WAVES;
        if (a.whole_q) {
#pragma unroll
            for (int x = 0; x < (kPieces + kThreads - 1) / kThreads; ++x) {
                const int id = x * kThreads + (int)threadIdx.x, r = id / (4 * NB), f = id % (4 * NB) * 8;
                if (kPieces % kThreads && id >= kPieces) break;
                T y[8] = {};
                if (r < rows && f < d) __builtin_memcpy(y, __builtin_assume_aligned(q + at(r) + f, 16), sizeof(y));
#pragma unroll
                for (int e = 0; e < 8; ++e) to[r * kPitch + f + e] = to_f32(y[e]) * a.qsign;
            }
        } else {
#pragma unroll 4
            for (int id = threadIdx.x; id < 8 * kPieces; id += kThreads) {
                const int r = id / (32 * NB), f = id % (32 * NB);
                to[r * kPitch + f] = r < rows && f < d ? to_f32(q[at(r) + f]) * a.qsign : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void queries(const float *from, int lane) {
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int s = 0; s < NB; ++s) {
                float x[8];
                __builtin_memcpy(x, __builtin_assume_aligned(from + (16 * t + i) * kPitch + F * g + 8 * s, 16), sizeof(x));
                if constexpr (NP > 1) {  // an infinity is its first summand alone
                    float inf[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        inf[e] = __builtin_fabsf(x[e]) == INFINITY ? x[e] : 0.0f;
                        if (inf[e] != 0.0f) x[e] = 0.0f;
                    }
                    split(x, q[t][s]);
                    uint32_t w[4] = {q[t][s][0].v.x, q[t][s][0].v.y, q[t][s][0].v.z, q[t][s][0].v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] |= high(__float_as_uint(inf[2 * e]), __float_as_uint(inf[2 * e + 1]));
                    q[t][s][0].v = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    split(x, q[t][s]);
                }
            }
    }

    // One summand in bfloat16, rounded; or three that hold all 24 bits, each what is left cut off to 8.
    static __device__ __forceinline__ void split(float (&x)[8], Frag<uint16_t> (&f)[NP]) {
        if constexpr (NP == 1) {
            f[0] = pack8(x, uint16_t{});
        } else {
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __float_as_uint(x[e]);
                    x[e] -= __uint_as_float(w[e] & 0xffff0000u);
                }
                f[p].v = make_uint4(high(w[0], w[1]), high(w[2], w[3]), high(w[4], w[5]), high(w[6], w[7]));
            }
        }
    }
    static __device__ __forceinline__ uint32_t high(uint32_t lo, uint32_t hi) {
        return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
    }

    __device__ __forceinline__ void load(const Cache &c, int64_t b, int64_t kh, int j0, int len, int lane, C &w) const {
        const int i = lane & 15, g = lane >> 4;
        const Granule gk = granule(c, b, j0 + 8 * (i >> 2), len), gv = granule(c, b, j0 + 8 * g, len);
        const uint8_t *k = c.k.codes + gk.first * c.k.cf + kh * c.k.ch + (gk.row + (i & 3)) * c.k.cr;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int s = 0; s < C::KS; ++s) load_words(w.k[t][s], k + 4 * t * c.k.cr + koff[s]);
        const uint8_t *ks = c.k.scales + gk.first * c.k.sf + kh * c.k.sh + gk.row;
#pragma unroll
        for (int s = 0; s < C::KS; ++s) w.ks[s] = *reinterpret_cast<const uint2 *>(ks + kblock[s] * c.k.sb);
        const uint8_t *v = c.v.codes + gv.first * c.v.cf + kh * c.v.ch + gv.row * c.v.cr + voff;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if constexpr (NB * BITS < 16)
                w.v[u][0] = *reinterpret_cast<const uint16_t *>(v + u * c.v.cr);
            else
                load_words(w.v[u], v + u * c.v.cr);
        }
        w.vs = *reinterpret_cast<const uint2 *>(c.v.scales + gv.first * c.v.sf + kh * c.v.sh + vblock * c.v.sb + gv.row);
        w.live = gv.live;
    }

    // Added values (natural units) and what a boolean mask leaves, for keys j .. j + 7 of row t.
    __device__ __forceinline__ void masked(const Args &a, int64_t b, int t, int j, float (&s)[8]) const {
        const int64_t at = b * a.mb + qh[t] * a.mh + (qi[t] < 0 ? 0 : qi[t]) * a.mn + j * a.mm;
        if constexpr (BIAS) {
            float x[8];
            if (a.mask_bf16) {
                const uint16_t *p = reinterpret_cast<const uint16_t *>(a.mask) + at;
                uint16_t y[8];
                if (a.mm == 1) {
                    __builtin_memcpy(y, p, 16);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = p[e * a.mm];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = bf16_to_f32(y[e]);
            } else {
                const float *p = reinterpret_cast<const float *>(a.mask) + at;
                if (a.mm == 1) {
                    __builtin_memcpy(x, p, 32);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = p[e * a.mm];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = x[e] == -INFINITY ? -INFINITY : s[e] * a.scale + x[e];
        } else {
            const uint8_t *p = reinterpret_cast<const uint8_t *>(a.mask) + at;
            uint8_t y[8];
            if (a.mm == 1) {
                __builtin_memcpy(y, p, 8);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = p[e * a.mm];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = y[e] ? s[e] : -INFINITY;
        }
    }

    // 32 keys from j0 on.
    __device__ __forceinline__ void use(const Args &a, int64_t b, C &w, int j0, int len, int lane) {
        const int i = lane & 15, g = lane >> 4, j = j0 + 8 * g;
        if (j0 + 32 > len || !__all(w.live)) {  // values that are not there: zeros
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint32_t there = w.live && j + u < len ? 0xffffffffu : 0u;
#pragma unroll
                for (int x = 0; x < C::VW; ++x) w.v[u][x] &= there;
                uint32_t &s = u < 4 ? w.vs.x : w.vs.y;
                s &= there | ~(0xffu << (8 * (u & 3)));
            }
        }
        f32x4 s[2][RT];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < RT; ++r) s[t][r] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                constexpr int kSteps = NB / C::KS;  // products of a block
                const uint2 by = w.ks[k / kSteps];
                const float scale = cache::scale_of(((t ? by.y : by.x) >> (8 * (i & 3))) & 0xffu);
                Eight<BITS> e;
#pragma unroll
                for (int x = 0; x < BITS / 4; ++x) e.w[x] = w.k[t][k / kSteps][k % kSteps * (BITS / 4) + x];
                const bf16x8 f = __builtin_bit_cast(bf16x8, e.bf16(scale));
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p)
                        s[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(bf16x8, q[r][k][p].v),
                                                                          s[t][r], 0, 0, 0);
            }
        }
        Frag<uint16_t> pr[RT][NP];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = s[e / 4][r][e % 4];
            if constexpr (BIAS) {
                masked(a, b, r, j < len ? j : 0, x);
            } else {
                if (a.mask) masked(a, b, r, j < len ? j : 0, x);
            }
            const int end = w.live ? lim[r] - j : 0;  // of the lane's eight keys, those the row sees
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
            // bfloat16 queries: probabilities rounded to bfloat16 (within 2^-9 of each), their sum is not
            split(x, pr[r]);
        }
        float vscale[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) vscale[u] = cache::scale_of(((u < 4 ? w.vs.x : w.vs.y) >> (8 * (u & 3))) & 0xffu);
        values(w, vscale, pr, std::make_integer_sequence<int, NB>{});
    }

    static __device__ __forceinline__ float unit() { return BIAS ? kLog2e : 1.0f; }
    static constexpr float kSlack = BIAS ? 5.0f : 8.0f;

    template <int... P>
    __device__ __forceinline__ void values(const C &w, const float (&scale)[8], const Frag<uint16_t> (&pr)[RT][NP],
                                           std::integer_sequence<int, P...>) {
        (pair<P>(w, scale, pr), ...);
    }
    // Features 2 P and 2 P + 1 of the lane's.
    template <int P>
    __device__ __forceinline__ void pair(const C &w, const float (&scale)[8], const Frag<uint16_t> (&pr)[RT][NP]) {
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
            for (int p = NP - 1; p >= 0; --p) {
                const bf16x8 f = __builtin_bit_cast(bf16x8, pr[r][p].v);
                o[r][2 * P] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3])), f, o[r][2 * P], 0, 0, 0);
                o[r][2 * P + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3])), f, o[r][2 * P + 1], 0, 0, 0);
            }
    }
};

// One block: the rows of a (sequence, key head), over the keys of one part; its waves take 32 keys in turn and
// are joined at the end, in an order that the sizes fix.
template <int BITS, int NB, int NP, int RT, bool BIAS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void cache_rows_kernel(const Args a, const Cache c) {
    using R = Rows<BITS, NB, NP, RT, BIAS, WAVES>;
    constexpr int V = R::V, H = WAVES / 2;
    constexpr int kHalf = H * RT * V * 64 * 4, kQueries = RT * 16 * R::kPitch;
    __shared__ __attribute__((aligned(16))) float smem[kHalf > kQueries ? kHalf : kQueries];
    f32x4(*half)[RT * V][64] = reinterpret_cast<f32x4(*)[RT * V][64]>(smem);
    __shared__ float stat[2][WAVES][RT][16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    int64_t t = xcd_linear(blockIdx.x, gridDim.x);
    const int64_t part = t % a.splits;
    t /= a.splits;
    const int64_t b = t / a.key_heads, kh = t % a.key_heads;
    const int len = (int)key_end(a, b), chunks = (int)cdiv_dev(len, 32);
    const int c0 = (int)((int64_t)chunks * part / a.splits), c1 = (int)((int64_t)chunks * (part + 1) / a.splits);

    R r;
    r.init(a, c, b, kh, 0, len, lane);
    typename R::C w, next;
    int x = c0 + wave;
    if (x < c1) r.load(c, b, kh, 32 * x, len, lane, w);
    R::stage(a, b, kh, smem);
    __syncthreads();
    r.queries(smem, lane);
    for (; x < c1; x += WAVES) {
        if (x + WAVES < c1) r.load(c, b, kh, 32 * (x + WAVES), len, lane, next);
        r.use(a, b, w, 32 * x, len, lane);
        w = next;
    }

    float top[RT], sum[RT];
#pragma unroll
    for (int q = 0; q < RT; ++q) {
        const float s = over_groups_sum<16>(r.sum[q]);
        if (g == 0) stat[0][wave][q][i] = r.base[q];
        if (g == 0) stat[1][wave][q][i] = s;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < RT; ++q) {
        top[q] = -INFINITY;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) top[q] = __builtin_fmaxf(top[q], stat[0][v][q][i]);
        const float base = top[q] == -INFINITY ? 0.0f : top[q];
        sum[q] = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v)
            sum[q] += stat[1][v][q][i] * __builtin_amdgcn_exp2f((stat[0][v][q][i] - base) * R::unit());
        const float f = __builtin_amdgcn_exp2f((r.base[q] - base) * R::unit());
#pragma unroll
        for (int k = 0; k < V; ++k) r.o[q][k] *= f;
    }
#pragma unroll
    for (int h = H; h >= 1; h /= 2) {
        if (wave >= h && wave < 2 * h) {
#pragma unroll
            for (int q = 0; q < RT; ++q)
#pragma unroll
                for (int k = 0; k < V; ++k) half[wave - h][q * V + k][lane] = r.o[q][k];
        }
        __syncthreads();
        if (wave < h) {
#pragma unroll
            for (int q = 0; q < RT; ++q)
#pragma unroll
                for (int k = 0; k < V; ++k) r.o[q][k] += half[wave][q * V + k][lane];
        }
        if (h > 1) __syncthreads();
    }
    if (wave > 0) return;

#pragma unroll
    for (int q = 0; q < RT; ++q) {
        if (r.qi[q] < 0) continue;
        const int64_t row = (b * a.heads + r.qh[q]) * a.n + r.qi[q], all = a.batch * a.heads * a.n;
        const float inv = sum[q] > 0.0f || sum[q] != sum[q] ? 1.0f / sum[q] : 0.0f;
        const int width = (int)quads4(a.dv);
        if (a.splits > 1 && g == 0) {
            a.part_stats[part * 2 * all + row] = top[q];
            a.part_stats[(part * 2 + 1) * all + row] = sum[q];
        }
        float *p = a.part + (part * all + row) * width;
        const int64_t at = b * a.o.b + r.qh[q] * a.o.h + r.qi[q] * a.o.n;
        // register e of accumulator k is feature V (4 g + e) + k
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const int f = V * (4 * g + e) + k;
                const f32x4 v = {r.o[q][k][e], r.o[q][k + 1][e], r.o[q][k + 2][e], r.o[q][k + 3][e]};
                if (a.splits > 1)
                    store4(p, f, width, v);
                else if constexpr (NP == 1)
                    store4(reinterpret_cast<uint16_t *>(const_cast<void *>(a.o.p)) + at, f, (int)a.dv, v * inv);
                else
                    store4(reinterpret_cast<float *>(const_cast<void *>(a.o.p)) + at, f, (int)a.dv, v * inv);
            }
    }
}

constexpr int kWaves = 4;

template <int BITS, int NB, int NP, int RT>
int launch(const Args &a, const Cache &c, bool bias, unsigned blocks, hipStream_t s) {
    if (bias)
        hipLaunchKernelGGL((cache_rows_kernel<BITS, NB, NP, RT, true, kWaves>), dim3(blocks), dim3(64 * kWaves), 0, s, a, c);
    else
        hipLaunchKernelGGL((cache_rows_kernel<BITS, NB, NP, RT, false, kWaves>), dim3(blocks), dim3(64 * kWaves), 0, s, a, c);
    return check_launch("cache_rows_kernel");
}
template <int BITS, int NP, int RT>
int by_blocks(const Args &a, const Cache &c, bool bias, unsigned blocks, hipStream_t s) {
    const int most = c.k.blocks > c.v.blocks ? c.k.blocks : c.v.blocks;
    if (most <= 2) return launch<BITS, 2, NP, RT>(a, c, bias, blocks, s);
    if constexpr (NP > 1 && RT > 1)
        return launch<BITS, 4, NP, RT>(a, c, bias, blocks, s);
    else
        return most <= 4 ? launch<BITS, 4, NP, RT>(a, c, bias, blocks, s)
                         : launch<BITS, 8, NP, RT>(a, c, bias, blocks, s);
}
template <int BITS>
int by_rows(const Args &a, const Cache &c, int dtype, bool bias, unsigned blocks, hipStream_t s) {
    const bool one = a.n * a.group <= 16;
    // wider float32 caches come with 16 rows at most, blocks without a query or an output uncounted
    if (dtype == TPW_BF16)
        return one ? by_blocks<BITS, 1, 1>(a, c, bias, blocks, s) : by_blocks<BITS, 1, 2>(a, c, bias, blocks, s);
    return one ? by_blocks<BITS, 3, 1>(a, c, bias, blocks, s) : by_blocks<BITS, 3, 2>(a, c, bias, blocks, s);
}

}  // namespace

void plan_rows(Args &a) {
    const int64_t bk = a.batch * a.key_heads, chunks = cdiv(a.m, 32);
    int64_t splits = bk > 0 ? cdiv(256 * 3, bk) : 1;
    const int64_t most = cdiv(chunks, kWaves);
    splits = splits > most ? most : splits;
    a.splits = (int)(splits < 1 ? 1 : splits > kMaxParts ? kMaxParts : splits);
    a.tiles = 1;
}

int cache_rows(const Args &a, const Cache &c, int bits, int dtype, bool bias, hipStream_t s) {
    const int64_t blocks = a.batch * a.key_heads * a.splits;
    TPW_REQUIRE(blocks < (int64_t(1) << 31), "attention: too many rows");
    return bits == 4 ? by_rows<4>(a, c, dtype, bias, (unsigned)blocks, s)
                     : by_rows<8>(a, c, dtype, bias, (unsigned)blocks, s);
}

}  // namespace attn
}  // namespace tpw
