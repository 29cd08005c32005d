// Attention forward: o_i = sum_j softmax_j(scale q_i . k_j + mask_ij) v_j in one pass over the keys
// with the running maximum and sum of every row (layouts: attention.hpp).
#include <math.h>

#include "attention.hpp"

namespace tpw {
namespace attn {

// Per-row running softmax of one wave's W rows and the loop over one key tile.
template <typename T, int W, int DP, int BN, int MM, bool DWORDS>
struct Forward {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    using CR = ColReader<T, DP, W>;
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
            q[s] = load_row8(row, M::KS * s + 8 * (lane / W), (int)a.d, DWORDS);
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
                    for (int i = 0; i < NB; ++i) M::mma1(s[i], f[i], q[k], e);
            } else {
#pragma unroll
                for (int i = 0; i < NB; ++i) M::mma(s[i], rr.read(kt, i, k), q[k]);
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
            const Frag<T> p = pack8(x, T{});
#pragma unroll
            for (int c = 0; c < CR::kPieces; ++c) CR::use(o, c, cr.read(vt, t, c), p);
        }
    }
};

// One block: kWaves * W query rows of the rows that share a key head, over the keys of one part.  The
// next tile of keys and values travels by DMA while this one is worked on, one barrier a tile.
// Bound by the matrix cores beside the softmax: a 32 x 64 tile of scores at 128 features is 1024 cycles
// of products and about 900 of maxima, exponentials, sums and packing, which the two waves of a SIMD
// overlap.  bf16, not causal: 2 x 16 (4) x 8192^2 x 128 in 1.09 to 1.19 ms (0.92 to 1.01 PFLOP/s), 8 x
// 8192^2 x 256 in 0.55 (0.99), 32 x 4096^2 x 64 in 0.18 (0.77: exponentials).  fp32: 8 x 8192^2 x 256 in
// 4.2 ms (130 TFLOP/s).  One token of 16 x 16 (2) heads over 32768 keys: 4.6 TB/s.  Priorities (s_setprio)
// around the products or the softmax changed nothing.
template <typename T, int W, int DP, int BN, int MM, bool DWORDS, int kWaves, int OCC>
__global__ __launch_bounds__(64 * kWaves, OCC) void attention_kernel(const Args a) {
    using F = Forward<T, W, DP, BN, MM, DWORDS>;
    using M = typename F::M;
    constexpr uint32_t kTileBytes = BN * Tile<T, DP>::kRowBytes;
    // two buffers of a key tile and a value tile
    __shared__ __attribute__((aligned(256))) uint4 smem[4 * kTileBytes / 16];
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
    Stager<T, DP, BN, kWaves, DWORDS> sk, sv;
    sk.init(a.k.n, (int)a.d, wave, lane);
    sv.init(a.v.n, (int)a.dv, wave, lane);
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
        const int width = (int)quads4(a.dv);
        float *p = a.part + (part * all + row) * width;
        F::CR::each(f.o, lane, [&](int at, f32x4 v) { store4(p, at, width, v); });
        return;
    }
    if (g == 0 && a.stats) {
        a.stats[row] = f.top;
        a.stats[a.batch * a.heads * a.n + row] = sum;
    }
    const OutRow<T> out(a, b, f.qh, f.qi);
    F::CR::each(f.o, lane, [&](int at, f32x4 v) { out.store(at, v * inv); });
}

// Joins the parts of every row: m = max m_s, l = sum l_s 2^(m_s - m), o = sum o_s 2^(m_s - m) / l.
// One block per row: lane s of every wave holds part s's weight; then LANES lanes of four features
// each, 256 / LANES parts at a time, in an order that the sizes fix.
template <typename T, bool BIAS, int LANES>
__global__ __launch_bounds__(256) void attention_join_kernel(const Args a) {
    constexpr int G = 256 / LANES, U = kMaxParts / G < 8 ? kMaxParts / G : 8;
    __shared__ f32x4 waves[3][LANES];
    const int64_t rows = a.batch * a.heads * a.n, row = blockIdx.x, pitch = quads4(a.dv);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, f = lane % LANES * 4;
    const float top_s = lane < a.splits ? a.part_stats[2 * lane * rows + row] : -INFINITY;
    const float sum_s = lane < a.splits ? a.part_stats[(2 * lane + 1) * rows + row] : 0.0f;
    const float top = over_groups_max<1>(top_s);
    const float base = top == -INFINITY ? 0.0f : top;
    const float w = __builtin_amdgcn_exp2f(BIAS ? (top_s - base) * kLog2e : top_s - base);
    const float sum = over_groups_sum<1>(lane < a.splits ? w * sum_s : 0.0f);
    const float *p = a.part + row * pitch + f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < a.splits; s0 += G * U) {
        f32x4 x[U];
        float c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + G * u + (int)threadIdx.x / LANES;
            const bool in = s < a.splits;
            c[u] = __shfl(w, in ? s : 0, 64);
            x[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (in && f < a.dv) x[u] = *reinterpret_cast<const f32x4 *>(p + s * rows * pitch);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) o += x[u] * c[u];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = over_groups_sum<LANES>(o[e]);
    if (wave > 0 && lane < LANES) waves[wave - 1][lane] = o;
    __syncthreads();
    if ((int)threadIdx.x >= LANES) return;
#pragma unroll
    for (int v = 0; v < 3; ++v) o += waves[v][lane];
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    if (lane == 0 && a.stats) {
        a.stats[row] = top;
        a.stats[rows + row] = sum;
    }
    const int64_t i = row % a.n, h = row / a.n % a.heads, b = row / a.n / a.heads;
    OutRow<T>(a, b, h, i).store(f, o * inv);
}

// The same for at most PARTS parts: one thread per four features, every load in flight at once
// (32 x 4096 rows of 64 features in two parts: 30 us, where a wave per row takes 80).  Of 9 to 32 parts it
// takes over where there are enough quads to fill the card (whole calls; 16 parts: 16 x 500 rows of 64, 128000
// quads, 58.7 us, with a block per row 63.4; 8 x 200 of 128, 51200 quads, 25.6, 27.0; 256 of 128, 8192 quads,
// equal; 32 parts: 16 x 128 of 64, 32768 quads, 23.9, 25.0; 26 parts: 64 of 128, 2048 quads, 12.2, 11.5).
constexpr int64_t kManyQuads = 32768;
template <typename T, bool BIAS, int PARTS>
__global__ __launch_bounds__(256) void attention_join_few_kernel(const Args a) {
    const int64_t rows = a.batch * a.heads * a.n, quads = cdiv_dev(a.dv, 4);
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / quads;
    if (row >= rows) return;
    const int f = (int)(id % quads) * 4;
    float top_s[PARTS], sum_s[PARTS];
    f32x4 x[PARTS];
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        top_s[s] = -INFINITY;
        sum_s[s] = 0.0f;
        x[s] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (s >= a.splits) continue;
        top_s[s] = a.part_stats[2 * s * rows + row];
        sum_s[s] = a.part_stats[(2 * s + 1) * rows + row];
        x[s] = *reinterpret_cast<const f32x4 *>(a.part + (s * rows + row) * (4 * quads) + f);
    }
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int s = 0; s < PARTS; ++s) top = __builtin_fmaxf(top, top_s[s]);
    const float base = top == -INFINITY ? 0.0f : top;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < PARTS; ++s) {
        const float w = __builtin_amdgcn_exp2f(BIAS ? (top_s[s] - base) * kLog2e : top_s[s] - base);
        sum += w * sum_s[s];
        o += x[s] * w;
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    if (f == 0 && a.stats) {
        a.stats[row] = top;
        a.stats[rows + row] = sum;
    }
    const int64_t i = row % a.n, h = row / a.n % a.heads, b = row / a.n / a.heads;
    OutRow<T>(a, b, h, i).store(f, o * inv);
}

namespace {

int64_t round_up(int64_t x, int64_t to) { return cdiv(x, to) * to; }

bool whole_pieces(const View &v, int64_t width, int64_t size) {
    const auto whole = [&](int64_t elements) { return elements * size % 16 == 0; };
    return aligned16(v.p) && whole(width) && whole(v.b) && whole(v.h) && whole(v.n);
}
// Strides of dimensions of one entry reach nothing: whatever they are, they ask for no copy.
View view_of(const void *p, const int64_t *strides, int64_t batch, int64_t heads, int64_t rows, int64_t width,
             int64_t size) {
    return {p, batch == 1 ? 0 : strides[0], heads == 1 ? 0 : strides[1],
            rows == 1 ? cdiv(width * size, 16) * 16 / size : strides[2]};
}

constexpr int kPadded = 6;  // q, k, v, do, o and its rest
struct PadArgs {
    View from[kPadded];
    void *to[kPadded];
    int64_t heads[kPadded], rows[kPadded], width[kPadded], pieces[kPadded], first[kPadded + 1];
    int count;
};

// Dense copies [batch, heads, rows, whole pieces] of operands, zeros past their width; one thread per
// 16-byte piece.  Staging such rows element by element inside the kernels took 200 to 300 us where the
// copies of 4 x 3001 rows of 90 take 6 to 12.
template <typename T>
__global__ void pad_kernel(const PadArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= a.first[a.count]) return;
    int t = 0;
    while (id >= a.first[t + 1]) ++t;
    id -= a.first[t];
    const int64_t c = id % a.pieces[t], r = id / a.pieces[t], i = r % a.rows[t], bh = r / a.rows[t];
    const View v = a.from[t];
    const T *row = reinterpret_cast<const T *>(v.p) + bh / a.heads[t] * v.b + bh % a.heads[t] * v.h + i * v.n;
    T x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = c * E + e < a.width[t] ? row[c * E + e] : T(0);
    uint4 w;
    __builtin_memcpy(&w, x, 16);
    reinterpret_cast<uint4 *>(a.to[t])[id] = w;
}

// Whether the forward's operands that are not whole pieces are whole dwords, to be read as they lie, and
// the call is one where that takes less than copying them: each key is read by one tile of rows (one token of
// 8 x 16 (4) heads over 16000 keys of 90 bf16: 52 us against 127 + 38), or there are few pairs (2^22: 4 x 8 x
// 128 x 1000 x 50 fp32 23 against 13 + 18, 2 x 8 x 300 x 900 x 118 fp32 46 against 13 + 32; 2^25: 4 x 8 x
// 1024^2 x 90 bf16 51 against 14 + 33).  The backward's kernels have no registers left for it.
bool reads_dwords(const Args &a, int64_t size) {
    bool pieces = true, dwords = true;
    const auto look = [&](const View &v, int64_t width) {
        pieces = pieces && whole_pieces(v, width, size);
        dwords = dwords && reinterpret_cast<uintptr_t>(v.p) % 4 == 0 && (width | v.b | v.h | v.n) * size % 4 == 0;
    };
    look(a.q, a.d);
    look(a.k, a.d);
    look(a.v, a.dv);
    return !pieces && dwords && (a.n * a.group <= 64 || a.batch * a.heads * a.n * a.m <= int64_t(1) << 22);
}

// The operands to copy, their addresses from `at` on; returns the bytes they take.
size_t plan_padding(Args &a, int dtype, bool backward, uint8_t *at, PadArgs *p) {
    const int64_t size = dtype == TPW_F32 ? 4 : 2, e = 16 / size;
    size_t bytes = 0;
    if (a.dwords) return 0;
    const auto take = [&](View &v, int64_t heads, int64_t rows, int64_t width, bool always = false) {
        if ((!always && whole_pieces(v, width, size)) || a.batch * heads * rows == 0) return;
        const int64_t pieces = cdiv(width, e), n = a.batch * heads * rows * pieces;
        if (p) {
            const int t = p->count++;
            p->from[t] = v;
            p->to[t] = at + bytes;
            p->heads[t] = heads, p->rows[t] = rows, p->width[t] = width, p->pieces[t] = pieces;
            p->first[t + 1] = p->first[t] + n;
            v = {p->to[t], heads * rows * pieces * e, rows * pieces * e, pieces * e};
        }
        bytes += (size_t)n * 16;
    };
    take(a.q, a.heads, a.n, a.d);
    take(a.k, a.key_heads, a.m, a.d);
    take(a.v, a.key_heads, a.m, a.dv);
    if (backward) {
        take(a.go, a.heads, a.n, a.dv);
        View rest = {a.rest, a.o.b, a.o.h, a.o.n};
        const bool both = a.rest && !(whole_pieces(a.o, a.dv, size) && whole_pieces(rest, a.dv, size));
        take(a.o, a.heads, a.n, a.dv, both);
        if (both) take(rest, a.heads, a.n, a.dv, both);  // strides of o
        a.rest = const_cast<void *>(rest.p);
    }
    return bytes;
}

struct BitArgs {
    const uint8_t *mask;
    uint32_t *bits, *cols;
    int64_t mb, mh, mn, mm, heads, n, m, lead, words;
};

// Bits of a boolean mask, one row of words for each of its distinct rows (a broadcast dimension
// counts once): the kernels test a bit of a word where they would load a byte, and the heads that
// share a mask read an eighth of it (3001^2: 9 us, for 110 to 230 less in each kernel).  For the
// backward also by column: word (i / 32, j) holds rows
// 32 (i / 32) .. + 31 of key j.  One wave per 64 keys x 32 rows; all of its loads are in flight at once.
__global__ __launch_bounds__(256) void pack_mask_kernel(const BitArgs a) {
    const int64_t pairs = a.words / 2, steps = cdiv_dev(a.n, 32), id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t w = id % pairs * 2, t = id / pairs, i0 = t % steps * 32, bh = t / steps;
    if (bh >= a.lead) return;
    const int lane = threadIdx.x & 63;
    const int64_t j = 32 * w + lane;
    const uint8_t *p = a.mask + bh / a.heads * a.mb + bh % a.heads * a.mh + i0 * a.mn + j * a.mm;
    const int rows = a.n - i0 < 32 ? (int)(a.n - i0) : 32;
    uint8_t x[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) x[r] = r < rows && j < a.m ? p[r * a.mn] : 0;
    uint32_t col = 0, mine = 0;
#pragma unroll
    for (int r = 0; r < 32; ++r) {
        const uint64_t all = __ballot(x[r] != 0);
        if (lane % 32 == r) mine = lane < 32 ? (uint32_t)all : (uint32_t)(all >> 32);
        col |= x[r] != 0 ? 1u << r : 0u;
    }
    if (lane % 32 < rows) a.bits[(bh * a.n + i0 + lane % 32) * a.words + w + lane / 32] = mine;
    // one row for all: every row of the column
    if (a.cols && j < a.m) a.cols[(bh * steps + i0 / 32) * a.m + j] = a.mn ? col : col ? 0xffffffffu : 0u;
}

// The bits' layout, its strides into the arguments; returns the bytes they take.
int64_t plan_bits(Args &a, bool backward, uint8_t *at, BitArgs *p) {
    const int64_t words = round_up(cdiv(a.m, 32), 2);  // whole tiles of 64 keys
    const int64_t n = a.mn ? a.n : 1, heads = a.mh ? a.heads : 1;
    const int64_t lead = heads * (a.mb ? a.batch : 1), steps = cdiv(n, 32);
    const int64_t rows = round_up(lead * n * words * 4, 16);
    if (p)
        *p = {reinterpret_cast<const uint8_t *>(a.mask), reinterpret_cast<uint32_t *>(at),
              backward ? reinterpret_cast<uint32_t *>(at + rows) : nullptr,
              a.mb, a.mh, a.mn, a.mm, heads, n, a.m, lead, words};
    a.mask = at;
    a.mask_cols = backward ? reinterpret_cast<uint32_t *>(at + rows) : nullptr;
    a.cn = a.mn ? a.m : 0;
    a.ch = a.mh ? steps * a.m : 0;
    a.cb = a.mb ? heads * steps * a.m : 0;
    a.mb = a.mb ? heads * n * words : 0;
    a.mh = a.mh ? n * words : 0;
    a.mn = a.mn ? words : 0;
    a.mm = 0;
    return rows + (backward ? round_up(lead * steps * a.m * 4, 16) : 0);
}

// Sets tiles and splits for the element type and width.
template <typename T, int DP>
void plan(Args &a) {
    using L = Tiles<T, DP>;
    constexpr int64_t kOwn = L::kWaves * L::kWidth;
    a.tiles = cdiv(a.n * a.group, kOwn);
    a.splits = (int)parts_for(a.batch * a.key_heads * a.tiles, cdiv(a.m, L::kKeys), L::kPerCu, uneven(a),
                              step_us<T, DP>(kOwn, L::kKeys, 2, L::kPerCu),
                              part_us(a.batch * a.heads * a.n, quads4(a.dv)));
}

}  // namespace

size_t prepared_bytes(const Args &a, const tpw_attention_desc *d, bool backward) {
    Args b = a;
    const size_t bits = mask_mode(d) == kKeep ? (size_t)plan_bits(b, backward, nullptr, nullptr) : 0;
    return plan_padding(b, d->dtype, backward, nullptr, nullptr) + bits;
}
int prepare_operands(Args &a, const tpw_attention_desc *d, bool backward, void *at, hipStream_t s) {
    PadArgs p = {};
    uint8_t *next = reinterpret_cast<uint8_t *>(at);
    if (const size_t bytes = plan_padding(a, d->dtype, backward, next, &p)) {
        const int64_t blocks = cdiv(p.first[p.count], 256);
        TPW_REQUIRE(blocks < (int64_t(1) << 31), "attention: too many rows");
        bool pairs = d->dtype == TPW_BF16;  // bf16 rows of whole dwords: copied by dwords
        for (int t = 0; t < p.count; ++t)
            pairs = pairs && (p.width[t] | p.from[t].b | p.from[t].h | p.from[t].n) % 2 == 0 &&
                    reinterpret_cast<uintptr_t>(p.from[t].p) % 4 == 0;
        for (int t = 0; pairs && t < p.count; ++t) {
            p.width[t] /= 2;
            p.from[t].b /= 2, p.from[t].h /= 2, p.from[t].n /= 2;
        }
        if (d->dtype == TPW_F32 || pairs)
            hipLaunchKernelGGL((pad_kernel<uint32_t>), dim3((unsigned)blocks), dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((pad_kernel<uint16_t>), dim3((unsigned)blocks), dim3(256), 0, s, p);
        if (const int rc = check_launch("pad_kernel")) return rc;
        next += bytes;
    }
    if (mask_mode(d) == kKeep) {
        BitArgs m = {};
        plan_bits(a, backward, next, &m);
        const int64_t blocks = cdiv(m.lead * cdiv(m.n, 32) * (m.words / 2), 4);
        TPW_REQUIRE(blocks < (int64_t(1) << 31), "attention: mask too large");
        hipLaunchKernelGGL(pack_mask_kernel, dim3((unsigned)blocks), dim3(256), 0, s, m);
        return check_launch("pack_mask_kernel");
    }
    return TPW_OK;
}

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
    a.q = view_of(d->query, d->query_strides, d->batch, d->heads, d->n, d->d, size);
    a.k = view_of(d->key, d->key_strides, d->batch, d->key_heads, d->m, d->d, size);
    a.v = view_of(d->value, d->value_strides, d->batch, d->key_heads, d->m, d->dv, size);
    a.o = view_of(d->out, d->out_strides, d->batch, d->heads, d->n, d->dv, size);
    a.stats = d->stats;
    a.lengths = d->lengths;
    a.mask = d->mask_type == TPW_MASK_NONE ? nullptr : d->mask;
    a.mb = d->mask_strides[0];
    a.mh = d->mask_strides[1];
    a.mn = d->mask_strides[2];
    a.mm = d->mask_strides[3];
    a.mask_bf16 = d->mask_type == TPW_MASK_ADD_BF16;
    const bool bias = mask_mode(d) == kBias;
    // a scale that 32 bits hold as zero is zero: it would turn the -inf of a key that is left out to NaN
    a.scale = (float)(fabs(d->scale) * (bias ? 1.0 : 1.4426950408889634));
    a.qsign = a.scale == 0.0f ? 0.0f : d->scale > 0 ? 1.0f : -1.0f;
    if (a.scale == 0.0f) a.scale = 1.0f;
    a.gscale = (float)d->scale;
    a.rest = d->dtype == TPW_BF16 ? d->out_rest : nullptr;
    const auto streamed = [&](const View &v, int64_t rows, int64_t width) {
        return a.batch * a.heads * a.n * a.m == 0 || rows <= 1 || (v.n >= width && v.n * size <= (int64_t(1) << 23));
    };
    bool ok = streamed(a.k, d->m, d->d) && streamed(a.v, d->m, d->dv);
    if (backward) {
        a.go = view_of(d->grad_out, d->grad_out_strides, d->batch, d->heads, d->n, d->dv, size);
        a.gq = view_of(d->grad_query, d->grad_query_strides, d->batch, d->heads, d->n, d->d, size);
        a.gk = view_of(d->grad_key, d->grad_key_strides, d->batch, d->key_heads, d->m, d->d, size);
        a.gv = view_of(d->grad_value, d->grad_value_strides, d->batch, d->key_heads, d->m, d->dv, size);
        ok = ok && streamed(a.q, d->n, d->d) && streamed(a.go, d->n, d->dv);
    }
    TPW_REQUIRE(ok, "attention: rows of an operand overlap or lie more than 8 MiB apart");
    a.dwords = !backward && reads_dwords(a, size);
    return TPW_OK;
}

}  // namespace attn
}  // namespace tpw

using namespace tpw;
using namespace tpw::attn;

namespace {

size_t forward_workspace(const Args &a) {
    return a.splits > 1 ? (size_t)a.splits * a.batch * a.heads * a.n * (quads4(a.dv) + 2) * 4 : 0;
}

}  // namespace

extern "C" size_t tpw_attention_workspace_size(const tpw_attention_desc *d) {
    Args a = {};
    if (read_args(d, false, a) != TPW_OK || a.batch * a.heads * a.n == 0) return 0;
    size_t bytes = 0;
    by_type(a, d->dtype, kNoMask, [&](auto t, auto dp, auto) {
        plan<decltype(t), decltype(dp)::value>(a);
        bytes = prepared_bytes(a, d, false) + forward_workspace(a);
        return TPW_OK;
    });
    return bytes;
}

extern "C" int tpw_attention(const tpw_attention_desc *d, void *workspace, void *stream) {
    Args a = {};
    if (const int rc = read_args(d, false, a)) return rc;
    if (a.batch * a.heads * a.n == 0) return TPW_OK;
    TPW_REQUIRE(a.q.p && a.o.p && (a.m == 0 || (a.k.p && a.v.p)), "attention: null operand");
    TPW_REQUIRE(mask_mode(d) == kNoMask || a.mask, "attention: null mask");
    hipStream_t s = as_stream(stream);
    const size_t prepared = prepared_bytes(a, d, false);
    if (prepared) {
        TPW_REQUIRE(workspace && aligned16(workspace), "attention: null or unaligned workspace");
        if (const int rc = prepare_operands(a, d, false, workspace, s)) return rc;
    }
    return by_type(a, d->dtype, mask_mode(d), [&](auto t, auto dp, auto mode) {
        using T = decltype(t);
        constexpr int DP = decltype(dp)::value, MM = decltype(mode)::value, W = Tiles<T, DP>::kWidth;
        plan<T, DP>(a);
        const int64_t blocks = a.batch * a.key_heads * a.tiles * a.splits, rows = a.batch * a.heads * a.n;
        TPW_REQUIRE(blocks < (int64_t(1) << 31), "attention: too many rows");
        if (a.splits > 1) {
            TPW_REQUIRE(workspace && aligned16(workspace), "attention: null or unaligned workspace");
            a.part = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + prepared);
            a.part_stats = a.part + a.splits * rows * quads4(a.dv);
        }
        constexpr int kOcc = 2;
        constexpr int kWaves = Tiles<T, DP>::kWaves;
        constexpr int kKeys = Tiles<T, DP>::kKeys;
        // a kernel of its own: the branch alone would cost the others 2 %
        if (a.dwords)
            hipLaunchKernelGGL((attention_kernel<T, W, DP, kKeys, MM, true, kWaves, kOcc>), dim3((unsigned)blocks),
                               dim3(64 * kWaves), 0, s, a);
        else
            hipLaunchKernelGGL((attention_kernel<T, W, DP, kKeys, MM, false, kWaves, kOcc>), dim3((unsigned)blocks),
                               dim3(64 * kWaves), 0, s, a);
        if (const int rc = check_launch("attention_kernel")) return rc;
        if (a.splits > 1) {
            const int64_t quads = rows * cdiv(a.dv, 4);
            const dim3 few((unsigned)cdiv(quads, 256));
            if (a.splits <= 8)
                hipLaunchKernelGGL((attention_join_few_kernel<T, MM == kBias, 8>), few, dim3(256), 0, s, a);
            else if (a.splits <= 16 && quads >= kManyQuads)
                hipLaunchKernelGGL((attention_join_few_kernel<T, MM == kBias, 16>), few, dim3(256), 0, s, a);
            else if (a.splits <= 32 && quads >= kManyQuads)
                hipLaunchKernelGGL((attention_join_few_kernel<T, MM == kBias, 32>), few, dim3(256), 0, s, a);
            else
                hipLaunchKernelGGL((attention_join_kernel<T, MM == kBias, Tile<T, DP>::P / 4>), dim3((unsigned)rows),
                                   dim3(256), 0, s, a);
            return check_launch("attention_join_kernel");
        }
        return TPW_OK;
    });
}
