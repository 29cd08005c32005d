// Attention backward.  The probabilities are formed again from q, k and the saved row maxima and
// sums; no [n, m] matrix is written and nothing is added atomically, so results do not depend on
// the order of blocks:
//   p_ij = exp(s_ij - m_i) / l_i,  dp_ij = do_i . v_j,  delta_i = do_i . o_i,
//   ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = scale sum_j ds_ij k_j                    attention_dq_kernel: a wave owns query rows
//   dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i   attention_dkv_kernel: a wave owns keys
// Seven products where five would do with dq summed in memory: the two scores' products are formed
// in both kernels.
#include <math.h>

#include "attention.hpp"

namespace tpw {
namespace attn {

// Runs N steps of `use` on fragments that `load` reads from LDS, the next step's reads issued before
// this step's products.  The compiler may not move the reads further ahead: left alone it hoists
// them all and spills the accumulators.
template <int N, int F, typename Piece, typename Load, typename Use>
__device__ __forceinline__ void stream_steps(Load load, Use use) {
    Piece f[2][F];
    load(0, f[0]);
#pragma unroll
    for (int x = 0; x < N; ++x) {
        if (x + 1 < N) load(x + 1, f[(x + 1) & 1]);
        asm volatile("" ::: "memory");
        use(x, f[x & 1]);
    }
}

constexpr int kUnit = 32;  // rows (keys) of the streamed operand that are worked on at a time

template <typename T, int W, int DP, int BN, int MM, int kWaves, int OCC>
__global__ __launch_bounds__(64 * kWaves, OCC) void attention_dq_kernel(const Args a) {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    using CR = ColReader<T, DP, W>;
    constexpr int DB = DP / W, QS = DP / M::KS, NU = kUnit / W, ST = kUnit / M::KS;
    constexpr uint32_t kTileBytes = BN * DP * sizeof(T);
    __shared__ __attribute__((aligned(256))) uint4 smem[4 * kTileBytes / 16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane / W;
    int64_t t = xcd_linear(blockIdx.x, gridDim.x);
    const int64_t part = t % a.splits;
    t /= a.splits;
    const int64_t tile = a.tiles - 1 - t % a.tiles;
    const int64_t bk = t / a.tiles, b = bk / a.key_heads, kh = bk % a.key_heads;
    const int64_t len = key_end(a, b), rows = a.n * a.group, all = a.batch * a.heads * a.n;
    const int64_t row0 = tile * (kWaves * W), row1 = row0 + kWaves * W < rows ? row0 + kWaves * W : rows;

    const int64_t r = row0 + wave * W + lane % W;
    const bool live = r < rows;
    const int64_t qh = kh * a.group + (live ? r / a.n : 0), qi = live ? r % a.n : -1;
    const int lim = (int)(live ? row_limit(a, len, qi) : 0);
    int wmax = lim, wmin = live ? lim : 0x7fffffff;
#pragma unroll
    for (int s = 1; s < W; s <<= 1) {
        const int x = __shfl_xor(wmax, s, 64), y = __shfl_xor(wmin, s, 64);
        wmax = wmax > x ? wmax : x;
        wmin = wmin < y ? wmin : y;
    }
    wmax = __builtin_amdgcn_readfirstlane(wmax);
    wmin = __builtin_amdgcn_readfirstlane(wmin);

    Frag<T> q[QS], go[QS];
    float delta = 0.0f;
    {
        const T *qr = live ? reinterpret_cast<const T *>(a.q.p) + b * a.q.b + qh * a.q.h + qi * a.q.n : nullptr;
        const T *gr = live ? reinterpret_cast<const T *>(a.go.p) + b * a.go.b + qh * a.go.h + qi * a.go.n : nullptr;
        const T *orow = live ? reinterpret_cast<const T *>(a.o.p) + b * a.o.b + qh * a.o.h + qi * a.o.n : nullptr;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            const int f = M::KS * s + 8 * g;
            q[s] = load_row8(qr, f, (int)a.d);
            go[s] = load_row8(gr, f, (int)a.dv);
            float x[8], y[8];
            if (a.qsign != 1.0f) {
                unpack8(q[s], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= a.qsign;
                q[s] = pack8(x, T{});
            }
            unpack8(go[s], x);
            unpack8(load_row8(orow, f, (int)a.dv), y);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(x[e], y[e], delta);
        }
        delta = over_groups_sum<W>(delta);
    }
    const int64_t row = live ? (b * a.heads + qh) * a.n + qi : 0;
    float base = 0.0f, inv = 0.0f;
    if (live) {
        const float top = a.stats[row], sum = a.stats[all + row];
        base = top == -INFINITY ? 0.0f : top;
        inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
        if (g == 0 && part == 0) {
            a.rows[row] = base;
            a.rows[all + row] = inv;
            a.rows[2 * all + row] = delta;
        }
    }

    Acc dq[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) dq[i] = Acc{};

    int64_t end = len;
    if (a.causal && row0 / a.n == (row1 - 1) / a.n) end = row_limit(a, len, (row1 - 1) % a.n);
    const int nt = (int)cdiv_dev(end, BN);
    const int t0 = (int)((int64_t)nt * part / a.splits), t1 = (int)((int64_t)nt * (part + 1) / a.splits);

    const uint32_t lds = tile::lds_addr(smem);
    Stager<T, DP, BN, kWaves> sk, sv;
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
    const RowReader<T, DP, W> rr(lane);
    const CR cr(lane);
    if (t0 < t1) fetch(t0);
    for (int it = t0; it < t1; ++it) {
        tile::barrier_all();
        if (it + 1 < t1) fetch(it + 1);
        const uint32_t kt = lds + (uint32_t)((it - t0) & 1) * 2 * kTileBytes, vt = kt + kTileBytes;
#pragma unroll
        for (int u = 0; u < BN / kUnit; ++u) {
            const int j0 = it * BN + u * kUnit;
            if (j0 >= wmax) break;
            Acc s[NU], dp[NU];
#pragma unroll
            for (int i = 0; i < NU; ++i) s[i] = dp[i] = Acc{};
#pragma unroll
            for (int k = 0; k < QS; ++k)
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    M::mma(s[i], rr.read(kt, u * NU + i, k), q[k]);
                    M::mma(dp[i], rr.read(vt, u * NU + i, k), go[k]);
                }
            if constexpr (MM == kBias) {
                const void *mr = mask_row(a, b, qh, qi);
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w) {
                        const int j = j0 + W * i + 4 * M::NG * w + 4 * g;
                        f32x4 add = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (j < lim) add = mask_bias4(a, mr, j);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool off = add[e] == -INFINITY;
                            s[i][4 * w + e] = off ? -INFINITY : s[i][4 * w + e] * a.scale + add[e];
                            if (off) dp[i][4 * w + e] = 0.0f;
                        }
                    }
            }
            if constexpr (MM == kKeep) {
                const uint32_t keep = j0 < lim ? mask_words(a, b, qh, qi)[j0 / 32] >> (4 * g) : 0;
#pragma unroll
                for (int x = 0; x < 32 / (4 * M::NG); ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(keep & (1u << (4 * M::NG * x + e)))) {
                            const int at = 4 * M::NG * x;
                            s[at / W][4 * (at % W / (4 * M::NG)) + e] = -INFINITY;
                            dp[at / W][4 * (at % W / (4 * M::NG)) + e] = 0.0f;
                        }
            }
            if (j0 + kUnit > wmin) {
                asm volatile("");  // a branch: most units skip this
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (j0 + W * i + 4 * M::NG * w + 4 * g + e >= lim) {
                                s[i][4 * w + e] = -INFINITY;
                                dp[i][4 * w + e] = 0.0f;
                            }
            }
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int e = 0; e < 4 * M::Q; ++e) {
                    const float p = MM == kBias ? __builtin_amdgcn_exp2f((s[i][e] - base) * kLog2e)
                                                : __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e], a.scale, -base));
                    s[i][e] = p * inv * (dp[i][e] - delta);
                }
            // ds of bf16 inputs is rounded to bf16 for the matrix cores, as p is
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                float x[8];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[4 * v + e] = s[(2 * st + v) / M::Q][4 * ((2 * st + v) % M::Q) + e];
                const Frag<T> ds = pack8(x, T{});
#pragma unroll
                for (int c = 0; c < CR::kPieces; ++c) CR::use(dq, c, cr.read(kt, u * ST + st, c), ds);
            }
        }
    }
    if (!live) return;
    if (a.splits > 1) {
        float *p = a.part + (part * all + row) * quads4(a.d);
        CR::each(dq, lane, [&](int at, f32x4 v) { store4(p, at, (int)a.d, 1, v); });
        return;
    }
    T *p = reinterpret_cast<T *>(const_cast<void *>(a.gq.p)) + b * a.gq.b + qh * a.gq.h + qi * a.gq.n;
    CR::each(dq, lane, [&](int at, f32x4 v) { store4(p, at, (int)a.d, a.vec_out, v * a.gscale); });
}

template <typename T, int W, int DP, int BM, int MM, int kWaves, int OCC, bool VLDS, int OUT>
__global__ __launch_bounds__(64 * kWaves, OCC) void attention_dkv_kernel(const Args a) {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    using CR = ColReader<T, DP, W>;
    constexpr int DB = DP / W, QS = DP / M::KS, NU = kUnit / W, ST = kUnit / M::KS;
    constexpr uint32_t kTileBytes = BM * DP * sizeof(T), kBuf = 2 * kTileBytes + 3 * 64 * 4;
    static_assert(BM <= 64, "one DMA of row values per array");
    constexpr uint32_t kValues = VLDS ? kWaves * W * DP * sizeof(T) : 0;
    // two buffers of a q tile, a do tile and the row values; the block's value rows
    __shared__ __attribute__((aligned(256))) uint4 smem[(2 * kBuf + kValues) / 16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane / W;
    int64_t t = xcd_linear(blockIdx.x, gridDim.x);
    const int64_t part = t % a.splits;
    t /= a.splits;
    const int64_t tile = t % a.tiles;  // first keys of a causal call first: most rows see them
    const int64_t bk = t / a.tiles, b = bk / a.key_heads, kh = bk % a.key_heads;
    const int64_t len = key_end(a, b), all = a.batch * a.heads * a.n;
    const int rows = (int)a.n;
    const int64_t key0 = tile * (kWaves * W), j = key0 + wave * W + lane % W;
    const bool live = j < len, stored = j < a.m;

    constexpr bool DK = (OUT & 1) != 0, DV = (OUT & 2) != 0, VREG = DK && !VLDS;
    Frag<T> k[QS], v[VREG ? QS : 1];
    {
        const T *kr = live ? reinterpret_cast<const T *>(a.k.p) + b * a.k.b + kh * a.k.h + j * a.k.n : nullptr;
        const T *vr = live ? reinterpret_cast<const T *>(a.v.p) + b * a.v.b + kh * a.v.h + j * a.v.n : nullptr;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            k[s] = load_row8(kr, M::KS * s + 8 * g, (int)a.d);
            if constexpr (VREG) v[s] = load_row8(vr, M::KS * s + 8 * g, (int)a.dv);
            if (a.qsign != 1.0f) {
                float x[8];
                unpack8(k[s], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= a.qsign;
                k[s] = pack8(x, T{});
            }
        }
    }
    // the first row that sees key j; no row sees a key past the length
    int64_t first64 = !live ? 0x7fffffff : a.causal ? j - (len - a.n) : 0;
    const int first = (int)(first64 < 0 ? 0 : first64 > 0x7fffffff ? 0x7fffffff : first64);
    int wfirst = first, wlast = first;
#pragma unroll
    for (int s = 1; s < W; s <<= 1) {
        const int x = __shfl_xor(wfirst, s, 64), y = __shfl_xor(wlast, s, 64);
        wfirst = wfirst < x ? wfirst : x;
        wlast = wlast > y ? wlast : y;
    }
    wfirst = __builtin_amdgcn_readfirstlane(wfirst);
    wlast = __builtin_amdgcn_readfirstlane(wlast);

    Acc dk[DK ? DB : 1], dv[DV ? DB : 1];
#pragma unroll
    for (int i = 0; i < DB; ++i) {
        if constexpr (DK) dk[i] = Acc{};
        if constexpr (DV) dv[i] = Acc{};
    }

    // row tiles of each head from the first that sees a key of this block
    const int nt = (int)cdiv_dev(a.n, BM);
    int64_t skip = key0 >= len ? a.n : a.causal ? key0 - (len - a.n) : 0;
    skip = skip < 0 ? 0 : skip > a.n ? a.n : skip;
    const int tf = skip >= a.n ? nt : (int)(skip / BM), per = nt - tf;
    const int64_t total = a.group * per;
    const int64_t i0 = total * part / a.splits, i1 = total * (part + 1) / a.splits;

    const uint32_t lds = tile::lds_addr(smem);
    Stager<T, DP, BM, kWaves> sq, sg;
    sq.init(a.q.n, (int)a.d, wave, lane);
    sg.init(a.go.n, (int)a.dv, wave, lane);
    int hd = per ? (int)(i0 / per) : 0, rt = per ? tf + (int)(i0 % per) : 0;  // the next tile to fetch
    const auto fetch = [&](int64_t it) {
        const int64_t qh = kh * a.group + hd, r0 = (int64_t)rt * BM;
        const uint32_t buf = lds + (uint32_t)((it - i0) & 1) * kBuf;
        sq.load(reinterpret_cast<const T *>(a.q.p) + b * a.q.b + qh * a.q.h + r0 * a.q.n, a.n - r0, buf);
        sg.load(reinterpret_cast<const T *>(a.go.p) + b * a.go.b + qh * a.go.h + r0 * a.go.n, a.n - r0, buf + kTileBytes);
        if (wave < 3) {  // rows past the end read the last row's values, which are masked below
            int64_t i = r0 + (lane < BM ? lane : BM - 1);
            i = i < a.n ? i : a.n - 1;
            tile::dma4(uniform(a.rows + wave * all + (b * a.heads + qh) * a.n + r0), (uint32_t)((i - r0) * 4),
                       buf + 2 * kTileBytes + (uint32_t)wave * 256);
        }
    };
    const RowReader<T, DP, W> rr(lane);
    const CR cr(lane);
    const uint32_t vt = lds + 2 * kBuf;
    if constexpr (VLDS) {
        Stager<T, DP, kWaves * W, kWaves> sv;
        sv.init(a.v.n, (int)a.dv, wave, lane);
        sv.load(reinterpret_cast<const T *>(a.v.p) + b * a.v.b + kh * a.v.h + key0 * a.v.n, len - key0, vt);
    }
    if (i0 < i1) fetch(i0);
    for (int64_t it = i0; it < i1; ++it) {
        const int64_t qh = kh * a.group + hd;
        const int r0 = rt * BM;
        if (++rt == nt) {
            rt = tf;
            ++hd;
        }
        tile::barrier_all();
        if (it + 1 < i1) fetch(it + 1);
        const uint32_t qt = lds + (uint32_t)((it - i0) & 1) * kBuf, gt = qt + kTileBytes, vals = gt + kTileBytes;
#pragma unroll
        for (int u = 0; u < BM / kUnit; ++u) {
            const int u0 = r0 + u * kUnit;
            if (u0 + kUnit <= wfirst || u0 >= rows) continue;
            // the mask's bits of this key, rows u0 .. u0 + 31
            const uint32_t word = MM == kKeep && live ? a.mask_cols[b * a.cb + qh * a.ch + u0 / 32 * a.cn + j] : 0;
            Acc s[NU], dp[NU];
#pragma unroll
            for (int i = 0; i < NU; ++i) s[i] = dp[i] = Acc{};
            constexpr int F1 = DK ? VLDS ? 3 : 2 : 1, F2 = DK && DV ? 2 : 1;
            stream_steps<QS * NU, F1, Frag<T>>(
                [&](int x, Frag<T>(&f)[F1]) {
                    f[0] = rr.read(qt, u * NU + x % NU, x / NU);
                    if constexpr (DK) f[1] = rr.read(gt, u * NU + x % NU, x / NU);
                    if constexpr (DK && VLDS) f[2] = rr.read(vt, wave, x / NU);
                },
                [&](int x, const Frag<T>(&f)[F1]) {
                    M::mma(s[x % NU], f[0], k[x / NU]);
                    if constexpr (VREG) M::mma(dp[x % NU], f[1], v[x / NU]);
                    if constexpr (DK && VLDS) M::mma(dp[x % NU], f[1], f[2]);
                });
            if constexpr (MM == kKeep) {
                const uint32_t keep = word >> (4 * g);
#pragma unroll
                for (int x = 0; x < 32 / (4 * M::NG); ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!(keep & (1u << (4 * M::NG * x + e)))) {
                            const int at = 4 * M::NG * x;
                            s[at / W][4 * (at % W / (4 * M::NG)) + e] = -INFINITY;
                            dp[at / W][4 * (at % W / (4 * M::NG)) + e] = 0.0f;
                        }
            }
            if constexpr (MM == kBias) {
                const uint8_t *mr = reinterpret_cast<const uint8_t *>(mask_row(a, b, qh, 0));
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = u0 + W * i + 4 * M::NG * w + 4 * g + e;
                            const int64_t at = r * a.mn + j * a.mm;
                            const float add = !(live && r < rows) ? 0.0f
                                              : a.mask_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(mr)[at])
                                                            : reinterpret_cast<const float *>(mr)[at];
                            const bool off = add == -INFINITY;
                            s[i][4 * w + e] = off ? -INFINITY : s[i][4 * w + e] * a.scale + add;
                            if (off) dp[i][4 * w + e] = 0.0f;
                        }
            }
            if (u0 < wlast || u0 + kUnit > rows) {
                asm volatile("");  // a branch: most units skip this
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = u0 + W * i + 4 * M::NG * w + 4 * g + e;
                            if (r < first || r >= rows) {
                                s[i][4 * w + e] = -INFINITY;
                                dp[i][4 * w + e] = 0.0f;
                            }
                        }
            }
            float x[NU * M::Q][4];
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int w = 0; w < M::Q; ++w) {
                    const uint32_t at = vals + (uint32_t)((u * kUnit + W * i + 4 * M::NG * w + 4 * g) * 4);
                    const f32x4 base = __builtin_bit_cast(f32x4, lds_read16(at));
                    const f32x4 inv = __builtin_bit_cast(f32x4, lds_read16(at + 256));
                    const f32x4 delta = __builtin_bit_cast(f32x4, lds_read16(at + 512));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float sv = s[i][4 * w + e];
                        const float p = inv[e] * (MM == kBias ? __builtin_amdgcn_exp2f((sv - base[e]) * kLog2e)
                                                              : __builtin_amdgcn_exp2f(__builtin_fmaf(sv, a.scale, -base[e])));
                        x[i * M::Q + w][e] = p;
                        s[i][4 * w + e] = p * (dp[i][4 * w + e] - delta[e]);
                    }
                }
            Frag<T> p[ST], ds[ST];
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                float y[8], z[8];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[4 * h + e] = x[2 * st + h][e];
                        z[4 * h + e] = s[(2 * st + h) / M::Q][4 * ((2 * st + h) % M::Q) + e];
                    }
                p[st] = pack8(y, T{});
                ds[st] = pack8(z, T{});
            }
            constexpr int kPieces = CR::kPieces;
            stream_steps<ST * kPieces, F2, typename CR::Piece>(
                [&](int x, typename CR::Piece(&f)[F2]) {
                    if constexpr (DV) f[0] = cr.read(gt, u * ST + x / kPieces, x % kPieces);
                    if constexpr (DK) f[F2 - 1] = cr.read(qt, u * ST + x / kPieces, x % kPieces);
                },
                [&](int x, const typename CR::Piece(&f)[F2]) {
                    if constexpr (DV) CR::use(dv, x % kPieces, f[0], p[x / kPieces]);
                    if constexpr (DK) CR::use(dk, x % kPieces, f[F2 - 1], ds[x / kPieces]);
                });
        }
    }
    if (!stored) return;
    const int64_t keys = a.batch * a.key_heads * a.m, row = (b * a.key_heads + kh) * a.m + j;
    const auto store = [&](const Acc *acc, int64_t width, int64_t at, const View &out, float scale) {
        float *part_row = a.part + (part * keys + row) * (quads4(a.d) + quads4(a.dv)) + at;
        T *out_row = reinterpret_cast<T *>(const_cast<void *>(out.p)) + b * out.b + kh * out.h + j * out.n;
        CR::each(acc, lane, [&](int f, f32x4 x) {
            if (a.splits > 1)
                store4(part_row, f, (int)width, 1, x);
            else
                store4(out_row, f, (int)width, a.vec_out, x * scale);
        });
    };
    if constexpr (DK) store(dk, a.d, 0, a.gk, a.gscale);
    if constexpr (DV) store(dv, a.dv, quads4(a.d), a.gv, 1.0f);
}

// Sums the parts of one or two gradients, in their order, one thread per four features: rows of fp32
// quads, the first output's features, then the second's.
struct SumArgs {
    const float *part;
    View out[2];
    int64_t width[2];
    float scale[2];
    int64_t rows, heads, n;
    int splits, vec_out;
};
template <typename T>
__global__ __launch_bounds__(256) void attention_sum_kernel(const SumArgs a) {
    constexpr int U = 8;
    const int64_t q0 = cdiv_dev(a.width[0], 4), quads = q0 + cdiv_dev(a.width[1], 4);
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, row = id / quads;
    if (row >= a.rows) return;
    const int which = id % quads >= q0, f = (int)(id % quads - (which ? q0 : 0)) * 4;
    const int64_t pitch = 4 * quads;
    const float *p = a.part + row * pitch + (which ? 4 * q0 : 0) + f;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < a.splits; s0 += U) {
        f32x4 y[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            y[u] = s0 + u < a.splits ? *reinterpret_cast<const f32x4 *>(p + (s0 + u) * a.rows * pitch)
                                     : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < U; ++u) x += y[u];
    }
    const int64_t i = row % a.n, h = row / a.n % a.heads, b = row / a.n / a.heads;
    const View out = which ? a.out[1] : a.out[0];
    store4(reinterpret_cast<T *>(const_cast<void *>(out.p)) + b * out.b + h * out.h + i * out.n, f,
           (int)(which ? a.width[1] : a.width[0]), a.vec_out,
           x * (which ? a.scale[1] : a.scale[0]));
}

}  // namespace attn
}  // namespace tpw

using namespace tpw;
using namespace tpw::attn;

namespace {

struct BackwardPlan {
    int64_t q_tiles, k_tiles;
    int q_splits, k_splits;
};
template <typename T, int DP>
BackwardPlan backward_plan(const Args &a) {
    BackwardPlan p;
    using L = Tiles<T, DP>;
    const int64_t bk = a.batch * a.key_heads;
    p.q_tiles = cdiv(a.n * a.group, (int64_t)L::kWaves * L::kWidth);
    p.k_tiles = cdiv(a.m, (int64_t)L::kRowWaves * L::kWidth);
    p.q_splits = (int)parts_for(bk * p.q_tiles, cdiv(a.m, L::kKeys), L::kPerCuQ, uneven(a));
    p.k_splits = (int)parts_for(bk * p.k_tiles, a.group * cdiv(a.n, L::kRows), L::kPerCuK, uneven(a));
    return p;
}
size_t backward_workspace(const Args &a, const BackwardPlan &p) {
    const int64_t rows = a.batch * a.heads * a.n;
    const int64_t q = p.q_splits > 1 ? p.q_splits * rows * quads4(a.d) : 0;
    const int64_t k = p.k_splits > 1 ? p.k_splits * a.batch * a.key_heads * a.m * (quads4(a.d) + quads4(a.dv)) : 0;
    return (size_t)(quads4(3 * rows) + (q > k ? q : k)) * 4;
}

template <typename T>
int sum_parts(const SumArgs &a, hipStream_t s) {
    const int64_t threads = a.rows * (cdiv(a.width[0], 4) + cdiv(a.width[1], 4));
    hipLaunchKernelGGL((attention_sum_kernel<T>), dim3((unsigned)cdiv(threads, 256)), dim3(256), 0, s, a);
    return check_launch("attention_sum_kernel");
}

}  // namespace

extern "C" size_t tpw_attention_backward_workspace_size(const tpw_attention_desc *d) {
    Args a = {};
    if (read_args(d, true, a) != TPW_OK) return 0;
    size_t bytes = 0;
    by_type(a, d->dtype, kNoMask, [&](auto t, auto dp, auto) {
        bytes = prepared_bytes(a, d, true) + backward_workspace(a, backward_plan<decltype(t), decltype(dp)::value>(a));
        return TPW_OK;
    });
    return bytes;
}

extern "C" int tpw_attention_backward(const tpw_attention_desc *d, void *workspace, void *stream) {
    Args a = {};
    if (const int rc = read_args(d, true, a)) return rc;
    const int64_t rows = a.batch * a.heads * a.n, keys = a.batch * a.key_heads * a.m;
    if (rows + keys == 0) return TPW_OK;
    TPW_REQUIRE(rows == 0 || (a.q.p && a.o.p && a.go.p && a.gq.p && a.stats), "attention backward: null operand");
    TPW_REQUIRE(keys == 0 || (a.k.p && a.v.p && a.gk.p && a.gv.p), "attention backward: null operand");
    TPW_REQUIRE(d->mask_type == TPW_MASK_NONE || a.mask || a.m == 0, "attention: null mask");
    TPW_REQUIRE(workspace && aligned16(workspace), "attention backward: null or unaligned workspace");
    hipStream_t s = as_stream(stream);
    const size_t prepared = prepared_bytes(a, d, true);
    if (prepared)
        if (const int rc = prepare_operands(a, d, true, workspace, s)) return rc;
    return by_type(a, d->dtype, mask_mode(d), [&](auto t, auto dp, auto mode) {
        using T = decltype(t);
        constexpr int DP = decltype(dp)::value, MM = decltype(mode)::value, W = Tiles<T, DP>::kWidth;
        constexpr int kOcc = sizeof(T) == 2 && DP == 256 ? 1 : 2, kOccKv = DP == 256 ? 1 : 2;
        const BackwardPlan p = backward_plan<T, DP>(a);
        const int64_t bk = a.batch * a.key_heads;
        TPW_REQUIRE(bk * p.q_tiles * p.q_splits < (int64_t(1) << 31) && bk * p.k_tiles * p.k_splits < (int64_t(1) << 31),
                    "attention: too many rows");
        a.rows = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + prepared);
        a.part = a.rows + quads4(3 * rows);
        if (rows) {
            a.tiles = p.q_tiles;
            a.splits = p.q_splits;
            constexpr int kWaves = Tiles<T, DP>::kWaves;
            hipLaunchKernelGGL((attention_dq_kernel<T, W, DP, Tiles<T, DP>::kKeys, MM, kWaves, kOcc>),
                               dim3((unsigned)(bk * a.tiles * a.splits)), dim3(64 * kWaves), 0, s, a);
            if (const int rc = check_launch("attention_dq_kernel")) return rc;
            if (a.splits > 1)
                if (const int rc = sum_parts<T>(
                        {a.part, {a.gq, {}}, {a.d, 0}, {a.gscale, 0.0f}, rows, a.heads, a.n, a.splits, a.vec_out}, s))
                    return rc;
        }
        if (keys) {
            a.tiles = p.k_tiles;
            a.splits = p.k_splits;
            const dim3 grid((unsigned)(bk * a.tiles * a.splits)), block(64 * Tiles<T, DP>::kRowWaves);
            // bf16 at 256 features: dk and dv would take all 256 accumulation registers and leave none for
            // the scores, so each is a launch of its own
            constexpr bool kApart = sizeof(T) == 2 && DP == 256;
            constexpr int kRows = Tiles<T, DP>::kRows, kWaves = Tiles<T, DP>::kRowWaves;
            if constexpr (kApart) {
                hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, kRows, MM, kWaves, 2, false, 2>), grid, block, 0, s, a);
                hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, kRows, MM, kWaves, 1, false, 1>), grid, block, 0, s, a);
            } else {
                hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, kRows, MM, kWaves, kOccKv, DP == 128, 3>), grid, block, 0, s, a);
            }
            if (const int rc = check_launch("attention_dkv_kernel")) return rc;
            if (a.splits > 1)
                return sum_parts<T>({a.part, {a.gk, a.gv}, {a.d, a.dv}, {a.gscale, 1.0f}, keys, a.key_heads, a.m, a.splits,
                                     a.vec_out}, s);
        }
        return TPW_OK;
    });
}
