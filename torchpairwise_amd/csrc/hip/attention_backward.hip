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

constexpr int kUnit = 32;  // rows (keys) of the streamed operand that are worked on at a time

template <typename T, int W, int DP, int BN, int MM, int OCC>
__global__ __launch_bounds__(kThreads, OCC) void attention_dq_kernel(const Args a) {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    constexpr int DB = DP / W, QS = DP / M::KS, NU = kUnit / W, ST = kUnit / M::KS;
    constexpr uint32_t kTileBytes = BN * DP * sizeof(T);
    __shared__ uint4 smem[4 * kTileBytes / 16];
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
            q[s] = load_row8(qr, f, (int)a.d, a.vec);
            go[s] = load_row8(gr, f, (int)a.dv, a.vec);
            float x[8], y[8];
            if (a.qsign != 1.0f) {
                unpack8(q[s], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] *= a.qsign;
                q[s] = pack8(x, T{});
            }
            unpack8(go[s], x);
            unpack8(load_row8(orow, f, (int)a.dv, a.vec), y);
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
    const RowReader<T, DP, W> rr(lane);
    const ColReader<T, DP, W> cr(lane);
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
                const void *mr = mask_row(a, b, qh, qi, a.mask_bf16 ? 2 : 4);
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
                const uint8_t *mr = reinterpret_cast<const uint8_t *>(mask_row(a, b, qh, qi, 1));
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w) {
                        const int j = j0 + W * i + 4 * M::NG * w + 4 * g;
                        uint32_t keep = 0;
                        if (j < lim) keep = mask_keep4(a, mr, j);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!(keep & (0xffu << (8 * e)))) {
                                s[i][4 * w + e] = -INFINITY;
                                dp[i][4 * w + e] = 0.0f;
                            }
                    }
            }
            if (j0 + kUnit > wmin) {
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
                for (int i = 0; i < DB; ++i) M::mma(dq[i], cr.read(kt, u * ST + st, i), ds);
            }
        }
    }
    if (!live) return;
    if (a.splits > 1) {
        float *p = a.part + (part * all + row) * a.d;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int w = 0; w < M::Q; ++w) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = dq[i][4 * w + e];
                store4(p, W * i + 4 * M::NG * w + 4 * g, (int)a.d, a.d % 4 == 0, v);
            }
        return;
    }
    T *p = reinterpret_cast<T *>(const_cast<void *>(a.gq.p)) + b * a.gq.b + qh * a.gq.h + qi * a.gq.n;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int w = 0; w < M::Q; ++w) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = dq[i][4 * w + e] * a.gscale;
            store4(p, W * i + 4 * M::NG * w + 4 * g, (int)a.d, a.vec_out, v);
        }
}

template <typename T, int W, int DP, int BM, int MM, int OCC>
__global__ __launch_bounds__(kThreads, OCC) void attention_dkv_kernel(const Args a) {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    constexpr int DB = DP / W, QS = DP / M::KS, NU = kUnit / W, ST = kUnit / M::KS;
    constexpr uint32_t kTileBytes = BM * DP * sizeof(T), kBuf = 2 * kTileBytes + 3 * 64 * 4;
    static_assert(BM <= 64, "one DMA of row values per array");
    __shared__ uint4 smem[2 * kBuf / 16];  // two buffers of a q tile, a do tile and the row values
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane / W;
    int64_t t = xcd_linear(blockIdx.x, gridDim.x);
    const int64_t part = t % a.splits;
    t /= a.splits;
    const int64_t tile = t % a.tiles;  // first keys of a causal call first: most rows see them
    const int64_t bk = t / a.tiles, b = bk / a.key_heads, kh = bk % a.key_heads;
    const int64_t len = key_end(a, b), all = a.batch * a.heads * a.n;
    const int64_t key0 = tile * (kWaves * W), j = key0 + wave * W + lane % W;
    const bool live = j < len, stored = j < a.m;

    Frag<T> k[QS], v[QS];
    {
        const T *kr = live ? reinterpret_cast<const T *>(a.k.p) + b * a.k.b + kh * a.k.h + j * a.k.n : nullptr;
        const T *vr = live ? reinterpret_cast<const T *>(a.v.p) + b * a.v.b + kh * a.v.h + j * a.v.n : nullptr;
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            k[s] = load_row8(kr, M::KS * s + 8 * g, (int)a.d, a.vec);
            v[s] = load_row8(vr, M::KS * s + 8 * g, (int)a.dv, a.vec);
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

    Acc dk[DB], dv[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) dk[i] = dv[i] = Acc{};

    // row tiles of each head from the first that sees a key of this block
    const int nt = (int)cdiv_dev(a.n, BM);
    int64_t skip = key0 >= len ? a.n : a.causal ? key0 - (len - a.n) : 0;
    skip = skip < 0 ? 0 : skip > a.n ? a.n : skip;
    const int tf = skip >= a.n ? nt : (int)(skip / BM), per = nt - tf;
    const int64_t total = a.group * per;
    const int64_t i0 = total * part / a.splits, i1 = total * (part + 1) / a.splits;

    const uint32_t lds = tile::lds_addr(smem);
    Stager<T, DP, BM, kWaves> sq, sg;
    sq.init(a.q.n, (int)a.d, a.vec, wave, lane);
    sg.init(a.go.n, (int)a.dv, a.vec, wave, lane);
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
    const ColReader<T, DP, W> cr(lane);
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
            if (u0 + kUnit <= wfirst || u0 >= a.n) continue;
            Acc s[NU], dp[NU];
#pragma unroll
            for (int i = 0; i < NU; ++i) s[i] = dp[i] = Acc{};
#pragma unroll
            for (int f = 0; f < QS; ++f)
#pragma unroll
                for (int i = 0; i < NU; ++i) {
                    M::mma(s[i], rr.read(qt, u * NU + i, f), k[f]);
                    M::mma(dp[i], rr.read(gt, u * NU + i, f), v[f]);
                }
            if constexpr (MM != kNoMask) {
                const uint8_t *mr = reinterpret_cast<const uint8_t *>(
                    mask_row(a, b, qh, 0, MM == kKeep ? 1 : a.mask_bf16 ? 2 : 4));
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int64_t r = u0 + W * i + 4 * M::NG * w + 4 * g + e;
                            const bool in = live && r < a.n;
                            const int64_t at = r * a.mn + j * a.mm;
                            float x = s[i][4 * w + e];
                            bool off;
                            if constexpr (MM == kKeep) {
                                off = !in || !mr[at];
                            } else {
                                const float add = !in ? 0.0f
                                                  : a.mask_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(mr)[at])
                                                                : reinterpret_cast<const float *>(mr)[at];
                                off = add == -INFINITY;
                                x = x * a.scale + add;
                            }
                            s[i][4 * w + e] = off ? -INFINITY : x;
                            if (off) dp[i][4 * w + e] = 0.0f;
                        }
            }
            if (u0 < wlast || u0 + kUnit > a.n) {
#pragma unroll
                for (int i = 0; i < NU; ++i)
#pragma unroll
                    for (int w = 0; w < M::Q; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int r = u0 + W * i + 4 * M::NG * w + 4 * g + e;
                            if (r < first || r >= a.n) {
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
                const Frag<T> p = pack8(y, T{}), ds = pack8(z, T{});
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    M::mma(dv[i], cr.read(gt, u * ST + st, i), p);
                    M::mma(dk[i], cr.read(qt, u * ST + st, i), ds);
                }
            }
        }
    }
    if (!stored) return;
    if (a.splits > 1) {
        const int64_t keys = a.batch * a.key_heads * a.m, row = (b * a.key_heads + kh) * a.m + j;
        float *pk = a.part + (part * keys + row) * (a.d + a.dv), *pv = pk + a.d;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int w = 0; w < M::Q; ++w) {
                f32x4 x, y;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = dk[i][4 * w + e];
                    y[e] = dv[i][4 * w + e];
                }
                const int f = W * i + 4 * M::NG * w + 4 * g;
                const int v4 = a.d % 4 == 0 && a.dv % 4 == 0;
                store4(pk, f, (int)a.d, v4, x);
                store4(pv, f, (int)a.dv, v4, y);
            }
        return;
    }
    T *pk = reinterpret_cast<T *>(const_cast<void *>(a.gk.p)) + b * a.gk.b + kh * a.gk.h + j * a.gk.n;
    T *pv = reinterpret_cast<T *>(const_cast<void *>(a.gv.p)) + b * a.gv.b + kh * a.gv.h + j * a.gv.n;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int w = 0; w < M::Q; ++w) {
            f32x4 x, y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = dk[i][4 * w + e] * a.gscale;
                y[e] = dv[i][4 * w + e];
            }
            const int f = W * i + 4 * M::NG * w + 4 * g;
            store4(pk, f, (int)a.d, a.vec_out, x);
            store4(pv, f, (int)a.dv, a.vec_out, y);
        }
}

// Sums the parts of the gradients, in their order, one thread per four features: rows of `width`
// fp32 values of which this output takes `d` from `at`, times `scale`.
template <typename T>
__global__ void attention_sum_kernel(const float *part, int splits, int64_t rows, int64_t width, int64_t at, int64_t d,
                                     float scale, View out, int64_t heads, int64_t n, int vec) {
    const int64_t quads = (d + 3) / 4, id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= rows * quads) return;
    const int64_t row = id / quads;
    const int f = (int)(id % quads) * 4;
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < splits; ++s) {
        const float *p = part + (s * rows + row) * width + at + f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (f + e < d) x[e] += p[e];
    }
    const int64_t i = row % n, h = row / n % heads, b = row / n / heads;
    x *= scale;
    store4(reinterpret_cast<T *>(const_cast<void *>(out.p)) + b * out.b + h * out.h + i * out.n, f, (int)d, vec, x);
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
    const int64_t own = (int64_t)kWaves * Tiles<T, DP>::kWidth, bk = a.batch * a.key_heads;
    p.q_tiles = cdiv(a.n * a.group, own);
    p.k_tiles = cdiv(a.m, own);
    p.q_splits = (int)parts_for(bk * p.q_tiles, cdiv(a.m, Tiles<T, DP>::kKeys));
    p.k_splits = (int)parts_for(bk * p.k_tiles, a.group * cdiv(a.n, Tiles<T, DP>::kRows));
    return p;
}
int64_t round4(int64_t x) { return (x + 3) / 4 * 4; }
size_t backward_workspace(const Args &a, const BackwardPlan &p) {
    const int64_t rows = a.batch * a.heads * a.n;
    const int64_t q = p.q_splits > 1 ? p.q_splits * rows * a.d : 0;
    const int64_t k = p.k_splits > 1 ? p.k_splits * a.batch * a.key_heads * a.m * (a.d + a.dv) : 0;
    return (size_t)(round4(3 * rows) + (q > k ? q : k)) * 4;
}

template <typename T>
int sum_parts(const Args &a, int64_t rows, int64_t width, int64_t at, int64_t d, float scale, const View &out,
              int64_t heads, int64_t n, hipStream_t s) {
    hipLaunchKernelGGL((attention_sum_kernel<T>), dim3((unsigned)cdiv(rows * cdiv(d, 4), 256)), dim3(256), 0, s, a.part,
                       a.splits, rows, width, at, d, scale, out, heads, n, a.vec_out);
    return check_launch("attention_sum_kernel");
}

}  // namespace

extern "C" size_t tpw_attention_backward_workspace_size(const tpw_attention_desc *d) {
    Args a = {};
    if (read_args(d, true, a) != TPW_OK) return 0;
    size_t bytes = 0;
    by_type(a, d->dtype, kNoMask, [&](auto t, auto dp, auto) {
        bytes = backward_workspace(a, backward_plan<decltype(t), decltype(dp)::value>(a));
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
    return by_type(a, d->dtype, mask_mode(d), [&](auto t, auto dp, auto mode) {
        using T = decltype(t);
        constexpr int DP = decltype(dp)::value, MM = decltype(mode)::value, W = Tiles<T, DP>::kWidth;
        constexpr int kOcc = DP == 256 ? 1 : 2;
        const BackwardPlan p = backward_plan<T, DP>(a);
        const int64_t bk = a.batch * a.key_heads;
        TPW_REQUIRE(bk * p.q_tiles * p.q_splits < (int64_t(1) << 31) && bk * p.k_tiles * p.k_splits < (int64_t(1) << 31),
                    "attention: too many rows");
        a.rows = reinterpret_cast<float *>(workspace);
        a.part = a.rows + round4(3 * rows);
        if (rows) {
            a.tiles = p.q_tiles;
            a.splits = p.q_splits;
            hipLaunchKernelGGL((attention_dq_kernel<T, W, DP, Tiles<T, DP>::kKeys, MM, kOcc>),
                               dim3((unsigned)(bk * a.tiles * a.splits)), dim3(attn::kThreads), 0, s, a);
            if (const int rc = check_launch("attention_dq_kernel")) return rc;
            if (a.splits > 1)
                if (const int rc = sum_parts<T>(a, rows, a.d, 0, a.d, a.gscale, a.gq, a.heads, a.n, s)) return rc;
        }
        if (keys) {
            a.tiles = p.k_tiles;
            a.splits = p.k_splits;
            hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, Tiles<T, DP>::kRows, MM, kOcc>),
                               dim3((unsigned)(bk * a.tiles * a.splits)), dim3(attn::kThreads), 0, s, a);
            if (const int rc = check_launch("attention_dkv_kernel")) return rc;
            if (a.splits > 1) {
                if (const int rc = sum_parts<T>(a, keys, a.d + a.dv, 0, a.d, a.gscale, a.gk, a.key_heads, a.m, s)) return rc;
                return sum_parts<T>(a, keys, a.d + a.dv, a.d, a.dv, 1.0f, a.gv, a.key_heads, a.m, s);
            }
        }
        return TPW_OK;
    });
}
