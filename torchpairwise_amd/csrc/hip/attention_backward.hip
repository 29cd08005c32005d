// Attention backward.  The probabilities are formed again from q, k and the saved row maxima and
// sums; no [n, m] matrix is written and nothing is added atomically, so results do not depend on
// the order of blocks:
//   p_ij = exp(s_ij - m_i) / l_i,  dp_ij = do_i . v_j,  delta_i = do_i . o_i,
//   ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = scale sum_j ds_ij k_j                    attention_dq_kernel: a wave owns query rows
//   dk_j = scale sum_i ds_ij q_i, dv_j = sum_i p_ij do_i   attention_dkv_kernel: a wave owns keys
// Seven products where five would do with dq summed in memory: the two scores' products are formed
// in both kernels (eight for bf16 rows of more than 128 features, whose dk and dv are a launch each: the
// scores of q and k once more).  On the fp32 matrix cores two products of wide rows cost more than writing
// and reading ds: there (see keeps_ds) the kernel that owns keys keeps ds in the workspace, for as many
// heads at a time as 1 GiB holds, and dk and dq are one product each (attention_ds_product_kernel), five
// in all.
#include <math.h>

#include "attention.hpp"

namespace tpw {
namespace attn {

// Runs N steps of `use` on fragments that `load` reads from LDS, the next step's reads issued before
// this step's products.  FENCED: the compiler may not move the reads further ahead; left alone it hoists
// them all, which spills the accumulators where registers are scarce.
template <int N, int F, typename Piece, bool FENCED = true, typename Load, typename Use>
__device__ __forceinline__ void stream_steps(Load load, Use use) {
    Piece f[2][F];
    load(0, f[0]);
#pragma unroll
    for (int x = 0; x < N; ++x) {
        if (x + 1 < N) load(x + 1, f[(x + 1) & 1]);
        if constexpr (FENCED) asm volatile("" ::: "memory");
        use(x, f[x & 1]);
    }
}

constexpr int kUnit = 32;  // rows (keys) of the streamed operand that are worked on at a time

// dq: the forward's structure with a second product of scores (v, do) and one of keys.  It also leaves
// base, 1 / sum and delta of every row for the kernel below.  bf16 2 x 16 (4) x 8192^2 x 128: 1.45 to 1.55
// ms (1.06 to 1.14 PFLOP/s over three products); at 256 features one wave per SIMD holds q, do and dq, and
// softmax and products alternate (8 x 8192^2: 0.98 to 1.15 ms, 720 to 840 TFLOP/s); at 192 two waves hold
// them but for 54 to 74 spilled registers (8 x 8192^2: 0.78 ms, 790 TFLOP/s).  fp32 forms it at 8 x 4096^2 x
// 64 in 0.43 ms (120 TFLOP/s).  Added values are loaded behind the scores' products (16 x 4096^2 x 128 bf16
// with values per head: 0.37 ms, 1 GiB of them).
template <typename T, int W, int DP, int BN, int MM, int kWaves, int OCC>
__global__ __launch_bounds__(64 * kWaves, OCC) void attention_dq_kernel(const Args a) {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    using CR = ColReader<T, DP, W>;
    constexpr int DB = DP / W, QS = DP / M::KS, NU = kUnit / W, ST = kUnit / M::KS;
    constexpr bool kFenced = DP == 192 || sizeof(T) == 4;
    constexpr uint32_t kTileBytes = BN * Tile<T, DP>::kRowBytes;
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
        const int64_t oat = b * a.o.b + qh * a.o.h + qi * a.o.n;
        const T *orow = live ? reinterpret_cast<const T *>(a.o.p) + oat : nullptr;
        const T *rest = live && a.rest ? reinterpret_cast<const T *>(a.rest) + oat : nullptr;
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
            if constexpr (sizeof(T) == 2) {
                unpack8(load_row8(rest, f, (int)a.dv), y);
#pragma unroll
                for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(x[e], y[e], delta);
            }
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
            stream_steps<QS, 2 * NU, Frag<T>, kFenced>(
                [&](int x, Frag<T>(&f)[2 * NU]) {
#pragma unroll
                    for (int i = 0; i < NU; ++i) {
                        f[2 * i] = rr.read(kt, u * NU + i, x);
                        f[2 * i + 1] = rr.read(vt, u * NU + i, x);
                    }
                },
                [&](int x, const Frag<T>(&f)[2 * NU]) {
                    if constexpr (sizeof(T) == 4) {  // independent products side by side
#pragma unroll
                        for (int e = 0; e < 8; ++e)
#pragma unroll
                            for (int i = 0; i < NU; ++i) {
                                M::mma1(s[i], f[2 * i], q[x], e);
                                M::mma1(dp[i], f[2 * i + 1], go[x], e);
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < NU; ++i) {
                            M::mma(s[i], f[2 * i], q[x]);
                            M::mma(dp[i], f[2 * i + 1], go[x]);
                        }
                    }
                });
            if constexpr (MM == kBias) {
                constexpr int N = NU * M::Q;
                f32x4 add[N];
                mask_bias<N, 4 * M::NG>(a, mask_row(a, b, qh, qi < 0 ? 0 : qi), j0, 4 * g, kUnit, add);
#pragma unroll
                for (int x = 0; x < N; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool off = add[x][e] == -INFINITY;
                        const float y = s[x / M::Q][4 * (x % M::Q) + e] * a.scale + add[x][e];
                        s[x / M::Q][4 * (x % M::Q) + e] = off ? -INFINITY : y;
                        if (off) dp[x / M::Q][4 * (x % M::Q) + e] = 0.0f;
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
            Frag<T> ds[ST];
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                float x[8];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[4 * v + e] = s[(2 * st + v) / M::Q][4 * ((2 * st + v) % M::Q) + e];
                ds[st] = pack8(x, T{});
            }
            stream_steps<ST * CR::kPieces, 1, typename CR::Piece, kFenced>(
                [&](int x, typename CR::Piece(&f)[1]) { f[0] = cr.read(kt, u * ST + x / CR::kPieces, x % CR::kPieces); },
                [&](int x, const typename CR::Piece(&f)[1]) { CR::use(dq, x % CR::kPieces, f[0], ds[x / CR::kPieces]); });
        }
    }
    if (!live) return;
    if (a.splits > 1) {
        const int width = (int)quads4(a.d);
        float *p = a.part + (part * all + row) * width;
        CR::each(dq, lane, [&](int at, f32x4 v) { store4(p, at, width, v); });
        return;
    }
    T *p = reinterpret_cast<T *>(const_cast<void *>(a.gq.p)) + b * a.gq.b + qh * a.gq.h + qi * a.gq.n;
    CR::each(dq, lane, [&](int at, f32x4 v) { store4(p, at, (int)a.d, v * a.gscale); });
}

// dk, dv (or one of them, or dv with ds kept): a wave owns 32 keys (fp32: 16), streams q and do, and needs
// 2 DP accumulators a lane beside its keys and values.  To stay at two waves per SIMD, bf16 at 65 to 128
// features reads the block's values from LDS (VLDS: 2.0 ms where spilled registers took 2.9), and at more
// takes dk and dv in a launch each; dk at 192 spills 38 to 59 registers all the same, and with added values
// 128 features spill 14 and dv at 256 24.  fp32 at 96 and 128 reads its values from LDS too, at one wave per
// SIMD.  bf16 2 x 16 (4) x 8192^2 x 128: 2.04 to 2.3 ms (0.95 to 1.08 PFLOP/s over four products); 8 x 8192^2
// x 192: dv 0.46, dk 0.88; x 256: dv 0.53, dk 1.36 to 1.5 (one wave per SIMD).  fp32 8 x 4096^2 x 64: 0.59 ms
// (117 TFLOP/s over four), 2 x 4096^2 x 128 0.34 (102).  Added values come one by one behind the scores'
// products: 16 x 4096^2 x 128 bf16 with values per head 0.64 ms.
template <typename T, int W, int DP, int BM, int MM, int kWaves, int OCC, bool VLDS, int OUT>
__global__ __launch_bounds__(64 * kWaves, OCC) void attention_dkv_kernel(const Args a) {
    using M = Mma<T, W>;
    using Acc = typename M::Acc;
    using CR = ColReader<T, DP, W>;
    constexpr int DB = DP / W, QS = DP / M::KS, NU = kUnit / W, ST = kUnit / M::KS;
    constexpr uint32_t kTileBytes = BM * Tile<T, DP>::kRowBytes, kBuf = 2 * kTileBytes + 3 * 64 * 4;
    static_assert(BM <= 64, "one DMA of row values per array");
    constexpr uint32_t kValues = VLDS ? kWaves * W * Tile<T, DP>::kRowBytes : 0;
    // two buffers of a q tile, a do tile and the row values; the block's value rows
    __shared__ __attribute__((aligned(256))) uint4 smem[(2 * kBuf + kValues) / 16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane / W;
    int64_t t = xcd_linear(blockIdx.x, gridDim.x);
    const int64_t part = t % a.splits;
    t /= a.splits;
    const int64_t tile = t % a.tiles;  // first keys of a causal call first: most rows see them
    const int64_t bk = a.first_bk + t / a.tiles, b = bk / a.key_heads, kh = bk % a.key_heads;
    const int64_t len = key_end(a, b), all = a.batch * a.heads * a.n;
    const int rows = (int)a.n;
    const int64_t key0 = tile * (kWaves * W), j = key0 + wave * W + lane % W;
    const bool live = j < len, stored = j < a.m;

    // OUT: 1 dk, 2 dv, 4 ds kept in a.ds
    constexpr bool DK = (OUT & 1) != 0, DV = (OUT & 2) != 0, DS = (OUT & 5) != 0, VREG = DS && !VLDS;
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
            constexpr int R = DS ? 2 : 1, F1 = R * NU + (DS && VLDS), F2 = DK && DV ? 2 : 1;
            stream_steps<QS, F1, Frag<T>>(
                [&](int x, Frag<T>(&f)[F1]) {
#pragma unroll
                    for (int i = 0; i < NU; ++i) {
                        f[R * i] = rr.read(qt, u * NU + i, x);
                        if constexpr (DS) f[R * i + 1] = rr.read(gt, u * NU + i, x);
                    }
                    if constexpr (DS && VLDS) f[F1 - 1] = rr.read(vt, wave, x);
                },
                [&](int x, const Frag<T>(&f)[F1]) {
                    const Frag<T> &vv = VLDS ? f[F1 - 1] : v[VREG ? x : 0];
                    if constexpr (sizeof(T) == 4) {  // independent products side by side
#pragma unroll
                        for (int e = 0; e < 8; ++e)
#pragma unroll
                            for (int i = 0; i < NU; ++i) {
                                M::mma1(s[i], f[R * i], k[x], e);
                                if constexpr (DS) M::mma1(dp[i], f[R * i + R - 1], vv, e);
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < NU; ++i) {
                            M::mma(s[i], f[R * i], k[x]);
                            if constexpr (DS) M::mma(dp[i], f[R * i + R - 1], vv);
                        }
                    }
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
                // rows and keys past the end read the last ones, and are masked below
                const void *mr = mask_row(a, b, qh, 0);
                const int64_t at = (j < a.m ? j : a.m - 1) * a.mm;
#pragma unroll
                for (int x = 0; x < NU * M::Q; ++x) {
                    float add[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = u0 + 4 * M::NG * x + 4 * g + e;
                        add[e] = mask_value(a, mr, (r < rows ? r : rows - 1) * a.mn + at);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool off = add[e] == -INFINITY;
                        const float y = s[x / M::Q][4 * (x % M::Q) + e] * a.scale + add[e];
                        s[x / M::Q][4 * (x % M::Q) + e] = off ? -INFINITY : y;
                        if (off) dp[x / M::Q][4 * (x % M::Q) + e] = 0.0f;
                    }
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
                        const float p = inv[e] * __builtin_amdgcn_exp2f(MM == kBias ? (sv - base[e]) * kLog2e
                                                                                    : __builtin_fmaf(sv, a.scale, -base[e]));
                        x[i * M::Q + w][e] = p;
                        s[i][4 * w + e] = p * (dp[i][4 * w + e] - delta[e]);
                    }
                }
            if constexpr ((OUT & 4) != 0) {
                if (live) {
                    const int64_t head = (bk - a.first_bk) * a.group + qh - kh * a.group;
                    float *kept = a.ds + (head * a.m + j) * a.ds_pitch + u0 + 4 * g;
#pragma unroll
                    for (int i = 0; i < NU; ++i)
#pragma unroll
                        for (int w = 0; w < M::Q; ++w) {
                            f32x4 y;
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[e] = s[i][4 * w + e];
                            *reinterpret_cast<f32x4 *>(kept + W * i + 4 * M::NG * w) = y;
                        }
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
                store4(part_row, f, (int)quads4(width), x);
            else
                store4(out_row, f, (int)width, x * scale);
        });
    };
    if constexpr (DK) store(dk, a.d, 0, a.gk, a.gscale);
    if constexpr (DV) store(dv, a.dv, quads4(a.d), a.gv, 1.0f);
}

// base, 1 / sum and delta of every row, one wave per row (the dq kernel forms them where it runs).
// Bound by memory: 8 x 8192 rows of 256 in 34 us (4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void attention_rows_kernel(const Args a) {
    const int64_t all = a.batch * a.heads * a.n, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= all) return;
    const int lane = threadIdx.x & 63;
    const int64_t i = row % a.n, h = row / a.n % a.heads, b = row / a.n / a.heads;
    const T *o = reinterpret_cast<const T *>(a.o.p) + b * a.o.b + h * a.o.h + i * a.o.n;
    const T *g = reinterpret_cast<const T *>(a.go.p) + b * a.go.b + h * a.go.h + i * a.go.n;
    float delta = 0.0f;
    for (int f = lane; f < a.dv; f += 64) delta = __builtin_fmaf(to_f32(o[f]), to_f32(g[f]), delta);
    delta = over_groups_sum<1>(delta);
    if (lane) return;
    const float top = a.stats[row], sum = a.stats[all + row];
    a.rows[row] = top == -INFINITY ? 0.0f : top;
    a.rows[all + row] = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    a.rows[2 * all + row] = delta;
}

// dk (KEYS) or dq from the kept ds: a wave owns 16 keys (query rows) and streams q (k) through LDS.
// Only units that the kernel above wrote are read; what no row sees counts as zero.  fp32 4 x 8192^2 x
// 256: 1.19 and 1.24 ms (115 and 111 TFLOP/s beside reading 1 GiB).
template <int DP, bool KEYS>
__global__ __launch_bounds__(512, 2) void attention_ds_product_kernel(const Args a) {
    constexpr int W = 16, kWaves = 8;
    using M = Mma<float, W>;
    using CR = ColReader<float, DP, W>;
    constexpr uint32_t kTileBytes = kUnit * Tile<float, DP>::kRowBytes;
    __shared__ __attribute__((aligned(256))) uint4 smem[2 * kTileBytes / 16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane / W;
    const int64_t t = xcd_linear(blockIdx.x, gridDim.x), own_tiles = cdiv_dev(KEYS ? a.m : a.n, kWaves * W);
    // longest first: a causal call's first keys and last rows
    const int64_t tile = KEYS ? t % own_tiles : own_tiles - 1 - t % own_tiles;
    const int64_t head = KEYS ? 0 : t / own_tiles % a.group, local = KEYS ? t / own_tiles : t / own_tiles / a.group;
    const int64_t bk = a.first_bk + local, b = bk / a.key_heads, kh = bk % a.key_heads;
    const int64_t len = key_end(a, b), own0 = tile * (kWaves * W), o = own0 + wave * W + lane % W;

    // KEYS: the first row that sees the key; else the keys that the row sees
    int bound;
    if (KEYS) {
        const int64_t first = o >= len ? 0x7fffffff : a.causal ? o - (len - a.n) : 0;
        bound = (int)(first < 0 ? 0 : first);
    } else {
        bound = o < a.n ? (int)row_limit(a, len, o) : 0;
    }
    int far = bound;  // over the wave: KEYS the least, else the greatest
#pragma unroll
    for (int s = 1; s < W; s <<= 1) {
        const int x = __shfl_xor(far, s, 64);
        far = (KEYS ? x < far : x > far) ? x : far;
    }
    far = __builtin_amdgcn_readfirstlane(far);

    // units of the streamed rows: KEYS of every head of the group, from the first that sees a key
    int64_t skip = own0 >= len ? a.n : a.causal ? own0 - (len - a.n) : 0;
    skip = skip < 0 ? 0 : skip > a.n ? a.n : skip;
    const int64_t last = own0 + kWaves * W < a.n ? own0 + kWaves * W - 1 : a.n - 1;
    const int nt = (int)cdiv_dev(KEYS ? a.n : row_limit(a, len, last), kUnit);
    const int tf = !KEYS ? 0 : skip >= a.n ? nt : (int)(skip / kUnit), per = nt - tf;
    const int total = KEYS ? (int)a.group * per : per;

    const uint32_t lds = tile::lds_addr(smem);
    Stager<float, DP, kUnit, kWaves> st;
    const View &x = KEYS ? a.q : a.k;
    st.init(x.n, (int)a.d, wave, lane);
    const float *xb = reinterpret_cast<const float *>(x.p) + b * x.b + kh * (KEYS ? a.group : 1) * x.h;
    const float *db = a.ds + (local * a.group + head) * a.m * a.ds_pitch;
    int fh = 0, ft = tf;  // head and unit to fetch next
    Frag<float> next = {}, now = {};
    const auto fetch = [&](int i) {
        const int64_t r0 = (int64_t)ft * kUnit;
        st.load(xb + fh * x.h + r0 * x.n, (KEYS ? a.n : len) - r0, lds + (uint32_t)(i & 1) * kTileBytes);
        next = Frag<float>{};
        if (KEYS) {
            if (o < len && r0 + kUnit > far) {
                const float *p = db + (fh * a.m + o) * a.ds_pitch + r0 + 4 * g;
                next.v[0] = *reinterpret_cast<const f32x4 *>(p);
                next.v[1] = *reinterpret_cast<const f32x4 *>(p + 16);
            }
        } else if (r0 < far) {
            const float *p = db + (o < a.n ? o : 0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t key = r0 + 16 * (e >> 2) + 4 * g + (e & 3);
                const float y = p[(key < bound ? key : 0) * a.ds_pitch];
                next.v[e >> 2][e & 3] = key < bound ? y : 0.0f;
            }
        }
        if (++ft == nt) {
            ft = tf;
            ++fh;
        }
    };
    M::Acc acc[CR::kBlocks];
#pragma unroll
    for (int i = 0; i < CR::kBlocks; ++i) acc[i] = M::Acc{};
    const CR cr(lane);
    if (total > 0) fetch(0);
    int ct = tf;
    for (int i = 0; i < total; ++i) {
        tile::barrier_all();
        now = next;
        const int r0 = ct * kUnit;
        if (++ct == nt) ct = tf;
        if (i + 1 < total) fetch(i + 1);
        if (KEYS ? r0 + kUnit <= far : r0 >= far) continue;
        const uint32_t at = lds + (uint32_t)(i & 1) * kTileBytes;
#pragma unroll
        for (int c = 0; c < CR::kPieces; ++c) CR::use(acc, c, cr.read(at, 0, c), now);
    }
    if (o >= (KEYS ? a.m : a.n)) return;
    const View &out = KEYS ? a.gk : a.gq;
    float *row = reinterpret_cast<float *>(const_cast<void *>(out.p)) + b * out.b +
                 (KEYS ? kh : kh * a.group + head) * out.h + o * out.n;
    CR::each(acc, lane, [&](int f, f32x4 v) { store4(row, f, (int)a.d, v * a.gscale); });
}

// Sums the parts of one or two gradients, in their order, one thread per four features: rows of fp32
// quads, the first output's features, then the second's.
struct SumArgs {
    const float *part;
    View out[2];
    int64_t width[2];
    float scale[2];
    int64_t rows, heads, n;
    int splits;
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
           (int)(which ? a.width[1] : a.width[0]),
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
    int64_t kept;  // (batch, key head)s whose ds is kept at a time; 0: formed again
};
// fp32 rows of more than 64 features keep ds where a 1 GiB workspace holds enough heads for a block on
// most CUs (8 x 8192^2 x 256: 11.3 ms where forming them again takes 15.5; 8 x 4096^2 x 128: 1.56, 2.07)
constexpr int64_t kKeptBytes = int64_t(1) << 30, kKeptKeys = 128;
int64_t ds_bytes(const Args &a) { return a.group * a.m * (cdiv(a.n, kUnit) * kUnit) * 4; }  // of one key head
template <typename T, int DP>
int64_t keeps_ds(const Args &a) {
    const int64_t bk = a.batch * a.key_heads;
    // nothing to keep of empty calls; the bytes of a key head are compared without their product
    if (sizeof(T) != 4 || DP == 64 || bk * a.group == 0 || a.n == 0 || a.m == 0 ||
        a.group > kKeptBytes / 4 / (cdiv(a.n, kUnit) * kUnit) / a.m)
        return 0;
    const int64_t most = kKeptBytes / ds_bytes(a), kept = cdiv(bk, cdiv(bk, most));
    return kept * cdiv(a.m, kKeptKeys) >= 192 && kept * a.group * cdiv(a.n, kKeptKeys) >= 192 ? kept : 0;
}
template <typename T, int DP>
BackwardPlan backward_plan(const Args &a) {
    BackwardPlan p;
    using L = Tiles<T, DP>;
    const int64_t bk = a.batch * a.key_heads;
    p.q_tiles = cdiv(a.n * a.group, (int64_t)L::kWaves * L::kWidth);
    p.k_tiles = cdiv(a.m, (int64_t)L::kRowWaves * L::kWidth);
    p.q_splits = (int)parts_for(bk * p.q_tiles, cdiv(a.m, L::kKeys), L::kPerCuQ, uneven(a),
                                step_us<T, DP>((int64_t)L::kWaves * L::kWidth, L::kKeys, 3, L::kPerCuQ),
                                part_us(a.batch * a.heads * a.n, quads4(a.d)));
    // four products: what one launch for dk and dv has.  Of a launch each (wide bf16 rows) dk has three and
    // dv two; the parts were not measured with those.
    p.k_splits = (int)parts_for(bk * p.k_tiles, a.group * cdiv(a.n, L::kRows), L::kPerCuK, uneven(a),
                                step_us<T, DP>((int64_t)L::kRowWaves * L::kWidth, L::kRows, 4, L::kPerCuK),
                                part_us(bk * a.m, quads4(a.d) + quads4(a.dv)));
    p.kept = keeps_ds<T, DP>(a);
    return p;
}
size_t backward_workspace(const Args &a, const BackwardPlan &p) {
    const int64_t rows = a.batch * a.heads * a.n;
    if (p.kept) return (size_t)(quads4(3 * rows) * 4 + p.kept * ds_bytes(a));
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

template <int DP, int MM>
int backward_kept(Args &a, int64_t kept, int64_t rows, hipStream_t s) {
    const int64_t bk = a.batch * a.key_heads, k_tiles = cdiv(a.m, kKeptKeys), q_tiles = cdiv(a.n, kKeptKeys);
    hipLaunchKernelGGL((attention_rows_kernel<float>), dim3((unsigned)cdiv(rows, 4)), dim3(256), 0, s, a);
    if (const int rc = check_launch("attention_rows_kernel")) return rc;
    a.ds = a.part;
    a.ds_pitch = cdiv(a.n, kUnit) * kUnit;
    a.tiles = k_tiles;
    a.splits = 1;
    for (a.first_bk = 0; a.first_bk < bk; a.first_bk += kept) {
        const int64_t now = bk - a.first_bk < kept ? bk - a.first_bk : kept;
        const dim3 keys((unsigned)(now * k_tiles)), queries((unsigned)(now * a.group * q_tiles));
        hipLaunchKernelGGL((attention_dkv_kernel<float, 16, DP, 32, MM, 8, 2, false, 6>), keys, dim3(512), 0, s, a);
        hipLaunchKernelGGL((attention_ds_product_kernel<DP, true>), keys, dim3(512), 0, s, a);
        hipLaunchKernelGGL((attention_ds_product_kernel<DP, false>), queries, dim3(512), 0, s, a);
        if (const int rc = check_launch("attention_ds_product_kernel")) return rc;
    }
    return TPW_OK;
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
    TPW_REQUIRE(mask_mode(d) == kNoMask || a.mask, "attention: null mask");
    TPW_REQUIRE(workspace && aligned16(workspace), "attention backward: null or unaligned workspace");
    hipStream_t s = as_stream(stream);
    const size_t prepared = prepared_bytes(a, d, true);
    if (prepared)
        if (const int rc = prepare_operands(a, d, true, workspace, s)) return rc;
    return by_type(a, d->dtype, mask_mode(d), [&](auto t, auto dp, auto mode) {
        using T = decltype(t);
        constexpr int DP = decltype(dp)::value, MM = decltype(mode)::value, W = Tiles<T, DP>::kWidth;
        constexpr int kOcc = sizeof(T) == 2 && DP == 256 ? 1 : 2, kOccKv = Tile<T, DP>::P == 256 ? 1 : 2;
        constexpr bool kValuesInLds = Tile<T, DP>::P == 128;
        const BackwardPlan p = backward_plan<T, DP>(a);
        const int64_t bk = a.batch * a.key_heads;
        TPW_REQUIRE(bk * p.q_tiles * p.q_splits < (int64_t(1) << 31) && bk * p.k_tiles * p.k_splits < (int64_t(1) << 31),
                    "attention: too many rows");
        a.rows = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + prepared);
        a.part = a.rows + quads4(3 * rows);
        if constexpr (sizeof(T) == 4 && DP > 64) {
            if (p.kept) return backward_kept<DP, MM>(a, p.kept, rows, s);
        }
        if (rows) {
            a.tiles = p.q_tiles;
            a.splits = p.q_splits;
            constexpr int kWaves = Tiles<T, DP>::kWaves;
            hipLaunchKernelGGL((attention_dq_kernel<T, W, DP, Tiles<T, DP>::kKeys, MM, kWaves, kOcc>),
                               dim3((unsigned)(bk * a.tiles * a.splits)), dim3(64 * kWaves), 0, s, a);
            if (const int rc = check_launch("attention_dq_kernel")) return rc;
            if (a.splits > 1)
                if (const int rc = sum_parts<T>(
                        {a.part, {a.gq, {}}, {a.d, 0}, {a.gscale, 0.0f}, rows, a.heads, a.n, a.splits}, s))
                    return rc;
        }
        if (keys) {
            a.tiles = p.k_tiles;
            a.splits = p.k_splits;
            const dim3 grid((unsigned)(bk * a.tiles * a.splits)), block(64 * Tiles<T, DP>::kRowWaves);
            // bf16 at more than 128 features: dk and dv together would take 192 or all 256 accumulation
            // registers and leave too few for the scores, so each is a launch of its own
            constexpr bool kApart = sizeof(T) == 2 && DP > 128;
            constexpr int kRows = Tiles<T, DP>::kRows, kWaves = Tiles<T, DP>::kRowWaves;
            if constexpr (kApart) {
                constexpr int kOccK = DP == 256 ? 1 : 2;
                hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, kRows, MM, kWaves, 2, false, 2>), grid, block, 0, s,
                                   a);
                hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, kRows, MM, kWaves, kOccK, false, 1>), grid, block, 0,
                                   s, a);
            } else {
                hipLaunchKernelGGL((attention_dkv_kernel<T, W, DP, kRows, MM, kWaves, kOccKv, kValuesInLds, 3>), grid,
                                   block, 0, s, a);
            }
            if (const int rc = check_launch("attention_dkv_kernel")) return rc;
            if (a.splits > 1)
                return sum_parts<T>(
                    {a.part, {a.gk, a.gv}, {a.d, a.dv}, {a.gscale, 1.0f}, keys, a.key_heads, a.m, a.splits}, s);
        }
        return TPW_OK;
    });
}
