// Shared pieces of the attention kernels (attention.hip, attention_backward.hip).
//
//   s_ij = scale q_i . k_j (+ mask_ij),  p_ij = exp(s_ij - m_i) / l_i,  o_i = sum_j p_ij v_j
//
// with the row maximum m_i and sum l_i over the keys that the mask, the causal limit and the
// lengths leave; a row that none is left to gives zeros.  No [n, m] matrix is written (but for the score
// gradients of wide fp32 rows, a bounded number of heads at a time).
//
// Products run on the matrix cores, transposed so that a lane owns one row: a block of W x W
// scores is K (first operand, from LDS) times Q (second operand, in registers), and its
// accumulator holds row c = lane % W, keys 4 NG a + 4 g + e in register 4 a + e, g = lane / W,
// NG = 64 / W.  Each row's softmax is then a loop over the lane's own registers and one exchange
// between its NG lanes.  The probabilities are the second operand of the next product as they
// lie: in a step of KS = 8 NG keys a lane holds quads 2 t and 2 t + 1, and the order of keys
// within a step is free as long as both operands agree, so V is read in that order (rows
// 4 NG (2 t + u) + 4 g .. + 3: transposing LDS reads for bf16, plain ones for fp32).
//
//   bf16: v_mfma_f32_32x32x16_bf16, W = 32;  fp32: 8 x v_mfma_f32_16x16x4_f32 per step, W = 16.
#pragma once

#include "tile_mfma.hpp"

namespace tpw {
namespace attn {

constexpr float kLog2e = 1.44269504088896340736f;

enum MaskMode { kNoMask = 0, kKeep = 1, kBias = 2 };

// One operand: element strides of [batch, heads, rows, features] (features dense).  The kernels read
// rows as 16-byte pieces at 16-byte aligned addresses, a last partial piece filled up with zeros.
// Operands that do not lie so are copied first (pad_kernel), or read by dwords (Args::dwords).
struct View {
    const void *p;
    int64_t b, h, n;
};

struct Args {
    View q, k, v;
    View o, go;          // output; upstream gradient (backward)
    View gq, gk, gv;     // gradients (backward)
    float *stats;        // [2, b, h, n]: row maxima, row sums
    void *rest;          // bf16: what the outputs' rounding left, strides of o; or null
    float *rows;         // [3, b, h, n] (backward): base and 1 / sum of the softmax, delta
    const void *mask;    // kKeep: words of 32 keys' bits (pack_mask_kernel); kBias: fp32 or bf16 values
    int64_t mb, mh, mn, mm;  // its strides, in words or values (0: broadcast; words: mm is 0)
    int mask_bf16;
    const uint32_t *mask_cols;  // kKeep, backward: bits by column, word (row / 32, key)
    int64_t cb, ch, cn;         // its strides over batch, heads and row / 32
    const int64_t *lengths;  // [b] or null
    int64_t batch, heads, key_heads, group, n, m, d, dv;
    float scale;   // |scale| * log2(e) (kBias: |scale|), 1 where scale is 0
    float qsign;   // -1, 0 or 1: the sign of scale, folded into q as it is loaded
    float gscale;  // scale (backward)
    int causal;
    int cached;     // keys and values lie in a cache in 4 or 8 bits: k and v are no operands
    int whole_q;    // (few rows over a cache) queries are whole pieces of 8 features
    int whole_rows; // (few rows over a cache) not in parts, by more waves
    int dwords;     // (forward) operands of whole dwords that are not whole pieces, read as they lie
    int64_t tiles;  // row tiles (dk / dv: key tiles) per (batch, key head)
    int splits;     // parts of the summed axis
    float *ds;      // kept score gradients (backward of wide fp32 rows): [key heads' heads, m, ds_pitch]
    int64_t ds_pitch, first_bk;  // rows rounded up to whole units; first (batch, key head) of this launch
    float *part;    // [splits, rows, features] partial results where splits > 1, rows of whole quads
    float *part_stats;  // [splits, 2, rows]
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T, int W>
struct Mma;

// Eight consecutive elements of a lane, as the matrix instructions take them.
template <typename T>
struct Frag;
template <>
struct Frag<uint16_t> {
    uint4 v;
};
template <>
struct Frag<float> {
    f32x4 v[2];
};

template <int W_>
struct Shape {
    static constexpr int W = W_, NG = 64 / W_, KS = 8 * NG, Q = W_ / (4 * NG);  // quads per block
};

template <>
struct Mma<uint16_t, 32> : Shape<32> {
    typedef floatx16 Acc;
    static __device__ __forceinline__ void mma(Acc &acc, const Frag<uint16_t> &a, const Frag<uint16_t> &b) {
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v),
                                                      acc, 0, 0, 0);
    }
};
template <>
struct Mma<float, 16> : Shape<16> {
    typedef f32x4 Acc;
    // element e of every lane makes one instruction: its four k are elements e of the four groups
    static __device__ __forceinline__ void mma1(Acc &acc, const Frag<float> &a, const Frag<float> &b, int e) {
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e >> 2][e & 3], b.v[e >> 2][e & 3], acc, 0, 0, 0);
    }
    static __device__ __forceinline__ void mma(Acc &acc, const Frag<float> &a, const Frag<float> &b) {
#pragma unroll
        for (int e = 0; e < 8; ++e) mma1(acc, a, b, e);
    }
};

__device__ __forceinline__ Frag<uint16_t> pack8(const float (&x)[8], uint16_t) {
    return {make_uint4(f32x2_to_bf16x2_rne(x[0], x[1]), f32x2_to_bf16x2_rne(x[2], x[3]),
                       f32x2_to_bf16x2_rne(x[4], x[5]), f32x2_to_bf16x2_rne(x[6], x[7]))};
}
__device__ __forceinline__ Frag<float> pack8(const float (&x)[8], float) {
    return {{{x[0], x[1], x[2], x[3]}, {x[4], x[5], x[6], x[7]}}};
}
__device__ __forceinline__ void unpack8(const Frag<uint16_t> &f, float (&x)[8]) {
    const uint32_t w[4] = {f.v.x, f.v.y, f.v.z, f.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack8(const Frag<float> &f, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f.v[i >> 2][i & 3];
}

// The upper halves of two words.
__device__ __forceinline__ uint32_t high2(uint32_t lo, uint32_t hi) {
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}
// fp32 values as three bf16 summands that hold all 24 bits, each what is left cut off to 8 (products with values that
// are exact in bf16 then run at its rate).
__device__ __forceinline__ void split3(float (&x)[8], Frag<uint16_t> (&f)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e] = __float_as_uint(x[e]);
            x[e] -= __uint_as_float(w[e] & 0xffff0000u);
        }
        f[p].v = make_uint4(high2(w[0], w[1]), high2(w[2], w[3]), high2(w[4], w[5]), high2(w[6], w[7]));
    }
}
// As two: rounded, and what that left, rounded.
__device__ __forceinline__ void split2(float (&x)[8], Frag<uint16_t> (&f)[2]) {
    f[0] = pack8(x, uint16_t{});
    float y[8];
    unpack8(f[0], y);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= y[e];
    f[1] = pack8(x, uint16_t{});
}
// As three, where an infinity may be among them: its first summand alone.
__device__ __forceinline__ void split3_any(float (&x)[8], Frag<uint16_t> (&f)[3]) {
    uint32_t inf[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool is = __builtin_fabsf(x[e]) == INFINITY;
        inf[e] = is ? __float_as_uint(x[e]) : 0u;
        x[e] = is ? 0.0f : x[e];
    }
    split3(x, f);
    f[0].v.x |= high2(inf[0], inf[1]);
    f[0].v.y |= high2(inf[2], inf[3]);
    f[0].v.z |= high2(inf[4], inf[5]);
    f[0].v.w |= high2(inf[6], inf[7]);
}

// ---- LDS tiles -----------------------------------------------------------------------------
// A tile of ROWS rows of DP features, with room for a power of two of them, lies as 16-byte pieces,
// piece c of row r at position c ^ swz(r).  Every 16 consecutive rows put one piece into the 16
// different 16-byte slots of the 64 banks (row fragments), and four consecutive rows put a run of four
// pieces into four different quarters of them (transposing reads), so that either read moves 256 bytes a
// cycle (with eight slots in use, conflicts took 22 to 27 % of the bf16 kernels' cycles; now none).
template <typename T, int DP>
struct Tile {
    static constexpr int P = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;  // features a row has room for
    static constexpr int E = 16 / (int)sizeof(T);                    // elements per piece
    static constexpr int C = P / E;                                  // pieces per row
    static constexpr int kRowBytes = P * (int)sizeof(T);
    static constexpr int kMask = C >= 16 ? 15 : 7;  // bits of a piece's index that swz reaches
    static_assert(C >= 8, "rows of 128 bytes at least");
    // rows of 128 bytes: two rows share the banks, so the pairs of rows take turns
    static __host__ __device__ constexpr int swz(int r) {
        return C >= 16 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    }
    // Address of piece c ^ (what `base` holds): base is 256-byte aligned but for a lane's own bits of
    // the piece, which differ from c's.
    static __device__ __forceinline__ uint32_t piece(uint32_t base, int c, int far) {
        return (base ^ (uint32_t)((c & kMask) * 16)) + (uint32_t)((c & ~kMask) * 16 + far);
    }
};

constexpr uint32_t kRange = 0x7ffffff0u;  // bytes a tile's buffer resource spans at most
constexpr uint32_t kBeyond = 0xfffffff0u;  // an offset that no range holds: the load gives zeros

// 16 bytes per lane from the resource into LDS at lds_base + 16 * lane, zeros where the offset is
// past the range.  Inline asm for the reason given at tile::dma16.
__device__ __forceinline__ void dma16(tpw_u32x4 rsrc, uint32_t voff, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds_base)
                 : "memory", "m0");
}
__device__ __forceinline__ void dma4(tpw_u32x4 rsrc, uint32_t voff, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(lds_base)
                 : "memory", "m0");
}
__device__ __forceinline__ tpw_u32x4 resource(const void *base, int64_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)base;
    const uint32_t num = bytes <= 0 ? 0u : bytes > (int64_t)kRange ? kRange : (uint32_t)bytes;
    return tpw_u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)),
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)num), 0x00020000u};
}

// The same address in every lane, in scalar registers.
__device__ __forceinline__ const void *uniform(const void *p) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
    return reinterpret_cast<const void *>((uintptr_t)((uint64_t)hi << 32 | lo));
}

// Moves rows [0, ROWS) of a tile into LDS; rows at or past `rows` and features at or past `d`
// become zeros and are not read.
template <typename T, int DP, int ROWS, int WAVES, bool DWORDS = false>
struct Stager {
    using L = Tile<T, DP>;
    static constexpr int kSlots = ROWS * L::C / (64 * WAVES);
    static_assert(ROWS * L::C % (64 * WAVES) == 0, "whole instructions");
    uint32_t off[kSlots];
    int64_t stride;  // bytes between rows
    int wave, width;  // width: bytes of a row (DWORDS)

    __device__ __forceinline__ void init(int64_t row_stride, int d, int wave_, int lane) {
        stride = row_stride * (int64_t)sizeof(T);
        wave = wave_;
        width = d * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const int s = (i * WAVES + wave) * 64 + lane, r = s / L::C, c = (s % L::C) ^ L::swz(r);
            off[i] = c * L::E < d ? (uint32_t)(r * stride + c * 16) : kBeyond;
        }
    }
    __device__ __forceinline__ void load(const T *base, int64_t rows, uint32_t to) const {
        const uint32_t lds = DWORDS ? (uint32_t)__builtin_amdgcn_readfirstlane((int)to) : to;
        const tpw_u32x4 r = resource(base, rows * stride);
        if constexpr (DWORDS) {  // four times the instructions, their offsets formed as they go
            const int lane = threadIdx.x & 63;
#pragma unroll 2
            for (int i = 0; i < 4 * kSlots; ++i) {
                const int s = (i * WAVES + wave) * 64 + lane, row = s / (4 * L::C);
                const int byte = ((s / 4 % L::C) ^ L::swz(row)) * 16 + (s & 3) * 4;
                dma4(r, byte < width ? (uint32_t)(row * stride + byte) : kBeyond,
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)(lds + (uint32_t)((i * WAVES + wave) * 256))));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kSlots; ++i) dma16(r, off[i], lds + (uint32_t)((i * WAVES + wave) * 1024));
        }
    }
};

__device__ __forceinline__ tpw_u32x4 lds_read16(uint32_t a) {
    return *reinterpret_cast<__attribute__((address_space(3))) const tpw_u32x4 *>((uintptr_t)a);
}

// Row fragments: features KS s + 8 g .. + 7 of row lane % W of a block of W rows.  A lane's own part
// of the address is one register; pieces differ from it by an exclusive or of a constant.
template <typename T, int DP, int W>
struct RowReader {
    using L = Tile<T, DP>;
    using S = Shape<W>;
    static constexpr int P = 8 / L::E;  // pieces per fragment
    uint32_t at;
    __device__ __forceinline__ RowReader(int lane) {
        const int r = lane % W;
        at = (uint32_t)(r * L::kRowBytes + ((P * (lane / W)) ^ L::swz(r)) * 16);
    }
    // block `blk` of the tile at `tile` (swz(r) depends on r mod 16 only, and W is a multiple of 16)
    __device__ __forceinline__ Frag<T> read(uint32_t tile, int blk, int s) const {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            f.v = __builtin_bit_cast(uint4, lds_read16(L::piece(tile + at, S::NG * s, blk * W * L::kRowBytes)));
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                f.v[u] = __builtin_bit_cast(
                    f32x4, lds_read16(L::piece(tile + at, 2 * S::NG * s + u, blk * W * L::kRowBytes)));
        }
        return f;
    }
};

// Column pieces, the first operands of the second products (sums over rows): a step t covers KS rows
// in kPieces pieces, each of which `use` multiplies into the accumulators of its feature blocks.
// Element 4 u + e of the second operand is row 4 NG (2 t + u) + 4 g + e of the tile.
//   bf16: piece c is block c of W features, by two transposing reads: lane i of a group of 16 points
//   at four features of row i / 4 and receives feature i % 16 of the four rows.
//   fp32: piece c is rows u = c % 2 of features 64 (c / 2) .. + 63.  A lane reads features 4 (lane %
//   16) .. + 3 of each row, so block 4 B + k holds features 64 B + 4 i + k: one 16-byte read feeds
//   four products.  The last 32 of 96 features go two by two.
// `each` gives the results back as quads of consecutive features.
template <typename T, int DP, int W>
struct ColReader;
template <int DP>
struct ColReader<uint16_t, DP, 32> {
    static constexpr int W = 32;
    using L = Tile<uint16_t, DP>;
    using M = Mma<uint16_t, W>;
    static constexpr int kBlocks = DP / W, kPieces = kBlocks;
    typedef uint4 Piece;
    uint32_t at;
    __device__ __forceinline__ ColReader(int lane) {
        const int i = lane & 15, r0 = 4 * (lane / W) + (i >> 2), col = 16 * ((lane % W) >> 4) + 4 * (i & 3);
        at = (uint32_t)(r0 * L::kRowBytes + ((col >> 3) ^ L::swz(r0)) * 16 + (col & 4) * 2);
    }
    __device__ __forceinline__ Piece read(uint32_t tile, int t, int c) const {
        uint2 v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // swz(8 (2 t + u) + r0) = swz(r0) ^ 2 u
            const uint32_t a = L::piece(tile + at, (4 * c) ^ (2 * u), 8 * (2 * t + u) * L::kRowBytes);
            v[u] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                 (__attribute__((address_space(3))) s16x4 *)(uintptr_t)a));
        }
        return make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
    }
    static __device__ __forceinline__ void use(typename M::Acc *acc, int c, const Piece &a, const Frag<uint16_t> &p) {
        M::mma(acc[c], Frag<uint16_t>{a}, p);
    }
    template <typename F>
    static __device__ __forceinline__ void each(const typename M::Acc *acc, int lane, F &&f) {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int w = 0; w < M::Q; ++w)
                f(W * i + 4 * M::NG * w + 4 * (lane / W),
                  f32x4{acc[i][4 * w], acc[i][4 * w + 1], acc[i][4 * w + 2], acc[i][4 * w + 3]});
    }
};
template <int DP>
struct ColReader<float, DP, 16> {
    using L = Tile<float, DP>;
    using M = Mma<float, 16>;
    static constexpr int kWhole = DP / 64, kHalf = DP % 64 / 32;
    static constexpr int kBlocks = DP / 16, kPieces = 2 * (kWhole + kHalf);
    static_assert(DP % 32 == 0, "pieces of 64 features and one of 32");
    struct Piece {
        f32x4 v[4];
    };
    uint32_t at, half;
    __device__ __forceinline__ ColReader(int lane) {
        const int r0 = 4 * (lane / 16), i = lane % 16;
        at = (uint32_t)(r0 * L::kRowBytes + (i ^ L::swz(r0)) * 16);
        half = (uint32_t)(r0 * L::kRowBytes + ((i >> 1) ^ L::swz(r0)) * 16 + (i & 1) * 8);
    }
    __device__ __forceinline__ Piece read(uint32_t tile, int t, int c) const {
        Piece p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // swz(r0 + e) = swz(r0) ^ 4 e
            const int index = (c / 2 * 16) ^ (4 * e), far = (16 * (2 * t + c % 2) + e) * L::kRowBytes;
            if (c / 2 < kWhole) {
                p.v[e] = __builtin_bit_cast(f32x4, lds_read16(L::piece(tile + at, index, far)));
            } else {
                const f32x2 x = *reinterpret_cast<__attribute__((address_space(3))) const f32x2 *>(
                    (uintptr_t)L::piece(tile + half, index, far));
                p.v[e] = f32x4{x[0], x[1], 0.0f, 0.0f};
            }
        }
        return p;
    }
    static __device__ __forceinline__ void use(M::Acc *acc, int c, const Piece &a, const Frag<float> &p) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int k = 0; k < (c / 2 < kWhole ? 4 : 2); ++k)
                acc[4 * (c / 2) + k] =
                    __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e][k], p.v[c % 2][e], acc[4 * (c / 2) + k], 0, 0, 0);
    }
    template <typename F>
    static __device__ __forceinline__ void each(const M::Acc *acc, int lane, F &&f) {
#pragma unroll
        for (int b = 0; b < kWhole; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                f(64 * b + 16 * (lane / 16) + 4 * r,
                  f32x4{acc[4 * b][r], acc[4 * b + 1][r], acc[4 * b + 2][r], acc[4 * b + 3][r]});
        if constexpr (kHalf)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto &x = acc[4 * kWhole], &y = acc[4 * kWhole + 1];
                f(64 * kWhole + 8 * (lane / 16) + 4 * h, f32x4{x[2 * h], y[2 * h], x[2 * h + 1], y[2 * h + 1]});
            }
    }
};

// Features f .. f + 7 of a row in global memory (null: zeros).
template <typename T>
__device__ __forceinline__ Frag<T> load_row8(const T *row, int f, int d, bool dwords = false) {
    constexpr int E = 16 / (int)sizeof(T), D = 4 / (int)sizeof(T);
    T x[8];
    if (dwords) {
#pragma unroll
        for (int u = 0; u < 8 / D; ++u) {
            uint32_t w = 0;
            if (row && f + u * D < d) w = *reinterpret_cast<const uint32_t *>(row + f + u * D);
            __builtin_memcpy(x + u * D, &w, 4);
        }
        Frag<T> r;
        __builtin_memcpy(&r, x, sizeof(r));
        return r;
    }
#pragma unroll
    for (int u = 0; u < 8 / E; ++u) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (row && f + u * E < d) w = *reinterpret_cast<const uint4 *>(row + f + u * E);
        __builtin_memcpy(x + u * E, &w, 16);
    }
    Frag<T> r;
    __builtin_memcpy(&r, x, sizeof(r));
    return r;
}

// Four consecutive features of an output row: one store of any alignment (global memory takes it),
// element by element past the last whole quad.
__device__ __forceinline__ void store4(float *row, int f, int d, f32x4 v) {
    if (f + 4 <= d) {
        __builtin_memcpy(row + f, &v, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (f + e < d) row[f + e] = v[e];
    }
}
__device__ __forceinline__ void store4(uint16_t *row, int f, int d, f32x4 v) {
    if (f + 4 <= d) {
        const uint2 w = make_uint2(f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]));
        __builtin_memcpy(row + f, &w, 8);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (f + e < d) row[f + e] = f32_to_bf16_rne(v[e]);
    }
}

// What rounding the four values above left, rounded in turn.  delta = do . o of a row that rests on few
// keys meets ds = p (dp - delta) with everything cancelled: from o alone, 2^-8 of each value off, dq and
// dk of short or sparse rows would lose a quarter of their precision.
__device__ __forceinline__ void store_rest4(uint16_t *row, int f, int d, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] -= bf16_to_f32(f32_to_bf16_rne(v[e]));
    store4(row, f, d, v);
}
// Output row of head h, row i: values, and their rest where it is wanted.
template <typename T>
struct OutRow {
    T *row, *rest;
    int d;
    __device__ __forceinline__ OutRow(const Args &a, int64_t b, int64_t h, int64_t i) : d((int)a.dv) {
        const int64_t at = b * a.o.b + h * a.o.h + i * a.o.n;
        row = reinterpret_cast<T *>(const_cast<void *>(a.o.p)) + at;
        rest = a.rest ? reinterpret_cast<T *>(a.rest) + at : nullptr;
    }
    __device__ __forceinline__ void store(int f, f32x4 v) const {
        store4(row, f, d, v);
        if constexpr (sizeof(T) == 2)
            if (rest) store_rest4(rest, f, d, v);
    }
};

template <int W>
__device__ __forceinline__ float over_groups_max(float v) {
#pragma unroll
    for (int o = W; o < 64; o <<= 1) v = __builtin_fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
template <int W>
__device__ __forceinline__ float over_groups_sum(float v) {
#pragma unroll
    for (int o = W; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Keys of an entry that may be read.
__device__ __forceinline__ int64_t key_end(const Args &a, int64_t b) {
    if (!a.lengths) return a.m;
    const int64_t l = a.lengths[b];
    return l < 0 ? 0 : l > a.m ? a.m : l;
}
// Keys that query i sees, of `len`: the last query sees all of them.
__device__ __forceinline__ int64_t row_limit(const Args &a, int64_t len, int64_t i) {
    if (!a.causal) return len;
    const int64_t l = i + 1 + len - a.n;
    return l < 0 ? 0 : l;
}

// kKeep: bits of keys 32 w .. 32 w + 31 of a row.  kBias: values of a row (any alignment; keys past m are
// not read).
__device__ __forceinline__ const uint32_t *mask_words(const Args &a, int64_t b, int64_t h, int64_t i) {
    return reinterpret_cast<const uint32_t *>(a.mask) + b * a.mb + h * a.mh + i * a.mn;
}
__device__ __forceinline__ const void *mask_row(const Args &a, int64_t b, int64_t h, int64_t i) {
    return reinterpret_cast<const uint8_t *>(a.mask) + (b * a.mb + h * a.mh + i * a.mn) * (a.mask_bf16 ? 2 : 4);
}
__device__ __forceinline__ float mask_value(const Args &a, const void *row, int64_t at) {
    return a.mask_bf16 ? bf16_to_f32(reinterpret_cast<const uint16_t *>(row)[at])
                       : reinterpret_cast<const float *>(row)[at];
}
// Values of keys j0 + STEP x + off + e, x < N, of one row (STEP keys apart, `span` of them from j0 for the
// wave).  Inside the row every load goes out at once, without a branch between them.
template <int N, int STEP>
__device__ __forceinline__ void mask_bias(const Args &a, const void *row, int j0, int off, int span, f32x4 (&v)[N]) {
    if (a.mm == 1 && j0 + span <= a.m) {
        if (a.mask_bf16) {
            const uint16_t *p = reinterpret_cast<const uint16_t *>(row) + j0 + off;
            uint2 w[N];
#pragma unroll
            for (int x = 0; x < N; ++x) __builtin_memcpy(&w[x], p + STEP * x, 8);
#pragma unroll
            for (int x = 0; x < N; ++x)
                v[x] = f32x4{__uint_as_float(w[x].x << 16), __uint_as_float(w[x].x & 0xffff0000u),
                             __uint_as_float(w[x].y << 16), __uint_as_float(w[x].y & 0xffff0000u)};
        } else {
            const float *p = reinterpret_cast<const float *>(row) + j0 + off;
#pragma unroll
            for (int x = 0; x < N; ++x) __builtin_memcpy(&v[x], p + STEP * x, 16);
        }
    } else {
#pragma unroll
        for (int x = 0; x < N; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t j = (int64_t)j0 + STEP * x + off + e;
                v[x][e] = j < a.m ? mask_value(a, row, j * a.mm) : 0.0f;
            }
    }
}

__device__ __forceinline__ int64_t cdiv_dev(int64_t a, int64_t b) { return (a + b - 1) / b; }
__host__ __device__ inline int64_t quads4(int64_t x) { return (x + 3) / 4 * 4; }

// Block id -> (tile, batch * key_heads + key head): ids go round-robin over the 8 XCDs, so where
// they divide, each XCD gets a contiguous range: the blocks that share keys share an L2.
__device__ __forceinline__ int64_t xcd_linear(int64_t bid, int64_t total) {
    return (total & 7) == 0 ? (bid & 7) * (total >> 3) + (bid >> 3) : bid;
}

// Blocks and tiles: waves per block, keys per LDS tile (rows per tile of the dk / dv kernel).  Two
// buffers of two tiles stay within 64 KiB, so two blocks of four waves share a CU; fp32 at 256
// features takes 128 KiB, and eight waves share them.
template <typename T, int DP>
struct Tiles {
    static constexpr int kWidth = sizeof(T) == 2 ? 32 : 16;  // W of the matrix instructions
    static constexpr int kRowBytes = Tile<T, DP>::kRowBytes;
    static constexpr int kWaves = kRowBytes == 1024 ? 8 : 4;
    static constexpr int kKeys = kRowBytes <= 256 ? 64 : 32;
    static constexpr int kRowWaves = 4, kRows = 32;          // dk / dv kernel
    // blocks that share a CU, as parts_for takes them: forward, dq, dk / dv.  What the registers and the LDS
    // of the kernels without added values leave (dk / dv of fp32 up to 64 features: three; of the two launches
    // for bf16 at 256 features: dk's one).
    static constexpr bool kNarrow = kRowBytes == 128;  // bf16 up to 64 features
    static constexpr int kPerCu = kNarrow ? 4 : kWaves == 8 ? 1 : 2;
    static constexpr int kPerCuQ = kNarrow ? 3 : kWaves == 8 || DP == 256 ? 1 : 2;
    static constexpr int kPerCuK = DP == 256 || (DP > 64 && sizeof(T) == 4) ? 1 : 2;
};

// Host side (attention.hip): reads a descriptor into the kernels' arguments; bytes that a call's
// prepared operands take (padded copies of those that need one, the bits of a boolean mask), and the
// launches that prepare them at `at` (16-byte aligned) and point the arguments to them.
int read_args(const tpw_attention_desc *d, bool backward, Args &a);
size_t prepared_bytes(const Args &a, const tpw_attention_desc *d, bool backward);
int prepare_operands(Args &a, const tpw_attention_desc *d, bool backward, void *at, hipStream_t s);
// Joins a.splits parts of every row into a.o (and a.stats).
int join_parts(const Args &a, int dtype, bool bias, hipStream_t s);

// Runs f(type tag, DP, mask mode) for the arguments' types and widths.
template <int V>
struct Const {
    static constexpr int value = V;
};
template <typename T, typename F>
int by_width(const Args &a, int mode, F &&f) {
    const int64_t w = a.d > a.dv ? a.d : a.dv;
    const auto by_mode = [&](auto dp) {
        if (mode == kNoMask) return f(T{}, dp, Const<kNoMask>{});
        if (mode == kKeep) return f(T{}, dp, Const<kKeep>{});
        return f(T{}, dp, Const<kBias>{});
    };
    // widths between the powers of two too, where up to half of the products would be of zeros
    if (w <= 64) return by_mode(Const<64>{});
    if (w <= 96) return by_mode(Const<96>{});
    if (w <= 128) return by_mode(Const<128>{});
    if (w <= 192) return by_mode(Const<192>{});
    return by_mode(Const<256>{});
}
template <typename F>
int by_type(const Args &a, int dtype, int mode, F &&f) {
    return dtype == TPW_BF16 ? by_width<uint16_t>(a, mode, f) : by_width<float>(a, mode, f);
}
// A mask over no pairs is none: it may have no address.
inline int mask_mode(const tpw_attention_desc *d) {
    if (d->batch == 0 || d->heads == 0 || d->n == 0 || d->m == 0) return kNoMask;
    return d->mask_type == TPW_MASK_NONE ? kNoMask : d->mask_type == TPW_MASK_KEEP ? kKeep : kBias;
}
// Parts of a summed axis of `steps` tiles for `blocks` blocks, `per_cu` of which share a CU: the least
// of the time that this model gives.
//   - A tile takes a block step_us with its CU full and less the fewer share it (bf16 at 128 features under a
//     boolean mask: 3.3 us two by two, 2.4 alone).
//   - Up to 256 per_cu blocks run at once, more as places come free: a started round costs a third of one.
//     A square causal call's differ in length, the longest twice the mean; they start with the longest,
//     which speeds up as it is left alone.
//   - Parts cost the launch that joins them (6 us, host and device) and their bytes, written and read
//     (part_us each).
// dk / dv of causal 2 x 4 key heads x 8192 keys x 128: 1.76 ms in 512 blocks, 1.23 + 0.035 in 1024;
// forward of causal 8 x 4 (2) x 587 x 128: 28 + 24 us in seven parts.
constexpr int kMaxParts = 64;  // the join gives each part a lane
inline bool uneven(const Args &a) { return a.causal && 2 * a.n > a.m; }
inline int64_t parts_for(int64_t blocks, int64_t steps, int64_t per_cu, bool uneven, double step_us, double part_us) {
    if (blocks <= 0) return 1;
    int64_t best = 1;
    double least = 0;
    for (int64_t p = 1; p <= steps && p <= kMaxParts; ++p) {
        const int64_t n = blocks * p, slots = 256 * per_cu, sharing = cdiv(n, 256) < per_cu ? cdiv(n, 256) : per_cu;
        const double step = step_us * (0.5 + 0.5 * (double)sharing / (double)per_cu), len = (double)cdiv(steps, p);
        const double flow = 0.5 * (double)steps * (double)blocks / (double)slots + 0.125 * len;
        const double rounds = (double)(n / slots), over = (double)(n % slots) / (double)slots;
        const double even = len * (rounds == 0 ? 1.0 : rounds + (over > 0 ? 0.35 + 0.65 * over : 0.0));
        double t = step * (!uneven ? even : 0.85 * len > flow ? 0.85 * len : flow);
        if (p > 1) t += 6.0 + (double)p * part_us;
        if (p == 1 || t < least) {
            least = t;
            best = p;
        }
        if (n >= 4 * slots) break;
    }
    return best;
}
// Microseconds of one tile with its CU full: `products` products of own x streamed x DP at the rate
// the kernels reach (0.9 PFLOP/s bf16, 120 TFLOP/s fp32).
template <typename T, int DP>
double step_us(int64_t own, int64_t streamed, int products, int64_t per_cu) {
    const double flops = 2.0 * products * (double)own * (double)streamed * DP;
    return flops * (double)per_cu * 256.0 / (sizeof(T) == 2 ? 0.9e9 : 0.12e9);
}
inline double part_us(int64_t rows, int64_t width) { return 2.0 * 4.0 * (double)rows * (double)width / 4.5e6; }

}  // namespace attn
}  // namespace tpw
