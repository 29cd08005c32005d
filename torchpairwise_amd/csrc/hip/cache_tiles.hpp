// Attention of many query rows a key head over a cache in 4 or 8 bits: the tiles of attention.hip's forward,
// formed from the codes on their way into LDS.
#pragma once

#include "attention_forward.hpp"
#include "cache_attention.hpp"

namespace tpw {
namespace attn {

using cache::Cache;
using cache::Eight;
using cache::Side;

// Brings tiles of BN keys and their values into LDS in bfloat16, which holds them exactly.  A slot is a block of 32 features
// of one row: threads of 64 (32) consecutive rows share a block, so that the 16-byte stores of 16 of them
// fall on 16 different slots of the banks.  Codes wait in registers while the tile before is worked on.
template <int DP, int BN, int WAVES, int BITS>
struct Decoder {
    using L = Tile<uint16_t, DP>;
    static constexpr int kThreads = 64 * WAVES, kBlocks = L::P / 32, kSlots = 2 * BN * kBlocks / kThreads;
    static_assert(2 * BN * kBlocks % kThreads == 0 && BN * kBlocks % 64 == 0, "whole waves of slots");
    uint4 codes[kSlots][BITS / 4];
    uint32_t scale[kSlots];
    uint64_t present;  // keys of the tile that have a place (bits past the length are set too)

    // Keys j0 .. j0 + BN - 1 of sequence b.  Rows at or past len, blocks past the row's and rows without a
    // place become zeros and are not read.
    __device__ __forceinline__ void load(const Cache &c, int64_t b, int64_t kh, int j0, int len, int tid) {
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const int id = i * kThreads + tid, r = id % BN, block = id / BN % kBlocks;
            const bool values = id / (BN * kBlocks) != 0;
            const Side &s = values ? c.v : c.k;
            const int j = j0 + r;
            const bool in = j < len && block < s.blocks;
            cache::Place p = {-1, 0};
            if (in) p = cache::place(c, b, j);
            scale[i] = 0;
#pragma unroll
            for (int x = 0; x < BITS / 4; ++x) codes[i][x] = make_uint4(0, 0, 0, 0);
            if (p.first >= 0) {
                const uint4 *at = reinterpret_cast<const uint4 *>(s.codes + p.first * s.cf + kh * s.ch + p.row * s.cr +
                                                                  block * (4 * BITS));
#pragma unroll
                for (int x = 0; x < BITS / 4; ++x) codes[i][x] = at[x];
                scale[i] = s.scales[p.first * s.sf + kh * s.sh + block * s.sb + p.row];
            }
        }
        present = ~uint64_t(0);
        if (c.pages) {  // every wave for itself
            const int j = j0 + (tid & 63);
            present = __ballot(j >= len || cache::place(c, b, j).first >= 0);
        }
    }

    // The tile into LDS, keys at `to`, values behind them.
    __device__ __forceinline__ void store(uint32_t to, int tid) const {
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const int id = i * kThreads + tid, r = id % BN, block = id / BN;  // blocks of the keys, then the values
            const int piece = block % kBlocks * 4;
            if (DP < L::P && block % kBlocks * 32 >= DP) continue;
            const uint32_t row = to + (uint32_t)(block / kBlocks * BN * L::kRowBytes + r * L::kRowBytes);
            const float f = cache::scale_of(scale[i]);
            const uint32_t w[8] = {codes[i][0].x, codes[i][0].y, codes[i][0].z, codes[i][0].w,
                                   codes[i][BITS / 8].x, codes[i][BITS / 8].y, codes[i][BITS / 8].z,
                                   codes[i][BITS / 8].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // eight features at a time
                Eight<BITS> e;
#pragma unroll
                for (int y = 0; y < BITS / 4; ++y) e.w[y] = w[x * (BITS / 4) + y];
                put(row, r, piece + x, e.bf16(f));
            }
        }
    }
    static __device__ __forceinline__ void put(uint32_t row, int r, int c, uint4 v) {
        *reinterpret_cast<__attribute__((address_space(3))) tpw_u32x4 *>((uintptr_t)(row + (uint32_t)((c ^ L::swz(r)) * 16))) =
            __builtin_bit_cast(tpw_u32x4, v);
    }
};

// One block: kWaves * W query rows of the rows that share a key head, over the keys of one part.  Codes are converted once
// a block, beside the softmax in the VALU: 2 x 16 (4) x 8192^2 x 128 causal 590 us (935 TFLOP/s, matrix cores 0.38 busy;
// with keys and values of bf16 in HBM 600 to 660), 500 rows over 16384 of 64 58 us (0.23 busy: half the products
// for as many exponentials).  float32 queries (QT) and probabilities are three bf16 summands each, three products
// for one at 16 times the rate of float32's: 2 x 16 (4) x 4096^2 x 128 causal 402 us, where those took 1250.
template <typename QT, int DP, int MM, int BITS, int kWaves, int kPerSimd>
__global__ __launch_bounds__(64 * kWaves, kPerSimd) void cache_tiles_kernel(const Args a, const Cache c) {
    using T = uint16_t;
    constexpr int W = Tiles<T, DP>::kWidth, BN = Tiles<T, DP>::kKeys;
    using F = Forward<T, W, DP, BN, MM, false, true, QT>;
    constexpr uint32_t kTileBytes = BN * Tile<T, DP>::kRowBytes;
    // two buffers of a key tile and a value tile
    __shared__ __attribute__((aligned(256))) uint4 smem[4 * kTileBytes / 16];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t all = gridDim.x, id = (all & 7) == 0 ? (blockIdx.x & 7) * (all >> 3) + (blockIdx.x >> 3) : blockIdx.x;
    const uint32_t part = id % (uint32_t)a.splits, t = id / (uint32_t)a.splits;
    const int64_t tile = a.tiles - 1 - t % (uint32_t)a.tiles;  // longest rows of a causal call first
    const uint32_t bk = t / (uint32_t)a.tiles;
    const int64_t b = bk / (uint32_t)a.key_heads, kh = bk % (uint32_t)a.key_heads;
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
    Decoder<DP, BN, kWaves, BITS> d;
    if (t0 < t1) {
        d.load(c, b, kh, t0 * BN, (int)len, threadIdx.x);
        d.store(lds, threadIdx.x);
    }
    for (int i = t0; i < t1; ++i) {
        const uint64_t present = d.present;
        if (i + 1 < t1) d.load(c, b, kh, (i + 1) * BN, (int)len, threadIdx.x);
        tile::barrier_lds();  // tile i is there, and nobody reads the other buffer any more
        const uint32_t buf = lds + (uint32_t)((i - t0) & 1) * 2 * kTileBytes;
        f.tile(a, b, buf, buf + kTileBytes, i * BN, lane, present);
        if (i + 1 < t1) d.store(lds + (uint32_t)((i + 1 - t0) & 1) * 2 * kTileBytes, threadIdx.x);
    }

    const float sum = over_groups_sum<W>(f.sum);
    if (f.qi < 0) return;
    const int g = lane / W;
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int64_t row = (b * a.heads + f.qh) * a.n + f.qi;
    if (a.splits > 1) {
        const int64_t lines = a.batch * a.heads * a.n, at = part;
        float *st = a.part_stats + at * 2 * lines;
        if (g == 0) {
            st[row] = f.top;
            st[lines + row] = sum;
        }
        const int width = (int)quads4(a.dv);
        float *p = a.part + (at * lines + row) * width;
        F::CR::each(f.o, lane, [&](int at, f32x4 v) { store4(p, at, width, v); });
        return;
    }
    const OutRow<QT> out(a, b, f.qh, f.qi);
    F::CR::each(f.o, lane, [&](int at, f32x4 v) { out.store(at, v * inv); });
}

template <int BITS, typename QT>
int launch_tiles_of(const Args &a, const Cache &c, int mode, hipStream_t s) {
    return by_width<QT>(a, mode, [&](auto, auto dp, auto mm) {
        constexpr int DP = decltype(dp)::value, MM = decltype(mm)::value, kWaves = Tiles<uint16_t, DP>::kWaves;
        const int64_t blocks = a.batch * a.key_heads * a.tiles * a.splits;
        TPW_REQUIRE(blocks * kWaves <= 4 * cache::kMostBlocks, "attention: too many rows");
        constexpr int kPerSimd = tiles_per_simd(sizeof(QT), DP);
        hipLaunchKernelGGL((cache_tiles_kernel<QT, DP, MM, BITS, kWaves, kPerSimd>), dim3((unsigned)blocks),
                           dim3(64 * kWaves), 0, s, a, c);
        return check_launch("cache_tiles_kernel");
    });
}
template <int BITS>
int launch_tiles(const Args &a, const Cache &c, int dtype, int mode, hipStream_t s) {
    return dtype == TPW_BF16 ? launch_tiles_of<BITS, uint16_t>(a, c, mode, s) : launch_tiles_of<BITS, float>(a, c, mode, s);
}

}  // namespace attn
}  // namespace tpw
