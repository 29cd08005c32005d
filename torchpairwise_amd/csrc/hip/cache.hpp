// Shared pieces of the kernels over a cache of keys and values in 4 or 8 bits (cache.hip, cache_rows.hpp,
// cache_tiles.hpp).
//
// A block of 32 features of a row shares a power of two 2^e, the first, from e = -127 on, with which the block's
// largest magnitude a is less than halfway from the last code to the one that would follow it:
//   4 bits: sign, 2 exponent and 1 mantissa bit, 0 .5 1 1.5 2 3 4 6;  a < 7 2^e
//   8 bits: sign, 4 and 3, largest 448;  a < 464 2^e  (464, a tie, would still round to 448: it takes the next power)
// so no value rounds past the last code, and each is off by at most half a step of its own binade, or of the block's
// smallest codes.  x / 2^e is exact, its rounding (to nearest, ties to even) the only one: the codes are the same on
// every machine.  (Magnitudes from 3.5 2^126, in 8 bits 1.9375 2^127 on round to 2^128, which float32 reads as
// infinity.)  The scale is kept as the byte e + 127, whose place in a float's bits is its exponent: gfx950's
// conversions (v_cvt_scalef32_*) take that float, read 0 as 2^-127 and 255 as NaN, whatever the code.  A block that
// holds NaN or an infinity has scale 255 and codes of zero.
// Every value is exact in bfloat16 (2 or 4 significant bits).
//
// Codes: [batch | pages, heads, rows, blocks] of 16 bytes (two features a byte, the even one low) or 32.
// Scales: [batch | pages, heads, blocks, rows], rows dense: eight bytes are eight keys' scales of a block.
// Rows come in multiples of 16, so that no read of 8 whole rows leaves the cache.
#pragma once

#include "common.hpp"

namespace tpw {
namespace cache {

struct Side {  // the keys or the values; strides in bytes
    uint8_t *codes, *scales;
    int64_t cf, ch, cr;  // codes: first dimension, heads, rows
    int64_t sf, sh, sb;  // scales: first dimension, heads, blocks
    int blocks;
};

struct Cache {
    Side k, v;
    const void *pages;  // table [batch, pages of a sequence] (dense in the second), or null
    int64_t pitch;      // its entries between sequences
    int64_t first;      // pages there are (without a table: sequences)
    int wide;           // its entries are 64-bit
    int shift, mask;    // rows of a page: 1 << shift, and less one (without a table: 31, all ones)
    int near;           // rows lie at most 8 MiB apart, the scales of a row's blocks 256 MiB: 32 bits reach over 32 rows
};

// Where row j of sequence b lies: entry of the first dimension (-1: nowhere) and row.
struct Place {
    int64_t first;
    int row;
};
__device__ __forceinline__ Place place(const Cache &c, int64_t b, int j) {
    if (!c.pages) return {b, j};
    const int64_t at = b * c.pitch + (j >> c.shift);
    const int64_t p = c.wide ? reinterpret_cast<const int64_t *>(c.pages)[at]
                             : (int64_t) reinterpret_cast<const int32_t *>(c.pages)[at];
    return {p >= 0 && p < c.first ? p : -1, j & c.mask};
}

// The same for a row that a wave's lanes agree on, in scalar registers.
__device__ __forceinline__ Place uniform_place(const Cache &c, int64_t b, int j) {
    if (!c.pages) return {b, j};
    const int64_t at = b * c.pitch + (j >> c.shift);
    typedef __attribute__((address_space(4))) const int64_t *Wide;
    typedef __attribute__((address_space(4))) const int32_t *Narrow;
    const int64_t p = c.wide ? reinterpret_cast<Wide>(reinterpret_cast<uintptr_t>(c.pages))[at]
                             : (int64_t) reinterpret_cast<Narrow>(reinterpret_cast<uintptr_t>(c.pages))[at];
    return {p >= 0 && p < c.first ? p : -1, j & c.mask};
}

// The float that the conversions take for scale byte `b`.
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b << 23); }
// The same for byte k of a word, by one shift: only the exponent's bits are read.
__device__ __forceinline__ float scale_in(uint32_t w, int k) {
    return __uint_as_float(k < 3 ? w << (23 - 8 * k) : w >> 1);
}

typedef float f2 __attribute__((ext_vector_type(2)));
typedef short s2 __attribute__((ext_vector_type(2)));

// Two values of four codes' word: 4 bits: features 2 C, 2 C + 1 of eight; 8 bits: of four.
template <int BITS, int C>
__device__ __forceinline__ uint32_t bf16_pair(uint32_t w, float scale) {
    if constexpr (BITS == 4)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, C));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, C != 0));
}
template <int BITS, int C>
__device__ __forceinline__ f2 f32_pair(uint32_t w, float scale) {
    if constexpr (BITS == 4)
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, C);
    else
        return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, C != 0);
}
// Eight consecutive features: one word of 4-bit codes, two of 8-bit ones.
template <int BITS>
struct Eight {
    uint32_t w[BITS / 4];
    __device__ __forceinline__ uint4 bf16(float s) const {
        if constexpr (BITS == 4)
            return make_uint4(bf16_pair<4, 0>(w[0], s), bf16_pair<4, 1>(w[0], s), bf16_pair<4, 2>(w[0], s),
                              bf16_pair<4, 3>(w[0], s));
        else
            return make_uint4(bf16_pair<8, 0>(w[0], s), bf16_pair<8, 1>(w[0], s), bf16_pair<8, 0>(w[1], s),
                              bf16_pair<8, 1>(w[1], s));
    }
    __device__ __forceinline__ void f32(float s, float (&x)[8]) const {
        f2 y[4];
        if constexpr (BITS == 4) {
            y[0] = f32_pair<4, 0>(w[0], s), y[1] = f32_pair<4, 1>(w[0], s);
            y[2] = f32_pair<4, 2>(w[0], s), y[3] = f32_pair<4, 3>(w[0], s);
        } else {
            y[0] = f32_pair<8, 0>(w[0], s), y[1] = f32_pair<8, 1>(w[0], s);
            y[2] = f32_pair<8, 0>(w[1], s), y[3] = f32_pair<8, 1>(w[1], s);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = y[i / 2][i % 2];
    }
};

// The largest of a block's magnitudes (as bits: NaN above infinity above all numbers) out of its 4 lanes'.
__device__ __forceinline__ uint32_t over_block(uint32_t top) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2
    top = a > top ? a : top;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true);  // lanes 2 3 0 1
    top = b > top ? b : top;
    return top;
}
// The scale byte of a block with that largest magnitude: one more from 7/4 (29/16) of a binade on.
template <int BITS>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    const int e = BITS == 4 ? (int)((top + 0x200000u) >> 23) - 2 : (int)((top + 0x180000u) >> 23) - 8;
    return top >= 0x7f800000u ? 255u : e < 0 ? 0u : (uint32_t)e;
}
// Eight features to codes.
__device__ __forceinline__ uint32_t to_fp4(const float (&x)[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}
__device__ __forceinline__ uint2 to_fp8(const float (&x)[8], float scale) {
    s2 lo = {0, 0}, hi = {0, 0};
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[0], x[1], scale, false);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, x[2], x[3], scale, true);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[4], x[5], scale, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, x[6], x[7], scale, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// Blocks of 256 threads that one dimension of a launch has room for: 2^32 threads.
constexpr int64_t kMostBlocks = (int64_t(1) << 24) - 1;

// Host side (cache.hip): checks a cache against its batch and reads it into the kernels' form.
int read_cache(const tpw_cache_desc *d, int64_t batch, Cache &c);

}  // namespace cache
}  // namespace tpw
