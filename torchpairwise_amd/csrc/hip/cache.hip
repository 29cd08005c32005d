// Rows into a cache of keys and values in 4 or 8 bits, and out of it (format and layouts: cache.hpp).
#include "cache.hpp"

namespace tpw {
namespace cache {
namespace {

struct RowsArgs {
    Cache c;
    const void *x[2];        // keys, values (written to the cache), or
    void *y[2];              // (read from it)
    int64_t xb[2], xh[2], xn[2];  // element strides of batch, heads, rows; features dense
    int width[2];
    int whole[2];            // rows are whole pieces of 8 features at 16-byte aligned addresses
    const int64_t *starts;   // [batch] or null (0)
    const int64_t *counts;   // [batch] or null (n)
    int64_t heads, n, m;     // rows of a call; rows that a sequence has room for
    int64_t tiles;           // blocks of 256 threads per (sequence, head), those of the wider side
};

// What one thread works on: 8 features (a piece) of row i; 4 consecutive lanes share a block of 32.
struct Piece {
    int64_t b, h, i;
    int piece;
    bool live;  // row i is one of the call's
    Place at;   // first < 0: no place in the cache
};
__device__ __forceinline__ bool piece_of(const RowsArgs &a, int side, Piece &p) {
    const Side &s = side ? a.c.v : a.c.k;
    const int pieces = 4 * s.blocks, per = 256 / pieces, t = (int)threadIdx.x, r = t / pieces;
    const int64_t id = blockIdx.x, bh = id / a.tiles;
    p.piece = t - r * pieces;
    p.b = bh / a.heads;
    p.h = bh - p.b * a.heads;
    p.i = (id - bh * a.tiles) * per + r;
    if (r >= per || p.i >= a.n) return false;
    p.live = !a.counts || p.i < a.counts[p.b];
    const int64_t j = (a.starts ? a.starts[p.b] : 0) + p.i;
    p.at = {-1, 0};
    if (p.live && j >= 0 && j < a.m) p.at = place(a.c, p.b, (int)j);
    return true;
}

// One thread per 8 features.  The largest magnitude is taken over the bits (NaN above infinity above all
// numbers) within the thread and over 4 lanes.  Bound by memory: 2 x 4 x 16 x 8192 x 128 bf16 (268 MB read,
// 71 MB written).
template <typename T, int BITS>
__global__ __launch_bounds__(256) void cache_write_kernel(const RowsArgs a) {
    const int side = blockIdx.y;
    Piece p;
    if (!piece_of(a, side, p) || p.at.first < 0) return;  // the four lanes of a block alike
    const T *row = reinterpret_cast<const T *>(a.x[side]) + p.b * a.xb[side] + p.h * a.xh[side] + p.i * a.xn[side];
    const int f = 8 * p.piece, d = a.width[side];
    T raw[8];
    if (a.whole[side] && f < d) {
        __builtin_memcpy(raw, __builtin_assume_aligned(row + f, 16), sizeof(raw));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e] = f + e < d ? row[f + e] : T(0);
    }
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = to_f32(raw[e]);
        const uint32_t m = __float_as_uint(x[e]) & 0x7fffffffu;
        top = m > top ? m : top;
    }
    const uint32_t byte = cache::scale_byte<BITS>(cache::over_block(top));
    const float scale = scale_of(byte);
    const bool finite = byte != 255;
    const Side &s = side ? a.c.v : a.c.k;
    uint8_t *codes = s.codes + p.at.first * s.cf + p.h * s.ch + p.at.row * s.cr;
    if constexpr (BITS == 4) {
        reinterpret_cast<uint32_t *>(codes)[p.piece] = finite ? to_fp4(x, scale) : 0u;
    } else {
        const uint2 w = to_fp8(x, scale);
        reinterpret_cast<uint2 *>(codes)[p.piece] = finite ? w : make_uint2(0u, 0u);
    }
    if (p.piece % 4 == 0)
        s.scales[p.at.first * s.sf + p.h * s.sh + p.piece / 4 * s.sb + p.at.row] = (uint8_t)byte;
}

// One thread per 8 features; rows that are not the call's, or that lie nowhere, are zeros.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void cache_read_kernel(const RowsArgs a) {
    const int side = blockIdx.y;
    Piece p;
    if (!piece_of(a, side, p)) return;
    T *row = reinterpret_cast<T *>(a.y[side]) + p.b * a.xb[side] + p.h * a.xh[side] + p.i * a.xn[side];
    const int f = 8 * p.piece, d = a.width[side];
    if (f >= d) return;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (p.at.first >= 0) {
        const Side &s = side ? a.c.v : a.c.k;
        const uint8_t *codes = s.codes + p.at.first * s.cf + p.h * s.ch + p.at.row * s.cr;
        Eight<BITS> w;
        __builtin_memcpy(&w, __builtin_assume_aligned(codes + BITS * p.piece, BITS), sizeof(w));
        w.f32(scale_of(s.scales[p.at.first * s.sf + p.h * s.sh + p.piece / 4 * s.sb + p.at.row]), x);
    }
    T out[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) from_f32(&out[e], x[e]);
    if (a.whole[side]) {
        __builtin_memcpy(__builtin_assume_aligned(row + f, 16), out, sizeof(out));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (f + e < d) row[f + e] = out[e];
    }
}

template <typename T, int BITS>
int launch(const RowsArgs &a, bool write, int64_t blocks, hipStream_t s) {
    const dim3 grid((unsigned)blocks, 2);
    if (write) {
        hipLaunchKernelGGL((cache_write_kernel<T, BITS>), grid, dim3(256), 0, s, a);
        return check_launch("cache_write_kernel");
    }
    hipLaunchKernelGGL((cache_read_kernel<T, BITS>), grid, dim3(256), 0, s, a);
    return check_launch("cache_read_kernel");
}

int move_rows(const tpw_cache_desc *d, bool write, int dtype, int64_t batch, int64_t n, const void *key, int64_t width,
              const int64_t *key_strides, const void *value, int64_t value_width, const int64_t *value_strides,
              const int64_t *starts, const int64_t *counts, void *stream) {
    RowsArgs a = {};
    if (const int rc = read_cache(d, batch, a.c)) return rc;
    TPW_REQUIRE(dtype == TPW_F32 || dtype == TPW_BF16, "cache: float32 or bfloat16 rows");
    TPW_REQUIRE(n >= 0 && n < (int64_t(1) << 31), "cache: invalid number of rows");
    TPW_REQUIRE(width >= 1 && width <= 32 * d->key_blocks && value_width >= 1 && value_width <= 32 * d->value_blocks,
                "cache: rows are wider than the cache's");
    if (batch * d->heads * n == 0) return TPW_OK;
    TPW_REQUIRE(key && value && key_strides && value_strides, "cache: null operand");
    const int64_t size = dtype == TPW_F32 ? 4 : 2;
    const void *rows[2] = {key, value};
    const int64_t *strides[2] = {key_strides, value_strides};
    const int64_t blocks = a.c.k.blocks > a.c.v.blocks ? a.c.k.blocks : a.c.v.blocks;
    for (int t = 0; t < 2; ++t) {
        a.x[t] = rows[t];
        a.y[t] = const_cast<void *>(rows[t]);
        a.xb[t] = batch == 1 ? 0 : strides[t][0];
        a.xh[t] = d->heads == 1 ? 0 : strides[t][1];
        a.xn[t] = n == 1 ? 0 : strides[t][2];
        a.width[t] = (int)(t ? value_width : width);
        a.whole[t] = a.width[t] % 8 == 0 && aligned16(rows[t]) && (a.xb[t] | a.xh[t] | a.xn[t]) * size % 16 == 0;
    }
    a.starts = starts;
    a.counts = counts;
    a.heads = d->heads;
    a.n = n;
    a.m = d->pages ? d->page_count * d->rows : d->rows;
    a.tiles = cdiv(n, 256 / (4 * blocks));
    const int64_t grid = a.tiles * batch * d->heads;
    TPW_REQUIRE(grid < (int64_t(1) << 31), "cache: too many rows");
    hipStream_t s = as_stream(stream);
    if (dtype == TPW_F32)
        return d->bits == 4 ? launch<float, 4>(a, write, grid, s) : launch<float, 8>(a, write, grid, s);
    return d->bits == 4 ? launch<uint16_t, 4>(a, write, grid, s) : launch<uint16_t, 8>(a, write, grid, s);
}

}  // namespace

int read_cache(const tpw_cache_desc *d, int64_t batch, Cache &c) {
    TPW_REQUIRE(d, "cache: null descriptor");
    TPW_REQUIRE(d->bits == 4 || d->bits == 8, "cache: 4 or 8 bits");
    TPW_REQUIRE(batch >= 0 && d->first >= 0 && d->heads >= 1 && d->rows >= 0, "cache: invalid sizes");
    TPW_REQUIRE(d->key_blocks >= 1 && d->key_blocks <= 8 && d->value_blocks >= 1 && d->value_blocks <= 8,
                "cache: rows have 1 to 8 blocks of 32 features");
    TPW_REQUIRE(d->rows % 16 == 0, "cache: rows must come in multiples of 16");
    int64_t m = d->rows;
    c.shift = 31;
    c.mask = 0x7fffffff;
    if (d->pages) {
        TPW_REQUIRE(d->rows >= 16 && (d->rows & (d->rows - 1)) == 0 && d->rows <= (int64_t(1) << 20),
                    "cache: pages have a power of two of rows, 16 to 2^20");
        TPW_REQUIRE(d->page_count >= 0 && d->page_count < (int64_t(1) << 31), "cache: invalid number of pages");
        m = d->page_count * d->rows;
        c.shift = __builtin_ctzll((unsigned long long)d->rows);
        c.mask = (int)d->rows - 1;
    } else {
        TPW_REQUIRE(d->first == batch, "cache: a cache without pages holds one entry per sequence");
    }
    TPW_REQUIRE(m < (int64_t(1) << 31) - 1024, "cache: too many rows");
    c.pages = d->pages;
    c.pitch = d->page_pitch;
    c.first = d->first;
    c.wide = d->pages_wide != 0;
    const auto side = [&](Side &s, void *codes, void *scales, const int64_t *cs, const int64_t *ss, int64_t blocks) {
        s.codes = reinterpret_cast<uint8_t *>(codes);
        s.scales = reinterpret_cast<uint8_t *>(scales);
        s.blocks = (int)blocks;
        // strides of dimensions of one entry reach nothing
        s.cf = d->first == 1 ? 0 : cs[0];
        s.ch = d->heads == 1 ? 0 : cs[1];
        s.cr = cs[2];
        s.sf = d->first == 1 ? 0 : ss[0];
        s.sh = d->heads == 1 ? 0 : ss[1];
        s.sb = blocks == 1 ? 0 : ss[2];
        return aligned16(codes) && aligned16(scales) && (s.cf | s.ch | s.cr | s.sf | s.sh | s.sb) % 16 == 0 &&
               (m * d->first == 0 || (codes && scales));
    };
    TPW_REQUIRE(side(c.k, d->key_codes, d->key_scales, d->key_code_strides, d->key_scale_strides, d->key_blocks) &&
                    side(c.v, d->value_codes, d->value_scales, d->value_code_strides, d->value_scale_strides,
                         d->value_blocks),
                "cache: codes and scales must lie at 16-byte aligned addresses and strides");
    return TPW_OK;
}

}  // namespace cache
}  // namespace tpw

using namespace tpw;
using namespace tpw::cache;

extern "C" int tpw_cache_write(const tpw_cache_desc *d, int dtype, int64_t batch, int64_t n, const void *key,
                               int64_t width, const int64_t *key_strides, const void *value, int64_t value_width,
                               const int64_t *value_strides, const int64_t *starts, const int64_t *counts,
                               void *stream) {
    return move_rows(d, true, dtype, batch, n, key, width, key_strides, value, value_width, value_strides, starts, counts,
                     stream);
}

extern "C" int tpw_cache_read(const tpw_cache_desc *d, int dtype, int64_t batch, int64_t n, void *key, int64_t width,
                              const int64_t *key_strides, void *value, int64_t value_width,
                              const int64_t *value_strides, const int64_t *starts, const int64_t *counts,
                              void *stream) {
    return move_rows(d, false, dtype, batch, n, key, width, key_strides, value, value_width, value_strides, starts,
                     counts, stream);
}
