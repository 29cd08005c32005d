// Rows into a cache of keys and values in 4 or 8 bits, and out of it (format and layouts: cache.hpp).
#include <type_traits>

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
    int64_t n, m;            // rows of a call; rows that a sequence has room for
    uint32_t heads, tiles;   // blocks of 256 threads per (sequence, head), those of the wider side
};

// A block's share: a thread works on PIECE features (a piece) of ROWS rows, consecutive ones (whose scales lie
// side by side: one word) or spread over the block; 4 (8) consecutive lanes share a block of 32 features.  What
// the call does not have is read from somewhere that exists and dropped: without branches between them all of a
// thread's loads are in flight at once.  The narrower side has more rows to a block, and none for the last ones:
// those return at once.
template <int ROWS, bool PAGED, int PIECE, bool SPREAD>
struct Share {
    static constexpr int kPieces = 32 / PIECE;  // of a block of 32 features
    int64_t b, h, first;  // first row of the block's
    int piece, r, per;    // the thread's piece and its place among the `per` threads of that
    int rows;             // of the call's (0: none left)
    int64_t entry[ROWS];  // where the thread's rows lie: entry of the cache's first dimension
    int row[ROWS];
    bool live[ROWS];      // the call has the row, and it has a place
    __device__ __forceinline__ Share(const RowsArgs &a, const Side &s) {
        // 32 bits: divisions in 64 would be most of a block's instructions
        const uint32_t pieces = kPieces * s.blocks, t = threadIdx.x;
        per = (int)(256 / pieces);
        r = (int)(t / pieces);
        piece = (int)(t % pieces);
        const uint32_t id = xcd_range(blockIdx.x, gridDim.x), bh = id / a.tiles;
        b = bh / a.heads;
        h = bh % a.heads;
        first = (int64_t)(id % a.tiles) * (ROWS * per);
        const int64_t left = a.n - first;
        rows = left <= 0 ? 0 : left < ROWS * per ? (int)left : ROWS * per;
        // starts so far out that none of the call's rows has a place count as -n: no sum passes 64 bits
        const int64_t from = a.starts ? a.starts[b] : 0, start = (from >= a.m || from < -a.n ? -a.n : from) + first;
        const int64_t counted = a.counts ? a.counts[b] : a.n;
        const int count = counted <= first ? 0 : counted - first < rows ? (int)(counted - first) : rows;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int64_t q = start + own(k);
            live[k] = r < per && own(k) < count && q >= 0 && q < a.m;
            row[k] = live[k] ? (int)q : 0;
            entry[k] = b;
        }
        if constexpr (PAGED) {
            if (a.m == 0) return;  // no table
            if (a.c.wide)
                look<int64_t>(a);
            else
                look<int32_t>(a);
        }
    }
    template <typename I>
    __device__ __forceinline__ void look(const RowsArgs &a) {
        const I *table = reinterpret_cast<const I *>(a.c.pages) + b * a.c.pitch;
        I page[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) page[k] = table[row[k] >> a.c.shift];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            live[k] = live[k] && page[k] >= 0 && (int64_t)page[k] < a.c.first;
            entry[k] = live[k] ? (int64_t)page[k] : 0;
            row[k] = live[k] ? row[k] & a.c.mask : 0;
        }
    }
    __device__ __forceinline__ uint8_t *codes(const Side &s, int k) const {
        return s.codes + entry[k] * s.cf + h * s.ch + (int64_t)row[k] * s.cr;
    }
    __device__ __forceinline__ uint8_t *scale(const Side &s, int k) const {
        return s.scales + entry[k] * s.sf + h * s.sh + piece / kPieces * s.sb + row[k];
    }
    // Row k of the thread's among the call's, and whether it is there.
    __device__ __forceinline__ int own(int k) const { return SPREAD ? k * per + r : r * ROWS + k; }
    __device__ __forceinline__ bool has(int k) const { return r < per && own(k) < rows; }
    // Ids go round-robin over the 8 XCDs: where they divide, each XCD gets a contiguous range, so that the
    // scales of neighbouring rows, a byte each, meet in one L2.
    static __device__ __forceinline__ uint32_t xcd_range(uint32_t id, uint32_t all) {
        return (all & 7) == 0 ? (id & 7) * (all >> 3) + (id >> 3) : id;
    }
};

// WHOLE: rows are whole pieces of 8 features at 16-byte aligned addresses.  Bound by memory: 2 x 4 x 16 x 8192 x
// 128 bf16 in 72 to 75 us back to back (4.6 TB/s read and written), behind a read of as much in 93.
template <typename T, int BITS, int ROWS, bool WHOLE, bool PAGED>
__global__ __launch_bounds__(256) void cache_write_kernel(const RowsArgs a) {
    const int side = blockIdx.y;
    const Side &s = side ? a.c.v : a.c.k;
    const Share<ROWS, PAGED, 8, false> p(a, s);
    if (p.rows == 0) return;
    const T *base = reinterpret_cast<const T *>(a.x[side]) + p.b * a.xb[side] + p.h * a.xh[side] + p.first * a.xn[side];
    const int f = 8 * p.piece, d = a.width[side];
    T raw[ROWS][8] = {};
    uint32_t bytes[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const T *row = base + (p.has(k) ? p.own(k) : 0) * a.xn[side];
        if constexpr (WHOLE) {
            __builtin_memcpy(raw[k], __builtin_assume_aligned(row + (f < d ? f : 0), 16), sizeof(raw[k]));
        } else if (d >= 8) {  // any alignment
            __builtin_memcpy(raw[k], row + (f + 8 <= d ? f : 0), sizeof(raw[k]));
        }
    }
    if (!WHOLE && f < d && f + 8 > d) {  // a row's last piece
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                raw[k][e] = base[(p.has(k) ? p.own(k) : 0) * a.xn[side] + (f + e < d ? f + e : d - 1)];
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        float x[8];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = (WHOLE ? f : f + e) < d ? to_f32(raw[k][e]) : 0.0f;
            const uint32_t m = __float_as_uint(x[e]) & 0x7fffffffu;
            top = m > top ? m : top;
        }
        const uint32_t byte = scale_byte<BITS>(over_block(top));
        const float scale = scale_of(byte);
        const bool finite = byte != 255;
        bytes[k] = byte;
        if (!p.live[k]) continue;  // the four lanes of a block alike
        if constexpr (BITS == 4) {
            reinterpret_cast<uint32_t *>(p.codes(s, k))[p.piece] = finite ? to_fp4(x, scale) : 0u;
        } else {
            const uint2 w = to_fp8(x, scale);
            reinterpret_cast<uint2 *>(p.codes(s, k))[p.piece] = finite ? w : make_uint2(0u, 0u);
        }
    }
    if (p.piece % 4 != 0) return;
    if constexpr (ROWS == 4) {  // four rows' scales of a block lie side by side: one store where they all go there
        if (p.live[0] && p.live[1] && p.live[2] && p.live[3] && p.row[0] % 4 == 0) {  // (pages: in one of them)
            *reinterpret_cast<uint32_t *>(p.scale(s, 0)) = bytes[0] | bytes[1] << 8 | bytes[2] << 16 | bytes[3] << 24;
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
        if (p.live[k]) *p.scale(s, k) = (uint8_t)bytes[k];
}

// What a thread reads of a row: 16 bytes out, so that a wave's stores cover whole lines.
constexpr int read_piece(size_t size) { return size == 4 ? 4 : 8; }
template <int BITS, int P>
struct Codes;
template <int BITS>
struct Codes<BITS, 8> {  // to bfloat16
    Eight<BITS> w;
    __device__ __forceinline__ void values(uint32_t byte, uint16_t (&out)[8]) const {
        const float scale = cache::scale_of(byte);
        if (__all(byte >= 32)) {  // exact
            const uint4 y = w.bf16(scale);
            __builtin_memcpy(out, &y, 16);
        } else {  // (below bfloat16's normal range: rounded)
            float x[8];
            w.f32(scale, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) from_f32(&out[e], x[e]);
        }
    }
};
template <int BITS>
struct Codes<BITS, 4> {  // to float32
    uint32_t w;
    __device__ __forceinline__ void values(uint32_t byte, float (&out)[4]) const {
        const float scale = cache::scale_of(byte);
        const f2 a = f32_pair<BITS, 0>(w, scale), b = f32_pair<BITS, 1>(w, scale);
        out[0] = a[0], out[1] = a[1], out[2] = b[0], out[3] = b[1];
    }
};

// Rows that are not the call's, or that lie nowhere, are zeros.  Bound by memory: 2 x 16 x 2 x 32768 x 128 bf16 in 122
// to 132 us (5 TB/s; one row a thread, with branches around its loads, took 205), 2 x 8 x 4 x 10240 x 128 fp32 in 73
// (5.2; 8 features a thread, a wave's store skipping every other 16 bytes: 106).  Rows that do not lie in 16-byte
// pieces are spread over the block, so that a store instruction's rows follow one another: 118 bf16 out of 8 bits 72 ->
// 56, 90 29 -> 26 (whole pieces: 33.6 -> 35.1); of fp32, 90 take 90 (3 TB/s): 16-byte stores at 8-byte addresses.
template <typename T, int BITS, int ROWS, bool WHOLE, bool PAGED>
__global__ __launch_bounds__(256) void cache_read_kernel(const RowsArgs a) {
    const int side = blockIdx.y;
    const Side &s = side ? a.c.v : a.c.k;
    constexpr int P = read_piece(sizeof(T));
    const Share<ROWS, PAGED, P, !WHOLE> p(a, s);
    T *base = reinterpret_cast<T *>(a.y[side]) + p.b * a.xb[side] + p.h * a.xh[side] + p.first * a.xn[side];
    const int f = P * p.piece, d = a.width[side];
    if (p.rows == 0 || f >= d || p.r >= p.per) return;
    Codes<BITS, P> w[ROWS] = {};
    uint32_t byte[ROWS] = {};
    if (a.m > 0 && a.c.first > 0) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            constexpr int kBytes = BITS * P / 8;
            __builtin_memcpy(&w[k], __builtin_assume_aligned(p.codes(s, k) + kBytes * p.piece, kBytes), kBytes);
            byte[k] = *p.scale(s, k);
        }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        T out[P];
        w[k].values(byte[k], out);
#pragma unroll
        for (int e = 0; e < P; ++e) out[e] = p.live[k] ? out[e] : T(0);
        if (!p.has(k)) continue;
        T *row = base + p.own(k) * a.xn[side] + f;
        if constexpr (WHOLE) {
            __builtin_memcpy(__builtin_assume_aligned(row, 16), out, sizeof(out));
        } else if (f + P <= d) {  // any alignment
            __builtin_memcpy(row, out, sizeof(out));
        } else {
#pragma unroll
            for (int e = 0; e < P; ++e)
                if (f + e < d) row[e] = out[e];
        }
    }
}

// Rows of a thread: several where every CU has a block all the same (4 x 4 x 1664 x 96 out of 8 bits: fp32 11.8 -> 6.9 us,
// bf16 7.3 -> 5.9, written 7.0 -> 5.6; 2 x 2 x 512 x 64, which have not: 3.1 where they would take 3.9).
constexpr int kManyRows = 4;
template <typename T, int BITS>
int launch(RowsArgs &a, bool write, int64_t batch, int64_t blocks, hipStream_t s) {
    const auto go = [&](auto rows, auto whole, auto paged) {
        constexpr int ROWS = decltype(rows)::value;
        constexpr bool WHOLE = decltype(whole)::value, PAGED = decltype(paged)::value;
        const int64_t piece = write ? 8 : read_piece(sizeof(T));
        const int64_t tiles = cdiv(a.n, ROWS * (256 / (32 / piece * blocks))), all = tiles * batch * a.heads;
        TPW_REQUIRE(all <= kMostBlocks, "cache: too many rows");
        a.tiles = (uint32_t)tiles;
        const dim3 grid((unsigned)all, 2);
        if (write) {
            hipLaunchKernelGGL((cache_write_kernel<T, BITS, ROWS, WHOLE, PAGED>), grid, dim3(256), 0, s, a);
            return check_launch("cache_write_kernel");
        }
        hipLaunchKernelGGL((cache_read_kernel<T, BITS, ROWS, WHOLE, PAGED>), grid, dim3(256), 0, s, a);
        return check_launch("cache_read_kernel");
    };
    const auto by_page = [&](auto rows, auto whole) {
        return a.c.pages ? go(rows, whole, std::true_type{}) : go(rows, whole, std::false_type{});
    };
    const auto by_row = [&](auto rows) {
        return a.whole[0] && a.whole[1] ? by_page(rows, std::true_type{}) : by_page(rows, std::false_type{});
    };
    const int64_t piece = write ? 8 : read_piece(sizeof(T));
    const int64_t all = cdiv(a.n, kManyRows * (256 / (32 / piece * blocks))) * batch * a.heads * 2;
    return all >= 256 ? by_row(std::integral_constant<int, kManyRows>{}) : by_row(std::integral_constant<int, 1>{});
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
    a.heads = (uint32_t)d->heads;
    a.n = n;
    a.m = d->pages ? d->page_count * d->rows : d->rows;
    if (write && (a.m == 0 || a.c.first == 0)) return TPW_OK;  // nowhere to go
    hipStream_t s = as_stream(stream);
    if (dtype == TPW_F32)
        return d->bits == 4 ? launch<float, 4>(a, write, batch, blocks, s) : launch<float, 8>(a, write, batch, blocks, s);
    return d->bits == 4 ? launch<uint16_t, 4>(a, write, batch, blocks, s) : launch<uint16_t, 8>(a, write, batch, blocks, s);
}

}  // namespace

int read_cache(const tpw_cache_desc *d, int64_t batch, Cache &c) {
    TPW_REQUIRE(d, "cache: null descriptor");
    TPW_REQUIRE(d->bits == 4 || d->bits == 8, "cache: 4 or 8 bits");
    TPW_REQUIRE(batch >= 0 && d->first >= 0 && d->heads >= 1 && d->rows >= 0, "cache: invalid sizes");
    TPW_REQUIRE(batch <= kMostBlocks && d->heads <= kMostBlocks && batch * d->heads <= kMostBlocks,
                "cache: too many sequences and heads");
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
    c.near = 1;
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
        c.near = c.near && s.cr <= (int64_t(1) << 23) && s.sb <= (int64_t(1) << 28);
        return s.cr >= 0 && s.sb >= 0 && aligned16(codes) && aligned16(scales) &&
               (s.cf | s.ch | s.cr | s.sf | s.sh | s.sb) % 16 == 0 && (m * d->first == 0 || (codes && scales));
    };
    TPW_REQUIRE(side(c.k, d->key_codes, d->key_scales, d->key_code_strides, d->key_scale_strides, d->key_blocks) &&
                    side(c.v, d->value_codes, d->value_scales, d->value_code_strides, d->value_scale_strides,
                         d->value_blocks),
                "cache: codes and scales must lie at 16-byte aligned addresses and strides, and those of rows and blocks "
                "must not be negative");
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
