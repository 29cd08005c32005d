// Attention over a cache in 4 or 8 bits: the two forms that cache_attention.hip chooses between.
#pragma once

#include <utility>

#include "attention.hpp"
#include "cache.hpp"

namespace tpw {
namespace attn {

// The form for few rows, up to kFewRows a key head (cache_rows.hpp).  4 bits, 128 features, 16 x 8 heads over 4096:
// 16 rows 22 us, 32 27 and, in tiles, 33 43; float32 25, 38 and 79.  (On short caches of few heads all are alike.)
constexpr int64_t kFewRows = 32;
constexpr int64_t kPackedRows = 4;  // of float32 whose summands share a product
// float32 rows of more than 128 features have no registers for a second 16: a block takes 16, and up to this many are
// done so, each 16 reading the keys again (256 features of 4 bits, 16 x 8 heads over 4096: 32 rows 68 us, 64 in two
// rounds 132; in tiles, which take up to 128 rows, 213).
constexpr int64_t kGroupedRows = 64;
constexpr bool in_groups(int nb, int np, bool pack) { return nb == 8 && np > 1 && !pack; }
constexpr int kRowWaves = 4;        // waves of a block that does one of several parts
constexpr int kWholeWaves = 8;      // .. that works alone on a sequence and head
// Blocks that share a CU, as their registers leave (NP: summands of a query, RT: 16 rows each).  Four of 64
// features would fit, and were slower where they fill the card (1664 keys of 16 x 8 heads 10.8 -> 11.8 us, with one
// summand of a probability; three with two of them: 11.4).
constexpr int rows_per_cu(int bits, int nb, int np, int rt) {
    if (np > 1 || rt > 1) return nb == 8 || (np > 1 && rt > 1) ? 1 : 2;
    return nb == 8 ? (bits == 4 ? 2 : 1) : bits == 4 ? 3 : 2;
}
// Up to 16 rows of bfloat16, 4 of float32, may be worked on by kWholeWaves (cache_attention.hip).
constexpr bool may_be_whole(int bits, int nb, int np, int rt) {
    return np == 1 && rt == 1 && rows_per_cu(bits, nb, np, rt) > 1;
}
// 64, 128 or 256 features.
constexpr int row_blocks(int most) { return most <= 2 ? 2 : most <= 4 ? 4 : 8; }
int cache_rows4(const Args &a, const cache::Cache &c, int dtype, int mode, hipStream_t s);
int cache_rows8(const Args &a, const cache::Cache &c, int dtype, int mode, hipStream_t s);

// The form for many rows (cache_tiles.hpp): waves that its registers leave a SIMD (blocks of four waves a CU).
constexpr int tiles_per_simd(int size, int dp) { return size == 4 && dp > 128 ? 1 : 2; }
int cache_tiles4(const Args &a, const cache::Cache &c, int dtype, int mode, hipStream_t s);
int cache_tiles8(const Args &a, const cache::Cache &c, int dtype, int mode, hipStream_t s);

}  // namespace attn
}  // namespace tpw
