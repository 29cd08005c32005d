// Attention over a cache in 4 or 8 bits: the two forms that cache_attention.hip chooses between.
#pragma once

#include <utility>

#include "attention.hpp"
#include "cache.hpp"

namespace tpw {
namespace attn {

// Rows of a key head up to which the form for few rows is taken (cache_rows.hip).
constexpr int64_t kFewRows = 32;
void plan_rows(Args &a);
int cache_rows(const Args &a, const cache::Cache &c, int bits, int dtype, bool bias, hipStream_t s);

// The form for many rows (cache_tiles4.hip, cache_tiles8.hip).
void plan_tiles(Args &a, int dtype);
int cache_tiles4(const Args &a, const cache::Cache &c, int dtype, int mode, hipStream_t s);
int cache_tiles8(const Args &a, const cache::Cache &c, int dtype, int mode, hipStream_t s);

}  // namespace attn
}  // namespace tpw
