// Attention over a cache in 4 or 8 bits: entry points and the choice of the form.
#include "attention_forward.hpp"
#include "cache_attention.hpp"

namespace tpw {
namespace attn {
namespace {

// Reads both descriptors.  The arguments' keys and values have no address: the cache has them.
int read_call(const tpw_attention_desc *d, const tpw_cache_desc *cd, tpw_attention_desc &own, Args &a, cache::Cache &c) {
    TPW_REQUIRE(d && cd, "null descriptor");
    own = *d;
    TPW_REQUIRE(!d->stats && !d->out_rest, "attention over a cache has no backward: stats and out_rest must be null");
    own.key = own.value = nullptr;
    const int64_t none[3] = {0, 0, 256};
    for (int i = 0; i < 3; ++i) own.key_strides[i] = own.value_strides[i] = none[i];
    if (const int rc = read_args(&own, false, a)) return rc;
    if (const int rc = cache::read_cache(cd, d->batch, c)) return rc;
    TPW_REQUIRE(d->key_heads == cd->heads, "attention: key_heads differ from the cache's heads");
    TPW_REQUIRE(d->m == (cd->pages ? cd->page_count * cd->rows : cd->rows), "attention: m differs from the cache's rows");
    TPW_REQUIRE(d->d <= 32 * cd->key_blocks && d->dv <= 32 * cd->value_blocks, "attention: rows are wider than the cache's");
    // blocks behind the call's features are not read: a NaN of theirs would spoil the scores
    c.k.blocks = (int)cdiv(d->d, 32);
    c.v.blocks = (int)cdiv(d->dv, 32);
    a.cached = 1;
    a.dwords = 0;
    const int64_t size = d->dtype == TPW_F32 ? 4 : 2;
    a.whole_q = a.d % 8 == 0 && aligned16(a.q.p) && (a.q.b | a.q.h | a.q.n) * size % 16 == 0;
    if (cd->first == 0) a.m = own.m = 0;  // a table without pages: no keys, and no mask over them
    return TPW_OK;
}

bool wide_f32(const Args &a, int dtype) { return dtype == TPW_F32 && (a.d > 128 || a.dv > 128); }

// The form for few rows reads a mask's keys side by side, and reaches its 32 rows and their scales by 32-bit offsets (the
// form for many addresses each row by itself, in 64 bits).
bool few_rows(const Args &a, const cache::Cache &c, int dtype, int mode) {
    return c.near && a.n * a.group <= (wide_f32(a, dtype) ? kGroupedRows : kFewRows) && (mode == kNoMask || a.mm == 1);
}

size_t parts_bytes(const Args &a) {
    return a.splits > 1 ? (size_t)a.splits * a.batch * a.heads * a.n * (quads4(a.dv) + 2) * 4 : 0;
}

// As many parts as fill the card's places once: a block's own time (queries, first loads, joining: 5 to 7 us) is that
// of many chunks of 32 keys, so a second round costs more than long parts do.  Short caches are left whole, by blocks
// of twice the waves, where a SIMD's chunks in turn are no more than those of a part and two: what the second launch
// and the parts' way through memory take (4 bits, 128 features, 16 x 8 heads: 256 keys 7.2 -> 5.7 us, 512 8.5 -> 7.4,
// 1024 11.6 -> 9.6, where 1664 stay at 13; one sequence: 256 keys 7.0 -> 5.6; both with one summand of a probability,
// with two the whole ones take 5.8, 7.6, 10.1 and 5.6).
void plan_rows(Args &a, const cache::Cache &c, int bits, int dtype) {
    const int nb = row_blocks(c.k.blocks > c.v.blocks ? c.k.blocks : c.v.blocks);
    const int64_t rows = a.n * a.group;
    const int np = dtype == TPW_F32 && rows > kPackedRows ? 3 : 1, rt = rows <= 16 || (nb == 8 && np > 1) ? 1 : 2;
    const int64_t per_cu = rows_per_cu(bits, nb, np, rt);
    a.tiles = in_groups(nb, np, false) ? cdiv(rows, 16) : 1;
    const int64_t bk = a.batch * a.key_heads * a.tiles, chunks = cdiv(a.m, 32), most = cdiv(chunks, kRowWaves);
    int64_t splits = bk > 0 ? 256 * per_cu / bk : 1;
    splits = splits > most ? most : splits;
    splits = splits > kMaxParts ? kMaxParts : splits;
    const int64_t shared = cdiv(bk * splits, 256);  // parts that share a CU, a wave of each on a SIMD
    a.whole_rows = splits > 1 && may_be_whole(bits, nb, np, rt) &&
                   kWholeWaves / 4 * cdiv(chunks, kWholeWaves) <= shared * cdiv(chunks, kRowWaves * splits) + 2;
    a.splits = a.whole_rows || splits < 1 ? 1 : (int)splits;
}

void plan_tiles(Args &a, int dtype) {
    by_width<uint16_t>(a, kNoMask, [&](auto t, auto dp, auto) {
        using T = decltype(t);
        constexpr int DP = decltype(dp)::value;
        if (dtype == TPW_BF16)
            plan<T, DP>(a);
        else
            plan<T, DP>(a, tiles_per_simd(4, DP), 6);
        return TPW_OK;
    });
}

}  // namespace
}  // namespace attn
}  // namespace tpw

using namespace tpw;
using namespace tpw::attn;

extern "C" size_t tpw_cache_attention_workspace_size(const tpw_attention_desc *d, const tpw_cache_desc *cd) {
    Args a = {};
    cache::Cache c = {};
    tpw_attention_desc own;
    if (read_call(d, cd, own, a, c) != TPW_OK || a.batch * a.heads * a.n == 0) return 0;
    if (few_rows(a, c, d->dtype, mask_mode(&own))) {
        plan_rows(a, c, cd->bits, d->dtype);
        return parts_bytes(a);
    }
    plan_tiles(a, d->dtype);
    return prepared_bytes(a, &own, false) + parts_bytes(a);
}

extern "C" int tpw_cache_attention(const tpw_attention_desc *d, const tpw_cache_desc *cd, void *workspace,
                                   void *stream) {
    Args a = {};
    cache::Cache c = {};
    tpw_attention_desc own;
    if (const int rc = read_call(d, cd, own, a, c)) return rc;
    if (a.batch * a.heads * a.n == 0) return TPW_OK;
    TPW_REQUIRE(a.q.p && a.o.p, "attention: null operand");
    const int mode = mask_mode(&own);
    TPW_REQUIRE(mode == kNoMask || a.mask, "attention: null mask");
    hipStream_t s = as_stream(stream);
    size_t prepared = 0;
    const bool few = few_rows(a, c, d->dtype, mode);
    if (few) {
        if (mode == kNoMask) a.mask = nullptr;
        plan_rows(a, c, cd->bits, d->dtype);
    } else {
        plan_tiles(a, d->dtype);
        prepared = prepared_bytes(a, &own, false);
    }
    TPW_REQUIRE(prepared + parts_bytes(a) == 0 || (workspace && aligned16(workspace)),
                "attention: null or unaligned workspace");
    if (prepared)
        if (const int rc = prepare_operands(a, &own, false, workspace, s)) return rc;
    if (a.splits > 1) {
        a.part = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + prepared);
        a.part_stats = a.part + a.splits * a.batch * a.heads * a.n * quads4(a.dv);
    }
    const int rc = few ? (cd->bits == 4 ? cache_rows4 : cache_rows8)(a, c, d->dtype, mode, s)
                       : (cd->bits == 4 ? cache_tiles4 : cache_tiles8)(a, c, d->dtype, mode, s);
    if (rc || a.splits == 1) return rc;
    return join_parts(a, d->dtype, mode == kBias, s);
}
