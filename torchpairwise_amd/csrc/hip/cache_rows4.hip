// The kernels of cache_rows.hpp for 4 bits.
#include "cache_rows.hpp"

namespace tpw {
namespace attn {

int cache_rows4(const Args &a, const Cache &c, int dtype, int mode, hipStream_t s) {
    return rows_by_type<4>(a, c, dtype, mode, s);
}

}  // namespace attn
}  // namespace tpw
