// The kernels of cache_tiles.hpp for 8 bits.
#include "cache_tiles.hpp"

namespace tpw {
namespace attn {

int cache_tiles8(const Args &a, const Cache &c, int dtype, int mode, hipStream_t s) {
    return launch_tiles<8>(a, c, dtype, mode, s);
}

}  // namespace attn
}  // namespace tpw
