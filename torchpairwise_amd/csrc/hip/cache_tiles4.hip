// The kernels of cache_tiles.hpp for 4 bits.
#include "cache_tiles.hpp"

namespace tpw {
namespace attn {

int cache_tiles4(const Args &a, const Cache &c, int dtype, int mode, hipStream_t s) {
    return launch_tiles<4>(a, c, dtype, mode, s);
}

}  // namespace attn
}  // namespace tpw
