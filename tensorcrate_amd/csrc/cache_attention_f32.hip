// The kernels of attention over a cache for f32.
#define TC_ATTENTION_TYPE float
#include "cache_attention.hpp"

namespace tc {
namespace cache {

const AttentionLaunches& attend_f32() {
    static const AttentionLaunches launches = {attend, join};
    return launches;
}

}  // namespace cache
}  // namespace tc
