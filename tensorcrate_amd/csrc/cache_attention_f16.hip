// The kernels of attention over a cache for f16.
#define TC_ATTENTION_TYPE _Float16
#include "cache_attention.hpp"

namespace tc {
namespace cache {

const AttentionLaunches& attend_f16() {
    static const AttentionLaunches launches = {attend, join};
    return launches;
}

}  // namespace cache
}  // namespace tc
