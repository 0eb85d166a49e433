// The kernels of attention over a cache for bf16.
#define TC_ATTENTION_TYPE ::tc::bf16_t
#include "cache_attention.hpp"

namespace tc {
namespace cache {

const AttentionLaunches& attend_bf16() {
    static const AttentionLaunches launches = {attend, join};
    return launches;
}

}  // namespace cache
}  // namespace tc
