// The attention kernels for bf16.
#define TC_ATTENTION_TYPE ::tc::bf16_t
#include "attention.hpp"

namespace tc {
namespace attention {

const Launches& bf16_launches() {
    static const Launches launches = {forward, backward};
    return launches;
}

}  // namespace attention
}  // namespace tc
