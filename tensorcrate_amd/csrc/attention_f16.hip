// The attention kernels for f16.
#define TC_ATTENTION_TYPE _Float16
#include "attention.hpp"

namespace tc {
namespace attention {

const Launches& f16_launches() {
    static const Launches launches = {forward, backward};
    return launches;
}

}  // namespace attention
}  // namespace tc
