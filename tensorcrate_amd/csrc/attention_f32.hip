// The attention kernels for f32.
#define TC_ATTENTION_TYPE float
#include "attention.hpp"

namespace tc {
namespace attention {

const Launches& f32_launches() {
    static const Launches launches = {forward, backward};
    return launches;
}

}  // namespace attention
}  // namespace tc
