// Instantiations of the 4-bit cache's decode attention for f32 Q and O.
#include "paged_decode_kv4.h"
#include "paged_decode_launch.h"

namespace xhip {

hipError_t launch_kv4_f32(const DecodeParams &p, int head_size, hipStream_t stream) {
    return launch_kv4_dtype<KV_F32>(p, head_size, stream);
}

}  // namespace xhip
