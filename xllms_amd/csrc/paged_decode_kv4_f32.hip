// Instantiations of the 4-bit cache's decode attention for f32 Q and O.
#include "paged_decode_kv4.h"

namespace xhip {

int kv4_occupancy_f32(int head_size, int head_tile, int group, size_t lds_bytes) {
    return kv4_occupancy_dtype<KV_F32>(head_size, head_tile, group, lds_bytes);
}

hipError_t launch_kv4_f32(const DecodeParams &p, int head_size, int head_tile, hipStream_t stream,
                         hipEvent_t ev_start, hipEvent_t ev_stop) {
    return launch_kv4_dtype<KV_F32>(p, head_size, head_tile, stream, ev_start, ev_stop);
}

}  // namespace xhip
