// Shared-prefix attention, head dim 96.
#include "da_prefix_kernel.h"

namespace da {
hipError_t launch_prefix_d96(const PrefixParams& p, bool is_bf16, bool wave_per_head, int own_wgs, hipStream_t stream) {
    return prefix::launch_dim<96>(p, is_bf16, wave_per_head, own_wgs, stream);
}
}  // namespace da
