// attention_f32.hip — the paged attention kernels of f32 caches.
#include "paged_attention.hpp"

namespace fmx {

int attention_f32(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s) {
    return launch_dim<float, 1>(A, scratch, type, s);
}

} // namespace fmx
