// attention_f16.hip — the paged attention kernels of f16 caches.
#include "paged_attention.hpp"

namespace fmx {

int attention_f16(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s) {
    return launch_type<_Float16>(A, scratch, type, s);
}

} // namespace fmx
