// attention_bf16.hip — the paged attention kernels of bf16 caches.
#include "paged_attention.hpp"

namespace fmx {

int attention_bf16(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s) {
    return launch_type<__bf16>(A, scratch, type, s);
}

} // namespace fmx
