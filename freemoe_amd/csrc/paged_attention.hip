// paged_attention.hip — fmx_attention_paged: the call's plan and its type's
// kernels (paged_attention.hpp, one source file per type to compile them side
// by side).
#include "paged_attention.hpp"

namespace fmx {

uint64_t attention_paged_scratch(const PagedArgs &a, uint32_t type, uint32_t heads) {
    const Plan p = plan_of(a, type, heads / a.kv_heads, kUnbounded); // (a window only lessens the splits)
    return p.splits > 1 ? scratch_of(p.tiles, a.kv_heads, p.splits, p.tile_rows, a.head_dim).total : 0;
}

int attention_paged(const PagedArgs &a, uint32_t type, const AttentionCall &c, hipStream_t s) {
    AttentionArgs A;
    A.a = a;
    A.q = static_cast<const uint8_t *>(c.q);
    A.out = static_cast<uint8_t *>(c.out);
    A.q_bytes = c.q_stride * element_bytes(type);
    A.out_bytes = c.out_stride * element_bytes(c.out_type);
    A.heads = c.heads;
    A.group = FastDiv(c.heads / a.kv_heads);
    constexpr double kLog2e = 1.4426950408889634;
    const double cap = c.options.softcap;
    A.negate = c.options.scale < 0.0;
    const double scale = A.negate ? -c.options.scale : c.options.scale;
    A.scale = static_cast<float>(cap != 0.0 ? scale / cap : 0.0);
    A.softcap = static_cast<float>(cap);
    A.per_score = static_cast<float>(cap != 0.0 ? kLog2e : scale * kLog2e);
    if (A.per_score == 0.0f) { // a scale of 0: all scores alike (0 times a hidden one's -inf would be NaN)
        A.softcap = 1.0f;
        A.per_score = static_cast<float>(kLog2e);
    }
    A.window = c.options.window == 0 || c.options.window > 0x7fffffffu ? kUnbounded : c.options.window;
    A.sinks = c.options.sinks;
    A.out_type = c.out_type;
    A.status = c.status;
    A.splits = 1;
    A.parts = nullptr;
    A.stats = nullptr;
    if (type == FMX_TYPE_F32) return attention_f32(A, c.scratch, type, s);
    if (type == FMX_TYPE_F16) return attention_f16(A, c.scratch, type, s);
    return attention_bf16(A, c.scratch, type, s);
}

} // namespace fmx
