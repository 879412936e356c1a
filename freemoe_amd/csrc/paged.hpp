// paged.hpp — a ragged batch over a paged cache: the descriptors as kernels
// take them, and how a workgroup finds its sequence and a position its row.
#pragma once

#include "fmx_internal.hpp"

namespace fmx {

// n / d for n < 2^31 by a multiplication: with s = ceil(log2 d) and m =
// floor(2^32 (2^s - d) / d) + 1, the quotient is (mulhi(m, n) + n) >> s
// (the sum stays below 2^32).
struct FastDiv {
    uint32_t d = 1, m = 1, s = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div) {
        while ((uint64_t{1} << s) < div) ++s;
        m = static_cast<uint32_t>((uint64_t{1} << 32) * ((uint64_t{1} << s) - div) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct PagedArgs {
    const uint8_t *k, *v;
    uint64_t page_bytes, position_bytes, head_bytes;
    uint32_t kv_heads, head_dim, pages;
    FastDiv page;
    uint32_t sequences, tokens, max_new, table_stride, max_length;
    const uint32_t *starts, *lengths, *table;
};

// A launch takes fewer than 2^32 threads in a dimension.
constexpr bool launch_fits(uint64_t workgroups, uint32_t threads) { return workgroups <= 0xffffffffu / threads; }
constexpr uint32_t kRopeThreads = 256;
constexpr uint32_t kSampleThreads = 512; // of a workgroup, where rows are many

inline uint32_t element_bytes(uint32_t type) {
    return type == FMX_TYPE_F32 ? 4 : type == FMX_TYPE_F16 || type == FMX_TYPE_BF16 ? 2 : 0;
}

// Checks both descriptors and fills `a`; FMX_OK with a->tokens == 0 for an
// empty batch.
int prepare_paged(const fmx_paged_cache *cache, const fmx_paged_batch *batch, PagedArgs *a);

// A sequence of the batch as its arrays name it, its bounds checked.
struct Sequence {
    uint32_t start, count, length; // rows, positions
    bool bad;
};

__device__ __forceinline__ Sequence sequence_at(const PagedArgs &a, uint32_t i) {
    Sequence q;
    const uint32_t s0 = a.starts[i], s1 = a.starts[i + 1], len = a.lengths[i];
    q.bad = s1 < s0 || s1 > a.tokens || s1 - s0 > a.max_new || len > a.max_length;
    q.start = s0;
    q.count = q.bad ? 0 : s1 - s0;
    q.length = q.bad ? 0 : len;
    return q;
}

// Position t's byte offset in the pools, kv head 0; `bad` where its page is
// not in the pool (the offset is then page 0's, so a read stays inside).
__device__ __forceinline__ uint64_t position_offset(const PagedArgs &a, uint32_t page, uint32_t place, bool &bad) {
    const bool off = page >= a.pages;
    bad |= off;
    return static_cast<uint64_t>(off ? 0 : page) * a.page_bytes + static_cast<uint64_t>(place) * a.position_bytes;
}

// Inclusive sums over the wavefront by DPP moves: within rows of 16 lanes, then
// each row's last sum into the rows behind it.
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
    int x = static_cast<int>(v);
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false); // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false); // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false); // row_bcast:31 into rows 2 and 3
    return static_cast<uint32_t>(x);
}

// Item `target` of the batch where sequence i holds per(sequence) items: the
// sequence and the item's number in it. Every lane of the wavefront calls it
// and gets the same answer; false past the last item. Sixty-four sequences at
// a time, one per lane. `bad`: a sequence passed on the way broke a bound.
template <class Per>
__device__ __forceinline__ bool find_item(const PagedArgs &a, uint32_t target, const Per &per, uint32_t &index,
                                          Sequence &q, uint32_t &item, bool &bad) {
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t b = 0; b < a.sequences; b += 64) {
        const uint32_t i = b + lane;
        Sequence mine{0, 0, 0, false};
        if (i < a.sequences) mine = sequence_at(a, i);
        bad |= __any(mine.bad);
        const uint32_t n = per(mine);
        const uint32_t incl = wave_scan_u32(n);
        const uint64_t hit = __ballot(incl > target);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            index = b + at;
            q.start = __builtin_amdgcn_readlane(mine.start, at);
            q.count = __builtin_amdgcn_readlane(mine.count, at);
            q.length = __builtin_amdgcn_readlane(mine.length, at);
            q.bad = false;
            item = target - __builtin_amdgcn_readlane(incl - n, at);
            return true;
        }
        target -= __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// Whether any sequence breaks a bound: for one workgroup of a call, since those
// behind the last item a wavefront looks for are not passed on its way.
__device__ __forceinline__ bool any_bad_sequence(const PagedArgs &a) {
    bool bad = false;
    for (uint32_t i = threadIdx.x & 63; i < a.sequences; i += 64) bad |= sequence_at(a, i).bad;
    return __any(bad);
}

// rope.hip, paged_attention.hip, sample.hip: the entry points after their
// pointer checks.
struct RopeCall {
    uint32_t heads, in_type;
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    void *q_out;
    uint64_t q_out_stride;
    uint32_t *status;
};
int rope_append(const PagedArgs &a, uint32_t type, const fmx_rope &rope, const RopeCall &c, hipStream_t s);

struct AttentionCall {
    uint32_t heads, out_type;
    const void *q;
    uint64_t q_stride;
    void *out;
    uint64_t out_stride;
    fmx_attention_options options;
    uint32_t *status;
    uint8_t *scratch;
};
uint64_t attention_paged_scratch(const PagedArgs &a, uint32_t type, uint32_t heads);
int attention_paged(const PagedArgs &a, uint32_t type, const AttentionCall &c, hipStream_t s);

constexpr uint32_t kSampleMaxVocab = 262144;
uint64_t sample_scratch(uint32_t rows, uint32_t vocab);
int sample(const float *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const fmx_sampling &p,
           const float *uniform, uint32_t *ids, float *probs, uint32_t *status, uint8_t *scratch, hipStream_t s);

} // namespace fmx
