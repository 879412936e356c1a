// rope.hip — rotary positions and the write of new keys and values into a
// paged cache (the place of FreeMoe's src/rope.cpp and of the cache rows
// engine.cpp:1075-1460 writes, for a ragged batch).
//
// Pair (x, y) of a head at position p becomes (x cos t - y sin t, x sin t +
// y cos t) with t = p * inv_freq[c]: formed in double, since p * inv_freq
// reaches 10^5 radians and more, where a float's last place is 2^-7; its
// cosine and sine are rounded to float once. A token's dims / 2 angles serve
// all of its heads, so a workgroup takes one token (or a part of one, where
// tokens are few), forms them once into LDS, and streams the heads: 16
// elements per thread and step, each row read once and written once.
//
// Memory-bound: 4096 tokens of 32 + 8 heads of 128, f32 to bf16, take 24 us at
// 6.3 TB/s of reads and writes together when called back to back, 31 us (4.9
// TB/s) out of cold caches, where a copy of 1 GiB reaches 5.1 TB/s; one token is
// a launch, 6 us.
#include "paged.hpp"

namespace fmx {

namespace {

constexpr uint32_t kThreads = kRopeThreads;
constexpr uint32_t kMaxPairs = 128;

struct RopeArgs {
    const uint8_t *q, *k, *v;
    uint64_t q_bytes, k_bytes, v_bytes, out_bytes; // row strides
    uint8_t *q_out;
    const double *inv_freq;
    const int32_t *positions;
    double magnitude;
    uint32_t heads, dims, half; // half: pairs (c, c + dims / 2)
    uint32_t units;             // of a q or k head
    FastDiv per_head, per_value;
    uint32_t *status;
};

template <typename T> struct Eight; // 8 elements, 16-byte aligned
template <> struct Eight<float> {
    static __device__ __forceinline__ void load(const void *p, float *x) {
        const uint4 a = ld16(p), b = ld16(static_cast<const uint8_t *>(p) + 16);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(float, w[i]);
    }
    static __device__ __forceinline__ void store(void *p, const float *x) {
        float4 *o = static_cast<float4 *>(p);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
};
template <typename T> struct Eight {
    typedef T vec __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ void load(const void *p, float *x) {
        const vec v = __builtin_bit_cast(vec, ld16(p));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
    }
    static __device__ __forceinline__ void store(void *p, const float *x) {
        vec v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[i]);
        *static_cast<uint4 *>(p) = __builtin_bit_cast(uint4, v);
    }
};

// grid: rows x parts of a row. kVector: dims is a multiple of 16, a unit of a q
// or k head is 8 pairs or, behind dims, 8 elements to copy; otherwise one pair
// or one element (the reads of a pair and its writes stay in one thread, so
// that q_out may be q).
template <typename TI, typename TO, bool kVector>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(PagedArgs a, RopeArgs r) {
    __shared__ float2 turn[kMaxPairs];
    const uint32_t tid = threadIdx.x;
    uint32_t index, item;
    Sequence seq;
    bool bad = false;
    const bool found =
        find_item(a, blockIdx.x, [](const Sequence &s) { return s.count; }, index, seq, item, bad);
    if (blockIdx.x == 0 && blockIdx.y == 0 && a.sequences > 64) bad |= any_bad_sequence(a);
    uint64_t at = 0;
    uint32_t row = 0;
    bool skip = !found;
    if (found) {
        row = seq.start + item;
        skip = seq.count - item > seq.length; // a position before the first
        bad |= skip;
        if (!skip) {
            const uint32_t position = seq.length - seq.count + item;
            const uint32_t page = a.page.div(position);
            at = position_offset(a, a.table[static_cast<uint64_t>(index) * a.table_stride + page],
                                 position - page * a.page.d, skip);
            bad |= skip;
            const int32_t turned = r.positions ? r.positions[row] : static_cast<int32_t>(position);
            if (tid < r.dims / 2) {
                double s, c;
                sincos(static_cast<double>(turned) * r.inv_freq[tid], &s, &c);
                turn[tid] = make_float2(static_cast<float>(c * r.magnitude), static_cast<float>(s * r.magnitude));
            }
        }
    }
    if (bad && tid == 0) atomicOr(r.status, STATUS_BAD_PAGE);
    if (skip) return; // the whole workgroup
    __syncthreads();
    const uint32_t H = r.heads, G = a.kv_heads, D = a.head_dim, R = r.dims, pairs = R / 2;
    const uint8_t *q = r.q + row * r.q_bytes, *k = r.k + row * r.k_bytes, *v = r.v + row * r.v_bytes;
    uint8_t *q_out = r.q_out + row * r.out_bytes;
    uint8_t *kc = const_cast<uint8_t *>(a.k) + at, *vc = const_cast<uint8_t *>(a.v) + at;
    const uint32_t turning = (H + G) * r.units, total = turning + G * (D / 8);
    for (uint32_t u = blockIdx.y * kThreads + tid; u < total; u += gridDim.y * kThreads) {
        if (u >= turning) { // values
            const uint32_t w = u - turning, head = r.per_value.div(w), d = (w - head * (D / 8)) * 8;
            float x[8];
            Eight<TI>::load(v + (static_cast<uint64_t>(head) * D + d) * sizeof(TI), x);
            Eight<TO>::store(vc + head * a.head_bytes + d * sizeof(TO), x);
            continue;
        }
        const uint32_t head = r.per_head.div(u), w = u - head * r.units;
        const uint8_t *from = (head < H ? q + static_cast<uint64_t>(head) * D * sizeof(TI)
                                        : k + static_cast<uint64_t>(head - H) * D * sizeof(TI));
        uint8_t *to = head < H ? q_out + static_cast<uint64_t>(head) * D * sizeof(TO) : kc + (head - H) * a.head_bytes;
        if constexpr (kVector) {
            if (w >= R / 16) {
                const uint32_t d = R + (w - R / 16) * 8;
                float x[8];
                Eight<TI>::load(from + d * sizeof(TI), x);
                Eight<TO>::store(to + d * sizeof(TO), x);
                continue;
            }
            const uint32_t d0 = r.half ? w * 8 : w * 16, d1 = d0 + (r.half ? pairs : 8);
            float x[16], y[16];
            Eight<TI>::load(from + d0 * sizeof(TI), x);
            Eight<TI>::load(from + d1 * sizeof(TI), x + 8);
            if (r.half) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 t = turn[w * 8 + i];
                    y[i] = x[i] * t.x - x[8 + i] * t.y;
                    y[8 + i] = x[i] * t.y + x[8 + i] * t.x;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 t = turn[w * 8 + i];
                    y[2 * i] = x[2 * i] * t.x - x[2 * i + 1] * t.y;
                    y[2 * i + 1] = x[2 * i] * t.y + x[2 * i + 1] * t.x;
                }
            }
            Eight<TO>::store(to + d0 * sizeof(TO), y);
            Eight<TO>::store(to + d1 * sizeof(TO), y + 8);
        } else {
            const TI *f = reinterpret_cast<const TI *>(from);
            TO *o = reinterpret_cast<TO *>(to);
            if (w >= pairs) {
                const uint32_t d = R + w - pairs;
                o[d] = static_cast<TO>(static_cast<float>(f[d]));
                continue;
            }
            const uint32_t d0 = r.half ? w : 2 * w, d1 = r.half ? w + pairs : 2 * w + 1;
            const float x = static_cast<float>(f[d0]), y = static_cast<float>(f[d1]);
            const float2 t = turn[w];
            o[d0] = static_cast<TO>(x * t.x - y * t.y);
            o[d1] = static_cast<TO>(x * t.y + y * t.x);
        }
    }
}

template <typename TI, typename TO>
int launch(const PagedArgs &a, const RopeArgs &r, hipStream_t s) {
    const uint32_t total = (r.heads + a.kv_heads) * r.units + a.kv_heads * (a.head_dim / 8);
    // one workgroup per token; where that leaves CUs idle, up to one per 256
    // units of a token
    const uint32_t most = div_up(total, kThreads), want = div_up(512, a.tokens);
    const dim3 grid(a.tokens, want < most ? want : most);
    if (r.dims % 16 == 0)
        hipLaunchKernelGGL((rope_append_kernel<TI, TO, true>), grid, dim3(kThreads), 0, s, a, r);
    else
        hipLaunchKernelGGL((rope_append_kernel<TI, TO, false>), grid, dim3(kThreads), 0, s, a, r);
    FMX_LAUNCH_CHECK();
    return FMX_OK;
}

} // namespace

int rope_append(const PagedArgs &a, uint32_t type, const fmx_rope &rope, const RopeCall &c, hipStream_t s) {
    RopeArgs r;
    const uint32_t in = element_bytes(c.in_type), out = element_bytes(type), D = a.head_dim;
    r.q = static_cast<const uint8_t *>(c.q);
    r.k = static_cast<const uint8_t *>(c.k);
    r.v = static_cast<const uint8_t *>(c.v);
    r.q_bytes = c.q_stride * in;
    r.k_bytes = c.k_stride * in;
    r.v_bytes = c.v_stride * in;
    r.out_bytes = c.q_out_stride * out;
    r.q_out = static_cast<uint8_t *>(c.q_out);
    r.inv_freq = rope.inv_freq;
    r.positions = rope.positions;
    r.magnitude = rope.magnitude;
    r.heads = c.heads;
    r.dims = rope.dims;
    r.half = rope.layout == FMX_ROPE_HALF;
    r.units = rope.dims % 16 == 0 ? rope.dims / 16 + (D - rope.dims) / 8 : rope.dims / 2 + (D - rope.dims);
    r.per_head = FastDiv(r.units);
    r.per_value = FastDiv(D / 8);
    r.status = c.status;
    if (type == FMX_TYPE_F32) return launch<float, float>(a, r, s);
    if (type == FMX_TYPE_F16)
        return c.in_type == FMX_TYPE_F32 ? launch<float, _Float16>(a, r, s) : launch<_Float16, _Float16>(a, r, s);
    return c.in_type == FMX_TYPE_F32 ? launch<float, __bf16>(a, r, s) : launch<__bf16, __bf16>(a, r, s);
}

} // namespace fmx
