// paged_attention.hpp — attention of a batch's new tokens over the pages their
// sequences hold.
//
// Query head h of the token at position p, over the visible positions j of its
// sequence (j <= p, and p - j < window where there is one):
//   s_j = scale q . k_j  (softcap c: c tanh(s_j / c)),
//   out = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink_h - m)),
// in one pass over j with the running maximum m and sum: where a later tile
// raises m, what was summed is multiplied by e^(m_old - m_new). Scores are kept
// in units of log 2 (scale times log2 e), so that e^x is one v_exp_f32.
//
// The query heads of one kv head read the same keys: a sequence's new tokens
// times those heads are the rows of one small matrix, row r being token r /
// group and head r % group.
#pragma once

#include "paged.hpp"

#include <algorithm>

namespace fmx {

struct AttentionArgs {
    PagedArgs a;
    const uint8_t *q;
    uint8_t *out;
    uint64_t q_bytes, out_bytes; // row strides
    uint32_t heads;
    FastDiv group;               // query heads of a kv head
    float scale, softcap;        // scale / softcap and softcap, or 0
    float per_score;             // log 2 units of a score, never negative: q's sign is turned instead
    bool negate;
    uint32_t window;             // or kUnbounded
    const float *sinks;
    uint32_t out_type;
    uint32_t *status;
    // splits > 1: a tile's keys go to that many workgroups at most, whose sums
    // meet in `parts` and `stats` (below)
    uint32_t splits;
    float *parts;  // [tile][kv head][split][row][head_dim]
    float2 *stats; // [tile][kv head][split][row]: maximum, sum
};

int attention_f32(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s);
int attention_f16(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s);
int attention_bf16(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
constexpr uint32_t kUnbounded = 0x80000000u; // a window: all positions before
constexpr uint32_t kWaves = 4;
constexpr uint32_t kThreads = 64 * kWaves;

// What one workgroup has of a tile of rows: its sequence, rows and keys.
struct Job {
    uint32_t index, start, r0, r1, kvh, slot; // slot: of its sums, where they are split
    int32_t before;                           // position of the sequence's first new token
    int32_t lo, hi;                           // this workgroup's keys
    bool whole;                               // all of the tile's keys are its
};

// The keys of a tile go out in equal pieces of whole `unit`s; the pieces that
// hold any number `pieces`.
struct Pieces {
    uint32_t size, count;
};
__device__ __forceinline__ Pieces pieces_of(uint32_t keys, uint32_t splits, uint32_t unit) {
    const uint32_t units = (keys + unit - 1) / unit, each = (units + splits - 1) / splits;
    return Pieces{each * unit, each ? (units + each - 1) / each : 0};
}

// The first position that position p sees (p may lie before the first one, far
// enough that p - window would pass -2^31).
__device__ __forceinline__ int32_t first_seen(const AttentionArgs &A, int32_t p) {
    const int32_t window = static_cast<int32_t>(A.window);
    return A.window != kUnbounded && p >= window ? p - window + 1 : 0;
}

// The visible keys of rows r0 .. r1 - 1: [lo, hi). lo is brought down to a
// multiple of 8, so that the keys of one load instruction share a page where its
// size allows, but not out of its page: an earlier one may have been given back.
// (A page whose size is a multiple of a load's rows, at most 8, starts at one.)
__device__ __forceinline__ void visible_keys(const AttentionArgs &A, int32_t before, uint32_t r0, uint32_t r1,
                                             int32_t &lo, int32_t &hi) {
    const int32_t first = before + static_cast<int32_t>(A.group.div(r0));
    hi = before + static_cast<int32_t>(A.group.div(r1 - 1)) + 1;
    hi = hi > 0 ? hi : 0;
    const int32_t seen = first_seen(A, first);
    const int32_t page = static_cast<int32_t>(A.a.page.div(seen) * A.a.page.d); // its first position
    lo = seen & ~7;
    lo = lo > page ? lo : page;
}

// Workgroup -> job: splits slowest (so that a tile's workgroups are spread over
// time as little as over the chip), kv heads fastest.
template <uint32_t kTileRows, uint32_t kUnit>
__device__ __forceinline__ bool find_job(const AttentionArgs &A, uint32_t block, Job &job, bool &bad) {
    const PagedArgs &a = A.a;
    const uint32_t G = A.group.d;
    job.kvh = block % a.kv_heads;
    const uint32_t rest = block / a.kv_heads, split = rest % A.splits, target = rest / A.splits;
    uint32_t item;
    Sequence seq;
    if (block == 0 && a.sequences > 64) bad |= any_bad_sequence(a);
    if (!find_item(a, target, [&](const Sequence &s) { return (s.count * G + kTileRows - 1) / kTileRows; }, job.index,
                   seq, item, bad))
        return false;
    const uint32_t rows = seq.count * G;
    job.start = seq.start;
    job.r0 = item * kTileRows;
    job.r1 = job.r0 + kTileRows < rows ? job.r0 + kTileRows : rows;
    job.before = static_cast<int32_t>(seq.length) - static_cast<int32_t>(seq.count);
    job.slot = (target * a.kv_heads + job.kvh) * A.splits + split;
    visible_keys(A, job.before, job.r0, job.r1, job.lo, job.hi);
    const Pieces p = pieces_of(job.hi - job.lo, A.splits, kUnit);
    job.whole = p.count <= 1;
    if (split >= p.count) return split == 0; // (a tile without keys is split 0's)
    job.lo += split * p.size;
    const int32_t end = job.lo + static_cast<int32_t>(p.size);
    job.hi = end < job.hi ? end : job.hi;
    return true;
}

// Element types: how many 16-bit parts carry a weight to f32 accuracy; kSlack,
// by how many powers of two a score may pass the maximum its row's sums are
// kept at before they are brought to a new one (any number near the maximum
// serves, and most tiles bring a slightly larger one for some row); kLift, the
// power of two the weights are kept at. A half's range ends at 2^-24, which
// would cost small weights their low bits: its weights are kept 2^9 times as
// large, 2^15 at most with the slack (the sum carries the same factor).
template <typename T> struct Element;
template <> struct Element<float> {
    static constexpr int kParts = 1;
    static constexpr float kLift = 0.0f, kSlack = 8.0f;
};
template <> struct Element<_Float16> {
    static constexpr int kParts = 2;
    static constexpr float kLift = 9.0f, kSlack = 6.0f;
    static constexpr uint32_t kExponent = 0x7c007c00u;
};
template <> struct Element<__bf16> {
    static constexpr int kParts = 3;
    static constexpr float kLift = 0.0f, kSlack = 8.0f;
    static constexpr uint32_t kExponent = 0x7f807f80u;
};

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

__device__ __forceinline__ f32x4 mma16(Vec8<__bf16>::type a, Vec8<__bf16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(Vec8<_Float16>::type a, Vec8<_Float16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's maximum or sum over the four 16-lane groups that hold its keys.
__device__ __forceinline__ float row_max(float v) {
    uint32_t a, b;
    lane_pair_u32<16>(__builtin_bit_cast(uint32_t, v), a, b);
    v = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    lane_pair_u32<32>(__builtin_bit_cast(uint32_t, v), a, b);
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float row_sum(float v) {
    uint32_t a, b;
    lane_pair_u32<16>(__builtin_bit_cast(uint32_t, v), a, b);
    v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    lane_pair_u32<32>(__builtin_bit_cast(uint32_t, v), a, b);
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

// One wavefront's 16 rows against kKeys keys, everything in registers: the
// scores are formed transposed (keys x rows), so that lane (c = lane % 16, g =
// lane / 16) holds row c's scores of the keys the next product wants from it,
// and the weights never move. The keys' order inside a product's k dimension
// is free as long as both operands agree: slot 8 g + x of the 32 is key 4 g + x
// (x < 4) or 16 + 4 g + x - 4, as the score registers have them.
// Keys and values come straight from global memory: a lane loads 16 bytes of
// key c per step, and of the 8 keys of its slots kE = DP / 16 consecutive
// elements, from kE c on: value product m has element kE c + m in its row c, so
// the transposition is one v_perm per two elements and whole rows are read.
template <typename T, int DP> struct Tile16 {
    static constexpr int kKeys = 32, kScores = 8, kE = DP / 16, kSteps = DP / 32;
    static constexpr int kLoads = kE * 2 / 16 ? kE * 2 / 16 : 1; // 16-byte (or one 8-byte) pieces of a value row
    typedef typename Vec8<T>::type v8;
    v8 q[kSteps], k[2][kSteps];
    uint32_t v[kScores][kE / 2];
    f32x4 acc[kE];

    static __device__ __forceinline__ uint32_t key(uint32_t g, int x) { return (x < 4 ? 0 : 12) + 4 * g + x; }

    __device__ __forceinline__ void load_q(const uint8_t *row, uint32_t g, uint32_t D, bool negate) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = v8{};
            if (32 * s + 8 * g < D) q[s] = __builtin_bit_cast(v8, ld16(row + (32 * s + 8 * g) * 2));
            if (negate) q[s] = -q[s];
        }
    }
    __device__ __forceinline__ void load(const uint8_t *kp, const uint8_t *vp, const uint64_t *offset, uint32_t c,
                                         uint32_t g, uint32_t D) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t *row = kp + offset[16 * t + c] + 16 * g;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                if (D != DP) k[t][s] = v8{};
                if (D == DP || 32 * s + 8 * g < D) k[t][s] = __builtin_bit_cast(v8, ld16(row + 64 * s));
            }
        }
#pragma unroll
        for (int x = 0; x < kScores; ++x) {
            const uint8_t *row = vp + offset[key(g, x)] + kE * 2 * c;
            if constexpr (kE == 4) {
                uint2 w = make_uint2(0, 0);
                if (D == DP || kE * c < D) w = ld8(row);
                v[x][0] = w.x;
                v[x][1] = w.y;
            } else {
#pragma unroll
                for (int h = 0; h < kLoads; ++h) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (D == DP || kE * c + 8 * h < D) w = ld16(row + 16 * h);
                    v[x][4 * h] = w.x;
                    v[x][4 * h + 1] = w.y;
                    v[x][4 * h + 2] = w.z;
                    v[x][4 * h + 3] = w.w;
                }
            }
        }
    }
    __device__ __forceinline__ void scores(float *s) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) r = mma16(k[t][i], q[i], r);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * t + i] = r[i];
        }
    }
    __device__ __forceinline__ void clear_values(uint32_t g, uint32_t first_hidden) {
#pragma unroll
        for (int x = 0; x < kScores; ++x)
            if (key(g, x) >= first_hidden)
#pragma unroll
                for (int w = 0; w < kE / 2; ++w) v[x][w] = 0;
    }
    static __device__ __forceinline__ v8 columns(const uint32_t (&w)[kScores][kE / 2], int m) {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r[j] = __builtin_amdgcn_perm(w[2 * j + 1][m / 2], w[2 * j][m / 2], m % 2 ? 0x07060302u : 0x05040100u);
        return __builtin_bit_cast(v8, r);
    }
    template <int kParts> __device__ __forceinline__ void add(const float *p) {
        float rest[kScores];
#pragma unroll
        for (int x = 0; x < kScores; ++x) rest[x] = p[x];
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            v8 w;
#pragma unroll
            for (int x = 0; x < kScores; ++x) {
                w[x] = static_cast<T>(rest[x]);
                if (part + 1 < kParts) rest[x] -= static_cast<float>(w[x]); // exact
            }
#pragma unroll
            for (int m = 0; m < kE; ++m) acc[m] = mma16(columns(v, m), w, acc[m]);
        }
    }
    // Infinities and NaN among the values of a tile that some row sees only in
    // part: a zero weight would not keep them out of that row's sums. They leave
    // the values, and the sums of the rows that see one become NaN, found by a
    // product of 0 / 1 matrices.
    __device__ __forceinline__ void split_nonfinite(const bool *seen) {
        constexpr uint32_t kHalf = Element<T>::kExponent & 0xffffu, kOne = sizeof(T) == 2 && kHalf == 0x7f80 ? 0x3f80 : 0x3c00;
        bool any = false;
#pragma unroll
        for (int x = 0; x < kScores; ++x)
#pragma unroll
            for (int w = 0; w < kE / 2; ++w)
                any |= (v[x][w] & kHalf) == kHalf || (v[x][w] >> 16 & kHalf) == kHalf;
        if (!__any(any)) return;
        uint32_t odd[kScores][kE / 2];
#pragma unroll
        for (int x = 0; x < kScores; ++x)
#pragma unroll
            for (int w = 0; w < kE / 2; ++w) {
                odd[x][w] = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if ((v[x][w] >> (16 * h) & kHalf) == kHalf) {
                        odd[x][w] |= kOne << (16 * h);
                        v[x][w] &= ~(0xffffu << (16 * h));
                    }
            }
        v8 w;
#pragma unroll
        for (int x = 0; x < kScores; ++x) w[x] = static_cast<T>(seen[x] ? 1.0f : 0.0f);
#pragma unroll
        for (int m = 0; m < kE; ++m) {
            const f32x4 n = mma16(columns(odd, m), w, f32x4{});
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = n[i] > 0.0f ? __builtin_nanf("") : acc[m][i];
        }
    }
};

// The same on v_mfma_f32_16x16x4_f32, 16 keys at a time: product i of a score
// step takes element 16 s + 4 g + i of key c, product i of the values slot g =
// key 4 g + i.
template <int DP> struct Tile16<float, DP> {
    static constexpr int kKeys = 16, kScores = 4, kE = DP / 16, kSteps = DP / 16;
    f32x4 q[kSteps], k[kSteps], v[kScores][kE / 4], acc[kE];

    static __device__ __forceinline__ uint32_t key(uint32_t g, int x) { return 4 * g + x; }

    __device__ __forceinline__ void load_q(const uint8_t *row, uint32_t g, uint32_t D, bool negate) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = f32x4{};
            if (16 * s + 4 * g < D) q[s] = __builtin_bit_cast(f32x4, ld16(row + (16 * s + 4 * g) * 4));
            if (negate) q[s] = -q[s];
        }
    }
    __device__ __forceinline__ void load(const uint8_t *kp, const uint8_t *vp, const uint64_t *offset, uint32_t c,
                                         uint32_t g, uint32_t D) {
        const uint8_t *row = kp + offset[c] + 16 * g;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (D != DP) k[s] = f32x4{};
            if (D == DP || 16 * s + 4 * g < D) k[s] = __builtin_bit_cast(f32x4, ld16(row + 64 * s));
        }
#pragma unroll
        for (int x = 0; x < kScores; ++x) {
            const uint8_t *from = vp + offset[key(g, x)] + kE * 4 * c;
#pragma unroll
            for (int h = 0; h < kE / 4; ++h) {
                if (D != DP) v[x][h] = f32x4{};
                if (D == DP || kE * c + 4 * h < D) v[x][h] = __builtin_bit_cast(f32x4, ld16(from + 16 * h));
            }
        }
    }
    __device__ __forceinline__ void scores(float *s) const {
        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < kSteps; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) r = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][i], q[t][i], r, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = r[i];
    }
    __device__ __forceinline__ void clear_values(uint32_t g, uint32_t first_hidden) {
#pragma unroll
        for (int x = 0; x < kScores; ++x)
            if (key(g, x) >= first_hidden)
#pragma unroll
                for (int h = 0; h < kE / 4; ++h) v[x][h] = f32x4{};
    }
    template <int kParts> __device__ __forceinline__ void add(const float *p) {
#pragma unroll
        for (int m = 0; m < kE; ++m)
#pragma unroll
            for (int x = 0; x < kScores; ++x)
                acc[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[x][m / 4][m % 4], p[x], acc[m], 0, 0, 0);
    }
    __device__ __forceinline__ void split_nonfinite(const bool *seen) {
        bool any = false;
#pragma unroll
        for (int x = 0; x < kScores; ++x)
#pragma unroll
            for (int m = 0; m < kE; ++m) any |= !__builtin_isfinite(v[x][m / 4][m % 4]);
        if (!__any(any)) return;
#pragma unroll
        for (int m = 0; m < kE; ++m) {
            f32x4 n = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < kScores; ++x) {
                const bool finite = __builtin_isfinite(v[x][m / 4][m % 4]);
                n = __builtin_amdgcn_mfma_f32_16x16x4f32(finite ? 0.0f : 1.0f, seen[x] ? 1.0f : 0.0f, n, 0, 0, 0);
                if (!finite) v[x][m / 4][m % 4] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][i] = n[i] > 0.0f ? __builtin_nanf("") : acc[m][i];
        }
    }
};

// Scores from q . k, in units of 1 / per_score of log 2: q . k itself, or the
// capped score. Below 1 / 4, where scores mostly lie, the hyperbolic tangent is
// its Taylor sum to x^9 (the next term is below 2^-26 of it), a fifth of
// tanhf's instructions. Which of the two a score takes goes by that score alone,
// whatever the others of the wavefront are (keys its row does not see among
// them); their vote only decides whether tanhf has to be computed at all. (A
// prompt of 4096 in bf16: 159 us without a cap, 196 with scores of a thirtieth of
// it, 420 with scores about as large as it.)
template <class Scores> __device__ __forceinline__ void cap_scores(const AttentionArgs &A, Scores &s) {
    constexpr int kN = sizeof(Scores) / sizeof(float);
    if (A.softcap == 0.0f) return;
    constexpr float kNear = 0.25f;
    const auto near = [](float x) {
        const float q = x * x;
        float t = fma_rn(q, 62.0f / 2835.0f, -17.0f / 315.0f);
        t = fma_rn(t, q, 2.0f / 15.0f);
        t = fma_rn(t, q, -1.0f / 3.0f);
        return fma_rn(t * q, x, x);
    };
    float most = 0.0f;
#pragma unroll
    for (int x = 0; x < kN; ++x) {
        s[x] *= A.scale;
        most = fmaxf(most, fabsf(s[x])); // (a NaN is dropped here and kept by either form)
    }
    if (__any(most > kNear)) {
#pragma unroll
        for (int x = 0; x < kN; ++x) s[x] = (fabsf(s[x]) > kNear ? tanhf(s[x]) : near(s[x])) * A.softcap;
    } else {
#pragma unroll
        for (int x = 0; x < kN; ++x) s[x] = near(s[x]) * A.softcap;
    }
}

__device__ __forceinline__ void store4(uint8_t *row, uint32_t d, uint32_t type, f32x4 x) {
    if (type == FMX_TYPE_F32) {
        *reinterpret_cast<f32x4 *>(row + d * 4) = x;
    } else if (type == FMX_TYPE_F16) {
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<h4 *>(row + d * 2) = __builtin_convertvector(x, h4);
    } else {
        typedef __bf16 b4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<b4 *>(row + d * 2) = __builtin_convertvector(x, b4);
    }
}

// Four elements of a row's sums with their maximum and the sum of weights: to
// the output, with the sink's weight and divided, or, of a split tile, to where
// attention_join_kernel takes them up. A row at a position before the first sees
// nothing and is zero; any other sees itself, and without a score above -inf
// (NaN, or -inf alone) its sums make it NaN, as they should.
__device__ __forceinline__ void finish(const AttentionArgs &A, const Job &job, uint32_t tile_rows, uint32_t r,
                                       uint32_t head, uint32_t token, uint32_t d, float top, float mass, f32x4 o,
                                       float lift) {
    const uint32_t D = A.a.head_dim;
    if (!job.whole) {
        const uint64_t at = static_cast<uint64_t>(job.slot) * tile_rows + r;
        *reinterpret_cast<f32x4 *>(A.parts + at * D + d) = o;
        if (d == 0) A.stats[at] = make_float2(top, mass);
        return;
    }
    const bool sees = job.before + static_cast<int32_t>(token - job.start) >= 0;
    if (A.sinks && sees) {
        const float sink = A.sinks[head] * 0x1.715476p+0f; // log2 e
        const float best = fmaxf(top, sink), f = exp2_fast(top - best);
        mass = mass * f + exp2_fast(sink - best + lift);
        o *= f;
    }
    if (sees) o /= mass;
    else o = f32x4{};
    const uint32_t size = A.out_type == FMX_TYPE_F32 ? 4 : 2;
    store4(A.out + token * A.out_bytes + static_cast<uint64_t>(head) * D * size, d, A.out_type, o);
}

constexpr uint32_t kRows = 16;

// 16 rows of one sequence and kv head per workgroup; its wavefronts take tiles
// of keys in turn and join their sums through LDS.
// Bound by the cache's way from memory: keys and values go straight into
// registers, 16 KiB a wavefront and step at head_dim 128, with enough
// wavefronts (kFillRows workgroups) to cover the latency instead of a
// pipeline. One token over 131072 positions, 32 / 8 heads of 128, f16: 116 us,
// 4.6 TB/s; 64 tokens of sequences up to 8192 long, bf16: 222 us, 4.8 TB/s (a
// copy of 1 GiB: 5.1); one token over 2000 positions in f32: 12 us, of which 7.5
// here and 3.3 the join, both latency (the batch's entries, the page, the rows:
// reads that wait for each other). The weights meet the values in all their
// parts whatever the result's type: the second part costs the f16 case nothing
// (116.6 us with and without).
// grid: row tiles x splits x kv heads, the heads fastest.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_rows_kernel(AttentionArgs A) {
    using Tile = Tile16<T, DP>;
    constexpr int kParts = Element<T>::kParts;
    constexpr float kLift = Element<T>::kLift;
    constexpr uint32_t kStride = DP + 4;
    extern __shared__ __align__(16) char lds[];
    float *sums = reinterpret_cast<float *>(lds); // [waves][rows][kStride]
    __shared__ __align__(16) uint64_t offsets[kWaves][32];
    __shared__ float top_s[kWaves][kRows], mass_s[kWaves][kRows];
    const PagedArgs &a = A.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const uint32_t G = A.group.d, D = a.head_dim;
    bool bad = false;
    Job job;
    if (!find_job<kRows, Tile::kKeys * kWaves>(A, blockIdx.x, job, bad)) {
        if (bad && tid == 0) atomicOr(A.status, STATUS_BAD_PAGE);
        return;
    }
    const uint32_t r0 = job.r0, r1 = job.r1, kvh = job.kvh;
    const int32_t lo = job.lo, hi = job.hi;
    const int32_t p_first = job.before + static_cast<int32_t>(A.group.div(r0));
    const int32_t p_last = job.before + static_cast<int32_t>(A.group.div(r1 - 1));
    const uint32_t row = r0 + c < r1 ? r0 + c : r1 - 1, token = A.group.div(row), head = kvh * G + row - token * G;
    const int32_t p = job.before + static_cast<int32_t>(token);
    const int32_t from = first_seen(A, p);
    // every row of the tile sees these
    const int32_t all_lo = first_seen(A, p_last), all_hi = p_first + 1;

    Tile tile;
    tile.load_q(A.q + (job.start + token) * A.q_bytes + static_cast<uint64_t>(head) * D * sizeof(T), g, D, A.negate);
#pragma unroll
    for (int m = 0; m < Tile::kE; ++m) tile.acc[m] = f32x4{};
    float top = kNegInf, mass = 0.0f;
    const uint8_t *kp = a.k + kvh * a.head_bytes, *vp = a.v + kvh * a.head_bytes;
    const uint32_t *table = a.table + static_cast<uint64_t>(job.index) * a.table_stride;
    for (int32_t base = lo + static_cast<int32_t>(wave) * Tile::kKeys; base < hi; base += kWaves * Tile::kKeys) {
        const int32_t mine = base + static_cast<int32_t>(lane & (Tile::kKeys - 1));
        const uint32_t t = mine < hi ? mine : hi - 1; // reads stay in the sequence
        const uint32_t page = a.page.div(t);
        __builtin_amdgcn_wave_barrier();
        offsets[wave][lane & (Tile::kKeys - 1)] = position_offset(a, table[page], t - page * a.page.d, bad);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        tile.load(kp, vp, offsets[wave], c, g, D);
        float s[Tile::kScores];
        tile.scores(s);
        if (base + Tile::kKeys > hi) tile.clear_values(g, hi - base);
        cap_scores(A, s);
        float high = kNegInf;
        if (base < all_lo || base + Tile::kKeys > all_hi) {
            bool seen[Tile::kScores];
#pragma unroll
            for (int x = 0; x < Tile::kScores; ++x) {
                const int32_t j = base + static_cast<int32_t>(Tile::key(g, x));
                seen[x] = j <= p && j >= from;
                s[x] = seen[x] ? s[x] : kNegInf;
            }
            tile.split_nonfinite(seen);
        }
#pragma unroll
        for (int x = 0; x < Tile::kScores; ++x) high = fmaxf(high, s[x]);
        high = row_max(high) * A.per_score;
        const float next = fmaxf(top, high), at = next == kNegInf ? 0.0f : next;
        const float shrink = exp2_fast(top - at), shift = kLift - at;
        float w[Tile::kScores], sum = 0.0f;
#pragma unroll
        for (int x = 0; x < Tile::kScores; ++x) {
            w[x] = exp2_fast(fma_rn(s[x], A.per_score, shift));
            sum += w[x];
        }
        top = next;
        mass = mass * shrink + sum; // this lane's keys
        if (__any(shrink != 1.0f))
#pragma unroll
            for (int m = 0; m < Tile::kE; ++m) tile.acc[m] *= shrink;
        tile.template add<kParts>(w);
    }
    if (__any(bad) && lane == 0) atomicOr(A.status, STATUS_BAD_PAGE);
    mass = row_sum(mass);
    if (g == 0) {
        top_s[wave][c] = top;
        mass_s[wave][c] = mass;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < Tile::kE; m += 4)
            *reinterpret_cast<f32x4 *>(sums + (wave * kRows + c) * kStride + Tile::kE * (4 * g + i) + m) =
                f32x4{tile.acc[m][i], tile.acc[m + 1][i], tile.acc[m + 2][i], tile.acc[m + 3][i]};
    __syncthreads();
    for (uint32_t u = tid; u < kRows * DP / 4; u += kThreads) {
        const uint32_t r = u / (DP / 4), d = u % (DP / 4) * 4;
        if (r0 + r >= r1 || d >= D) continue;
        const uint32_t tok = A.group.div(r0 + r), h = kvh * G + r0 + r - tok * G;
        float best = kNegInf;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) best = fmaxf(best, top_s[i][r]);
        const float at = best == kNegInf ? 0.0f : best;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        float total = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) {
            const float f = exp2_fast(top_s[i][r] - at);
            total += f * mass_s[i][r];
            o += f * *reinterpret_cast<const f32x4 *>(sums + (i * kRows + r) * kStride + d);
        }
        finish(A, job, kRows, r, h, job.start + tok, d, best, total, o, kLift);
    }
}

// ------------------------------------------------------------ many rows --

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mma32(Vec8<__bf16>::type a, Vec8<__bf16>::type b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(Vec8<_Float16>::type a, Vec8<_Float16>::type b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Key of score x of lane half h within a block of 32.
__device__ __forceinline__ uint32_t score_key(uint32_t h, int x) { return x / 4 * 8 + 4 * h + x % 4; }

// One wavefront's 32 rows against a block of 32 keys in LDS. The scores are
// formed transposed as above: lane (c = lane % 32, h = lane / 32) holds row c's
// scores, register 8 u + x being key 16 u + 8 (x / 4) + 4 h + x % 4 (score_key),
// which as they stand are slots 8 h + x of the value product's step u.
//
// LDS holds keys and values as memory does, a row of DP elements per position,
// its 16-byte granules permuted so that every pass of a wavefront's reads
// touches all 64 banks: the key operand takes one granule of 16 consecutive
// rows, the value operand (ds_read_b64_tr_b16: 16 lanes read 4 rows x 16
// elements and each gets one column) a 64-byte piece of 4 rows. DC of the DP
// elements are multiplied.
template <typename T, int DP, int DC> struct Tile32 {
    static constexpr int kSteps = DC / 16, kD = DC / 32, kGranules = DP / 8, kGranule = 8;
    static constexpr int kRing = 4; // blocks in LDS; the next one's scores are formed beside this one's weights
    typedef typename Vec8<T>::type v8;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    v8 q[kSteps];
    f32x16 acc[kD];
    struct Keys {
        v8 k[kSteps];
    };

    static __device__ __forceinline__ uint32_t key_granule(uint32_t key, uint32_t granule) {
        return granule ^ (DP == 64 ? key >> 1 & 7 : key & 15);
    }
    static __device__ __forceinline__ uint32_t value_granule(uint32_t key, uint32_t granule) {
        return granule ^ (DP == 64 ? (key >> 1 & 1) * 4 : (key & 3) * 4);
    }
    __device__ __forceinline__ void load_q(const uint8_t *row, uint32_t h, uint32_t D, bool negate) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = v8{};
            if (16 * s + 8 * h < D) q[s] = __builtin_bit_cast(v8, ld16(row + (16 * s + 8 * h) * 2));
            if (negate) q[s] = -q[s];
        }
    }
    static __device__ __forceinline__ void read_keys(Keys &k, const char *keys, uint32_t c, uint32_t h) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            k.k[i] = *reinterpret_cast<const v8 *>(keys + c * (DP * 2) + key_granule(c, 2 * i + h) * 16);
    }
    __device__ __forceinline__ f32x16 scores(const Keys &k) const {
        f32x16 r = {};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) r = mma32(k.k[i], q[i], r);
        return r;
    }
    __device__ __forceinline__ f32x16 score_step(const Keys &k, int i, f32x16 r) const { return mma32(k.k[i], q[i], r); }
    // Value operand of step u, elements 32 d .. 32 d + 31.
    static __device__ __forceinline__ v8 value(const char *values, uint32_t lane, int u, int d) {
        typedef __attribute__((address_space(3))) s16x4 *ptr;
        const uint32_t g = lane >> 4, i = lane & 15, row = 16 * u + 4 * (g >> 1) + (i >> 2);
        const char *p = values + row * (DP * 2) + value_granule(row, 4 * d + 2 * (g & 1) + (i >> 1 & 1)) * 16 + 8 * (i & 1);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p + 8 * DP * 2));
        return __builtin_bit_cast(v8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    template <int kParts> __device__ __forceinline__ void add(const char *values, uint32_t lane, f32x16 p) {
        v8 w[kParts][2];
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const T t = static_cast<T>(p[x]);
                w[part][x / 8][x % 8] = t;
                if (part + 1 < kParts) p[x] -= static_cast<float>(t); // exact
            }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < kD; ++d) {
                const v8 v = value(values, lane, u, d);
#pragma unroll
                for (int part = 0; part < kParts; ++part) acc[d] = mma32(v, w[part][u], acc[d]);
            }
    }
    // The elements of a granule that are not finite, one bit each; they become 0.
    static __device__ __forceinline__ uint32_t take_nonfinite(uint4 &g) {
        constexpr uint32_t kHalf = Element<T>::kExponent & 0xffffu;
        uint32_t bits = 0, w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if ((w[i / 2] >> (i % 2 * 16) & kHalf) == kHalf) {
                bits |= 1u << i;
                w[i / 2] &= ~(0xffffu << (i % 2 * 16));
            }
        g = make_uint4(w[0], w[1], w[2], w[3]);
        return bits;
    }
    // Of a key's bits those of this lane's sums: elements 8 i + 4 h .. + 3 of each
    // 32 (register 4 i + b of acc[d]: bit 8 i + b of word d).
    static __device__ __forceinline__ uint32_t odd_word(const uint8_t *of_key, int d, uint32_t h) {
        return *reinterpret_cast<const uint32_t *>(of_key + 4 * d) >> (4 * h) & 0x0f0f0f0fu;
    }
};

// f32 on v_mfma_f32_32x32x2_f32: product e of a score step takes elements 8 s +
// 4 h + e, and register x of the scores is the value product's step x with no
// rearrangement at all, slot h being key score_key(h, x). A block's products
// take 64 cycles each, 16 times as long as its keys' way into LDS: two buffers
// do.
template <int DP, int DC> struct Tile32<float, DP, DC> {
    static constexpr int kSteps = DC / 8, kD = DC / 32, kGranules = DP / 4, kGranule = 4, kRing = 2;
    f32x4 q[kSteps];
    f32x16 acc[kD];
    struct Keys {
        const char *row;
        uint32_t c, h;
    };

    static __device__ __forceinline__ uint32_t key_granule(uint32_t key, uint32_t granule) { return granule ^ (key & 15); }
    static __device__ __forceinline__ uint32_t value_granule(uint32_t key, uint32_t granule) {
        return granule ^ (key >> 2 & 1) * 8;
    }
    __device__ __forceinline__ void load_q(const uint8_t *row, uint32_t h, uint32_t D, bool negate) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            q[s] = f32x4{};
            if (8 * s + 4 * h < D) q[s] = __builtin_bit_cast(f32x4, ld16(row + (8 * s + 4 * h) * 4));
            if (negate) q[s] = -q[s];
        }
    }
    static __device__ __forceinline__ void read_keys(Keys &k, const char *keys, uint32_t c, uint32_t h) {
        k = Keys{keys + c * (DP * 4), c, h};
    }
    __device__ __forceinline__ f32x16 scores(const Keys &k) const {
        f32x16 r = {};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(k.row + key_granule(k.c, 2 * i + k.h) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) r = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], q[i][e], r, 0, 0, 0);
        }
        return r;
    }
    template <int kParts> __device__ __forceinline__ void add(const char *values, uint32_t lane, const f32x16 &p) {
        const uint32_t c = lane & 31, h = lane >> 5;
#pragma unroll
        for (int x = 0; x < 16; ++x)
#pragma unroll
            for (int d = 0; d < kD; ++d) {
                const uint32_t key = score_key(h, x);
                const float v = *reinterpret_cast<const float *>(values + key * (DP * 4) +
                                                                 value_granule(key, 8 * d + c / 4) * 16 + c % 4 * 4);
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[x], acc[d], 0, 0, 0);
            }
    }
    static __device__ __forceinline__ uint32_t take_nonfinite(uint4 &g) {
        uint32_t bits = 0, w[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((w[i] & 0x7f800000u) == 0x7f800000u) {
                bits |= 1u << i;
                w[i] = 0;
            }
        g = make_uint4(w[0], w[1], w[2], w[3]);
        return bits;
    }
    static __device__ __forceinline__ uint32_t odd_word(const uint8_t *of_key, int d, uint32_t h) {
        const uint2 w = *reinterpret_cast<const uint2 *>(of_key + 8 * d); // a byte for each granule of 4
        const uint32_t lo = w.x >> (8 * h), hi = w.y >> (8 * h);
        return (lo & 15u) | (lo >> 8 & 15u << 8) | (hi & 15u) << 16 | (hi & 15u << 16) << 8;
    }
};

constexpr uint32_t kTileRows = 32 * kWaves;
constexpr uint32_t kBlock = 32; // keys

// 16 bytes per lane and side from global memory to LDS, `to` + 16 lane for the
// keys and `to` + side for the values (`to`: a byte offset in LDS,
// wave-uniform), for the lanes in the masks; all lanes are active again after
// it. In assembly, since the compiler waits for every load of the builtin
// before each transposing read of LDS, which would undo the ring; it has no
// result, and the waits for it are counted by hand below. (m0 is reserved: the
// compiler keeps nothing in it.)
struct LoadMasks {
    uint64_t k, v;
};
__device__ __forceinline__ void load_lds(const void *k, const void *v, uint32_t to, uint32_t side, const LoadMasks &m) {
    asm volatile("s_mov_b64 exec, %4\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off\n\t"
                 "s_mov_b64 exec, %5\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
                 "s_mov_b64 exec, -1" ::"v"(k),
                 "v"(v), "s"(to), "s"(to + side), "s"(m.k), "s"(m.v)
                 : "memory");
}
// The same from wave-uniform addresses and 32-bit offsets of the lanes. (The
// first s_nop: a scalar register a vector instruction wrote needs five cycles
// before a vector memory instruction reads it, which the compiler does not see
// here.)
__device__ __forceinline__ void load_lds(uint64_t k, uint64_t v, uint32_t k_lane, uint32_t v_lane, uint32_t to, uint32_t side,
                                         const LoadMasks &m) {
    asm volatile("s_nop 4\n\ts_mov_b64 exec, %6\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %0\n\t"
                 "s_mov_b64 exec, %7\n\ts_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %1\n\t"
                 "s_mov_b64 exec, -1" ::"s"(k),
                 "s"(v), "v"(k_lane), "v"(v_lane), "s"(to), "s"(to + side), "s"(m.k), "s"(m.v)
                 : "memory");
}

// Waits until at most N of this wavefront's vector memory operations are
// outstanding, then for the workgroup; no memory access moves across.
template <uint32_t N> __device__ __forceinline__ void wait_and_barrier() {
    static_assert(N < 64, "vmcnt has six bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15u) | ((N >> 4) << 14) | (7u << 4)); // vmcnt(N) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 128 rows of one sequence and kv head per workgroup, 32 a wavefront, all
// against the same keys, which pass through a ring of LDS blocks of 32: loads go
// straight into LDS, kRing - 1 blocks ahead, every wavefront issuing the same
// number for each block (behind the last one it loads that again), so that a
// count of outstanding operations tells which blocks have landed.
// kGrouped: the rows of a load instruction lie in one page (blocks start at
// multiples of 8 or of the page size, which is one of their number), less than
// 2^30 bytes apart. (A prompt of 4096, bf16: 159 us; pages of 6, 5 and 1 positions,
// whose rows are looked up one by one, 178, 180 and 195.)
// Bound by the matrix cores and the SIMDs' issue between their products: 32 rows
// a wavefront halve the LDS reads per product against 16, two workgroups share a
// CU, and while one wavefront of a SIMD forms its weights the other's products
// run. 2048 tokens at the end of 16384 positions, 32 / 8 heads of 128, bf16: 531 to
// 559 us on different cards, 0.97 to 0.92 PFLOP/s counted as two products per
// visible pair (a library product of 8192^3 reaches 1.14); a prompt of 4096: 159 to
// 166 us, 0.86 to 0.83; head_dim 256 (16 / 8 heads) keeps one workgroup a CU for its
// registers, 266 us, 0.52; f32, a ragged batch of 2544 tokens with a window of 1000,
// 16 / 8 heads of 96: 190 us, 65 TFLOP/s of the 153 a library product reaches: the
// tiles' unequal lengths leave CUs idle for a third of it. Of the chunk's time (531
// us), left out in a copy: the exponentials 35, the keys' LDS reads 35, the loads
// 70, three quarters of the value products 120.
// grid: row tiles x splits x kv heads, the heads fastest; the tiles with the
// most keys first.
template <typename T, int DP, int DC, int kParts, bool kGrouped>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void attention_tiles_kernel(AttentionArgs A) {
    using Tile = Tile32<T, DP, DC>;
    constexpr float kLift = Element<T>::kLift;
    constexpr uint32_t kRowBytes = DP * sizeof(T), kSide = kBlock * kRowBytes; // a block's keys or values
    constexpr uint32_t kRing = Tile::kRing, kRowsAtOnce = 1024 / kRowBytes; // rows of one load instruction
    constexpr uint32_t kLoads = kSide / 1024 / kWaves;                      // instructions a side and wavefront
    extern __shared__ __align__(16) char lds[];                             // ring of (keys, values); bits
    uint8_t *const bits = reinterpret_cast<uint8_t *>(lds) + kRing * 2 * kSide;
    const uint32_t ring = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds)));
    const PagedArgs &a = A.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t G = A.group.d, D = a.head_dim;
    bool bad = false;
    Job job;
    if (!find_job<kTileRows, kBlock>(A, gridDim.x - 1 - blockIdx.x, job, bad)) {
        if (bad && tid == 0) atomicOr(A.status, STATUS_BAD_PAGE);
        return;
    }
    const uint32_t w0 = job.r0 + 32 * wave, w1 = w0 + 32 < job.r1 ? w0 + 32 : job.r1; // this wavefront's rows
    const bool active = w0 < job.r1;
    const int32_t lo = job.lo, hi = job.hi;
    const uint32_t row = w0 + c < job.r1 ? w0 + c : job.r1 - 1, token = A.group.div(row);
    const uint32_t head = job.kvh * G + row - token * G;
    const int32_t p = job.before + static_cast<int32_t>(token);
    const int32_t p_first = job.before + static_cast<int32_t>(A.group.div(active ? w0 : job.r0));
    const int32_t p_last = job.before + static_cast<int32_t>(A.group.div(active ? w1 - 1 : job.r0));
    const int32_t from = first_seen(A, p);
    // what every row of the workgroup sees, what every row of the wavefront, and
    // where the last of these ends
    const int32_t tile_hi = job.before + static_cast<int32_t>(A.group.div(job.r0)) + 1;
    const int32_t tile_lo = first_seen(A, job.before + static_cast<int32_t>(A.group.div(job.r1 - 1)));
    const int32_t all_lo = first_seen(A, p_last), all_hi = p_first + 1;
    const int32_t any_hi = active ? p_last + 1 : 0;

    Tile tile;
    tile.load_q(A.q + (job.start + token) * A.q_bytes + static_cast<uint64_t>(head) * D * sizeof(T), h, D, A.negate);
#pragma unroll
    for (int d = 0; d < Tile::kD; ++d) tile.acc[d] = f32x16{};
    float top = kNegInf, mass = 0.0f;
    uint32_t spoiled[Tile::kD] = {}; // sums that met a value that is not finite

    // Loads: instruction n of this wavefront covers rows (4 n + wave) kRowsAtOnce
    // on of a block; lane l writes granule l of those bytes, so it reads the
    // element granule that belongs there.
    const uint32_t in_row = lane / Tile::kGranules, slot = lane % Tile::kGranules;
    uint32_t kg[kLoads], vg[kLoads];
    LoadMasks masks[kLoads];
#pragma unroll
    for (uint32_t n = 0; n < kLoads; ++n) {
        const uint32_t r = (kWaves * n + wave) * kRowsAtOnce + in_row;
        kg[n] = Tile::key_granule(r, slot);
        vg[n] = Tile::value_granule(r, slot);
        masks[n] = LoadMasks{__ballot(kg[n] * Tile::kGranule < D), __ballot(vg[n] * Tile::kGranule < D)};
    }
    const uint32_t *table = a.table + static_cast<uint64_t>(job.index) * a.table_stride;
    const uint8_t *kp = a.k + job.kvh * a.head_bytes, *vp = a.v + job.kvh * a.head_bytes;
    const auto first_row = [&](int32_t base, uint32_t n) {
        return base + static_cast<int32_t>((kWaves * n + wave) * kRowsAtOnce);
    };
    // kGrouped: the offsets of the next 64 / kLoads blocks' instructions, one a
    // lane, found at once; a block's come out by v_readlane. (Rows behind the last
    // position, in its page: read and never used.)
    constexpr uint32_t kBatch = 64 / kLoads;
    uint64_t offsets = 0;
    uint32_t batch = kBatch;
    const auto find_offsets = [&](int32_t base) {
        const int32_t j = first_row(base + static_cast<int32_t>(lane / kLoads * kBlock), lane % kLoads);
        const int32_t last = (hi - 1) & ~static_cast<int32_t>(kRowsAtOnce - 1), t = j < last ? j : last;
        const uint32_t page = a.page.div(t);
        offsets = position_offset(a, table[page], t - page * a.page.d, bad);
        batch = 0;
    };
    const uint32_t row_at = in_row * static_cast<uint32_t>(a.position_bytes); // (kGrouped: below 2^30)
    auto request = [&](int32_t base, uint32_t at) { // into the ring's block `at`
        if (kGrouped && batch == kBatch) find_offsets(base);
#pragma unroll
        for (uint32_t n = 0; n < kLoads; ++n) {
            const uint32_t to = ring + at * 2 * kSide + (kWaves * n + wave) * kRowsAtOnce * kRowBytes;
            if constexpr (kGrouped) {
                const uint32_t from = batch * kLoads + n;
                const uint64_t o = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(offsets >> 32), from)) << 32 |
                                   static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(offsets), from));
                load_lds(reinterpret_cast<uint64_t>(kp) + o, reinterpret_cast<uint64_t>(vp) + o, row_at + kg[n] * 16,
                         row_at + vg[n] * 16, to, kSide, masks[n]);
            } else {
                const int32_t j = first_row(base, n) + static_cast<int32_t>(in_row), t = j < hi ? j : hi - 1;
                const uint32_t page = a.page.div(t);
                const uint64_t o = position_offset(a, table[page], t - page * a.page.d, bad);
                load_lds(kp + o + kg[n] * 16, vp + o + vg[n] * 16, to, kSide, masks[n]);
            }
        }
        ++batch;
    };
    f32x16 s = {};
    if (lo < hi) {
        if (D != DP) { // the granules behind head_dim: zeros that no load touches
            for (uint32_t i = tid; i < kRing * 2 * kSide / 16; i += kThreads)
                reinterpret_cast<uint4 *>(lds)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
#pragma unroll
        for (uint32_t i = 0; i + 1 < kRing; ++i) request(lo + i * kBlock, i);
        if constexpr (kRing > 2) {
            wait_and_barrier<0>();
            typename Tile::Keys k;
            Tile::read_keys(k, lds, c, h);
            s = tile.scores(k);
        }
    }
    uint32_t at = 0;
    for (int32_t base = lo; base < hi; base += kBlock, at = at + 1 == kRing ? 0 : at + 1) {
        const uint32_t next = at + 1 == kRing ? 0 : at + 1, free = at == 0 ? kRing - 1 : at - 1;
        // the next block (kRing = 2: this one) has landed for every wavefront, and
        // none reads the block before this one any more
        wait_and_barrier<kRing == 2 ? 0 : 2 * kLoads * (kRing - 3)>();
        request(base + (kRing - 1) * kBlock, free);
        const char *keys = lds + at * 2 * kSide, *next_keys = lds + next * 2 * kSide;
        char *values = lds + at * 2 * kSide + kSide;
        // Infinities and NaN among the values of a block that some row sees only in
        // part: a zero weight would not keep them out of that row's sums. They
        // become 0 with a bit each, and the rows that see one get NaN in the end.
        bool odd = false;
        if (base < tile_lo || base + static_cast<int32_t>(kBlock) > tile_hi) {
            uint32_t any = 0;
#pragma unroll
            for (uint32_t i = tid; i < kSide / 16; i += kThreads) {
                uint4 g = reinterpret_cast<const uint4 *>(values)[i];
                const uint32_t b = Tile::take_nonfinite(g), r = i / Tile::kGranules;
                bits[r * Tile::kGranules + Tile::value_granule(r, i % Tile::kGranules)] = b;
                if (b) reinterpret_cast<uint4 *>(values)[i] = g;
                any |= b;
            }
            odd = __syncthreads_or(any);
        }
        if (base >= any_hi) continue; // no row of the wavefront sees it or a later one
        if constexpr (kRing == 2) {
            typename Tile::Keys k;
            Tile::read_keys(k, keys, c, h);
            s = tile.scores(k);
        }
        typename Tile::Keys k;
        if constexpr (kRing > 2) Tile::read_keys(k, next_keys, c, h);
        cap_scores(A, s);
        if (base < all_lo || base + static_cast<int32_t>(kBlock) > all_hi) {
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const int32_t j = base + static_cast<int32_t>(score_key(h, x));
                s[x] = j <= p && j >= from && j < hi ? s[x] : kNegInf;
            }
        }
        float high = s[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) high = fmaxf(high, s[x]);
        uint32_t u, v;
        lane_pair_u32<32>(__builtin_bit_cast(uint32_t, high), u, v);
        high = fmaxf(__builtin_bit_cast(float, u), __builtin_bit_cast(float, v)) * A.per_score;
        const bool raise = high > top + Element<T>::kSlack; // (also from -inf)
        if (__any(raise)) {
            const float shrink = raise ? exp2_fast(top - high) : 1.0f;
            top = raise ? high : top;
            mass *= shrink;
#pragma unroll
            for (int d = 0; d < Tile::kD; ++d) tile.acc[d] *= shrink;
        }
        const float shift = kLift - (top == kNegInf ? 0.0f : top);
        float sum = 0.0f;
        const auto weigh = [&](int x) {
            s[x] = exp2_fast(fma_rn(s[x], A.per_score, shift));
            sum += s[x];
        };
        f32x16 following = {};
        __builtin_amdgcn_s_setprio(1);
        if constexpr (kRing > 2) {
            // the next block's products run while the weights' exponentials issue:
            // a few of these behind each product, in that order
#pragma unroll
            for (int i = 0; i < Tile::kSteps; ++i) {
                following = tile.score_step(k, i, following);
#pragma unroll
                for (int x = i * 16 / Tile::kSteps; x < (i + 1) * 16 / Tile::kSteps; ++x) weigh(x);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) weigh(x);
        }
        mass += sum; // this lane's keys
        tile.template add<kParts>(values, lane, s);
        s = following;
        __builtin_amdgcn_s_setprio(0);
        if (odd)
#pragma unroll 1
            for (int32_t j = base > from ? base : from; j <= p && j < base + static_cast<int32_t>(kBlock) && j < hi; ++j)
#pragma unroll
                for (int d = 0; d < Tile::kD; ++d) spoiled[d] |= Tile::odd_word(bits + (j - base) * Tile::kGranules, d, h);
    }
    wait_and_barrier<0>(); // no load into LDS outlives the workgroup
    if (__any(bad) && lane == 0) atomicOr(A.status, STATUS_BAD_PAGE);
    uint32_t u, v;
    lane_pair_u32<32>(__builtin_bit_cast(uint32_t, mass), u, v);
    mass = __builtin_bit_cast(float, u) + __builtin_bit_cast(float, v);
    if (!active || w0 + c >= job.r1) return;
#pragma unroll
    for (int d = 0; d < Tile::kD; ++d)
        if (spoiled[d])
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (spoiled[d] >> (i / 4 * 8 + i % 4) & 1) tile.acc[d][i] = __builtin_nanf("");
#pragma unroll
    for (int d = 0; d < Tile::kD; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t e = 32 * d + 8 * i + 4 * h;
            if (e < D)
                finish(A, job, kTileRows, 32 * wave + c, head, job.start + token, e, top, mass,
                       f32x4{tile.acc[d][4 * i], tile.acc[d][4 * i + 1], tile.acc[d][4 * i + 2], tile.acc[d][4 * i + 3]},
                       kLift);
        }
}

// A split tile's sums joined: DP / 4 lanes hold a row of one head, kGroups such
// groups take its pieces in turn, in the same order at every call. grid: row
// tiles x kv heads x workgroups of a tile, these fastest. Latency: 3.3 us for 32
// pieces of one token's rows, 6.4 for 256.
template <int DP, uint32_t kGroups>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(AttentionArgs A, uint32_t tile_rows, uint32_t unit,
                                                                  float lift) {
    constexpr uint32_t kLanes = DP / 4, kSlots = kThreads / kLanes, kRowsHere = kSlots / kGroups;
    __shared__ f32x4 sum_s[kThreads];
    __shared__ float2 stat_s[kSlots];
    const PagedArgs &a = A.a;
    const uint32_t G = A.group.d, D = a.head_dim, here = tile_rows / kRowsHere;
    const uint32_t rest = blockIdx.x / here, kvh = rest % a.kv_heads, target = rest / a.kv_heads;
    const uint32_t tid = threadIdx.x, d = tid % kLanes * 4, slot = tid / kLanes, group = slot % kGroups;
    const uint32_t r = blockIdx.x % here * kRowsHere + slot / kGroups;
    Job job;
    uint32_t item;
    Sequence seq;
    bool bad = false; // (the tiles' own kernel reports it)
    if (!find_item(a, target, [&](const Sequence &s) { return (s.count * G + tile_rows - 1) / tile_rows; }, job.index,
                   seq, item, bad))
        return;
    const uint32_t rows = seq.count * G;
    job.r0 = item * tile_rows;
    job.r1 = job.r0 + tile_rows < rows ? job.r0 + tile_rows : rows;
    job.start = seq.start;
    job.before = static_cast<int32_t>(seq.length) - static_cast<int32_t>(seq.count);
    visible_keys(A, job.before, job.r0, job.r1, job.lo, job.hi);
    const uint32_t count = pieces_of(job.hi - job.lo, A.splits, unit).count;
    if (count <= 1) return;
    job.whole = true;
    const bool mine = job.r0 + r < job.r1 && d < D;
    const uint64_t first = static_cast<uint64_t>(target * a.kv_heads + kvh) * A.splits;
    float top = kNegInf, mass = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine)
#pragma unroll 4
        for (uint32_t i = group; i < count; i += kGroups) {
            const uint64_t at = (first + i) * tile_rows + r;
            const float2 st = A.stats[at];
            const f32x4 x = *reinterpret_cast<const f32x4 *>(A.parts + at * D + d);
            const float next = fmaxf(top, st.x), safe = next == kNegInf ? 0.0f : next;
            const float f = exp2_fast(top - safe), g = exp2_fast(st.x - safe);
            mass = mass * f + st.y * g;
            o = o * f + x * g;
            top = next;
        }
    if constexpr (kGroups > 1) {
        sum_s[tid] = o;
        if (d == 0) stat_s[slot] = make_float2(top, mass);
        __syncthreads();
        if (group != 0) return;
        for (uint32_t i = 1; i < kGroups; ++i) {
            const float2 st = stat_s[slot + i];
            const f32x4 x = sum_s[tid + i * kLanes];
            const float next = fmaxf(top, st.x), safe = next == kNegInf ? 0.0f : next;
            const float f = exp2_fast(top - safe), g = exp2_fast(st.x - safe);
            mass = mass * f + st.y * g;
            o = o * f + x * g;
            top = next;
        }
    }
    if (!mine) return;
    const uint32_t tok = A.group.div(job.r0 + r), head = kvh * G + job.r0 + r - tok * G;
    finish(A, job, tile_rows, r, head, seq.start + tok, d, top, mass, o, lift);
}

// A split is worth its second launch and its sums' way through memory where
// the tiles alone leave CUs idle; never into pieces below one unit of keys.
// Workgroups that a split aims at; an f32 call, whose blocks take 16 times as
// long, aims at kFillLong where the pieces stay of kLongPiece keys and more, so
// that tiles of unequal length end together. (us at 512 / 1280: f32, 11 new tokens
// of 4 sequences over up to 60376 positions, 2 kv heads, 352 / 259; a ragged batch
// of 2544 with a window of 1000, 8 kv heads, 198 / 190; 709 over 1512, 8 heads,
// whose pieces would be shorter than kLongPiece and which so stays at 512, 67 / 75;
// bf16, a prompt of 4096 tokens, 8 kv heads, 159 / 209, for the sums' way through
// memory.)
constexpr uint32_t kFillRows = 2048, kFillTiles = 512, kFillLong = 1280, kLongPiece = 256;
// Rows of a sequence up to which the 16-row kernel takes a call. 32, 64 and 128
// rows of 16 sequences over 4096 positions, 8 kv heads of 128, 16-row / 128-row
// kernel, us: bf16 80 / 57, 126 / 59, 211 / 71; f32 160 / 226, 268 / 407, 485 /
// 420 (an f32 block takes a wavefront's 32 rows as long as its 128-row tile's
// idle wavefronts wait for it; in 16 bits the keys' way to the CU counts).
constexpr uint32_t rows_most(uint32_t type) { return type == FMX_TYPE_F32 ? 64 : 16; }

// Scratch of a split call: stats, then sums.
struct Scratch {
    uint64_t stats, total;
};
Scratch scratch_of(uint64_t tiles, uint32_t kv_heads, uint32_t splits, uint32_t tile_rows, uint32_t head_dim) {
    const uint64_t rows = tiles * kv_heads * splits * tile_rows;
    const uint64_t stats = align_up(rows * sizeof(float2), 256);
    return Scratch{stats, stats + align_up(rows * head_dim * sizeof(float), 256)};
}

uint64_t tiles_of(const PagedArgs &a, uint32_t group, uint32_t tile_rows) {
    return static_cast<uint64_t>(a.tokens) * group / tile_rows + (a.sequences < a.tokens ? a.sequences : a.tokens);
}

template <typename T, int DP> int launch_join(const AttentionArgs &A, uint64_t tiles, uint32_t tile_rows, uint32_t unit,
                                              hipStream_t s) {
    if (A.splits <= 1) return FMX_OK;
    constexpr uint32_t kSlots = kThreads / (DP / 4);
    const bool many = A.splits > 8;
    // (a call is split while its tiles times kv heads are below the workgroups
    // aimed at: a small grid)
    const uint64_t blocks = tiles * A.a.kv_heads * (tile_rows / (many ? 1 : kSlots));
    const auto kernel = many ? attention_join_kernel<DP, kSlots> : attention_join_kernel<DP, 1>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), 0, s, A, tile_rows, unit,
                       Element<T>::kLift);
    FMX_LAUNCH_CHECK();
    return FMX_OK;
}

// Which kernel takes a call, and what it splits into: 16 rows a workgroup while
// a sequence's rows fit few such tiles, else 128.
struct Plan {
    uint32_t tile_rows, unit, splits;
    uint64_t tiles;
};
Plan plan_of(const PagedArgs &a, uint32_t type, uint32_t group, uint32_t window) {
    Plan p;
    const bool rows = static_cast<uint64_t>(a.max_new) * group <= rows_most(type);
    p.tile_rows = rows ? kRows : kTileRows;
    p.unit = rows ? (type == FMX_TYPE_F32 ? 16 : 32) * kWaves : kBlock;
    p.tiles = tiles_of(a, group, p.tile_rows);
    // keys that a tile's rows see, at most
    const uint64_t near = static_cast<uint64_t>(window) + p.tile_rows / group + 8;
    const uint32_t keys = near < a.max_length ? static_cast<uint32_t>(near) : a.max_length;
    const uint64_t blocks = p.tiles * a.kv_heads;
    uint64_t want = ((rows ? kFillRows : kFillTiles) + blocks - 1) / blocks;
    if (!rows && type == FMX_TYPE_F32) {
        const uint64_t finer = (kFillLong + blocks - 1) / blocks, pieces = keys / kLongPiece;
        want = std::max(want, std::min(finer, pieces));
    }
    p.splits = static_cast<uint32_t>(std::min<uint64_t>(want, div_up(keys, p.unit)));
    return p;
}

template <typename T, int DP, int DC, int kParts>
int launch_one(AttentionArgs A, uint8_t *scratch, uint32_t type, hipStream_t s) {
    using Tile = Tile32<T, DP, DC>;
    const Plan p = plan_of(A.a, type, A.group.d, A.window);
    A.splits = p.splits;
    A.stats = reinterpret_cast<float2 *>(scratch);
    A.parts = reinterpret_cast<float *>(scratch + scratch_of(p.tiles, A.a.kv_heads, p.splits, p.tile_rows, A.a.head_dim).stats);
    const uint64_t blocks = p.tiles * A.a.kv_heads * p.splits;
    if (!launch_fits(blocks, kThreads)) return FMX_ERR_SHAPE_MISMATCH;
    const bool rows = p.tile_rows == kRows;
    const size_t lds = rows ? kWaves * kRows * (DP + 4) * sizeof(float)
                            : kBlock * (Tile::kRing * 2 * DP * sizeof(T) + Tile::kGranules);
    // (f32 waits for its loads at every block anyway, so one kernel serves)
    constexpr uint32_t kRowsAtOnce = 1024 / (DP * sizeof(T));
    const bool grouped = sizeof(T) == 2 && A.a.page.d % kRowsAtOnce == 0 && A.a.position_bytes < 1u << 27;
    const auto kernel = rows ? attention_rows_kernel<T, DP>
                        : grouped ? attention_tiles_kernel<T, DP, DC, kParts, sizeof(T) == 2>
                                  : attention_tiles_kernel<T, DP, DC, kParts, false>;
    if (int rc = allow_lds(reinterpret_cast<const void *>(kernel), lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), lds, s, A);
    FMX_LAUNCH_CHECK();
    return launch_join<T, DP>(A, p.tiles, p.tile_rows, p.unit, s);
}

template <typename T, int kParts> int launch_dim(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s) {
    const uint32_t D = A.a.head_dim;
    if (D <= 64) return launch_one<T, 64, 64, kParts>(A, scratch, type, s);
    if (D <= 96) return launch_one<T, 128, 96, kParts>(A, scratch, type, s);
    if (D <= 128) return launch_one<T, 128, 128, kParts>(A, scratch, type, s);
    return launch_one<T, 256, 256, kParts>(A, scratch, type, s);
}

// The prompt kernels' weights go to the matrix cores in all their parts for an
// f32 result. A 16-bit one takes a single part, a weight rounded by half a step at
// most (2^-8 of it in bf16, 2^-11 in f16), since the products bound these kernels:
// one, two and three parts, bf16, 2048 tokens at the end of 16384 positions, 531,
// 690 and 863 us, a prompt of 4096 159, 203 and 250. The error against 64 bits is then
// 1.3 to 1.4 times the result's own rounding, where two parts would leave that.
template <typename T> int launch_type(const AttentionArgs &A, uint8_t *scratch, uint32_t type, hipStream_t s) {
    return A.out_type == FMX_TYPE_F32 ? launch_dim<T, Element<T>::kParts>(A, scratch, type, s)
                                      : launch_dim<T, 1>(A, scratch, type, s);
}

} // namespace

} // namespace fmx
