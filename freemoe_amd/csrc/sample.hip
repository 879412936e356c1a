// sample.hip — one token per row of logits by temperature, top-k, top-p and
// min-p (the choice of FreeMoe's engine.cpp:471-631 from a given uniform
// number).
//
// Tokens in falling order of logit x (equal ones by rising id) carry weights
// w = e^((x - M) / T), M the largest logit. Each filter keeps a prefix of that
// order, so what is kept is the shortest of three prefixes and its mass the
// least of three masses, and the token is the first whose cumulated mass
// exceeds uniform x that mass. A place in the order where a count or a mass
// crosses a target is found by a histogram over equal steps of x, then by the 64
// parts of the one step that holds it, then among that part's few elements, each
// against every other. A small top-k needs no masses but its own: the k-th
// largest of the threads' maxima bounds the k-th logit from below, and what lies
// above that bound is listed in one pass and ordered.
//
// Masses are integers in steps of 2^-44: their sums do not depend on the order
// of the additions (LDS atomics, whichever wavefront comes first).
//
// One workgroup a row, so that a row's passes meet in LDS. One row of 32000 with
// top-k takes 13 us (5.4 to the maximum, launch included, 5 to list what passes
// the bound, 2 to order it); 64 rows of 131072 take 24 us with top-k and 52 with
// top-p alone, 512 rows of 32001 46 us, where a copy would take 6.6, 6.6 and 13:
// the histogram's pass issues some 17 instructions an element on the one CU that
// has the row (18 us for 131072), and each pass after the first waits for L2.
#include "paged.hpp"

namespace fmx {

namespace {

constexpr uint32_t kMaxWaves = 16;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kList = 1024; // elements set aside; as many as a workgroup has threads are compared pair by pair
constexpr uint32_t kMassBits = 44;
static_assert(kSampleMaxVocab <= 1u << 18, "sums of that many masses of at most 2^44 stay below 2^63");

// A top-k up to here is listed through the threads' maxima.
constexpr uint32_t kListedTopK = 256;

struct SampleArgs {
    const float *logits;
    uint64_t row_stride;
    uint32_t vocab;
    fmx_sampling p;
    const float *uniform;
    uint32_t *ids;
    float *probs;
    uint32_t *status;
};

// 2^t for t <= 0 to about 2^-52 of its value: t = i / 64 + r with |r| <= 1 / 128,
// 2^(i / 64 mod 1) from a table times the Taylor sum of 2^r to r^5 (the sixth
// term is below 2^-54).
__device__ __forceinline__ double exp2_table(double t, const double *table) {
    const double n = rint(t * 64.0), r = fma(n, -1.0 / 64.0, t);
    const int i = static_cast<int>(n);
    double s = 0x1.5d87fe78a6731p-10; // ln2^5 / 120
    s = fma(s, r, 0x1.3b2ab6fba4e77p-7);
    s = fma(s, r, 0x1.c6b08d704a0cp-5);
    s = fma(s, r, 0x1.ebfbdff82c58fp-3);
    s = fma(s, r, 0x1.62e42fefa39efp-1);
    const double base = table[i & 63];
    return ldexp(fma(s * r, base, base), i >> 6);
}

// A row's weights. Those of about 1 / 8 of the largest and more, and those next
// to min-p's border, come from double arithmetic ("heavy"); the others, a body
// that matters by its sum, from v_exp_f32 on an exponent t that carries two
// roundings: to (2 |t| ln 2 + 2) 2^-24 of itself, so 2^-24 of the largest weight
// at the very most and 2^-20 of a weight of 2^-10. Weights below 2^-46 are none.
struct Weights {
    float M, c_hi, c_lo;          // log 2 units per logit in two floats
    float heavy, border, passed;  // logits: from `heavy` on, and `border` to `passed` (2^-10 around it), in double
    double M_d, c;
    const double *table;

    __device__ __forceinline__ float exponent(float x) const {
        const float d = x - M;
        return fma_rn(d, c_hi, d * c_lo);
    }
    // d = -inf times a zero c is NaN: no weight, as any exponent not above -46
    static __device__ __forceinline__ bool any(float t) { return t > -46.0f; }
    __device__ __forceinline__ bool is_heavy(float x) const { return x >= heavy || (x >= border && x <= passed); }
    __device__ __forceinline__ double exact(float x) const {
        const double t = (static_cast<double>(x) - M_d) * c;
        return t > -46.0 ? exp2_table(t, table) : 0.0;
    }
    // an integer below 2^45 through the mantissa of 2^52 + it
    static __device__ __forceinline__ uint64_t mass(double w) {
        return __builtin_bit_cast(uint64_t, fma(w, 0x1p44, 0x1p52)) & 0xfffffffffffffull;
    }
    static __device__ __forceinline__ uint64_t light(float t) {
        return mass(static_cast<double>(__builtin_amdgcn_exp2f(t)));
    }
    __device__ __forceinline__ uint64_t of(float x) const {
        const float t = exponent(x);
        if (!any(t)) return 0;
        return is_heavy(x) ? mass(exact(x)) : light(t);
    }
};

// An element's place in the order, as a number: falling logits, then rising ids.
__device__ __forceinline__ uint64_t place_of(float x, uint32_t id) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f); // (-0 is 0)
    return static_cast<uint64_t>(b >> 31 ? b : ~(b | 0x80000000u)) << 32 | id;
}
__device__ __forceinline__ float logit_of(uint64_t place) {
    const uint32_t b = static_cast<uint32_t>(place >> 32);
    return __builtin_bit_cast(float, b >> 31 ? b : ~b & 0x7fffffffu);
}

enum Mode : uint32_t { kCount, kReach, kExceed }; // count >= n; mass >= m; mass > m

struct Target {
    Mode mode;
    uint32_t count;
    double mass;
    __device__ __forceinline__ bool met(uint32_t c, uint64_t m) const {
        return mode == kCount ? c >= count : mode == kReach ? static_cast<double>(m) >= mass
                                                            : static_cast<double>(m) > mass;
    }
};

struct __align__(16) Listed {
    uint64_t place, mass;
};

struct Shared {
    Listed list[kList], few[kList];
    uint64_t mass[kBins];
    uint32_t count[kBins];
    double table[64];
    uint64_t wave_mass[kMaxWaves];
    uint32_t wave_count[kMaxWaves];
    float wave_a[kMaxWaves], wave_b[kMaxWaves];
    bool wave_bad[kMaxWaves];
    uint64_t part_mass[64];
    uint32_t part_count[64];
    uint32_t n, n2, step;
    uint64_t cut_place, cut_mass, kept_by_min;
};

// Steps of x: element x lies in step floor((top - x) * scale), the last one
// taking the rest; monotonic in x, so the steps are stretches of the order.
// (An infinite difference at an infinite temperature: the last, without a weight.)
struct Steps {
    float top, scale;
    __device__ __forceinline__ uint32_t of(float x) const {
        const float d = (top - x) * scale;
        return static_cast<uint32_t>(fminf(d, kBins - 1)); // (a NaN: the last)
    }
    // A step's 64 parts.
    __device__ __forceinline__ uint32_t part(float x, uint32_t step) const {
        const float d = ((top - x) * scale - static_cast<float>(step)) * 64.0f;
        return static_cast<uint32_t>(fminf(fmaxf(d, 0.0f), 63.0f));
    }
    // Logits outside [lo, hi] are not in the step: d above comes to within 2^-22
    // of itself, and a bound rounded to the nearest float passes no float by.
    __device__ __forceinline__ void reach(uint32_t step, float &lo, float &hi) const {
        const double of = scale, t = top;
        lo = scale == 0.0f || step == kBins - 1 ? -__builtin_inff()
                                                : static_cast<float>(t - (step + 1) * (1.0 + 0x1p-20) / of);
        hi = scale == 0.0f || step == 0 ? __builtin_inff() : static_cast<float>(t - step * (1.0 - 0x1p-20) / of);
    }
};

// Inclusive sums over the wavefront, of numbers below 2^63 whose sum is.
__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
    constexpr uint32_t k21 = (1u << 21) - 1;
    const uint64_t a = wave_scan_u32(static_cast<uint32_t>(v) & k21), b = wave_scan_u32(static_cast<uint32_t>(v >> 21) & k21),
                   c = wave_scan_u32(static_cast<uint32_t>(v >> 42));
    return a + (b << 21) + (c << 42);
}

// Inclusive sums of the steps' counts and, kMasses, masses, in place.
template <uint32_t kThreads, bool kMasses = true> __device__ __forceinline__ void scan_steps(Shared &s) {
    constexpr uint32_t kPer = kBins / kThreads, kWaves = kThreads / 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t m[kPer], mi = 0;
    uint32_t c[kPer], ci = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        if (kMasses) mi += s.mass[tid * kPer + i];
        ci += s.count[tid * kPer + i];
        m[i] = mi;
        c[i] = ci;
    }
    const uint64_t own_m = mi;
    const uint32_t own_c = ci;
    ci = wave_scan_u32(ci);
    if (kMasses) mi = wave_scan_u64(mi);
    if (lane == 63) {
        s.wave_mass[wave] = mi;
        s.wave_count[wave] = ci;
    }
    __syncthreads();
    mi -= own_m;
    ci -= own_c;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        if (kMasses) mi += i < wave ? s.wave_mass[i] : 0;
        ci += i < wave ? s.wave_count[i] : 0;
    }
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        if (kMasses) s.mass[tid * kPer + i] = mi + m[i];
        s.count[tid * kPer + i] = ci + c[i];
    }
    __syncthreads();
}

// The row in memory, one element at a time, for the passes few rows need.
template <uint32_t kThreads> struct SlowRow {
    const float *from;
    uint32_t vocab;
    template <class F> __device__ __forceinline__ void each(const F &f) const {
        float next = threadIdx.x < vocab ? from[threadIdx.x] : 0.0f;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
            const float x = next;
            if (i + kThreads < vocab) next = from[i + kThreads];
            f(x, i);
        }
    }
};

// The row, from memory at the first pass and from L2 at the others (held in
// registers, 32 elements a thread, one row of 32000 took 17 us for 12). kWide:
// in 16-byte pieces, kAhead of a thread at a time: piece v holds elements 4 v -
// skew .. + 3, skew being what the row's start lacks to the next lower multiple
// of 16 bytes. Else an element at a time, so that a short row meets every
// thread. A thread's elements come in batches of kBatch; -inf where one
// reaches past the row.
template <uint32_t kThreads, bool kWide> struct Row {
    static constexpr uint32_t kAhead = 8, kBatch = kWide ? 4 * kAhead : 4;
    static constexpr uint32_t kPieces = (kWide ? kAhead : kBatch) * kThreads; // of a batch, all threads
    const float *from;
    uint32_t vocab, skew, pieces;

    __device__ __forceinline__ Row(const float *row, uint32_t n) : from(row), vocab(n) {
        skew = kWide ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) >> 2 & 3) : 0;
        pieces = kWide ? (skew + n + 3) / 4 : n;
    }
    // element r of this thread's batch whose first pieces are b0 on
    __device__ __forceinline__ uint32_t id(uint32_t b0, uint32_t r) const {
        const uint32_t v0 = b0 + threadIdx.x;
        return kWide ? 4 * (v0 + r / 4 * kThreads) + r % 4 - skew : v0 + r * kThreads;
    }
    __device__ __forceinline__ void load(float (&x)[kBatch], uint32_t b0) const {
        if constexpr (!kWide) {
#pragma unroll
            for (uint32_t r = 0; r < kBatch; ++r) x[r] = id(b0, r) < vocab ? from[id(b0, r)] : -__builtin_inff();
        } else {
            const float *const base = from - skew + 4 * static_cast<uint64_t>(b0 + threadIdx.x);
#pragma unroll
            for (uint32_t r = 0; r < kAhead; ++r) {
                const uint32_t v = b0 + r * kThreads; // the workgroup's first piece
                if ((v != 0 || skew == 0) && 4 * (v + kThreads) - skew <= vocab) {
                    const uint4 w = ld16(base + 4 * r * kThreads);
                    x[4 * r] = __builtin_bit_cast(float, w.x);
                    x[4 * r + 1] = __builtin_bit_cast(float, w.y);
                    x[4 * r + 2] = __builtin_bit_cast(float, w.z);
                    x[4 * r + 3] = __builtin_bit_cast(float, w.w);
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t i = id(b0, 4 * r + j); // (below 0: a large number)
                        x[4 * r + j] = i < vocab ? from[i] : -__builtin_inff();
                    }
                }
            }
        }
    }
    template <class F> __device__ __forceinline__ void batches(const F &f) const { // f(elements, first piece)
        for (uint32_t b0 = 0; b0 < pieces; b0 += kPieces) {
            float x[kBatch];
            load(x, b0);
            f(x, b0);
        }
    }
    // f(element, id) for those from lo to hi: few, so four at a time are passed over
    template <class F> __device__ __forceinline__ void between(float lo, float hi, const F &f) const {
        batches([&](const float (&x)[kBatch], uint32_t b0) {
#pragma unroll
            for (uint32_t r = 0; r < kBatch; r += 4) {
                bool in[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) in[j] = x[r + j] >= lo && x[r + j] <= hi;
                if (!(in[0] || in[1] || in[2] || in[3])) continue;
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (in[j]) f(x[r + j], id(b0, r + j));
            }
        });
    }
    template <class F> __device__ __forceinline__ void each(const F &f) const { // f(element, id)
        batches([&](const float (&x)[kBatch], uint32_t b0) {
#pragma unroll
            for (uint32_t r = 0; r < kBatch; ++r) f(x[r], id(b0, r));
        });
    }
};

__device__ __forceinline__ void put(Shared &s, float x, uint32_t i) {
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kList) s.list[at].place = place_of(x, i);
}

// Of the listed elements, whose predecessors hold m0 and number c0: the one at
// which `t` is first met, to s.cut_*. Each against every other, 2^k lanes next
// to each other taking an element's comparisons in turn, as many as the threads
// allow.
template <uint32_t kThreads>
__device__ __forceinline__ void rank_list(Shared &s, const Listed *list, const Target &t, uint32_t listed, uint64_t m0,
                                          uint32_t c0) {
    const uint32_t tid = threadIdx.x;
    uint32_t lanes = 1;
    while (lanes < 32 && listed * lanes * 2 <= kThreads) lanes *= 2;
    const uint32_t e = tid / lanes;
    const uint64_t place = list[e < listed ? e : 0].place;
    uint64_t m = 0;
    uint32_t c = 0;
#pragma unroll 4
    for (uint32_t j = tid % lanes; j < listed; j += lanes) {
        const Listed o = list[j];
        const bool before = o.place < place;
        m += before ? o.mass : 0;
        c += before;
    }
    for (uint32_t d = 1; d < lanes; d <<= 1) {
        m += __shfl_xor(m, d);
        c += __shfl_xor(c, d);
    }
    if (tid % lanes == 0 && e < listed) {
        const uint64_t with = m0 + m + list[e].mass;
        if (t.met(c0 + c + 1, with) && !t.met(c0 + c, m0 + m)) {
            s.cut_place = list[e].place;
            s.cut_mass = with;
        }
    }
    __syncthreads();
}

// The same for a step's elements: the part of the step that meets the target
// first, then that part's few. (s.part_* and s.n2 are 0.)
template <uint32_t kThreads>
__device__ __forceinline__ void rank_step(Shared &s, const Steps &steps, uint32_t step, const Target &t, uint32_t listed,
                                          uint64_t m0, uint32_t c0) {
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t part = tid < listed ? steps.part(logit_of(s.list[tid].place), step) : 64;
    if (tid < listed) {
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.part_mass[part]), s.list[tid].mass);
        atomicAdd(&s.part_count[part], 1u);
    }
    __syncthreads();
    const uint64_t own = s.part_mass[lane];
    const uint32_t own_c = s.part_count[lane];
    const uint64_t m = m0 + wave_scan_u64(own);
    const uint32_t c = c0 + wave_scan_u32(own_c);
    const uint64_t met = __ballot(t.met(c, m));
    const int at = met ? __builtin_ctzll(met) : 63;
    if (part == static_cast<uint32_t>(at)) s.few[atomicAdd(&s.n2, 1u)] = s.list[tid];
    __syncthreads();
    rank_list<kThreads>(s, s.few, t, s.n2, __shfl(m - own, at), __shfl(c - own_c, at));
}

// A stretch of the order with more elements than the list takes, those with lo
// <= x <= hi: narrowed by finer and finer steps, or, where all are equal,
// counted off by id. Fills s.cut_* and returns true, or leaves the stretch's
// bounds, mass and count for the list.
template <uint32_t kThreads>
__device__ __forceinline__ bool narrow(Shared &s, SlowRow<kThreads> row, Weights w, Target t, float &hi, float &lo, uint64_t &m0,
                                    uint32_t &c0, uint32_t &n) {
    constexpr uint32_t kWaves = kThreads / 64;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr float kInf = __builtin_inff();
    // (the steps' sums have served; their arrays hold the finer ones)
    const auto bounds = [&](float &a, float &b, auto in) {
        a = -kInf;
        b = kInf;
        row.each([&](float x, uint32_t) {
            if (in(x) && Weights::any(w.exponent(x))) {
                a = fmaxf(a, x);
                b = fminf(b, x);
            }
        });
        for (uint32_t d = 32; d >= 1; d >>= 1) {
            a = fmaxf(a, __shfl_xor(a, d));
            b = fminf(b, __shfl_xor(b, d));
        }
        __syncthreads();
        if (lane == 0) {
            s.wave_a[wave] = a;
            s.wave_b[wave] = b;
        }
        __syncthreads();
        for (uint32_t i = 0; i < kWaves; ++i) {
            a = fmaxf(a, s.wave_a[i]);
            b = fminf(b, s.wave_b[i]);
        }
    };
    while (n > kThreads) {
        float a, b;
        bounds(a, b, [&](float x) { return x <= hi && x >= lo; });
        if (a == b) {
            const uint64_t m = w.of(a);
            uint32_t least = 1, most = n; // the smallest count that meets the target
            while (least < most) {
                const uint32_t mid = (least + most) / 2;
                if (t.met(c0 + mid, m0 + mid * m)) most = mid;
                else least = mid + 1;
            }
            uint32_t left = least;
            for (uint32_t i0 = 0; i0 < row.vocab; i0 += kThreads) {
                const uint32_t i = i0 + tid;
                const bool here = i < row.vocab && row.from[i] == a;
                const uint64_t vote = __ballot(here);
                __syncthreads();
                if (lane == 0) s.wave_count[wave] = __builtin_popcountll(vote);
                __syncthreads();
                uint32_t before = 0, all = 0;
                for (uint32_t k = 0; k < kWaves; ++k) {
                    before += k < wave ? s.wave_count[k] : 0;
                    all += s.wave_count[k];
                }
                if (left > all) {
                    left -= all;
                    continue;
                }
                before += __builtin_popcountll(vote & ((uint64_t{1} << lane) - 1));
                if (here && before + 1 == left) {
                    s.cut_place = place_of(a, i);
                    s.cut_mass = m0 + least * m;
                }
                break;
            }
            __syncthreads();
            return true;
        }
        __syncthreads();
        for (uint32_t i = tid; i < kBins; i += kThreads) {
            s.mass[i] = 0;
            s.count[i] = 0;
        }
        __syncthreads();
        const double per = (kBins - 1) / (static_cast<double>(a) - static_cast<double>(b));
        const auto step_of = [&](float x) {
            const double d = (static_cast<double>(a) - static_cast<double>(x)) * per;
            return d < kBins - 1 ? static_cast<uint32_t>(d) : kBins - 1;
        };
        row.each([&](float x, uint32_t) {
            if (!(x <= hi && x >= lo)) return;
            if (!Weights::any(w.exponent(x))) return;
            const uint32_t f = step_of(x);
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[f]), w.of(x));
            atomicAdd(&s.count[f], 1u);
        });
        __syncthreads();
        scan_steps<kThreads>(s);
        for (uint32_t i = tid; i < kBins; i += kThreads)
            if (t.met(c0 + s.count[i], m0 + s.mass[i]) && (i == 0 || !t.met(c0 + s.count[i - 1], m0 + s.mass[i - 1])))
                s.step = i;
        __syncthreads();
        const uint32_t f = s.step;
        const uint64_t fm = f ? s.mass[f - 1] : 0;
        const uint32_t fc = f ? s.count[f - 1] : 0;
        n = s.count[f] - fc;
        m0 += fm;
        c0 += fc;
        const float was_hi = hi, was_lo = lo;
        bounds(hi, lo, [&](float x) { return x <= was_hi && x >= was_lo && step_of(x) == f; });
    }
    return false;
}

// grid: rows.
template <uint32_t kThreads, bool kWide> __global__ __launch_bounds__(kThreads, 4) void sample_kernel(SampleArgs A) {
    constexpr uint32_t kWaves = kThreads / 64;
    __shared__ Shared s;
    constexpr float kInf = __builtin_inff();
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, V = A.vocab;
    const Row<kThreads, kWide> row(A.logits + r * A.row_stride, V);
    const SlowRow<kThreads> slow{row.from, V};
    const float temperature = A.p.temperature ? A.p.temperature[r] : 1.0f;
    const uint32_t top_k = A.p.top_k ? A.p.top_k[r] : 0;
    const float top_p = A.p.top_p ? A.p.top_p[r] : 1.0f, min_p = A.p.min_p ? A.p.min_p[r] : 0.0f;
    const float uniform = A.uniform[r];
    for (uint32_t i = tid; i < kBins; i += kThreads) {
        s.mass[i] = 0;
        s.count[i] = 0;
    }
    if (tid < 64) s.table[tid] = exp2(tid / 64.0);
    if (tid == 0) {
        s.n = 0;
        s.kept_by_min = 0;
    }

    // the largest and the smallest logit
    float high = -kInf, low = kInf;
    bool bad = false;
    row.batches([&](const float (&x)[row.kBatch], uint32_t) {
#pragma unroll
        for (uint32_t i = 0; i < row.kBatch; i += 2) {
            bad |= x[i] != x[i] || x[i + 1] != x[i + 1];
            high = fmaxf(fmaxf(x[i], x[i + 1]), high);
            low = fminf(fminf(x[i], x[i + 1]), low);
        }
    });
    const float own_high = high;
    for (uint32_t d = 32; d >= 1; d >>= 1) {
        high = fmaxf(high, __shfl_xor(high, d));
        low = fminf(low, __shfl_xor(low, d));
    }
    bad = __any(bad);
    if (lane == 0) {
        s.wave_a[wave] = high;
        s.wave_b[wave] = low;
        s.wave_bad[wave] = bad;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        bad |= s.wave_bad[i];
        high = fmaxf(high, s.wave_a[i]);
        low = fminf(low, s.wave_b[i]);
    }
    bad |= !__builtin_isfinite(high) || !(temperature >= 0.0f) || top_p != top_p || min_p != min_p || uniform != uniform;
    if (bad) {
        if (tid == 0) {
            A.ids[r] = 0xffffffffu;
            if (A.probs) A.probs[r] = 0.0f;
            atomicOr(A.status, STATUS_NONFINITE_SCORE);
        }
        return;
    }
    if (temperature == 0.0f) { // the lowest id of the largest
        if (tid == 0) s.step = 0xffffffffu;
        __syncthreads();
        row.each([&](float x, uint32_t i) {
            if (x == high) atomicMin(&s.step, i);
        });
        __syncthreads();
        if (tid == 0) {
            A.ids[r] = s.step;
            if (A.probs) A.probs[r] = 1.0f;
        }
        return;
    }
    Weights w;
    w.M = high;
    w.M_d = high;
    w.c = 1.4426950408889634 / static_cast<double>(temperature);
    // (temperatures near 0, where a float does not hold the factor: all in double)
    const bool small = w.c < 0x1p100;
    w.c_hi = small ? static_cast<float>(w.c) : 0x1p100f;
    w.c_lo = small ? static_cast<float>(w.c - static_cast<double>(w.c_hi)) : 0.0f;
    w.heavy = small ? static_cast<float>(w.M_d - 3.0 / w.c) : -kInf;
    w.border = w.passed = kInf;
    if (min_p > 0.0f) {
        const double at = __builtin_amdgcn_logf(min_p); // (log 2)
        w.border = static_cast<float>(w.M_d + (at - 0x1p-10) / w.c);
        w.passed = static_cast<float>(w.M_d + (at + 0x1p-10) / w.c);
    }
    w.table = s.table;
    const double reach = 46.0 / w.c, span = fmin(static_cast<double>(high) - static_cast<double>(low), reach); // (low: -inf too)
    const Steps steps{high, span > 0.0 ? static_cast<float>(fmin((kBins - 1) / span, 0x1p126)) : 0.0f};
    const float u = fminf(fmaxf(uniform, 0.0f), 0x1.fffffep-1f);

    // A small top-k: the k-th largest of the threads' maxima, or one a little
    // below, bounds the k-th logit; what reaches it is listed. (Fewer than k
    // threads with a weight: all that have one.)
    if (top_k != 0 && top_k <= kListedTopK) {
        const uint32_t own_step = steps.of(own_high);
        const bool weighs = Weights::any(w.exponent(own_high));
        if (weighs) atomicAdd(&s.count[own_step], 1u);
        if (tid == 0) s.step = kBins - 1;
        __syncthreads();
        scan_steps<kThreads, false>(s);
        for (uint32_t i = tid; i < kBins; i += kThreads)
            if (s.count[i] >= top_k && (i == 0 || s.count[i - 1] < top_k)) s.step = i;
        __syncthreads();
        const bool enough = s.count[kBins - 1] >= top_k;
        float least = weighs && own_step <= s.step ? own_high : kInf;
        for (uint32_t d = 32; d >= 1; d >>= 1) least = fminf(least, __shfl_xor(least, d));
        if (lane == 0) s.wave_a[wave] = least;
        __syncthreads();
        for (uint32_t i = tid; i < kBins; i += kThreads) s.count[i] = 0;
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i) least = fminf(least, s.wave_a[i]);
        __syncthreads();
        row.between(enough ? least : -kInf, kInf, [&](float x, uint32_t i) {
            if (!Weights::any(w.exponent(x))) return;
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < kThreads) s.list[at] = Listed{place_of(x, i), atomicAdd(&s.count[steps.of(x)], 1u)};
        });
        __syncthreads();
        const uint32_t listed = s.n, k = top_k < listed ? top_k : listed;
        if (listed <= kThreads) {
            // sorted: by steps, each element's number within its step having come
            // with the count, then within a step against its few others
            scan_steps<kThreads, false>(s);
            uint64_t place = 0, own = 0, with = 0;
            uint32_t rank = 0, end = 0;
            if (tid < listed) {
                place = s.list[tid].place;
                const float x = logit_of(place);
                const uint32_t step = steps.of(x);
                own = w.of(x);
                rank = step ? s.count[step - 1] : 0;
                end = s.count[step];
                s.few[rank + s.list[tid].mass].place = place;
            }
            __syncthreads();
            if (tid < listed) {
                uint32_t to = rank;
                for (uint32_t j = rank; j < end; ++j) to += s.few[j].place < place;
                s.list[to] = Listed{place, own};
            }
            __syncthreads();
            double weight = 0.0;
            own = tid < listed ? s.list[tid].mass : 0;
            place = tid < listed ? s.list[tid].place : 0;
            with = wave_scan_u64(own);
            if (lane == 63) s.wave_mass[wave] = with;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kWaves; ++i) with += i < wave ? s.wave_mass[i] : 0;
            const uint64_t before = with - own;
            const bool mine = tid < k;
            if (mine) weight = w.exact(logit_of(place));
            if (tid + 1 == k) s.cut_mass = with;
            __syncthreads();
            uint64_t kept = s.cut_mass;
            __syncthreads();
            if (top_p < 1.0f) {
                const double least = fmax(static_cast<double>(top_p) * static_cast<double>(kept), 1.0);
                if (mine && static_cast<double>(with) >= least && static_cast<double>(before) < least) s.cut_mass = with;
                __syncthreads();
                kept = s.cut_mass < kept ? s.cut_mass : kept;
            }
            if (min_p > 0.0f) {
                if (mine && weight >= static_cast<double>(min_p))
                    atomicMax(reinterpret_cast<unsigned long long *>(&s.kept_by_min), with);
                __syncthreads();
                const uint64_t least = s.kept_by_min ? s.kept_by_min : uint64_t{1} << kMassBits; // the largest at least
                kept = least < kept ? least : kept;
            }
            const double exceed = static_cast<double>(u) * static_cast<double>(kept);
            if (mine && static_cast<double>(with) > exceed && !(static_cast<double>(before) > exceed)) {
                A.ids[r] = static_cast<uint32_t>(place);
                if (A.probs) A.probs[r] = static_cast<float>(weight * 0x1p44 / static_cast<double>(kept));
            }
            return;
        }
    }

    // The steps' masses (and counts, for a large top-k), and the mass that min-p
    // keeps. The heavy weights wait in the list, so that the others' code is
    // short; where they are more than it takes, they come from a pass of their
    // own.
    const bool counted = top_k != 0;
    __syncthreads();
    for (uint32_t i = tid; i < kBins; i += kThreads) s.count[i] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    uint64_t by_min = 0;
    const bool bordered = min_p > 0.0f;
    row.batches([&](const float (&x)[row.kBatch], uint32_t b0) {
#pragma unroll
        for (uint32_t q = 0; q < row.kBatch; q += 4) { // four side by side, since each is a chain of slow instructions
            const float most = fmaxf(fmaxf(x[q], x[q + 1]), fmaxf(x[q + 2], x[q + 3]));
            if (!Weights::any(w.exponent(most))) continue;
            float t[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) t[j] = fmaxf(w.exponent(x[q + j]), -64.0f); // (from -inf or NaN too)
            bool some = most >= w.heavy;
            if (bordered)
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) some |= x[q + j] >= w.border && x[q + j] <= w.passed;
            if (some)
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (w.is_heavy(x[q + j]) && Weights::any(t[j])) {
                        put(s, x[q + j], row.id(b0, q + j));
                        t[j] = -64.0f;
                    }
            uint64_t m[4];
            uint32_t b[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                m[j] = Weights::light(t[j]); // 0 up to -46
                b[j] = steps.of(x[q + j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[b[j]]), m[j]);
            if (counted)
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) atomicAdd(&s.count[b[j]], Weights::any(t[j]) ? 1u : 0u);
            if (bordered)
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) by_min += x[q + j] > w.passed ? m[j] : 0;
        }
    });
    __syncthreads();
    const auto heavy = [&](float x) {
        const double weight = w.exact(x);
        const uint64_t m = Weights::mass(weight);
        const uint32_t b = steps.of(x);
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[b]), m);
        if (counted) atomicAdd(&s.count[b], 1u);
        if (weight >= static_cast<double>(min_p)) by_min += m;
    };
    const uint32_t heavies = s.n;
    if (heavies <= kList) {
        for (uint32_t i = tid; i < heavies; i += kThreads) heavy(logit_of(s.list[i].place));
    } else {
        slow.each([&](float x, uint32_t) {
            const float t = w.exponent(x);
            if (Weights::any(t) && w.is_heavy(x)) heavy(x);
        });
    }
    if (min_p > 0.0f && by_min) atomicAdd(reinterpret_cast<unsigned long long *>(&s.kept_by_min), by_min);
    __syncthreads();
    scan_steps<kThreads>(s);
    uint64_t kept = s.mass[kBins - 1];
    const uint64_t kept_by_min = s.kept_by_min;
    const uint32_t weighted = s.count[kBins - 1];

    // top-k, top-p and the choice itself, each a target that some element first
    // meets
    bool spoiled = false; // narrow() has taken the steps' arrays
#pragma unroll 1
    for (uint32_t stage = 0; stage < 3; ++stage) {
        Target t;
        if (stage == 0) {
            if (!counted || top_k >= weighted) continue;
            t = Target{kCount, top_k, 0.0};
        } else if (stage == 1) {
            if (!(top_p < 1.0f)) continue;
            t = Target{kReach, 0, fmax(static_cast<double>(top_p) * static_cast<double>(kept), 1.0)};
        } else {
            if (min_p > 0.0f) {
                const uint64_t least = kept_by_min ? kept_by_min : uint64_t{1} << kMassBits; // the largest at least
                kept = least < kept ? least : kept;
            }
            t = Target{kExceed, 0, static_cast<double>(u) * static_cast<double>(kept)};
        }
        uint64_t m0 = 0;
        uint32_t c0 = 0, step = 0;
        float hi = high, lo = -kInf;
        if (tid == 0) s.n = s.n2 = 0;
        if (tid < 64) {
            s.part_mass[tid] = 0;
            s.part_count[tid] = 0;
        }
        if (!spoiled) {
            for (uint32_t i = tid; i < kBins; i += kThreads)
                if (t.met(s.count[i], s.mass[i]) && (i == 0 || !t.met(s.count[i - 1], s.mass[i - 1]))) s.step = i;
            __syncthreads();
            step = s.step;
            m0 = step ? s.mass[step - 1] : 0;
            c0 = step && counted ? s.count[step - 1] : 0;
            float from, to;
            steps.reach(step, from, to);
            row.between(from, to, [&](float x, uint32_t i) {
                if (steps.of(x) == step && Weights::any(w.exponent(x))) put(s, x, i);
            });
        } else {
            __syncthreads();
            slow.each([&](float x, uint32_t i) {
                if (Weights::any(w.exponent(x))) put(s, x, i);
            });
        }
        __syncthreads();
        uint32_t n = s.n;
        const bool in_step = !spoiled && n <= kThreads && n > 32;
        if (n > kThreads) {
            if (!spoiled) { // the step's bounds
                float a = -kInf, b = kInf;
                slow.each([&](float x, uint32_t) {
                    if (steps.of(x) == step && Weights::any(w.exponent(x))) {
                        a = fmaxf(a, x);
                        b = fminf(b, x);
                    }
                });
                for (uint32_t d = 32; d >= 1; d >>= 1) {
                    a = fmaxf(a, __shfl_xor(a, d));
                    b = fminf(b, __shfl_xor(b, d));
                }
                if (lane == 0) {
                    s.wave_a[wave] = a;
                    s.wave_b[wave] = b;
                }
                __syncthreads();
                for (uint32_t i = 0; i < kWaves; ++i) {
                    a = fmaxf(a, s.wave_a[i]);
                    b = fminf(b, s.wave_b[i]);
                }
                hi = a;
                lo = b;
            }
            spoiled = true;
            const bool found = narrow(s, slow, w, t, hi, lo, m0, c0, n);
            if (found) {
                if (stage < 2) kept = s.cut_mass < kept ? s.cut_mass : kept;
                __syncthreads();
                continue;
            }
            if (tid == 0) s.n = 0;
            __syncthreads();
            slow.each([&](float x, uint32_t i) {
                if (x <= hi && x >= lo && Weights::any(w.exponent(x))) put(s, x, i);
            });
            __syncthreads();
            n = s.n;
        }
        if (tid < n) s.list[tid].mass = w.of(logit_of(s.list[tid].place));
        __syncthreads();
        if (in_step) rank_step<kThreads>(s, steps, step, t, n, m0, c0);
        else rank_list<kThreads>(s, s.list, t, n, m0, c0);
        if (stage < 2) kept = s.cut_mass < kept ? s.cut_mass : kept;
        __syncthreads();
    }
    if (tid == 0) {
        A.ids[r] = static_cast<uint32_t>(s.cut_place);
        if (A.probs)
            A.probs[r] = static_cast<float>(w.exact(logit_of(s.cut_place)) * 0x1p44 / static_cast<double>(kept));
    }
}

} // namespace

uint64_t sample_scratch(uint32_t, uint32_t) { return 0; }

int sample(const float *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const fmx_sampling &p,
           const float *uniform, uint32_t *ids, float *probs, uint32_t *status, uint8_t *, hipStream_t s) {
    const SampleArgs A{logits, row_stride, vocab, p, uniform, ids, probs, status};
    // Two workgroups of 512 threads share a CU, one of 1024 fills it: 1024 where
    // every row has a CU to itself, 512 where rows are more than CUs. us at 1024 / 512
    // threads, top-p: 64 rows of 131072 54 / 66, 256 of 32001 36.5 / 34.6, 300 58 / 40,
    // 511 63 / 46, 1000 120 / 86; with top-k, 64 of 131072 24.6 / 27.5, 256 of 32001
    // 21.6 / 22.4, 300 31 / 22.
    constexpr uint32_t kCus = 256;
    const uint32_t threads = rows > kCus ? kSampleThreads : 1024;
    const bool wide = vocab > 4 * threads;
    constexpr uint32_t kMany = kSampleThreads;
    const auto kernel = threads == kMany ? (wide ? sample_kernel<kMany, true> : sample_kernel<kMany, false>)
                                         : (wide ? sample_kernel<1024, true> : sample_kernel<1024, false>);
    hipLaunchKernelGGL(kernel, dim3(rows), dim3(threads), 0, s, A);
    FMX_LAUNCH_CHECK();
    return FMX_OK;
}

} // namespace fmx
