// sample.hip — one token per row of logits by temperature, top-k, top-p and
// min-p (the choice of FreeMoe's engine.cpp:471-631 from a given uniform
// number).
//
// Tokens in falling order of logit x (equal ones by rising id) carry weights
// w = e^((x - M) / T), M the largest logit. Each filter keeps a prefix of that
// order, so what is kept is the shortest of three prefixes and its mass the
// least of three masses, and the token is the first whose cumulated mass
// exceeds uniform x that mass. Nothing is sorted: a place in the order where a
// count or a mass crosses a target is found by a histogram over equal steps of
// x, then among the elements of the one step that holds it, every one against
// every other. A small top-k needs no masses but its own: the steps down to
// the k-th logit are taken out at once.
//
// Masses are integers in steps of 2^-44: their sums do not depend on the order
// of the additions (LDS atomics, whichever wavefront comes first).
#include "paged.hpp"

namespace fmx {

namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWaves = kThreads / 64;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kList = 1024;  // elements compared pair by pair
constexpr uint32_t kMassBits = 44;
static_assert(kSampleMaxVocab <= 1u << 18, "sums of that many masses of at most 2^44 stay below 2^63");

// A top-k up to here is taken out by counts (the list holds it and the rest of
// its last step).
constexpr uint32_t kCountedTopK = 512;

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

// A row's weights. Those of at least 2^-8 of the largest, and all that min-p
// might keep, come from double arithmetic; the others, a body that matters by
// its sum, from v_exp_f32 on a product carried to 2^-24 of the exponent (about
// 2^-20 of each weight, at most 2^-28 of the largest, in either direction).
// Weights below 2^-46 are none.
struct Weights {
    float M, c_hi, c_lo, heavy; // log 2 units per logit in two floats; exponents from `heavy` on in double
    double M_d, c;
    const double *table;

    __device__ __forceinline__ float exponent(float x) const {
        const float d = x - M;
        return fma_rn(d, c_hi, d * c_lo);
    }
    // d = -inf times a zero c is NaN: no weight, as any exponent not above -46
    static __device__ __forceinline__ bool any(float t) { return t > -46.0f; }
    __device__ __forceinline__ uint64_t light(float t) const {
        return static_cast<uint64_t>(static_cast<uint32_t>(fma_rn(__builtin_amdgcn_exp2f(t), 0x1p40f, 0.5f))) << 4;
    }
    __device__ __forceinline__ double exact(float x) const {
        const double t = (static_cast<double>(x) - M_d) * c;
        return t > -46.0 ? exp2_table(t, table) : 0.0;
    }
    // an integer below 2^45 through the mantissa of 2^52 + it
    static __device__ __forceinline__ uint64_t mass(double w) {
        return __builtin_bit_cast(uint64_t, w * 0x1p44 + 0x1p52) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ uint64_t of(float x) const {
        const float t = exponent(x);
        if (!any(t)) return 0;
        return t >= heavy ? mass(exact(x)) : light(t);
    }
};

__device__ __forceinline__ bool precedes(float xa, uint32_t ia, float xb, uint32_t ib) {
    return xa > xb || (xa == xb && ia < ib);
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

struct Shared {
    uint64_t mass[kBins], list_mass[kList];
    uint32_t count[kBins];
    float list_x[kList];
    uint32_t list_id[kList];
    double table[64];
    uint64_t wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float wave_a[kWaves], wave_b[kWaves];
    uint32_t wave_id[kWaves];
    bool wave_bad[kWaves];
    uint32_t n, step;
    float cut_x;
    uint32_t cut_id;
    uint64_t cut_mass, kept_by_min;
};

// Steps of x: element x lies in step floor((top - x) * scale), the last one
// taking the rest; monotonic in x, so the steps are stretches of the order.
// (An infinite difference at an infinite temperature: scale 0, step 0.)
struct Steps {
    float top, scale;
    __device__ __forceinline__ uint32_t of(float x) const {
        const float d = (top - x) * scale;
        return d < static_cast<float>(kBins - 1) ? static_cast<uint32_t>(d) : d > 0.0f ? kBins - 1 : 0;
    }
};

// Inclusive sums of the steps' masses and counts, in place.
__device__ __forceinline__ void scan_steps(Shared &s) {
    constexpr uint32_t kPer = kBins / kThreads;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t m[kPer], mi = 0;
    uint32_t c[kPer], ci = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        mi += s.mass[tid * kPer + i];
        ci += s.count[tid * kPer + i];
        m[i] = mi;
        c[i] = ci;
    }
    const uint64_t own_m = mi;
    const uint32_t own_c = ci;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t mo = __shfl_up(mi, d);
        const uint32_t co = __shfl_up(ci, d);
        mi += lane >= d ? mo : 0;
        ci += lane >= d ? co : 0;
    }
    if (lane == 63) {
        s.wave_mass[wave] = mi;
        s.wave_count[wave] = ci;
    }
    __syncthreads();
    mi -= own_m;
    ci -= own_c;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        mi += i < wave ? s.wave_mass[i] : 0;
        ci += i < wave ? s.wave_count[i] : 0;
    }
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        s.mass[tid * kPer + i] = mi + m[i];
        s.count[tid * kPer + i] = ci + c[i];
    }
    __syncthreads();
}

// The row in memory, one element at a time, for the passes few rows need.
struct SlowRow {
    const float *from;
    uint32_t vocab;
    template <class F> __device__ __forceinline__ void each(const F &f) const {
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) f(from[i], i);
    }
};

// The row: kHeld elements a thread in registers, or (0) read again at each
// pass, from L2.
template <uint32_t kHeld> struct Row {
    float held[kHeld ? kHeld : 1];
    const float *from;
    uint32_t vocab;
    __device__ __forceinline__ void load() {
        if constexpr (kHeld > 0)
#pragma unroll
            for (uint32_t r = 0; r < kHeld; ++r) {
                const uint32_t i = r * kThreads + threadIdx.x;
                held[r] = i < vocab ? from[i] : -__builtin_inff();
            }
    }
    template <class F> __device__ __forceinline__ void each(const F &f) const {
        if constexpr (kHeld > 0) {
#pragma unroll
            for (uint32_t r = 0; r < kHeld; ++r) f(held[r], r * kThreads + threadIdx.x);
        } else {
            constexpr uint32_t kAhead = 8;
            for (uint32_t i0 = threadIdx.x; i0 < vocab; i0 += kAhead * kThreads) {
                float x[kAhead];
#pragma unroll
                for (uint32_t r = 0; r < kAhead; ++r) {
                    const uint32_t i = i0 + r * kThreads;
                    x[r] = i < vocab ? from[i] : -__builtin_inff();
                }
#pragma unroll
                for (uint32_t r = 0; r < kAhead; ++r) f(x[r], i0 + r * kThreads);
            }
        }
    }
};

__device__ __forceinline__ void put(Shared &s, float x, uint32_t i) {
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kList) {
        s.list_x[at] = x;
        s.list_id[at] = i;
    }
}

// Of the listed elements, whose predecessors hold m0 and number c0: the one at
// which `t` is first met, to s.cut_*.
__device__ __forceinline__ void rank_list(Shared &s, const Target &t, uint32_t listed, uint64_t m0, uint32_t c0) {
    const uint32_t tid = threadIdx.x;
    if (tid < listed) {
        const float x = s.list_x[tid];
        const uint32_t id = s.list_id[tid];
        uint64_t m = m0;
        uint32_t c = c0;
#pragma unroll 4
        for (uint32_t j = 0; j < listed; ++j)
            if (precedes(s.list_x[j], s.list_id[j], x, id)) {
                m += s.list_mass[j];
                ++c;
            }
        const uint64_t with = m + s.list_mass[tid];
        if (t.met(c + 1, with) && !t.met(c, m)) {
            s.cut_x = x;
            s.cut_id = id;
            s.cut_mass = with;
        }
    }
    __syncthreads();
}

// A stretch of the order with more elements than the list takes, those with lo
// <= x <= hi: narrowed by finer and finer steps, or, where all are equal,
// counted off by id. Fills s.cut_* and returns true, or leaves the stretch's
// bounds, mass and count for the list.
__device__ __forceinline__ bool narrow(Shared &s, SlowRow row, Weights w, Target t, float &hi, float &lo, uint64_t &m0,
                                    uint32_t &c0, uint32_t &n) {
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
    while (n > kList) {
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
                    s.cut_x = a;
                    s.cut_id = i;
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
        scan_steps(s);
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
template <uint32_t kHeld> __global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs A) {
    __shared__ Shared s;
    constexpr float kInf = __builtin_inff();
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, V = A.vocab;
    Row<kHeld> row;
    row.from = A.logits + r * A.row_stride;
    row.vocab = V;
    row.load();
    const SlowRow slow{row.from, V};
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

    // the largest logit (its lowest id) and the smallest finite one
    float high = -kInf, low = kInf;
    uint32_t high_id = 0xffffffffu;
    bool bad = false;
    row.each([&](float x, uint32_t i) {
        bad |= !(x < kInf);
        high_id = x > high ? i : high_id;
        high = fmaxf(high, x);
        low = fminf(low, x > -kInf ? x : kInf);
    });
    for (uint32_t d = 32; d >= 1; d >>= 1) {
        const float h = __shfl_xor(high, d);
        const uint32_t id = __shfl_xor(high_id, d);
        if (precedes(h, id, high, high_id)) {
            high = h;
            high_id = id;
        }
        low = fminf(low, __shfl_xor(low, d));
    }
    bad = __any(bad);
    if (lane == 0) {
        s.wave_a[wave] = high;
        s.wave_b[wave] = low;
        s.wave_id[wave] = high_id;
        s.wave_bad[wave] = bad;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) {
        bad |= s.wave_bad[i];
        if (precedes(s.wave_a[i], s.wave_id[i], high, high_id)) {
            high = s.wave_a[i];
            high_id = s.wave_id[i];
        }
        low = fminf(low, s.wave_b[i]);
    }
    bad |= high == -kInf || !(temperature >= 0.0f) || top_p != top_p || min_p != min_p || uniform != uniform;
    if (bad || temperature == 0.0f) {
        if (tid == 0) {
            A.ids[r] = bad ? 0xffffffffu : high_id;
            if (A.probs) A.probs[r] = bad ? 0.0f : 1.0f;
            if (bad) atomicOr(A.status, STATUS_NONFINITE_SCORE);
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
    w.heavy = !small ? -kInf : min_p > 0.0f ? fminf(-8.0f, __builtin_amdgcn_logf(min_p) - 0.125f) : -8.0f; // (log 2)
    w.table = s.table;
    const double reach = 46.0 / w.c, span = fmin(static_cast<double>(high) - static_cast<double>(low), reach);
    const Steps steps{high, span > 0.0 ? static_cast<float>(fmin((kBins - 1) / span, 0x1p126)) : 0.0f};
    const float u = fminf(fmaxf(uniform, 0.0f), 0x1.fffffep-1f);

    // A small top-k: count, and list the steps down to the one that holds the
    // k-th.
    if (top_k != 0 && top_k <= kCountedTopK) {
        row.each([&](float x, uint32_t) {
            if (Weights::any(w.exponent(x))) atomicAdd(&s.count[steps.of(x)], 1u);
        });
        __syncthreads();
        scan_steps(s); // (no masses)
        const uint32_t weighted = s.count[kBins - 1], k = top_k < weighted ? top_k : weighted;
        for (uint32_t i = tid; i < kBins; i += kThreads)
            if (s.count[i] >= k && (i == 0 || s.count[i - 1] < k)) s.step = i;
        __syncthreads();
        const uint32_t step = s.step, listed = s.count[step];
        if (listed <= kList) {
            row.each([&](float x, uint32_t i) {
                if (steps.of(x) <= step && Weights::any(w.exponent(x))) put(s, x, i);
            });
            __syncthreads();
            // every element's predecessors: their number and mass
            uint64_t m = 0, own = 0;
            uint32_t c = 0, id = 0;
            float x = 0.0f;
            const bool mine = tid < listed;
            double weight = 0.0;
            if (mine) {
                x = s.list_x[tid];
                id = s.list_id[tid];
                weight = w.exact(x);
                own = w.of(x);
                s.list_mass[tid] = own;
            }
            __syncthreads();
            if (mine)
#pragma unroll 4
                for (uint32_t j = 0; j < listed; ++j)
                    if (precedes(s.list_x[j], s.list_id[j], x, id)) {
                        m += s.list_mass[j];
                        ++c;
                    }
            if (mine && c + 1 == k) s.cut_mass = m + own;
            __syncthreads();
            uint64_t kept = s.cut_mass;
            const double reach_p = fmax(static_cast<double>(top_p) * static_cast<double>(kept), 1.0);
            __syncthreads();
            if (top_p < 1.0f) {
                if (mine && static_cast<double>(m + own) >= reach_p && static_cast<double>(m) < reach_p) s.cut_mass = m + own;
                __syncthreads();
                kept = s.cut_mass < kept ? s.cut_mass : kept;
            }
            if (min_p > 0.0f) {
                if (mine && weight >= static_cast<double>(min_p))
                    atomicMax(reinterpret_cast<unsigned long long *>(&s.kept_by_min), m + own);
                __syncthreads();
                const uint64_t least = s.kept_by_min ? s.kept_by_min : uint64_t{1} << kMassBits; // the largest at least
                kept = least < kept ? least : kept;
            }
            const double exceed = static_cast<double>(u) * static_cast<double>(kept);
            if (mine && static_cast<double>(m + own) > exceed && !(static_cast<double>(m) > exceed)) {
                A.ids[r] = id;
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
    row.each([&](float x, uint32_t i) {
        const float t = w.exponent(x);
        if (!Weights::any(t)) return;
        if (t >= w.heavy) {
            put(s, x, i);
            return;
        }
        const uint32_t b = steps.of(x);
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[b]), w.light(t));
        if (counted) atomicAdd(&s.count[b], 1u);
    });
    __syncthreads();
    uint64_t by_min = 0;
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
        if (tid < heavies) heavy(s.list_x[tid]);
    } else {
        slow.each([&](float x, uint32_t) {
            const float t = w.exponent(x);
            if (Weights::any(t) && t >= w.heavy) heavy(x);
        });
    }
    if (min_p > 0.0f && by_min) atomicAdd(reinterpret_cast<unsigned long long *>(&s.kept_by_min), by_min);
    __syncthreads();
    scan_steps(s);
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
        if (tid == 0) s.n = 0;
        if (!spoiled) {
            for (uint32_t i = tid; i < kBins; i += kThreads)
                if (t.met(s.count[i], s.mass[i]) && (i == 0 || !t.met(s.count[i - 1], s.mass[i - 1]))) s.step = i;
            __syncthreads();
            step = s.step;
            m0 = step ? s.mass[step - 1] : 0;
            c0 = step && counted ? s.count[step - 1] : 0;
            row.each([&](float x, uint32_t i) {
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
        if (n > kList) {
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
        if (tid < n) s.list_mass[tid] = w.of(s.list_x[tid]);
        __syncthreads();
        rank_list(s, t, n, m0, c0);
        if (stage < 2) kept = s.cut_mass < kept ? s.cut_mass : kept;
        __syncthreads();
    }
    if (tid == 0) {
        A.ids[r] = s.cut_id;
        if (A.probs) A.probs[r] = static_cast<float>(w.exact(s.cut_x) * 0x1p44 / static_cast<double>(kept));
    }
}

} // namespace

uint64_t sample_scratch(uint32_t, uint32_t) { return 0; }

int sample(const float *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const fmx_sampling &p,
           const float *uniform, uint32_t *ids, float *probs, uint32_t *status, uint8_t *, hipStream_t s) {
    const SampleArgs A{logits, row_stride, vocab, p, uniform, ids, probs, status};
    const auto kernel = vocab <= 8 * kThreads ? sample_kernel<8> : sample_kernel<0>;
    hipLaunchKernelGGL(kernel, dim3(rows), dim3(kThreads), 0, s, A);
    FMX_LAUNCH_CHECK();
    return FMX_OK;
}

} // namespace fmx
