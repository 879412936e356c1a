// sample.hip — one token per row of logits by temperature, top-k, top-p and
// min-p (the choice of FreeMoe's engine.cpp:471-631 from a given uniform
// number).
//
// Tokens in falling order of logit x (equal ones by rising id) carry weights
// w = e^((x - M) / T), M the largest logit. Each filter keeps a prefix of that
// order, so what is kept is the shortest of three prefixes and its mass the
// least of three masses, and the token is the first whose cumulated mass
// exceeds uniform x that mass. Nothing is sorted: a place in the order where a
// count or a mass crosses a target is found by a histogram of masses over
// equal steps of x, then among the elements of the one step that holds it.
//
// Masses are integers in steps of 2^-44: their sums do not depend on the order
// of the additions (LDS atomics, whichever wavefront comes first), and what
// they lose is 2^-45 of the largest weight per token.
#include "paged.hpp"

namespace fmx {

namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kWaves = kThreads / 64;
constexpr uint32_t kBins = 2048;     // of the first histogram
constexpr uint32_t kFineBins = 1024; // of those inside one of its steps
constexpr uint32_t kList = 1024;     // elements compared pair by pair
constexpr uint32_t kMassBits = 44;
static_assert(kSampleMaxVocab <= 1u << 18, "sums of that many masses of at most 2^44 stay below 2^63");

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

// An element's place in the order.
struct Place {
    float x;
    uint32_t id;
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
    uint64_t mass[kBins], fine_mass[kFineBins], list_mass[kList];
    uint32_t count[kBins], fine_count[kFineBins];
    float list_x[kList];
    uint32_t list_id[kList];
    double table[64];
    uint64_t wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float wave_a[kWaves], wave_b[kWaves];
    uint32_t wave_id[kWaves];
    bool wave_bad[kWaves];
    uint32_t n, step, found;
    Place cut;
    uint64_t cut_mass;
};

// Inclusive sums of n entries, a power of two from kThreads on, in place.
__device__ void scan_bins(Shared &s, uint64_t *mass, uint32_t *count, uint32_t n) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per = n / kThreads;
    uint64_t m = 0;
    uint32_t c = 0;
    for (uint32_t i = 0; i < per; ++i) {
        m += mass[tid * per + i];
        c += count[tid * per + i];
    }
    uint64_t mi = m;
    uint32_t ci = c;
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t mo = __shfl_up(mi, d);
        const uint32_t co = __shfl_up(ci, d);
        if (lane >= d) {
            mi += mo;
            ci += co;
        }
    }
    if (lane == 63) {
        s.wave_mass[wave] = mi;
        s.wave_count[wave] = ci;
    }
    __syncthreads();
    mi -= m;
    ci -= c;
    for (uint32_t i = 0; i < wave; ++i) {
        mi += s.wave_mass[i];
        ci += s.wave_count[i];
    }
    for (uint32_t i = 0; i < per; ++i) {
        mi += mass[tid * per + i];
        ci += count[tid * per + i];
        mass[tid * per + i] = mi;
        count[tid * per + i] = ci;
    }
    __syncthreads();
}

// The row, in registers where kHeld elements a thread hold it, else read again
// at each pass (from L2).
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

// Steps of x: element x lies in step floor((top - x) * scale), the last one
// taking the rest; monotonic in x, so the steps are stretches of the order.
struct Steps {
    double top, scale;
    uint32_t last;
    __device__ __forceinline__ uint32_t of(float x) const {
        const double d = (top - static_cast<double>(x)) * scale;
        return d < static_cast<double>(last) ? static_cast<uint32_t>(d) : last;
    }
};

// grid: rows.
template <uint32_t kHeld> __global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs A) {
    __shared__ Shared s;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x, V = A.vocab;
    Row<kHeld> row;
    row.from = A.logits + r * A.row_stride;
    row.vocab = V;
    row.load();
    const float temperature = A.p.temperature ? A.p.temperature[r] : 1.0f;
    const uint32_t top_k = A.p.top_k ? A.p.top_k[r] : 0;
    const float top_p = A.p.top_p ? A.p.top_p[r] : 1.0f, min_p = A.p.min_p ? A.p.min_p[r] : 0.0f;
    const float uniform = A.uniform[r];

    // the largest logit (its lowest id) and the smallest finite one
    float high = -__builtin_inff(), low = __builtin_inff();
    uint32_t high_id = 0xffffffffu;
    bool bad = false;
    row.each([&](float x, uint32_t i) {
        bad |= !(x < __builtin_inff());
        if (x > high) {
            high = x;
            high_id = i;
        }
        if (x > -__builtin_inff()) low = fminf(low, x);
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
    for (uint32_t i = tid; i < kBins; i += kThreads) {
        s.mass[i] = 0;
        s.count[i] = 0;
    }
    if (tid < 64) s.table[tid] = exp2(tid / 64.0);
    __syncthreads();
    for (uint32_t i = 0; i < kWaves; ++i) {
        bad |= s.wave_bad[i];
        if (precedes(s.wave_a[i], s.wave_id[i], high, high_id)) {
            high = s.wave_a[i];
            high_id = s.wave_id[i];
        }
        low = fminf(low, s.wave_b[i]);
    }
    bad |= high == -__builtin_inff() || !(temperature >= 0.0f) || top_p != top_p || min_p != min_p ||
           uniform != uniform;
    if (bad || temperature == 0.0f) {
        if (tid == 0) {
            A.ids[r] = bad ? 0xffffffffu : high_id;
            if (A.probs) A.probs[r] = bad ? 0.0f : 1.0f;
            if (bad) atomicOr(A.status, STATUS_NONFINITE_SCORE);
        }
        return;
    }
    const double M = high, per_x = 1.4426950408889634 / static_cast<double>(temperature);
    // log 2 of a weight; weights below 2^-46 are none
    constexpr double kLeast = -46.0;
    auto mass_of = [&](float x, double &w) -> uint64_t {
        const double t = (static_cast<double>(x) - M) * per_x;
        if (!(x > -__builtin_inff()) || !(t > kLeast)) return 0;
        w = exp2_table(t, s.table);
        // to an integer below 2^45 through the mantissa of 2^52 + it
        return __builtin_bit_cast(uint64_t, w * 0x1p44 + 0x1p52) & 0xfffffffffffffull;
    };

    // the histogram over the stretch that has weights, and min-p's mass
    const double reach = -kLeast / per_x, span = fmin(M - static_cast<double>(low), reach);
    const Steps steps{M, span > 0.0 ? (kBins - 1) / span : 0.0, kBins - 1};
    uint64_t kept_m = 0;
    row.each([&](float x, uint32_t) {
        double w;
        const uint64_t m = mass_of(x, w);
        if (m == 0) return;
        const uint32_t b = steps.of(x);
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[b]), m);
        atomicAdd(&s.count[b], 1u);
        if (w >= static_cast<double>(min_p)) kept_m += m;
    });
    for (uint32_t d = 32; d >= 1; d >>= 1) kept_m += __shfl_xor(kept_m, d);
    __syncthreads();
    scan_bins(s, s.mass, s.count, kBins);
    if (lane == 0) s.wave_mass[wave] = kept_m;
    __syncthreads();
    kept_m = 0;
    for (uint32_t i = 0; i < kWaves; ++i) kept_m += s.wave_mass[i];
    const uint64_t whole = s.mass[kBins - 1];
    const uint32_t weighted = s.count[kBins - 1];

    // The element at which `t` is first met: s.cut and the mass up to and with
    // it, s.cut_mass. Every thread calls it, with a target that the last
    // weighted element meets.
    auto find = [&](const Target &t) {
        __syncthreads();
        for (uint32_t i = tid; i < kBins; i += kThreads)
            if (t.met(s.count[i], s.mass[i]) && (i == 0 || !t.met(s.count[i - 1], s.mass[i - 1]))) s.step = i;
        __syncthreads();
        uint32_t step = s.step;
        uint64_t m0 = step ? s.mass[step - 1] : 0;
        uint32_t c0 = step ? s.count[step - 1] : 0, n = s.count[step] - c0;
        // elements of the current stretch: those of all steps so far
        float stretch_hi = high, stretch_lo = -__builtin_inff();
        bool first = true;
        auto inside = [&](float x) {
            return first ? x > -__builtin_inff() && steps.of(x) == step : x <= stretch_hi && x >= stretch_lo;
        };
        while (n > kList) { // many elements: the stretch's own bounds, then finer steps
            float a = -__builtin_inff(), b = __builtin_inff();
            row.each([&](float x, uint32_t) {
                double w;
                if (inside(x) && mass_of(x, w)) {
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
            for (uint32_t i = tid; i < kFineBins; i += kThreads) {
                s.fine_mass[i] = 0;
                s.fine_count[i] = 0;
            }
            __syncthreads();
            for (uint32_t i = 0; i < kWaves; ++i) {
                a = fmaxf(a, s.wave_a[i]);
                b = fminf(b, s.wave_b[i]);
            }
            if (a == b) { // equal logits: the r-th of them by id
                double w;
                const uint64_t m = mass_of(a, w);
                uint32_t lo = 1, hi = n; // the least count that meets the target
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (t.met(c0 + mid, m0 + mid * m)) hi = mid;
                    else lo = mid + 1;
                }
                uint32_t left = lo;
                for (uint32_t i0 = 0; i0 < V; i0 += kThreads) {
                    const uint32_t i = i0 + tid;
                    const bool here = i < V && row.from[i] == a;
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
                        s.cut = Place{a, i};
                        s.cut_mass = m0 + lo * m;
                    }
                    break;
                }
                __syncthreads();
                return;
            }
            const Steps fine{static_cast<double>(a), (kFineBins - 1) / (static_cast<double>(a) - static_cast<double>(b)),
                             kFineBins - 1};
            row.each([&](float x, uint32_t) {
                double w;
                if (!inside(x)) return;
                const uint64_t m = mass_of(x, w);
                if (m == 0) return;
                const uint32_t f = fine.of(x);
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.fine_mass[f]), m);
                atomicAdd(&s.fine_count[f], 1u);
            });
            __syncthreads();
            scan_bins(s, s.fine_mass, s.fine_count, kFineBins);
            for (uint32_t i = tid; i < kFineBins; i += kThreads)
                if (t.met(c0 + s.fine_count[i], m0 + s.fine_mass[i]) &&
                    (i == 0 || !t.met(c0 + s.fine_count[i - 1], m0 + s.fine_mass[i - 1])))
                    s.step = i;
            __syncthreads();
            const uint32_t f = s.step;
            const uint64_t fm = f ? s.fine_mass[f - 1] : 0;
            const uint32_t fc = f ? s.fine_count[f - 1] : 0;
            n = s.fine_count[f] - fc;
            m0 += fm;
            c0 += fc;
            // the elements of fine step f, as bounds on x
            float na = -__builtin_inff(), nb = __builtin_inff();
            row.each([&](float x, uint32_t) {
                double w;
                if (inside(x) && fine.of(x) == f && mass_of(x, w)) {
                    na = fmaxf(na, x);
                    nb = fminf(nb, x);
                }
            });
            for (uint32_t d = 32; d >= 1; d >>= 1) {
                na = fmaxf(na, __shfl_xor(na, d));
                nb = fminf(nb, __shfl_xor(nb, d));
            }
            __syncthreads();
            if (lane == 0) {
                s.wave_a[wave] = na;
                s.wave_b[wave] = nb;
            }
            __syncthreads();
            for (uint32_t i = 0; i < kWaves; ++i) {
                na = fmaxf(na, s.wave_a[i]);
                nb = fminf(nb, s.wave_b[i]);
            }
            stretch_hi = na;
            stretch_lo = nb;
            first = false;
        }
        if (tid == 0) s.n = 0;
        __syncthreads();
        row.each([&](float x, uint32_t i) {
            double w;
            if (!inside(x)) return;
            const uint64_t m = mass_of(x, w);
            if (m == 0) return;
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < kList) {
                s.list_x[at] = x;
                s.list_id[at] = i;
                s.list_mass[at] = m;
            }
        });
        __syncthreads();
        const uint32_t listed = s.n < kList ? s.n : kList;
        if (tid < listed) {
            const float x = s.list_x[tid];
            const uint32_t id = s.list_id[tid];
            uint64_t m = m0;
            uint32_t c = c0;
            for (uint32_t j = 0; j < listed; ++j)
                if (precedes(s.list_x[j], s.list_id[j], x, id)) {
                    m += s.list_mass[j];
                    ++c;
                }
            const uint64_t with = m + s.list_mass[tid];
            if (t.met(c + 1, with) && !t.met(c, m)) {
                s.cut = Place{x, id};
                s.cut_mass = with;
            }
        }
        __syncthreads();
    };

    uint64_t kept = whole;
    if (top_k != 0 && top_k < weighted) {
        find(Target{kCount, top_k, 0.0});
        kept = s.cut_mass;
    }
    if (top_p < 1.0f) {
        find(Target{kReach, 0, fmax(static_cast<double>(top_p) * static_cast<double>(kept), 1.0)});
        kept = s.cut_mass < kept ? s.cut_mass : kept;
    }
    if (min_p > 0.0f) {
        const uint64_t least = kept_m ? kept_m : uint64_t{1} << kMassBits; // the largest at least
        kept = least < kept ? least : kept;
    }
    const float u = fminf(fmaxf(uniform, 0.0f), 0x1.fffffep-1f);
    find(Target{kExceed, 0, static_cast<double>(u) * static_cast<double>(kept)});
    if (tid == 0) {
        double w = 0.0;
        (void)mass_of(s.cut.x, w);
        A.ids[r] = s.cut.id;
        if (A.probs) A.probs[r] = static_cast<float>(w * 0x1p44 / static_cast<double>(kept));
    }
}

} // namespace

uint64_t sample_scratch(uint32_t, uint32_t) { return 0; }

int sample(const float *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const fmx_sampling &p,
           const float *uniform, uint32_t *ids, float *probs, uint32_t *status, uint8_t *, hipStream_t s) {
    const SampleArgs A{logits, row_stride, vocab, p, uniform, ids, probs, status};
    const auto kernel = vocab <= 8 * kThreads ? sample_kernel<8> : vocab <= 32 * kThreads ? sample_kernel<32> : sample_kernel<0>;
    hipLaunchKernelGGL(kernel, dim3(rows), dim3(kThreads), 0, s, A);
    FMX_LAUNCH_CHECK();
    return FMX_OK;
}

} // namespace fmx
