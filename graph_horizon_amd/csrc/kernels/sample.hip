// Sampling of rows of logits: temperature, top-k, top-p, min-p and a draw by a given random number, as the host's
// gh_sample, in 64 bits.
//
// Tokens rank by (logit descending by f32 total order, index ascending), those with a finite logit. Token i has weight
// w = exp((l - M) / T), M the row's largest logit. Every filter keeps a prefix of the ranking, and the draw
// is the first rank whose running sum of weights passes u times the kept sum, so all a row needs are four searches in the
// running counts and sums. Sums are of whole numbers, w in fixed point: the same in any order. One word must leave room for
// `vocab` weights of 1: at a vocabulary of 2^17 a weight is off by 2^-46 at most, and a sum by 2^-29 of the largest weight. Larger
// vocabularies, where that grows with their square, take two words (Mass<true>): a sum is off by vocab 2^-54 at most, as in FP64.
// The second word costs 1 us of 22 for 1 row of 131072 and 5 of 47 for 64, so smaller ones do without.
//
// Four launches; a row's logits are read three times, from memory once (us of 1 / 8 / 64 rows of 131072):
//   gh_sample_max     the largest logit of each chunk of a row (3.8 / 4.3 / 10.3: 34 MB of 64 rows at half the rate of a
//                     long read, for a workgroup has one round of loads and ends);
//   gh_sample_bins    counts and sums over 1024 bins of the distance d = M - l, 64 per octave from 2^-9 to 2^7, so
//                     that a bin holds at most 3 % of any smooth distribution whatever its spread (5.6 / 6.9 / 13.7: three
//                     LDS operations a token, two of them atomic; a cheaper exponential, or fewer and larger workgroups, change nothing);
//   gh_sample_collect the tokens of the bins in which a search can end: the running sums up to the bins are known, and
//                     bound the top-k sum, then the kept sum, then the draw's target (7.5 / 8.5 / 11.9);
//   gh_sample_pick    searches these tokens, or, where they are more than the list takes, the row itself: one wave where they
//                     are 64 or fewer, else a workgroup of 16 waves, half of which look at the bins (4.8 / 12.6 / 11.2; all of
//                     them, before Mass, 5.6 / 14.0 / 12.3, 8 waves in all 4.7 / 14.9 / 12.6). The row itself is read four times or more by
//                     one workgroup: 131072 tokens within one bin 302 / 309 / 315.
// Chains of dependent loads and barriers bound the launches of few rows.
// What the device cannot trust is only the settings: any bits give a token of the row.
#include <type_traits>

#include "gh_wave64.h"

namespace {
constexpr uint32_t kBins = GH_SAMPLE_BINS, kList = GH_SAMPLE_LIST;
constexpr uint32_t kNone = 0xFFFFFFFFu;
constexpr uint32_t kLoads = 8;  // 16-byte loads that a thread has in flight
constexpr uint32_t kBlock = 256 * 4 * kLoads;

// f32 total order as unsigned order, and back
__device__ __forceinline__ uint32_t order_key(uint32_t bits) { return bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u); }
__device__ __forceinline__ float order_value(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
// Ascending in rank order.
__device__ __forceinline__ uint64_t rank_key(float l, uint32_t i) { return (uint64_t)~order_key(__float_as_uint(l)) << 32 | i; }
__device__ __forceinline__ float value_of(uint64_t key) { return order_value(~(uint32_t)(key >> 32)); }

// The bin of distance d >= 0.
__device__ __forceinline__ uint32_t bin_of(float d) {
    const int b = (int)(__float_as_uint(d) >> 17) - ((127 - 9) << 6) + 1;
    return (uint32_t)min(max(b, 0), (int)kBins - 1);
}

// A row's settings and what its chunks' maxima say.
struct Row {
    float temperature, top_p, min_p;
    uint32_t top_k;
    double u, inv;      // the draw's number, 1 / T
    float top;          // M
    uint32_t best;      // a greedy row's token: the index of the largest of all logits, infinite ones too
    bool greedy;        // T <= 0, or no finite logit
};
__device__ __forceinline__ Row row_of(const GhSampleArgs& a, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint4 p = gh_gp<uint4>(a.params)[row];
    const float u = gh_gp<float>(a.uniform)[row];
    ulonglong2 x = make_ulonglong2(0, 0);
    if (lane < a.chunks) x = gh_gp<ulonglong2>(a.part + (uint64_t)row * 64 * 16)[lane];
    const uint32_t fin = (uint32_t)gh_max64(x.y);
    Row r;
    r.temperature = __uint_as_float(p.x);
    r.top_p = __uint_as_float(p.y);
    r.top_k = p.z;
    r.min_p = __uint_as_float(p.w);
    r.u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    r.inv = 1.0 / (double)r.temperature;
    r.top = order_value(fin);
    r.greedy = !(r.temperature > 0.0f) || fin == 0;
    r.best = 0;
    if (r.greedy) {
        const uint64_t any = gh_max64(x.x);
        r.best = any ? ~(uint32_t)any : 0u;
    }
    return r;
}

// exp(x) of x <= 0 as 2^(n / 64) e^r, n the nearest whole number to 64 x / ln 2 and |r| <= ln 2 / 128: powers of two by
// 64ths from a table (Tang's method), e^r by its series to r^5 / 5!, whose rest is below 2^-57.
__device__ __forceinline__ void fill_exp(double* table) {
    if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x * 0x1p-6);
}
__device__ __forceinline__ double exp_scaled(const double* table, double x, int up) {
    x = x > -200.0 ? x : -200.0;  // (and what is not a number: none here)
    const double shift = 0x1.8p52;
    const double z = __builtin_fma(x, 0x1.71547652b82fep+6, shift), n = z - shift;
    const int whole = (int)(uint32_t)__builtin_bit_cast(uint64_t, z);
    // ln 2 / 64 in two parts, the first short enough for exact products with n
    double r = __builtin_fma(n, -0x1.62e42fefap-7, x);
    r = __builtin_fma(n, -0x1.cf79abc9e3b3ap-46, r);
    double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
    p = __builtin_fma(r, p, 1.0 / 6);
    p = __builtin_fma(r, p, 0.5);
    p = __builtin_fma(r * r, p, r);
    const double t = table[whole & 63];
    return __builtin_ldexp(__builtin_fma(t, p, t), (whole >> 6) + up);
}
__device__ __forceinline__ double weight(const Row& r, const double* table, float l) {
    return exp_scaled(table, ((double)l - (double)r.top) * r.inv, 0);
}
// What tokens weigh together, in fixed point, and their number. Whole parts are 2^-shift of the largest weight. FINE: above the count,
// in `count_bits` bits, `rest` holds further parts, of 2^-(shift + fine). All of a row's tokens fit both words.
template <bool FINE>
struct Mass {
    uint64_t whole;
    std::conditional_t<FINE, uint64_t, uint32_t> rest;
    __device__ __forceinline__ Mass operator+(const Mass& x) const { return Mass{whole + x.whole, rest + x.rest}; }
    __device__ __forceinline__ Mass operator-(const Mass& x) const { return Mass{whole - x.whole, rest - x.rest}; }
};
template <bool FINE>
__device__ __forceinline__ uint32_t count_of(const GhSampleArgs& a, const Mass<FINE>& m) {
    return FINE ? (uint32_t)m.rest & ((1u << a.count_bits) - 1) : (uint32_t)m.rest;
}
// In whole parts. No smaller for a mass with more tokens.
template <bool FINE>
__device__ __forceinline__ double sum_of(const GhSampleArgs& a, const Mass<FINE>& m) {
    if constexpr (FINE) return (double)m.whole + __builtin_ldexp((double)(m.rest >> a.count_bits), -a.fine);
    else return (double)m.whole;
}
template <bool FINE>
__device__ __forceinline__ Mass<FINE> scan_mass(const Mass<FINE>& m) {
    return Mass<FINE>{gh_scan64(m.whole), (decltype(m.rest))gh_scan64(m.rest)};
}
template <bool FINE>
__device__ __forceinline__ Mass<FINE> lane_mass(const Mass<FINE>& m, uint32_t lane) {
    if constexpr (FINE) return Mass<FINE>{gh_lane64(m.whole, lane), gh_lane64(m.rest, lane)};
    else return Mass<FINE>{gh_lane64(m.whole, lane), (uint32_t)__builtin_amdgcn_readlane(m.rest, lane)};
}
// A token's, its last part nearest. Both words' parts are at most 2^51, so that 2^52 more leaves them in the mantissa. (The
// largest weight, 1, has no further parts.)
template <bool FINE>
__device__ __forceinline__ Mass<FINE> fixed(const GhSampleArgs& a, const Row& r, const double* table, float l) {
    const double w = exp_scaled(table, ((double)l - (double)r.top) * r.inv, a.shift), whole = FINE ? __builtin_floor(w) : w;
    const uint64_t bits = 0xFFFFFFFFFFFFFull;
    Mass<FINE> m{__builtin_bit_cast(uint64_t, whole + 0x1p52) & bits, 1u};
    if constexpr (FINE) m.rest |= (__builtin_bit_cast(uint64_t, __builtin_ldexp(w - whole, a.fine) + 0x1p52) & bits) << a.count_bits;
    return m;
}

// The kernels have both forms, the one for two words behind the other, and an empty asm at its start keeps the compiler from drawing
// the first instructions of both together ahead of the branch (gh_sample_pick of 8 / 64 rows otherwise 13.0 / 11.7 us instead of
// 12.6 / 11.2: what is asked for there at once was waited for in turn).

// Masses of the bins, or of parts of one: 64 bits each for `rest`, or the first half of them 32.
template <bool FINE>
__device__ __forceinline__ Mass<FINE> mass_at(const uint64_t* whole, const uint64_t* rest, uint32_t i) {
    if constexpr (FINE) return Mass<FINE>{whole[i], rest[i]};
    else return Mass<FINE>{whole[i], ((const uint32_t*)rest)[i]};
}
template <bool FINE>
__device__ __forceinline__ void put_mass(uint64_t* whole, uint64_t* rest, uint32_t i, const Mass<FINE>& m) {
    whole[i] = m.whole;
    if constexpr (FINE) rest[i] = m.rest;
    else ((uint32_t*)rest)[i] = m.rest;
}
template <bool FINE>
__device__ __forceinline__ void add_mass(uint64_t* whole, uint64_t* rest, uint32_t i, const Mass<FINE>& m) {
    if constexpr (FINE) atomicAdd((unsigned long long*)rest + i, (unsigned long long)m.rest);
    else atomicAdd((uint32_t*)rest + i, m.rest);
    if (m.whole) atomicAdd((unsigned long long*)whole + i, (unsigned long long)m.whole);
}

// LOADS times four logits of a block of a row, the k-th four of a thread 4 THREADS k further on; NaN past `end`.
template <uint32_t THREADS, uint32_t LOADS>
__device__ __forceinline__ void load_block(const GhSampleArgs& a, uint32_t row, uint32_t block, uint32_t end, float4 (&v)[LOADS]) {
    const GH_GLOBAL float* l = gh_gp<float>(a.logits) + (uint64_t)row * a.stride;
#pragma unroll
    for (uint32_t k = 0; k < LOADS; ++k) {
        const uint32_t at = block + 4 * (threadIdx.x + THREADS * k);
        const float none = __uint_as_float(0x7FC00000u);
        v[k] = make_float4(none, none, none, none);
        if (a.wide && at + 4 <= end) {
            v[k] = *(const GH_GLOBAL float4*)(l + at);
        } else if (at < end) {
            v[k].x = l[at];
            if (at + 1 < end) v[k].y = l[at + 1];
            if (at + 2 < end) v[k].z = l[at + 2];
            if (at + 3 < end) v[k].w = l[at + 3];
        }
    }
}
// body(logit, index) for each of a block's tokens.
template <uint32_t THREADS, uint32_t LOADS, class F>
__device__ __forceinline__ void each_of(const float4 (&v)[LOADS], uint32_t block, F body) {
#pragma unroll
    for (uint32_t k = 0; k < LOADS; ++k) {
        const uint32_t at = block + 4 * (threadIdx.x + THREADS * k);
        body(v[k].x, at);
        body(v[k].y, at + 1);
        body(v[k].z, at + 2);
        body(v[k].w, at + 3);
    }
}
}  // namespace

// Grid (chunks, rows), 256 threads. Also clears the row's bins for the next launch.
GH_KERNEL __launch_bounds__(256) void gh_sample_max(GhSampleArgs a) {
    __shared__ uint64_t red[4][2];
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
    GH_GLOBAL uint32_t* bins = gh_gpw<uint32_t>(a.bins + (uint64_t)row * a.bin_bytes);
    for (uint32_t i = blockIdx.x * 256 + tid; i < a.bin_bytes / 4; i += gridDim.x * 256) bins[i] = 0u;
    uint32_t fin = 0;
    float4 v[kLoads];
    for (uint32_t block = first; block < end; block += kBlock) {
        load_block<256>(a, row, block, end, v);
        each_of<256>(v, block, [&](float l, uint32_t) __attribute__((always_inline)) {
            if (finite(l)) fin = max(fin, order_key(__float_as_uint(l)));
        });
    }
    // the index of the largest, infinite ones too, for rows that are or turn out greedy
    uint64_t any = 0;
    if (!(gh_gp<float4>(a.params)[row].x > 0.0f) || __syncthreads_or(fin) == 0) {
        for (uint32_t block = first; block < end; block += kBlock) {
            load_block<256>(a, row, block, end, v);
            each_of<256>(v, block, [&](float l, uint32_t i) __attribute__((always_inline)) {
                // -0 and 0 are equal here; a NaN is never the largest
                const uint64_t key = (uint64_t)order_key(__float_as_uint(l + 0.0f)) << 32 | (uint32_t)~i;
                if (l > -__builtin_inff()) any = any > key ? any : key;
            });
        }
    }
    any = gh_max64(any);
    const uint64_t top = gh_max64(fin);
    if ((tid & 63u) == 0) {
        red[tid >> 6][0] = any;
        red[tid >> 6][1] = top;
    }
    __syncthreads();
    if (tid == 0) {
        ulonglong2 x = make_ulonglong2(red[0][0], red[0][1]);
        for (uint32_t w = 1; w < 4; ++w) {
            x.x = x.x > red[w][0] ? x.x : red[w][0];
            x.y = x.y > red[w][1] ? x.y : red[w][1];
        }
        gh_gpw<ulonglong2>(a.part)[(uint64_t)row * 64 + blockIdx.x] = x;
    }
}

namespace {
template <bool FINE>
__device__ __forceinline__ void sample_bins(const GhSampleArgs& a, uint64_t* whole, uint64_t* rest, double* table) {
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
    float4 v[kLoads];
    load_block<256>(a, row, first, end, v);
    for (uint32_t i = tid; i < kBins; i += 256) put_mass(whole, rest, i, Mass<FINE>{0, 0});
    fill_exp(table);
    const Row r = row_of(a, row);
    if (r.greedy) return;
    __syncthreads();
    for (uint32_t block = first;;) {
        each_of<256>(v, block, [&](float l, uint32_t) __attribute__((always_inline)) {
            if (!finite(l)) return;
            add_mass(whole, rest, bin_of(r.top - l), fixed<FINE>(a, r, table, l));
        });
        block += kBlock;
        if (block >= end) break;
        load_block<256>(a, row, block, end, v);
    }
    __syncthreads();
    uint64_t* bins = (uint64_t*)(a.bins + (uint64_t)row * a.bin_bytes);
    for (uint32_t i = tid; i < kBins; i += 256) {
        const Mass<FINE> m = mass_at<FINE>(whole, rest, i);
        if (m.rest) add_mass(bins, bins + kBins, i, m);
    }
}
}  // namespace

// Grid (chunks, rows), 256 threads. Bins in LDS, added to the row's by atomics on whole numbers.
GH_KERNEL __launch_bounds__(256) void gh_sample_bins(GhSampleArgs a) {
    __shared__ uint64_t whole[kBins], rest[kBins];
    __shared__ double table[64];
    if (__builtin_expect(a.fine, 0)) {
        asm volatile("");
        sample_bins<true>(a, whole, rest, table);
    } else {
        sample_bins<false>(a, whole, rest, table);
    }
}

namespace {
// The bins in which a row's searches end.
struct Plan {
    uint32_t tokens;        // finite logits
    uint32_t keep;          // min(top_k, tokens)
    uint32_t k;             // bin of the last of them
    bool partly;            // not all of that bin's
    uint32_t p0, p1;        // top-p's, first and last (kNone: off)
    uint32_t m0, m1;        // min-p's
    uint32_t d0, d1;        // the draw's
    uint32_t listed;        // tokens in these bins
    __device__ __forceinline__ bool has(uint32_t b) const {
        return (partly && b == k) || (p0 != kNone && p0 <= b && b <= p1) || (m0 != kNone && m0 <= b && b <= m1) || (d0 <= b && b <= d1);
    }
};
// LDS of a plan: what the bins hold, running and inclusive.
struct PlanLds {
    uint64_t whole[kBins], rest[kBins];
    uint64_t wave_whole[16], wave_rest[16];
    uint32_t wave_listed[16];
    uint32_t found[5];
};
template <bool FINE>
__device__ __forceinline__ Mass<FINE> upto(const PlanLds& s, uint32_t b) { return mass_at<FINE>(s.whole, s.rest, b); }
template <bool FINE>
__device__ __forceinline__ Mass<FINE> before(const PlanLds& s, uint32_t b) { return b ? upto<FINE>(s, b - 1) : Mass<FINE>{0, 0}; }

// All threads of the workgroup get the same plan; the first THREADS look at the bins (of 16 waves, which take 16 cycles for
// an instruction, half). Sums are compared as doubles, as the searches compare them.
template <bool FINE, uint32_t THREADS, uint32_t ALL>
__device__ __forceinline__ Plan plan_of(const GhSampleArgs& a, const Row& r, uint32_t row, PlanLds& s) {
    constexpr uint32_t kEach = kBins / THREADS, kWaves = THREADS / 64;  // bins of a thread, in a row
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const GH_GLOBAL uint64_t* bins = gh_gp<uint64_t>(a.bins + (uint64_t)row * a.bin_bytes);
    const bool looks = THREADS == ALL || tid < THREADS;
    Mass<FINE> m[kEach], mu = {0, 0};
    uint32_t own[kEach];  // the bins' counts
    if (looks) {
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            m[j].whole = bins[tid * kEach + j];
            m[j].rest = ((const GH_GLOBAL decltype(mu.rest)*)(bins + kBins))[tid * kEach + j];
        }
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) own[j] = count_of(a, m[j]);
#pragma unroll
        for (uint32_t j = 1; j < kEach; ++j) m[j] = m[j - 1] + m[j];
        mu = scan_mass(m[kEach - 1]);
        if (lane == 63) put_mass(s.wave_whole, s.wave_rest, wave, mu);
        if (tid < 5) s.found[tid] = kBins - 1;
    }
    __syncthreads();
    Plan p;
    p.tokens = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) p.tokens += count_of(a, mass_at<FINE>(s.wave_whole, s.wave_rest, i));
    Mass<FINE> m0 = {0, 0};  // before the thread's bins
    if (looks) {
        m0 = mu - m[kEach - 1];
#pragma unroll
        for (uint32_t i = 0; i < kWaves; ++i)
            if (i < wave) m0 = m0 + mass_at<FINE>(s.wave_whole, s.wave_rest, i);
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            m[j] = m[j] + m0;
            put_mass(s.whole, s.rest, tid * kEach + j, m[j]);
        }
    }
    // The first bin up to which the running values satisfy `is`, which stays true once it is: one thread has it.
    auto first_bin = [&](uint32_t slot, auto is) __attribute__((always_inline)) {
        if (!looks || !is(m[kEach - 1]) || (tid && is(m0))) return;
        uint32_t j = 0;
#pragma unroll
        for (uint32_t i = 0; i + 1 < kEach; ++i) j += j == i && !is(m[i]);
        s.found[slot] = tid * kEach + j;
    };
    p.keep = r.top_k && r.top_k < p.tokens ? r.top_k : p.tokens;
    first_bin(0, [&](const Mass<FINE>& x) { return count_of(a, x) >= p.keep; });
    __syncthreads();
    p.k = s.found[0];
    p.partly = count_of(a, upto<FINE>(s, p.k)) > p.keep;
    // the sum of the first top_k lies between lo and hi
    double lo = sum_of(a, p.partly ? before<FINE>(s, p.k) : upto<FINE>(s, p.k)), hi = sum_of(a, upto<FINE>(s, p.k));
    uint32_t l0 = p.k, l1 = p.k;  // the last kept token's bins
    p.p0 = p.p1 = p.m0 = p.m1 = kNone;
    if (r.top_p < 1.0f) {
        const double want0 = r.top_p * lo, want1 = r.top_p * hi;
        first_bin(1, [&](const Mass<FINE>& x) { return sum_of(a, x) >= want0; });
        first_bin(2, [&](const Mass<FINE>& x) { return sum_of(a, x) >= want1; });
        __syncthreads();
        l0 = p.p0 = min(s.found[1], p.k);
        l1 = p.p1 = min(s.found[2], p.k);
    }
    if (r.min_p > 0.0f) {
        // w >= min_p up to a distance of -T ln min_p, and a little further, as weights next to 1 round to it; d is rounded to FP32
        const double d = r.min_p < 1.0f ? -log((double)r.min_p) * (double)r.temperature : 0.0;
        p.m0 = bin_of((float)(d * (1.0 - 1e-6)));
        p.m1 = bin_of((float)((d + (double)r.temperature * 0x1p-50) * (1.0 + 1e-6)));
        l0 = min(l0, p.m0);
        l1 = min(l1, p.m1);
    }
    // the kept sum lies between lo and hi
    if (p.partly || p.p0 != kNone || p.m0 != kNone) lo = sum_of(a, before<FINE>(s, l0));
    hi = sum_of(a, upto<FINE>(s, l1));
    const double want0 = r.u * lo, want1 = r.u * hi;
    first_bin(3, [&](const Mass<FINE>& x) { return sum_of(a, x) > want0; });
    first_bin(4, [&](const Mass<FINE>& x) { return sum_of(a, x) > want1; });
    __syncthreads();
    p.d0 = min(s.found[3], l1);
    p.d1 = min(s.found[4], l1);
    if (looks) {
        uint32_t listed = 0;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) listed += p.has(tid * kEach + j) ? own[j] : 0u;
        listed = (uint32_t)gh_scan64(listed);
        if (lane == 63) s.wave_listed[wave] = listed;
    }
    __syncthreads();
    p.listed = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWaves; ++i) p.listed += s.wave_listed[i];
    return p;
}
}  // namespace

namespace {
template <bool FINE>
__device__ __forceinline__ void sample_collect(const GhSampleArgs& a, PlanLds& s, uint32_t* need, uint32_t* places) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, row = blockIdx.y, first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
    float4 v[kLoads];
    load_block<256>(a, row, first, end, v);
    const Row r = row_of(a, row);
    if (r.greedy) return;
    const Plan p = plan_of<FINE, 256, 256>(a, r, row, s);
    if (p.listed > kList) return;
#pragma unroll
    for (uint32_t j = 0; j < kBins / 256; ++j) {
        const uint64_t has = __ballot(p.has(256 * j + tid));
        if (lane < 2) need[8 * j + 2 * wave + lane] = (uint32_t)(has >> (32 * lane));
    }
    __syncthreads();
    const uint64_t list = a.list + (uint64_t)row * kList * 8;
    uint32_t* length = (uint32_t*)(a.bins + (uint64_t)(row + 1) * a.bin_bytes - 16);
    for (uint32_t block = first;;) {
        uint32_t mine = 0, bit = 1;  // which of the thread's 32 are wanted
        each_of<256>(v, block, [&](float l, uint32_t) __attribute__((always_inline)) {
            const uint32_t b = bin_of(r.top - l);
            if (finite(l) && (need[b >> 5] >> (b & 31u) & 1u)) mine |= bit;
            bit <<= 1;
        });
        const uint32_t n = __popc(mine), mine_upto = (uint32_t)gh_scan64(n);
        if (lane == 63) places[wave] = mine_upto;
        __syncthreads();
        const uint32_t all = places[0] + places[1] + places[2] + places[3];
        if (all) {  // of the whole workgroup
            if (tid == 0) places[4] = atomicAdd(length, all);
            __syncthreads();
            uint32_t at = places[4] + mine_upto - n;
            for (uint32_t w = 0; w < wave; ++w) at += places[w];
            bit = 1;
            each_of<256>(v, block, [&](float l, uint32_t i) __attribute__((always_inline)) {
                if (mine & bit) {
                    if (at < kList) gh_gpw<uint64_t>(list)[at] = rank_key(l, i);
                    ++at;
                }
                bit <<= 1;
            });
        }
        block += kBlock;
        if (block >= end) break;
        load_block<256>(a, row, block, end, v);
        __syncthreads();
    }
}
}  // namespace

// Grid (chunks, rows), 256 threads. A block's tokens are counted first, so that it asks for its places in the list once.
GH_KERNEL __launch_bounds__(256) void gh_sample_collect(GhSampleArgs a) {
    __shared__ PlanLds s;
    __shared__ uint32_t need[kBins / 32], places[5];
    if (__builtin_expect(a.fine, 0)) {
        asm volatile("");
        sample_collect<true>(a, s, need, places);
    } else {
        sample_collect<false>(a, s, need, places);
    }
}

namespace {
// Threads, their waves; those that look at bins, their waves, bins of each.
constexpr uint32_t kPick = GH_SAMPLE_PICK, kPickWaves = kPick / 64, kLook = 512, kLookWaves = kLook / 64, kLookBins = kBins / kLook;
// A token found by its running values: its key, and the mass up to and with it.
template <bool FINE>
struct Hit {
    uint64_t key;
    Mass<FINE> mass;
};
struct PickLds {
    uint64_t list[kList];
    uint64_t few[64];       // the tokens among which a search ends
    uint64_t whole[kBins], rest[kBins];  // of a range of keys, in equal parts
    uint64_t lo[16], hi[16];
    uint64_t wave_whole[16], wave_rest[16];
    uint64_t hit_key, hit_whole, hit_rest;
    uint32_t found, fill;
};

// The tokens of the list, or of the row, by key.
struct Listed {
    const uint64_t* list;
    uint32_t n;
    template <class F>
    __device__ __forceinline__ void each(F body) const {
        for (uint32_t i = threadIdx.x; i < n; i += kPick) body(list[i]);
    }
};
struct Whole {
    const GhSampleArgs& a;
    uint32_t row;
    template <class F>
    __device__ __forceinline__ void each(F body) const {
        for (uint32_t block = 0; block < a.vocab; block += 8 * kPick) {
            float4 v[2];
            load_block<kPick>(a, row, block, a.vocab, v);
            each_of<kPick>(v, block, [&](float l, uint32_t i) __attribute__((always_inline)) {
                if (finite(l)) body(rank_key(l, i));
            });
        }
    }
};

// The first token in rank order up to which the mass satisfies `is`, which some token's do and stays true once it is. Its bin
// by the running values of the bins; then, while there are more than 64 tokens, in which 1024th of them it is, first by the next ten
// bits of their distance, then by parts of the range of their keys; then among these, by one wave.
template <bool FINE, class S, class F>
__device__ __forceinline__ Hit<FINE> search(const GhSampleArgs& a, const Row& r, const double* table, const PlanLds& s, PickLds& q, const S& source, F is) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    __syncthreads();
    if (tid == 0) q.found = kBins - 1;
    __syncthreads();
    const bool looks = tid < kLook;
    const uint32_t mine = tid * kLookBins;  // the thread's bins, or parts of a range
    if (looks && is(upto<FINE>(s, mine + kLookBins - 1)) && (tid == 0 || !is(upto<FINE>(s, mine - 1)))) {
        uint32_t b = mine;
#pragma unroll
        for (uint32_t j = 0; j + 1 < kLookBins; ++j) b += b == mine + j && !is(upto<FINE>(s, b));
        q.found = b;
    }
    __syncthreads();
    const uint32_t bin = q.found;
    __syncthreads();  // all have read it: the first round below writes it again
    Mass<FINE> base = before<FINE>(s, bin);
    uint64_t lo = 0, hi = ~0ull;
    uint32_t n = count_of(a, upto<FINE>(s, bin) - base);
    // (the first and the last bin hold distances of any exponent)
    bool bits = bin && bin < kBins - 1;
    uint32_t tenth = kNone;  // the distance's ten bits, once known
    auto ten = [&](uint64_t key) __attribute__((always_inline)) { return __float_as_uint(r.top - value_of(key)) >> 7 & 1023u; };
    auto inside = [&](uint64_t key) __attribute__((always_inline)) {
        return key >= lo && key <= hi && bin_of(r.top - value_of(key)) == bin && (tenth == kNone || ten(key) == tenth);
    };
    // (eight rounds narrow any range of keys to one: a bound for logits that another stream changes meanwhile)
    for (uint32_t round = 0; n > 64 && round < 8; ++round) {
        uint32_t shift = 0;
        for (uint32_t i = tid; i < kBins; i += kPick) put_mass(q.whole, q.rest, i, Mass<FINE>{0, 0});
        if (tid == 0) q.found = kBins - 1;
        if (!bits) {
            uint64_t least = ~0ull, most = 0;
            source.each([&](uint64_t key) __attribute__((always_inline)) {
                if (!inside(key)) return;
                least = min(least, key);
                most = max(most, key);
            });
            least = ~gh_max64(~least);
            most = gh_max64(most);
            if (lane == 0) {
                q.lo[wave] = least;
                q.hi[wave] = most;
            }
            __syncthreads();
            for (uint32_t i = 0; i < kPickWaves; ++i) {
                least = min(least, q.lo[i]);
                most = max(most, q.hi[i]);
            }
            lo = least;
            hi = most;
            const uint32_t width = 64 - __clzll((long long)(hi - lo));
            shift = width > 10 ? width - 10 : 0;
        } else {
            __syncthreads();
        }
        source.each([&](uint64_t key) __attribute__((always_inline)) {
            if (!inside(key)) return;
            const uint32_t part = bits ? ten(key) : (uint32_t)((key - lo) >> shift);
            add_mass(q.whole, q.rest, part, fixed<FINE>(a, r, table, value_of(key)));
        });
        __syncthreads();
        Mass<FINE> ms[kLookBins], all = {0, 0}, m = {0, 0};
        if (looks) {
#pragma unroll
            for (uint32_t j = 0; j < kLookBins; ++j) {
                ms[j] = mass_at<FINE>(q.whole, q.rest, mine + j);
                all = all + ms[j];
            }
            m = scan_mass(all);
            if (lane == 63) put_mass(q.wave_whole, q.wave_rest, wave, m);
        }
        __syncthreads();
        if (looks) {
            Mass<FINE> m0 = base + m - all;
#pragma unroll
            for (uint32_t i = 0; i + 1 < kLookWaves; ++i)
                if (i < wave) m0 = m0 + mass_at<FINE>(q.wave_whole, q.wave_rest, i);
            // one part: the first of those that hold a token and end where `is` is true
            const uint32_t none = count_of(a, base);
#pragma unroll
            for (uint32_t j = 0; j < kLookBins; ++j) {
                const Mass<FINE> next = m0 + ms[j];
                if (count_of(a, ms[j]) && is(next) && !(count_of(a, m0) > none && is(m0))) {
                    q.found = mine + j;
                    put_mass(&q.hit_whole, &q.hit_rest, 0, m0);
                }
                m0 = next;
            }
        }
        __syncthreads();
        const uint32_t part = q.found;
        base = mass_at<FINE>(&q.hit_whole, &q.hit_rest, 0);
        n = count_of(a, mass_at<FINE>(q.whole, q.rest, part));
        if (bits) {
            tenth = part;
            bits = false;
        } else {
            lo += (uint64_t)part << shift;
            hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
        }
        __syncthreads();
    }
    if (tid == 0) q.fill = 0;
    __syncthreads();
    source.each([&](uint64_t key) __attribute__((always_inline)) {
        if (!inside(key)) return;
        const uint32_t at = atomicAdd(&q.fill, 1u);
        if (at < 64) q.few[at] = key;
    });
    __syncthreads();
    if (wave == 0) {
        // each lane's token against all of them, which are few
        const uint32_t all = min(q.fill, 64u);
        const uint64_t key = lane < all ? q.few[lane] : ~0ull;
        Mass<FINE> own = {0, 0}, m = base;
        if (lane < all) own = fixed<FINE>(a, r, table, value_of(key));
        for (uint32_t i = 0; i < all; ++i) {
            const bool first = gh_lane64(key, i) <= key;
            const Mass<FINE> mi = lane_mass(own, i);
            if (first) m = m + mi;
        }
        const uint32_t rank = count_of(a, m) - count_of(a, base);
        const bool ends = is(m) && (rank == 1 || !is(m - own));
        const uint64_t good = __ballot(lane < all && ends), last = __ballot(lane < all && rank == all);
        if (lane == (uint32_t)__builtin_ctzll(good ? good : last | 1ull << 63)) {
            q.hit_key = key;
            put_mass(&q.hit_whole, &q.hit_rest, 0, m);
        }
    }
    __syncthreads();
    return Hit<FINE>{q.hit_key, mass_at<FINE>(&q.hit_whole, &q.hit_rest, 0)};
}

// The row's token; its share of the kept sum in *prob.
template <bool FINE, class S>
__device__ __forceinline__ uint32_t pick_by_search(const GhSampleArgs& a, const Row& r, const double* table, const Plan& p, const PlanLds& s,
                                                   PickLds& q, const S& source, double* prob) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    uint32_t keep = p.keep;
    Mass<FINE> mass = upto<FINE>(s, p.k);
    if (p.partly) mass = search<FINE>(a, r, table, s, q, source, [&](const Mass<FINE>& x) { return count_of(a, x) >= keep; }).mass;
    if (p.p0 != kNone) {
        const double want = r.top_p * sum_of(a, mass);
        const Hit<FINE> h = search<FINE>(a, r, table, s, q, source, [&](const Mass<FINE>& x) { return sum_of(a, x) >= want; });
        if (count_of(a, h.mass) < keep) {
            keep = count_of(a, h.mass);
            mass = h.mass;
        }
    }
    if (p.m0 != kNone) {
        Mass<FINE> in = {0, 0};
        source.each([&](uint64_t key) __attribute__((always_inline)) {
            const float l = value_of(key);
            const uint32_t b = bin_of(r.top - l);
            if (p.m0 <= b && b <= p.m1 && weight(r, table, l) >= (double)r.min_p) in = in + fixed<FINE>(a, r, table, l);
        });
        in = scan_mass(in);
        __syncthreads();
        if (lane == 63) put_mass(q.wave_whole, q.wave_rest, wave, in);
        __syncthreads();
        Mass<FINE> to = before<FINE>(s, p.m0);
        for (uint32_t i = 0; i < kPickWaves; ++i) to = to + mass_at<FINE>(q.wave_whole, q.wave_rest, i);
        if (count_of(a, to) == 0) to = fixed<FINE>(a, r, table, r.top);
        if (count_of(a, to) < keep) mass = to;
    }
    const double want = r.u * sum_of(a, mass);
    const Hit<FINE> h = search<FINE>(a, r, table, s, q, source, [&](const Mass<FINE>& x) { return sum_of(a, x) > want; });
    *prob = weight(r, table, value_of(h.key)) * a.scale / sum_of(a, mass);
    return (uint32_t)h.key;
}

// The same by one wave that has all of the list, at most 64 tokens: lane i the i-th in rank order, with the mass of the
// row's tokens up to it.
template <bool FINE>
__device__ __forceinline__ uint32_t pick_by_wave(const GhSampleArgs& a, const Row& r, const double* table, const Plan& p, const PlanLds& s,
                                                 uint64_t key, double* prob) {
    const uint32_t lane = threadIdx.x & 63u, n = p.listed;
    key = gh_sort64(key);
    const bool there = lane < n;
    const float l = value_of(key);
    const uint32_t bin = there ? bin_of(r.top - l) : kNone;
    Mass<FINE> own = {0, 0};
    if (there) own = fixed<FINE>(a, r, table, l);
    const Mass<FINE> run = scan_mass(own), ahead = run - own;
    // the first lane of the token's bin: what is before it in the list is not what is before it in the row
    const uint32_t left = (uint32_t)__shfl_up((int)bin, 1, 64);
    const uint64_t heads = __ballot(lane == 0 || bin != left);
    const uint32_t head = 63 - (uint32_t)__clzll((long long)(heads & (~0ull >> (63 - lane))));
    Mass<FINE> skip;
    skip.whole = __shfl((unsigned long long)ahead.whole, (int)head, 64);
    if constexpr (FINE) skip.rest = __shfl((unsigned long long)ahead.rest, (int)head, 64);
    else skip.rest = head;
    Mass<FINE> m = {0, 0};
    if (there) m = before<FINE>(s, bin) + run - skip;
    const double w = sum_of(a, m);
    auto first = [&](bool is) __attribute__((always_inline)) {
        const uint64_t good = __ballot(there && is);
        return good ? (uint32_t)__builtin_ctzll(good) : 64u;
    };
    uint32_t keep = p.keep;
    Mass<FINE> mass = upto<FINE>(s, p.k);
    if (p.partly) {
        const uint32_t i = min(first(count_of(a, m) >= keep), n - 1);
        mass = lane_mass(m, i);
    }
    if (p.p0 != kNone) {
        const uint32_t i = first(w >= r.top_p * sum_of(a, mass) && bin >= p.p0);
        const Mass<FINE> mi = lane_mass(m, i & 63u);
        if (i < n && count_of(a, mi) < keep) {
            keep = count_of(a, mi);
            mass = mi;
        }
    }
    if (p.m0 != kNone) {
        const bool in = there && p.m0 <= bin && bin <= p.m1 && weight(r, table, l) >= (double)r.min_p;
        Mass<FINE> to = before<FINE>(s, p.m0) + lane_mass(scan_mass(in ? own : Mass<FINE>{0, 0}), 63);
        if (count_of(a, to) == 0) to = fixed<FINE>(a, r, table, r.top);
        if (count_of(a, to) < keep) mass = to;
    }
    const uint32_t i = min(first(w > r.u * sum_of(a, mass) && bin >= p.d0), n - 1);
    const uint64_t hit = gh_lane64(key, i);
    *prob = weight(r, table, value_of(hit)) * a.scale / sum_of(a, mass);
    return (uint32_t)hit;
}
template <bool FINE>
__device__ __forceinline__ void sample_pick(const GhSampleArgs& a, PlanLds& s, PickLds& q, double* table) {
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const Row r = row_of(a, row);
    auto done = [&](uint32_t token, double prob) __attribute__((always_inline)) {
        gh_gpw<uint32_t>(a.tokens)[row] = token;
        if (a.probs) gh_gpw<float>(a.probs)[row] = (float)prob;
    };
    if (r.greedy) {
        if (tid == 0) done(r.best, 1.0);
        return;
    }
    fill_exp(table);
    const uint64_t list = a.list + (uint64_t)row * kList * 8;
    uint64_t key = ~0ull;
    if (tid < 64) key = gh_gp<uint64_t>(list)[tid];  // on its way while the plan is made
    const Plan p = plan_of<FINE, kLook, kPick>(a, r, row, s);
    double prob;
    uint32_t token;
    if (p.listed <= 64) {
        if (tid >= 64) return;
        token = pick_by_wave<FINE>(a, r, table, p, s, tid < p.listed ? key : ~0ull, &prob);
    } else if (p.listed <= kList) {
        for (uint32_t i = tid; i < p.listed; i += kPick) q.list[i] = gh_gp<uint64_t>(list)[i];
        token = pick_by_search<FINE>(a, r, table, p, s, q, Listed{q.list, p.listed}, &prob);
    } else {
        token = pick_by_search<FINE>(a, r, table, p, s, q, Whole{a, row}, &prob);
    }
    if (tid == 0) done(token, prob);
}
}  // namespace

// Grid (rows), kPick threads.
GH_KERNEL __launch_bounds__(kPick) void gh_sample_pick(GhSampleArgs a) {
    __shared__ PlanLds s;
    __shared__ PickLds q;
    __shared__ double table[64];
    if (__builtin_expect(a.fine, 0)) {
        asm volatile("");
        sample_pick<true>(a, s, q, table);
    } else {
        sample_pick<false>(a, s, q, table);
    }
}
