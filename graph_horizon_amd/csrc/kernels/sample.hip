// Sampling of rows of logits: temperature, top-k, top-p, min-p and a draw by a given random number, as the host's
// gh_sample, in 64 bits.
//
// Tokens rank by (logit descending by f32 total order, index ascending), those with a finite logit. Token i has weight
// w = exp((l - M) / T), M the row's largest logit. Every filter keeps a prefix of the ranking, and the draw
// is the first rank whose running sum of weights passes u times the kept sum, so all a row needs are four searches in the
// running counts and sums. Sums are of whole numbers, w in fixed point: the same in any order, and off by 2^-45 at a
// vocabulary of 2^17, so that what lies next to a border of the kept or drawn range falls where 64 bits put it.
//
// Four launches; a row's logits are read three times, from memory once:
//   gh_sample_max     the largest logit of each chunk of a row;
//   gh_sample_bins    counts and sums over 1024 bins of the distance d = M - l, 64 per octave from 2^-9 to 2^7, so
//                     that a bin holds at most 3 % of any smooth distribution whatever its spread;
//   gh_sample_collect the tokens of the bins in which a search can end: the running sums up to the bins are known, and
//                     bound the top-k sum, then the kept sum, then the draw's target;
//   gh_sample_pick    sorts these tokens and searches them. More than fit are searched in the row itself.
// What the device cannot trust is only the settings: any bits give a token of the row.
#include "gh_common.h"

namespace {
constexpr uint32_t kBins = GH_SAMPLE_BINS, kList = GH_SAMPLE_LIST;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// f32 total order as unsigned order, and back
__device__ __forceinline__ uint32_t order_key(uint32_t bits) { return bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u); }
__device__ __forceinline__ float order_value(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }

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
    uint32_t best;      // index of the largest of all logits, infinite ones too (what a greedy row takes)
    bool greedy;        // T <= 0, or no finite logit
};
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t y = __shfl_xor((unsigned long long)v, o, 64);
        v = v > y ? v : y;
    }
    return v;
}
__device__ __forceinline__ Row row_of(const GhSampleArgs& a, uint32_t row) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint4 p = gh_gp<uint4>(a.params)[row];
    const uint64_t part = a.part + (uint64_t)row * 64 * 16;
    uint64_t any = 0, fin = 0;
    if (lane < a.chunks) {
        const ulonglong2 x = gh_gp<ulonglong2>(part)[lane];
        any = x.x;
        fin = x.y;
    }
    any = wave_max64(any);
    fin = wave_max64(fin);
    Row r;
    r.temperature = __uint_as_float(p.x);
    r.top_p = __uint_as_float(p.y);
    r.top_k = p.z;
    r.min_p = __uint_as_float(p.w);
    const float u = gh_gp<float>(a.uniform)[row];
    r.u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    r.inv = 1.0 / (double)r.temperature;
    r.top = order_value((uint32_t)fin);
    r.best = any ? ~(uint32_t)any : 0u;
    r.greedy = !(r.temperature > 0.0f) || fin == 0;
    return r;
}
__device__ __forceinline__ double weight(const Row& r, float l) { return exp(((double)l - (double)r.top) * r.inv); }
__device__ __forceinline__ uint64_t fixed(const GhSampleArgs& a, double w) { return (uint64_t)__double2ull_rn(w * a.scale); }

// Calls body(logit, index) for the chunk's tokens, in no order.
template <class F>
__device__ __forceinline__ void each_logit(const GhSampleArgs& a, uint32_t row, uint32_t first, uint32_t end, uint32_t threads, F body) {
    const GH_GLOBAL float* l = gh_gp<float>(a.logits) + (uint64_t)row * a.stride;
    for (uint32_t i = first + 4 * threadIdx.x; i < end; i += 8 * threads) {
        float v[2][4];
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            const uint32_t at = i + 4 * threads * k;
            if (a.wide && at + 4 <= end) {
                const float4 x = *(const GH_GLOBAL float4*)(l + at);
                v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) v[k][j] = at + j < end ? l[at + j] : __uint_as_float(0x7FC00000u);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k)
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) body(v[k][j], i + 4 * threads * k + j);
    }
}
}  // namespace

// Grid (chunks, rows), 256 threads. Also clears the row's bins for the next launch.
GH_KERNEL __launch_bounds__(256) void gh_sample_max(GhSampleArgs a) {
    __shared__ uint64_t red[4][2];
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
    GH_GLOBAL uint32_t* bins = gh_gpw<uint32_t>(a.bins + (uint64_t)row * GH_SAMPLE_BIN_BYTES);
    for (uint32_t i = blockIdx.x * 256 + tid; i < GH_SAMPLE_BIN_BYTES / 4; i += gridDim.x * 256) bins[i] = 0u;
    uint64_t any = 0;
    uint32_t fin = 0;
    each_logit(a, row, first, end, 256, [&](float l, uint32_t i) __attribute__((always_inline)) {
        if (finite(l)) fin = max(fin, order_key(__float_as_uint(l)));
        // -0 and 0 are equal here; a NaN is never the largest
        const uint64_t key = (uint64_t)order_key(__float_as_uint(l + 0.0f)) << 32 | (uint32_t)~i;
        if (l > -__builtin_inff()) any = any > key ? any : key;
    });
    any = wave_max64(any);
    const uint64_t top = wave_max64(fin);
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

// Grid (chunks, rows), 256 threads. Bins in LDS, added to the row's by atomics on whole numbers.
GH_KERNEL __launch_bounds__(256) void gh_sample_bins(GhSampleArgs a) {
    __shared__ unsigned long long sum[kBins];
    __shared__ uint32_t count[kBins];
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
    for (uint32_t i = tid; i < kBins; i += 256) {
        sum[i] = 0;
        count[i] = 0;
    }
    const Row r = row_of(a, row);
    if (r.greedy) return;
    __syncthreads();
    each_logit(a, row, first, end, 256, [&](float l, uint32_t) __attribute__((always_inline)) {
        if (!finite(l)) return;
        const uint32_t b = bin_of(r.top - l);
        atomicAdd(&count[b], 1u);
        const uint64_t w = fixed(a, weight(r, l));
        if (w) atomicAdd(&sum[b], (unsigned long long)w);
    });
    __syncthreads();
    const uint64_t bins = a.bins + (uint64_t)row * GH_SAMPLE_BIN_BYTES;
    for (uint32_t i = tid; i < kBins; i += 256) {
        if (!count[i]) continue;
        atomicAdd((unsigned long long*)bins + i, sum[i]);
        atomicAdd((uint32_t*)(bins + kBins * 8) + i, count[i]);
    }
}

namespace {
// The bins in which a row's searches end.
struct Plan {
    uint32_t tokens;        // finite logits
    uint32_t keep;          // min(top_k, tokens)
    uint32_t k;             // bin of the last of them
    bool partly;            // not all of that bin's
    uint64_t all;           // sum over all tokens
    uint32_t p0, p1;        // top-p's, first and last (kNone: off)
    uint32_t m0, m1;        // min-p's
    uint32_t d0, d1;        // the draw's
    uint32_t listed;        // tokens in these bins
    __device__ __forceinline__ bool has(uint32_t b) const {
        return (partly && b == k) || (p0 != kNone && p0 <= b && b <= p1) || (m0 != kNone && m0 <= b && b <= m1) || (d0 <= b && b <= d1);
    }
};
// LDS of a plan: inclusive running counts and sums of the bins.
struct PlanLds {
    uint64_t sum[kBins];
    uint32_t count[kBins];
    uint64_t wave_sum[16];
    uint32_t wave_count[16];
    uint32_t found[5], listed;
};
__device__ __forceinline__ uint64_t before(const PlanLds& s, uint32_t b) { return b ? s.sum[b - 1] : 0; }
__device__ __forceinline__ uint32_t count_before(const PlanLds& s, uint32_t b) { return b ? s.count[b - 1] : 0; }

__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)v, o, 64);
        if (lane >= o) v += y;
    }
    return v;
}

// The first bin whose running value satisfies `is`, at most `last`; THREADS threads, each kBins / THREADS bins.
template <uint32_t THREADS, class F>
__device__ __forceinline__ void first_bin(uint32_t* found, F is) {
    constexpr uint32_t kEach = kBins / THREADS;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t b = threadIdx.x * kEach + j;
        if (is(b)) {
            atomicMin(found, b);
            break;
        }
    }
}

// All threads get the same plan. u64 sums are compared as doubles, as the searches compare them.
template <uint32_t THREADS>
__device__ __forceinline__ Plan plan_of(const GhSampleArgs& a, const Row& r, uint32_t row, PlanLds& s) {
    constexpr uint32_t kEach = kBins / THREADS;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint64_t bins = a.bins + (uint64_t)row * GH_SAMPLE_BIN_BYTES;
    uint64_t w[kEach], ws = 0;
    uint32_t c[kEach], cs = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        w[j] = gh_gp<uint64_t>(bins)[tid * kEach + j];
        c[j] = gh_gp<uint32_t>(bins + kBins * 8)[tid * kEach + j];
        ws += w[j];
        cs += c[j];
    }
    const uint64_t wu = wave_scan64(ws);
    const uint32_t cu = (uint32_t)wave_scan64(cs);
    if (lane == 63) {
        s.wave_sum[wave] = wu;
        s.wave_count[wave] = cu;
    }
    if (tid < 5) s.found[tid] = kBins - 1;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    uint64_t wat = wu - ws;
    uint32_t cat = cu - cs;
    for (uint32_t i = 0; i < wave; ++i) {
        wat += s.wave_sum[i];
        cat += s.wave_count[i];
    }
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        s.sum[tid * kEach + j] = wat += w[j];
        s.count[tid * kEach + j] = cat += c[j];
    }
    __syncthreads();
    Plan p;
    p.tokens = s.count[kBins - 1];
    p.all = s.sum[kBins - 1];
    p.keep = r.top_k && r.top_k < p.tokens ? r.top_k : p.tokens;
    first_bin<THREADS>(&s.found[0], [&](uint32_t b) { return s.count[b] >= p.keep; });
    __syncthreads();
    p.k = s.found[0];
    p.partly = s.count[p.k] > p.keep;
    // the sum of the first top_k lies between lo and hi
    uint64_t lo = p.partly ? before(s, p.k) : s.sum[p.k], hi = s.sum[p.k];
    uint32_t c0 = p.k, c1 = p.k;  // the last kept token's bins
    p.p0 = p.p1 = p.m0 = p.m1 = kNone;
    const bool nucleus = r.top_p < 1.0f;
    if (nucleus) {
        first_bin<THREADS>(&s.found[1], [&](uint32_t b) { return (double)s.sum[b] >= r.top_p * (double)lo; });
        first_bin<THREADS>(&s.found[2], [&](uint32_t b) { return (double)s.sum[b] >= r.top_p * (double)hi; });
    }
    __syncthreads();
    if (nucleus) {
        c0 = p.p0 = min(s.found[1], p.k);
        c1 = p.p1 = min(s.found[2], p.k);
    }
    if (r.min_p > 0.0f) {
        // w >= min_p up to a distance of -T ln min_p; d is rounded to FP32
        const double d = -log((double)r.min_p) * (double)r.temperature;
        p.m0 = d > 0.0 ? bin_of((float)(d * (1.0 - 1e-6))) : 0u;
        p.m1 = d > 0.0 ? bin_of((float)(d * (1.0 + 1e-6))) : 0u;
        c0 = min(c0, p.m0);
        c1 = min(c1, p.m1);
    }
    // the kept sum lies between lo and hi
    if (c0 != p.k || p.partly || nucleus || r.min_p > 0.0f) lo = before(s, c0);
    hi = s.sum[c1];
    first_bin<THREADS>(&s.found[3], [&](uint32_t b) { return (double)s.sum[b] > r.u * (double)lo; });
    first_bin<THREADS>(&s.found[4], [&](uint32_t b) { return (double)s.sum[b] > r.u * (double)hi; });
    __syncthreads();
    p.d0 = min(s.found[3], c1);
    p.d1 = min(s.found[4], c1);
    uint32_t listed = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) listed += p.has(tid * kEach + j) ? c[j] : 0u;
    if (listed) atomicAdd(&s.listed, listed);
    __syncthreads();
    p.listed = s.listed;
    return p;
}
}  // namespace

// Grid (chunks, rows), 256 threads.
GH_KERNEL __launch_bounds__(256) void gh_sample_collect(GhSampleArgs a) {
    __shared__ PlanLds s;
    __shared__ uint32_t need[kBins / 32];
    const uint32_t tid = threadIdx.x, row = blockIdx.y, first = blockIdx.x * a.per, end = min(a.vocab, first + a.per);
    const Row r = row_of(a, row);
    if (r.greedy) return;
    const Plan p = plan_of<256>(a, r, row, s);
    if (p.listed > kList) return;
    if (tid < kBins / 32) {
        uint32_t bits = 0;
        for (uint32_t j = 0; j < 32; ++j) bits |= (uint32_t)p.has(32 * tid + j) << j;
        need[tid] = bits;
    }
    __syncthreads();
    const uint64_t list = a.list + (uint64_t)row * kList * 8;
    uint32_t* length = (uint32_t*)(a.bins + (uint64_t)row * GH_SAMPLE_BIN_BYTES + kBins * 12);
    each_logit(a, row, first, end, 256, [&](float l, uint32_t i) __attribute__((always_inline)) {
        if (!finite(l)) return;
        const uint32_t b = bin_of(r.top - l);
        if (!(need[b >> 5] >> (b & 31u) & 1u)) return;
        const uint32_t at = atomicAdd(length, 1u);
        // ascending in rank order
        if (at < kList) gh_gpw<uint64_t>(list)[at] = (uint64_t)~order_key(__float_as_uint(l)) << 32 | i;
    });
}

namespace {
constexpr uint32_t kPick = 1024;  // threads
struct PickLds {
    uint64_t key[kList];  // (~order of the logit) << 32 | index, sorted
    uint64_t upto[kList]; // running sums
    uint64_t skip_sum[kBins];   // of a bin: what is before it and not listed
    uint32_t skip_count[kBins];
    uint32_t found[8];
    uint64_t value[8];
};
__device__ __forceinline__ float value_of(uint64_t key) { return order_value(~(uint32_t)(key >> 32)); }

// key[0 .. n) sorted, n a power of two.
__device__ __forceinline__ void sort_keys(uint64_t* key, uint32_t n) {
    for (uint32_t size = 2; size <= n; size <<= 1)
        for (uint32_t stride = size >> 1; stride > 0; stride >>= 1) {
            for (uint32_t t = threadIdx.x; t < n / 2; t += kPick) {
                const uint32_t i = 2 * t - (t & (stride - 1));
                const uint64_t x = key[i], y = key[i + stride];
                if ((x > y) == ((i & size) == 0)) {
                    key[i] = y;
                    key[i + stride] = x;
                }
            }
            __syncthreads();
        }
}
}  // namespace

namespace {
// Equal logits, and what ranks before them.
struct Ties {
    uint32_t key, count, count_before;
    uint64_t w, before;
    // how many of them it takes until `is` holds for the sum
    template <class F>
    __device__ __forceinline__ uint32_t until(F is) const {
        uint32_t lo = 1, hi = max(count, 1u);
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (is(before + mid * w)) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    }
};
// The first equal logits in rank order up to which the number and the sum of tokens satisfy `is`: eight bits of the logits'
// order at a time, over the whole row.
template <class F>
__device__ __forceinline__ Ties descend(const GhSampleArgs& a, const Row& r, uint32_t row, PlanLds& s, F is) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    Ties t{0, 0, 0, 0, 0};
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) {
            s.sum[tid] = 0;
            s.count[tid] = 0;
        }
        if (tid == 0) s.found[0] = 255;
        __syncthreads();
        each_logit(a, row, 0, a.vocab, kPick, [&](float l, uint32_t) __attribute__((always_inline)) {
            const uint32_t key = ~order_key(__float_as_uint(l));
            if (!finite(l) || (shift < 24 && key >> (shift + 8) != t.key)) return;
            atomicAdd(&s.count[key >> shift & 255u], 1u);
            atomicAdd((unsigned long long*)&s.sum[key >> shift & 255u], (unsigned long long)fixed(a, weight(r, l)));
        });
        __syncthreads();
        uint64_t wu = 0;
        uint32_t cu = 0;
        if (tid < 256) {
            wu = wave_scan64(s.sum[tid]);
            cu = (uint32_t)wave_scan64(s.count[tid]);
            if (lane == 63) {
                s.wave_sum[wave] = wu;
                s.wave_count[wave] = cu;
            }
        }
        __syncthreads();
        if (tid < 256) {
            for (uint32_t i = 0; i < wave; ++i) {
                wu += s.wave_sum[i];
                cu += s.wave_count[i];
            }
            s.sum[256 + tid] = wu;
            s.count[256 + tid] = cu;
            if (is(t.count_before + cu, t.before + wu)) atomicMin(&s.found[0], tid);
        }
        __syncthreads();
        const uint32_t b = s.found[0];
        t.key = t.key << 8 | b;
        t.count = s.count[b];
        t.count_before += s.count[256 + b] - s.count[b];
        t.before += s.sum[256 + b] - s.sum[b];
    }
    t.w = fixed(a, weight(r, order_value(~t.key)));
    return t;
}

// The searches of gh_sample_pick over the whole row. Returns the token, its weight over the kept sum in *prob.
__device__ __forceinline__ uint32_t pick_from_row(const GhSampleArgs& a, const Row& r, const Plan& p, uint32_t row, PlanLds& s, double* prob) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    uint32_t keep = p.keep;
    uint64_t sum = p.all;
    if (keep < p.tokens) {
        const Ties t = descend(a, r, row, s, [&](uint32_t c, uint64_t) { return c >= keep; });
        sum = t.before + (keep - t.count_before) * t.w;
    }
    if (r.top_p < 1.0f) {
        const double want = r.top_p * (double)sum;
        const Ties t = descend(a, r, row, s, [&](uint32_t, uint64_t w) { return (double)w >= want; });
        const uint32_t j = t.until([&](uint64_t w) { return (double)w >= want; });
        if (t.count_before + j < keep) {
            keep = t.count_before + j;
            sum = t.before + j * t.w;
        }
    }
    if (r.min_p > 0.0f) {
        __syncthreads();
        if (tid == 0) {
            s.sum[0] = 0;
            s.count[0] = 0;
        }
        __syncthreads();
        uint64_t w = 0;
        uint32_t c = 0;
        each_logit(a, row, 0, a.vocab, kPick, [&](float l, uint32_t) __attribute__((always_inline)) {
            if (!finite(l)) return;
            const double x = weight(r, l);
            if (x < (double)r.min_p) return;
            ++c;
            w += fixed(a, x);
        });
        atomicAdd(&s.count[0], c);
        atomicAdd((unsigned long long*)&s.sum[0], (unsigned long long)w);
        __syncthreads();
        const uint32_t rank = max(s.count[0], 1u);
        if (rank < keep) {
            keep = rank;
            sum = s.count[0] ? s.sum[0] : fixed(a, 1.0);
        }
    }
    const double want = r.u * (double)sum;
    const Ties t = descend(a, r, row, s, [&](uint32_t, uint64_t w) { return (double)w > want; });
    const uint32_t j = t.until([&](uint64_t w) { return (double)w > want; });
    *prob = weight(r, order_value(~t.key)) * a.scale / (double)sum;
    // the j-th of them by index: each thread counts in a part of the row
    const GH_GLOBAL uint32_t* l = gh_gp<uint32_t>(a.logits) + (uint64_t)row * a.stride;
    const uint32_t per = (a.vocab + kPick - 1) / kPick, from = min(tid * per, a.vocab), end = min(from + per, a.vocab);
    uint32_t mine = 0;
    for (uint32_t i = from; i < end; ++i) mine += ~order_key(l[i]) == t.key;
    const uint32_t upto = (uint32_t)wave_scan64(mine);
    __syncthreads();
    if (lane == 63) s.wave_count[wave] = upto;
    if (tid == 0) s.found[0] = r.best;
    __syncthreads();
    uint32_t at = upto - mine;
    for (uint32_t i = 0; i < wave; ++i) at += s.wave_count[i];
    if (at < j && j <= at + mine)
        for (uint32_t i = from; i < end; ++i)
            if (~order_key(l[i]) == t.key && ++at == j) s.found[0] = i;
    __syncthreads();
    return s.found[0];
}
}  // namespace

// Grid (rows), 1024 threads.
GH_KERNEL __launch_bounds__(1024) void gh_sample_pick(GhSampleArgs a) {
    __shared__ PlanLds s;
    __shared__ PickLds q;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, row = blockIdx.x;
    const Row r = row_of(a, row);
    auto done = [&](uint32_t token, double prob) __attribute__((always_inline)) {
        gh_gpw<uint32_t>(a.tokens)[row] = token;
        if (a.probs) gh_gpw<float>(a.probs)[row] = (float)prob;
    };
    if (r.greedy) {
        if (tid == 0) done(r.best, 1.0);
        return;
    }
    const Plan p = plan_of<kPick>(a, r, row, s);
    if (p.listed > kList) {
        double prob;
        const uint32_t token = pick_from_row(a, r, p, row, s, &prob);
        if (tid == 0) done(token, prob);
        return;
    }
    const uint32_t n = p.listed;
    uint32_t size = 64;
    while (size < n) size <<= 1;
    const uint64_t list = a.list + (uint64_t)row * kList * 8;
    for (uint32_t i = tid; i < size; i += kPick) q.key[i] = i < n ? gh_gp<uint64_t>(list)[i] : ~0ull;
    // of each bin: the sums and counts of the bins before it that are not listed
    {
        const uint32_t b = tid;  // kBins == kPick
        const bool in = p.has(b);
        const uint64_t w = in ? s.sum[b] - before(s, b) : 0;
        const uint32_t c = in ? s.count[b] - count_before(s, b) : 0;
        const uint64_t wu = wave_scan64(w);
        const uint32_t cu = (uint32_t)wave_scan64(c);
        __syncthreads();
        if (lane == 63) {
            s.wave_sum[wave] = wu;
            s.wave_count[wave] = cu;
        }
        __syncthreads();
        uint64_t wat = wu - w;
        uint32_t cat = cu - c;
        for (uint32_t i = 0; i < wave; ++i) {
            wat += s.wave_sum[i];
            cat += s.wave_count[i];
        }
        q.skip_sum[b] = before(s, b) - wat;
        q.skip_count[b] = count_before(s, b) - cat;
        if (tid < 8) q.found[tid] = kNone;
    }
    __syncthreads();
    sort_keys(q.key, size);
    // running sums: thread t has kList / kPick tokens in a row
    constexpr uint32_t kEach = kList / kPick;
    const uint32_t each = size > kPick ? size / kPick : 1;
    uint64_t own[kEach], mine = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t i = tid * each + j;
        own[j] = j < each && i < n ? fixed(a, weight(r, value_of(q.key[i]))) : 0;
        mine += own[j];
    }
    const uint64_t upto = wave_scan64(mine);
    if (lane == 63) s.wave_sum[wave] = upto;
    __syncthreads();
    uint64_t at = upto - mine;
    for (uint32_t i = 0; i < wave; ++i) at += s.wave_sum[i];
    // the thread's tokens: running sum of all tokens up to it, and its rank
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        const uint32_t i = tid * each + j;
        if (j < each && i < n) {
            at += own[j];
            q.upto[i] = at + q.skip_sum[bin_of(r.top - value_of(q.key[i]))];
        }
    }
    __syncthreads();
    auto bin_at = [&](uint32_t i) __attribute__((always_inline)) { return bin_of(r.top - value_of(q.key[i])); };
    auto rank_at = [&](uint32_t i) __attribute__((always_inline)) { return i + q.skip_count[bin_at(i)]; };
    // the first listed token for which `is`
    auto first = [&](uint32_t slot, auto is) __attribute__((always_inline)) {
        for (uint32_t i = tid; i < n; i += kPick)
            if (is(i)) {
                atomicMin(&q.found[slot], i);
                break;
            }
        __syncthreads();
        return q.found[slot];
    };
    // how many are kept, and their sum
    uint32_t keep = p.keep;
    uint64_t sum = s.sum[p.k];
    if (p.partly) sum = q.upto[first(0, [&](uint32_t i) { return rank_at(i) + 1 == p.keep; })];
    if (p.p0 != kNone) {
        const double want = r.top_p * (double)sum;
        const uint32_t i = first(1, [&](uint32_t i) { return (double)q.upto[i] >= want && bin_at(i) >= p.p0; });
        if (i < n && rank_at(i) + 1 < keep) {
            keep = rank_at(i) + 1;
            sum = q.upto[i];
        }
    }
    if (p.m0 != kNone) {
        const uint32_t i = first(2, [&](uint32_t i) {
            const uint32_t b = bin_at(i);
            return p.m0 <= b && b <= p.m1 && weight(r, value_of(q.key[i])) < (double)r.min_p;
        });
        uint32_t rank = i == kNone ? s.count[p.m1] : rank_at(i);
        uint64_t to = i == kNone ? s.sum[p.m1] : q.upto[i] - fixed(a, weight(r, value_of(q.key[i])));
        if (rank == 0) {
            rank = 1;
            to = fixed(a, 1.0);
        }
        if (rank < keep) {
            keep = rank;
            sum = to;
        }
    }
    const double want = r.u * (double)sum;
    const uint32_t i = min(first(3, [&](uint32_t i) { return (double)q.upto[i] > want && bin_at(i) >= p.d0; }), n - 1);
    if (tid == 0) {
        const uint64_t key = q.key[i];
        done((uint32_t)key, weight(r, value_of(key)) * a.scale / (double)sum);
    }
}
