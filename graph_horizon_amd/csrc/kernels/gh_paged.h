// Device code shared by the operators over paged caches, FP16 (paged.hip) and 4-bit (paged4.hip): what a row's
// length and table say, and decode attention's running sums, partials and scores.
#ifndef GH_PAGED_H
#define GH_PAGED_H
#include "gh_common.h"

namespace {
constexpr uint32_t kBad = 0xFFFFFFFFu;

__device__ __forceinline__ void fault(const GhPages& p, uint32_t what) { *gh_gpw<uint32_t>(p.fault) = what; }

// The row's length, 0 where it is longer than `most` (reported by the caller's first workgroup).
__device__ __forceinline__ uint32_t row_length(const GhPages& p, uint32_t row, uint32_t most, bool first) {
    const uint32_t n = gh_gp<uint32_t>(p.lengths)[row];
    if (n <= most) return n;
    if (first && threadIdx.x == 0) fault(p, GH_PAGED_LENGTH);
    return 0;
}

// Inclusive sum over the wave in DPP steps: within rows of 16 lanes, then the rows' totals onward.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t scan_step(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = scan_step<0x111, 0xF>(v);     // row_shr:1
    v = scan_step<0x112, 0xF>(v);     // row_shr:2
    v = scan_step<0x114, 0xF>(v);     // row_shr:4
    v = scan_step<0x118, 0xF>(v);     // row_shr:8
    v = scan_step<0x142, 0xA>(v);     // row_bcast:15 into rows 1 and 3
    return scan_step<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

// Slot of a row's position, kBad where the table's page is beyond the pool.
__device__ __forceinline__ uint32_t slot_of(const GhPages& p, uint32_t row, uint32_t pos) {
    const uint32_t page = gh_gp<uint32_t>(p.table)[(uint64_t)row * p.width + (pos >> p.shift)];
    if (page >= p.pages) {
        fault(p, GH_PAGED_PAGE);
        return kBad;
    }
    return (page << p.shift) + (pos & ((1u << p.shift) - 1));
}

// ---- decode attention ----
typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef float pf4 __attribute__((ext_vector_type(4)));
typedef uint16_t pu2 __attribute__((ext_vector_type(2)));
constexpr int kBufWord3 = 0x00020000;  // raw buffer, 32-bit data format
constexpr float kUp = 15.0f;
constexpr int kStream = 2;  // cache policy of reads that will not be wanted again soon (nt)

__device__ __forceinline__ float lanes4_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lanes4_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 2^(m - M), 0 for m = -inf whatever M is.
__device__ __forceinline__ float share(float m, float M) {
    return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - M);
}

// two outputs as FP16: sums times 1 / Σ weights (one division, where a quotient each takes ten instructions; two
// FP32 roundings before the one to FP16)
__device__ __forceinline__ uint32_t out2(float x, float y, float inv) {
    return (uint32_t)gh_f2h(x * inv) | (uint32_t)gh_f2h(y * inv) << 16;
}

// A wave's running sums: lane l holds head n = l % 16's maximum, its own part of Σ weights, and value dims
// 32 (l / 16) + 8 j + t in acc[t][j].
struct Sums {
    float m, l;
    pf4 acc[8];
    __device__ __forceinline__ void clear() {
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    }
};

// A row's output from whole sums, L the sum of the weights over the lanes.
__device__ __forceinline__ void store_out(const GhPagedAttnArgs& a, uint32_t row, uint32_t kvh, const Sums& x, float L) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
    const float inv = 1.0f / L;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) w[t] = out2(x.acc[2 * t][j], x.acc[2 * t + 1][j], inv);
        *gh_gpw<uint4>(a.out + ((uint64_t)row * a.q_heads + kvh * a.group + n) * 256 + 64 * g + 16 * j) =
            make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// The sums as partial `part` (of the lane's head).
__device__ __forceinline__ void store_partial(const GhPagedAttnArgs& a, uint64_t part, const Sums& x, float L) {
    const uint32_t g = (threadIdx.x & 63u) >> 4;
    GH_GLOBAL float4* to = gh_gpw<float4>(a.part_acc + part * 512 + 128 * g);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        to[2 * j] = make_float4(x.acc[0][j], x.acc[1][j], x.acc[2][j], x.acc[3][j]);
        to[2 * j + 1] = make_float4(x.acc[4][j], x.acc[5][j], x.acc[6][j], x.acc[7][j]);
    }
    if (g == 0) gh_gpw<float2>(a.part_ml)[part] = make_float2(x.m, L);
}

// The scores of four query heads h0 .. h0 + 3 (the last of G again past G) at positions pos .. pos + 3.
__device__ __forceinline__ void load_raw(const GhPagedAttnArgs& a, uint32_t row, uint32_t kvh, uint32_t h0, uint32_t pos, pf4 (&s)[4]) {
    const uint64_t raw = a.raw + ((uint64_t)row * a.p.kv_heads + kvh) * a.group * a.raw_len * 4;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) s[i] = *gh_gp<pf4>(raw + ((uint64_t)min(h0 + i, a.group - 1) * a.raw_len + pos) * 4);
}
// Adds the weights of positions pos .. + 3, pos + step .. + 3, ... < len to the scores of a row and kv head:
// 2^(s - M + 15) / L per query head, summed over the G heads in order. s: load_raw of the first four heads
// at the first position, where that is below len. Positions past the row keep their bits.
__device__ __forceinline__ void add_scores(const GhPagedAttnArgs& a, uint32_t row, uint32_t kvh, const float* M, const float* L,
                                           uint32_t pos, uint32_t step, uint32_t len, pf4 (&s)[4]) {
    const uint64_t to = a.p.score + ((uint64_t)row * a.p.kv_heads + kvh) * (a.p.width << a.p.shift) * 4;
    for (bool first = true; pos < len; pos += step, first = false) {
        GH_GLOBAL pf4* p = (GH_GLOBAL pf4*)gh_gpw<float>(to + (uint64_t)pos * 4);
        const pf4 old = *p;
        pf4 w = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t h0 = 0; h0 < a.group; h0 += 4) {
            if (h0 || !first) load_raw(a, row, kvh, h0, pos, s);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (h0 + i < a.group) {
                    const float up = kUp - M[h0 + i], inv = 1.0f / L[h0 + i];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] += __builtin_amdgcn_exp2f(s[i][j] + up) * inv;
                }
        }
        if (pos + 4 <= len) {
            *p = old + w;
        } else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (pos + j < len) gh_gpw<float>(to)[pos + j] = old[j] + w[j];
        }
    }
}

constexpr uint32_t kRows = 512;  // rows of a launch at most

// The rows' tiles one after the other: row r has tiles first[r] .. first[r + 1], of 16 positions or 32.
struct RowsLds {
    uint32_t len[kRows], first[kRows + 1];
    uint32_t sums[4];
};

// Fills sh from the rows' lengths (longer ones than max_len count 0); 256 threads. Up to 64 rows: lane r also gets
// the first tile behind row r. Tiles of 2^SHIFT positions.
template <int SHIFT>
__device__ __forceinline__ uint32_t lay_out_rows(const GhPagedAttnArgs& a, RowsLds& sh, bool report) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    if (a.rows <= 64) {  // each wave by itself, the same values
        uint32_t n = lane < a.rows ? gh_gp<uint32_t>(a.p.lengths)[lane] : 0u;
        if (n > a.max_len) {
            if (report) fault(a.p, GH_PAGED_LENGTH);
            n = 0;
        }
        const uint32_t upto = wave_scan((n + (1u << SHIFT) - 1) >> SHIFT);
        sh.len[lane] = n;
        if (lane == 0) sh.first[0] = 0;
        sh.first[lane + 1] = upto;
        // The wave reads what its other lanes wrote, and the other waves write the same values over it: nothing waits for
        // them, and the fence keeps the wave's own writes before its reads.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        return upto;
    }
    uint32_t n[2], t[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {  // rows 2 tid, 2 tid + 1
        const uint32_t r = 2 * tid + i;
        n[i] = r < a.rows ? gh_gp<uint32_t>(a.p.lengths)[r] : 0u;
        if (n[i] > a.max_len) {
            if (report) fault(a.p, GH_PAGED_LENGTH);
            n[i] = 0;
        }
        t[i] = (n[i] + (1u << SHIFT) - 1) >> SHIFT;
    }
    uint32_t upto = wave_scan(t[0] + t[1]);
    if (lane == 63) sh.sums[wave] = upto;
    sh.len[2 * tid] = n[0];
    sh.len[2 * tid + 1] = n[1];
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) upto += sh.sums[w];
    if (tid == 0) sh.first[0] = 0;
    sh.first[2 * tid + 1] = upto - t[1];
    sh.first[2 * tid + 2] = upto;
    __syncthreads();
    return 0;
}

// The end of a span of one row and kv head: the sums of the workgroup's four waves joined in `dyn` (per wave and head
// 132 floats of acc, then m and l), as an output with its scores where the row has one span, else as a partial.
template <bool SCORED>
__device__ __forceinline__ void split_finish(const GhPagedAttnArgs& a, const Sums& x, float* dyn, uint32_t row, uint32_t kvh,
                                             uint32_t split, uint32_t span, uint32_t len) {
    __shared__ float sM[16], sL[16];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t out = a.out + ((uint64_t)row * a.q_heads + kvh * G) * 256;
    // M = max m_w, L = Σ 2^(m_w - M) l_w, ACC likewise
    float* wm = dyn + 4 * G * 132;
    float* wl = wm + 4 * G;
    const float lt = lanes4_sum(x.l);
    if (n < G) {
        const uint32_t at = wave * G + n;
        if (g == 0) {
            wm[at] = x.m;
            wl[at] = lt;
        }
        float4* to = (float4*)(dyn + at * 132 + 32 * g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            to[2 * j] = make_float4(x.acc[0][j], x.acc[1][j], x.acc[2][j], x.acc[3][j]);
            to[2 * j + 1] = make_float4(x.acc[4][j], x.acc[5][j], x.acc[6][j], x.acc[7][j]);
        }
    }
    __syncthreads();
    const bool whole = len <= span;  // one split: the output itself
    const uint64_t part = ((uint64_t)row * a.chunks + split) * a.p.kv_heads * G + kvh * G;
    for (uint32_t i = tid; i < G * 64; i += 256) {
        const uint32_t h = i >> 6, d = 2 * (i & 63u);
        float M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, wm[w * G + h]);
        float L = 0.0f;
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float e = share(wm[w * G + h], M);
            const float2 y = *(const float2*)(dyn + (w * G + h) * 132 + d);
            L += e * wl[w * G + h];
            v.x += e * y.x;
            v.y += e * y.y;
        }
        if (whole) gh_gpw<uint32_t>(out)[i] = out2(v.x, v.y, 1.0f / L);
        else gh_gpw<float2>(a.part_acc)[part * 64 + i] = v;
        if (d == 0) {
            sM[h] = M;
            sL[h] = L;
            if (!whole) gh_gpw<float2>(a.part_ml)[part + h] = make_float2(M, L);
        }
    }
    if (!SCORED || !whole) return;
    __syncthreads();
    pf4 s[4];
    if (4 * tid < len) load_raw(a, row, kvh, 0, 4 * tid, s);
    add_scores(a, row, kvh, sM, sL, 4 * tid, 1024, len, s);
}
}  // namespace

#endif
