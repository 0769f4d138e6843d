// A batch of sequences over paged FP16 caches (gh_kv_paged): append with RoPE, decode attention, eviction.
//
// The pool is a cache [layer][slot][kv_heads][128]; position j of row r lives at slot
// (table[r][j >> shift] << shift) + (j & page_size - 1). Lengths, page numbers and positions are device data
// that the host has not seen: every kernel checks them before it forms an address, skips what does not fit
// and leaves a word in pinned host memory, which gh_submit reports.
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

// Slot of a row's position, kBad where the table's page is beyond the pool.
__device__ __forceinline__ uint32_t slot_of(const GhPages& p, uint32_t row, uint32_t pos) {
    const uint32_t page = gh_gp<uint32_t>(p.table)[(uint64_t)row * p.width + (pos >> p.shift)];
    if (page >= p.pages) {
        fault(p, GH_PAGED_PAGE);
        return kBad;
    }
    return (page << p.shift) + (pos & ((1u << p.shift) - 1));
}
}  // namespace

// ---- append ----------------------------------------------------------------------------------
// Thread = 8 values (16 bytes) of one head of one token: the token's query heads, then its key and value
// heads; a.groups workgroups per token. Rotation as in gh_rope: adjacent pairs turned by the (position, pair)
// table's (cos, sin) in FP32, queries times the post-scale, one rounding. Bound by launch latency at decode
// sizes and by memory at prompt sizes.
namespace {
__device__ __forceinline__ uint32_t turn(uint32_t v, float2 c, float scale) {
#pragma clang fp contract(off)
    const float x0 = gh_h2f(v & 0xFFFFu), x1 = gh_h2f(v >> 16);
    const float y0 = (x0 * c.x - x1 * c.y) * scale;
    const float y1 = (x0 * c.y + x1 * c.x) * scale;
    return (uint32_t)gh_f2h(y0) | ((uint32_t)gh_f2h(y1) << 16);
}
}  // namespace

GH_KERNEL __launch_bounds__(256) void gh_paged_write(GhPagedWriteArgs a) {
    const uint32_t token = blockIdx.x / a.groups, row = token / a.tokens, t = token % a.tokens;
    const uint32_t item = (blockIdx.x % a.groups) * 256 + threadIdx.x;
    const uint32_t head = item >> 4, part = item & 15u;  // 8 dims each
    const uint32_t n = row_length(a.p, row, a.p.width << a.p.shift, blockIdx.x % a.groups == 0);
    if (n + t < a.tokens) return;  // a free row, or before its first position
    const uint32_t at = n - a.tokens + t;
    uint32_t pos = 0;
    if (a.positions) {
        const uint32_t from = gh_gp<uint32_t>(a.positions)[row];
        if (from > a.max_pos || t > a.max_pos - from) {
            if (item == 0) fault(a.p, GH_PAGED_POSITION);
            return;
        }
        pos = from + t;
    }
    if (head >= a.q_heads + 2 * a.p.kv_heads) return;
    const bool query = head < a.q_heads, value = head >= a.q_heads + a.p.kv_heads;
    const uint32_t h = query ? head : head - a.q_heads - (value ? a.p.kv_heads : 0u);
    const uint32_t heads = query ? a.q_heads : a.p.kv_heads;
    const uint64_t in = ((uint64_t)token * heads + h) * 256 + 16 * part;
    uint4 x = *gh_gp<uint4>((query ? a.q : value ? a.v : a.k) + in);
    if (a.positions && !value && 4 * part < a.pairs) {
        const float scale = query ? gh_gp<float>(a.post)[pos] : 1.0f;
        const GH_GLOBAL float2* cs = gh_gp<float2>(a.table) + (uint64_t)pos * a.pairs + 4 * part;
        x.x = turn(x.x, cs[0], scale);
        if (4 * part + 1 < a.pairs) x.y = turn(x.y, cs[1], scale);
        if (4 * part + 2 < a.pairs) x.z = turn(x.z, cs[2], scale);
        if (4 * part + 3 < a.pairs) x.w = turn(x.w, cs[3], scale);
    }
    if (query) {
        *gh_gpw<uint4>(a.q_out + in) = x;
        return;
    }
    const uint32_t slot = slot_of(a.p, row, at);
    if (slot == kBad) return;
    *gh_gpw<uint4>((value ? a.p.vc : a.p.kc) + ((uint64_t)slot * a.p.kv_heads + h) * 256 + 16 * part) = x;
    if (a.p.score && !value && part == 0)
        gh_gpw<float>(a.p.score)[((uint64_t)row * a.p.kv_heads + h) * (a.p.width << a.p.shift) + at] = 0.0f;
}

// ---- decode attention ---------------------------------------------------------------------------
// Grid (kv heads, splits, rows), 256 threads: a workgroup takes the G query heads of one kv head over `span`
// positions of one row. Wave w owns tiles of 16 positions w, w + 4, ... of the span, each within one page
// (page_size >= 16): lane i holds the table entry of the wave's i-th tile, read once at the start, so a
// tile's address is a readlane away. Per tile, with FP32 accumulators and scores in base 2:
//   S^T = K·Q^T     4 x v_mfma_f32_16x16x32_f16: A = 16 K rows straight from memory (lane l: position l % 16,
//                   dims 32 s + 8 (l / 16) .. + 8), B = the query, column n = l % 16 is head n (zero
//                   past G); lane l receives head n's scores of positions 4 (l / 16) + i;
//   O^T += V^T·P^T  per 8-dim tile t one v_mfma_f32_16x16x32_f16 whose 32 k-slots are the 16 positions
//                   twice: a lane's weights split into FP16 hi + lo (truncated, so both are positive), so
//                   that P·V keeps 22 bits of each weight. Output row m stands for value dim 8 m + t.
// Weights are 2^(s - m + 15), m the running maximum: hi + lo then reach 2^-39 of the largest weight. Both
// parts are at least 2^-24, so that an infinite V gives an infinity and not infinity times 0.
// K and V are read through buffer resources whose range ends at the row's last position: what a page holds
// past it reads as zero, without a memory access, and has weight 0.
namespace {
typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef float pf4 __attribute__((ext_vector_type(4)));
typedef uint16_t pu2 __attribute__((ext_vector_type(2)));
constexpr int kBufWord3 = 0x00020000;  // raw buffer, 32-bit data format
constexpr float kUp = 15.0f;

struct Tile {
    uint4 k[4];  // position l % 16, dims 32 s + 8 (l / 16) .. + 8
    uint4 v[4];  // position 4 (l / 16) + i, dims 8 (l % 16) .. + 8
};

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

// element t of the 16-byte slices of four positions, twice (the hi and the lo slots)
__device__ __forceinline__ ph8 v_column(const uint4 (&v)[4], int t) {
    auto word = [&](int i) __attribute__((always_inline)) {
        return (t >> 1) == 0 ? v[i].x : (t >> 1) == 1 ? v[i].y : (t >> 1) == 2 ? v[i].z : v[i].w;
    };
    const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;  // the high or the low halves of two words
    const uint32_t d0 = __builtin_amdgcn_perm(word(1), word(0), sel), d1 = __builtin_amdgcn_perm(word(3), word(2), sel);
    return __builtin_bit_cast(ph8, make_uint4(d0, d1, d0, d1));
}

// two weights' FP16 hi parts in *hi, lo parts in *lo
__device__ __forceinline__ void weight_parts(float p0, float p1, uint32_t* hi, uint32_t* lo) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const pu2 one = {1, 1};
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    const h2 hv = __builtin_bit_cast(h2, h);
    const uint32_t l = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0 - (float)hv.x, p1 - (float)hv.y));
    *hi = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pu2, h), one));
    *lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pu2, l), one));
}

template <int GM>
struct AttnLds {
    float m[4][GM], l[4][GM];
    float acc[4][GM][132];
    float e[4][GM], M[GM], L[GM];
};

template <int GM, bool SCORED>
__device__ __forceinline__ void paged_attn(const GhPagedAttnArgs& a) {
    __shared__ AttnLds<GM> sh;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, row = blockIdx.z, G = a.group;
    const uint32_t begin = split * a.span;  // < max_len
    // the wave's table entries: tile i covers positions begin + 64 i + 16 wave .. + 16
    const uint32_t mine = begin + 64 * lane + 16 * wave;
    uint32_t entry = 0;
    if (64 * lane < a.span && mine < a.max_len)
        entry = gh_gp<uint32_t>(a.p.table)[(uint64_t)row * a.p.width + (mine >> a.p.shift)];
    ph8 qf[4];
    const GH_GLOBAL uint4* qp =
        gh_gp<uint4>(a.q + (((uint64_t)row * a.q_heads + kvh * G + min(n, G - 1)) * 128 + 8 * g) * 2);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint4 x = qp[4 * s];
        qf[s] = __builtin_bit_cast(ph8, n < G ? x : make_uint4(0u, 0u, 0u, 0u));
    }
    const uint32_t len = row_length(a.p, row, a.max_len, kvh == 0 && split == 0);
    const uint64_t out0 = a.out + ((uint64_t)row * a.q_heads + kvh * G) * 256;
    if (len == 0) {
        if (split == 0)
            for (uint32_t i = tid; i < G * 64; i += 256) gh_gpw<uint32_t>(out0)[i] = 0u;
        return;
    }
    if (begin >= len) return;
    const uint32_t end = min(len, begin + a.span);
    const bool bad = 64 * lane < a.span && mine < end && entry >= a.p.pages;
    if (bad) fault(a.p, GH_PAGED_PAGE);
    const uint64_t bad_tiles = __ballot(bad);
    const uint32_t first = begin + 16 * wave;
    const uint32_t tiles = first < end ? (end - first + 63) / 64 : 0u;
    const uint32_t row_bytes = a.p.kv_heads * 256;

    auto load = [&](uint32_t i, Tile& r) __attribute__((always_inline)) {
        const uint32_t pos = first + 64 * i;
        const uint32_t page = __builtin_amdgcn_readlane(entry, i & 63u);
        // a tile past the last or of a bad page has no range, and no address is formed from its entry
        const bool none = i >= tiles || (bad_tiles >> i & 1);
        const uint64_t slot = none ? 0 : ((uint64_t)page << a.p.shift) + (pos & ((1u << a.p.shift) - 1));
        const uint64_t at = slot * row_bytes + kvh * 256;
        const int range = none ? 0 : (int)((min(end - pos, 16u) - 1) * row_bytes + 256);
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.kc + at), 0, range, kBufWord3);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void*)(a.p.vc + at), 0, range, kBufWord3);
#pragma unroll
        for (int s = 0; s < 4; ++s)
            r.k[s] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(rk, n * row_bytes + 16 * g + 64 * s, 0, 0));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            r.v[j] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(rv, (4 * g + j) * row_bytes + 16 * n, 0, 0));
    };

    float m = -__builtin_inff(), l = 0.0f;
    pf4 acc[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[t] = pf4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint64_t raw = a.raw + (((uint64_t)row * a.p.kv_heads + kvh) * G + n) * a.raw_len * 4;

    auto step = [&](uint32_t i, const Tile& r) __attribute__((always_inline)) {
        const uint32_t pos = first + 64 * i + 4 * g;  // this lane's first position
        const uint32_t last = bad_tiles >> i & 1 ? 0u : end;
        pf4 st = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < 4; ++s)
            st = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, r.k[s]), qf[s], st, 0, 0, 0);
        float mx = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            st[j] = pos + (uint32_t)j < last ? st[j] * a.scale : -__builtin_inff();
            mx = fmaxf(mx, st[j]);
        }
        if (SCORED && n < G) *gh_gpw<float4>(raw + (uint64_t)pos * 4) = make_float4(st[0], st[1], st[2], st[3]);
        mx = fmaxf(m, lanes4_max(mx));
        const float f = share(m, mx);
        // nothing but -inf so far: every weight 0
        const float up = mx == -__builtin_inff() ? 0.0f : kUp - mx;
        m = mx;
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(st[j] + up);
        l = l * f + ((p[0] + p[1]) + (p[2] + p[3]));
        uint32_t h0, h1, l0, l1;
        weight_parts(p[0], p[1], &h0, &l0);
        weight_parts(p[2], p[3], &h1, &l1);
        const ph8 pv = __builtin_bit_cast(ph8, make_uint4(h0, h1, l0, l1));
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            acc[t] *= f;
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_column(r.v, t), pv, acc[t], 0, 0, 0);
        }
    };

    if (tiles) {
        Tile ra, rb;
        load(0, ra);
        for (uint32_t i = 0; i < tiles; i += 2) {
            load(i + 1, rb);
            step(i, ra);
            if (i + 1 >= tiles) break;
            load(i + 2, ra);
            step(i + 1, rb);
        }
    }

    // the four waves: M = max m_w, L = Σ 2^(m_w - M) l_w, ACC likewise
    const float lt = lanes4_sum(l);
    if (n < G) {
        if (g == 0) {
            sh.m[wave][n] = m;
            sh.l[wave][n] = lt;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < 8; ++t) sh.acc[wave][n][32 * g + 8 * j + t] = acc[t][j];
    }
    __syncthreads();
    if (tid < G) {
        const float M = fmaxf(fmaxf(sh.m[0][tid], sh.m[1][tid]), fmaxf(sh.m[2][tid], sh.m[3][tid]));
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float e = share(sh.m[w][tid], M);
            sh.e[w][tid] = e;
            L += e * sh.l[w][tid];
        }
        sh.M[tid] = M;
        sh.L[tid] = L;
    }
    __syncthreads();
    const bool whole = !SCORED && len <= a.span;  // one split: the output itself
    const uint64_t part = ((uint64_t)row * a.p.kv_heads + kvh) * a.splits + split;
    for (uint32_t i = tid; i < G * 64; i += 256) {
        const uint32_t h = i >> 6, d = 2 * (i & 63u);
        float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float e = sh.e[w][h];
            v.x += e * sh.acc[w][h][d];
            v.y += e * sh.acc[w][h][d + 1];
        }
        if (whole) {
            const float L = sh.L[h];
            gh_gpw<uint32_t>(out0)[i] = (uint32_t)gh_f2h(v.x / L) | (uint32_t)gh_f2h(v.y / L) << 16;
        } else {
            gh_gpw<float2>(a.part_acc)[part * G * 64 + i] = v;
        }
    }
    if (!whole && tid < G) gh_gpw<float2>(a.part_ml)[part * G + tid] = make_float2(sh.M[tid], sh.L[tid]);
}
}  // namespace

#define GH_PAGED_ATTN(GM)                                                                                  \
    GH_KERNEL __launch_bounds__(256) void gh_paged_attn_g##GM(GhPagedAttnArgs a) { paged_attn<GM, false>(a); } \
    GH_KERNEL __launch_bounds__(256) void gh_paged_attn_g##GM##_s(GhPagedAttnArgs a) { paged_attn<GM, true>(a); }
GH_PAGED_ATTN(4)
GH_PAGED_ATTN(8)
GH_PAGED_ATTN(16)

// The splits joined. Grid (q_heads + kv_heads·chunks, 1, rows), 256 threads.
// x < q_heads: the output of one query head: M = max m_s, out = Σ 2^(m_s - M) acc_s / Σ 2^(m_s - M) l_s; eight
// groups of 32 threads take every eighth split, four dims per thread, and add up in group order.
// Else: the scores of a kv head, every chunks-th 1024 positions: the weight of position j is
// 2^(s_j - M + 15) / L per query head, summed over the G heads in order and added to the row's score.
GH_KERNEL __launch_bounds__(256) void gh_paged_join(GhPagedAttnArgs a) {
    __shared__ float sm[16], sl[16];
    __shared__ float4 red[8][32];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, row = blockIdx.z, G = a.group;
    const uint32_t len = row_length(a.p, row, a.max_len, false);
    if (len == 0) return;
    const uint32_t ns = (len + a.span - 1) / a.span;
    const bool score = blockIdx.x >= a.q_heads;
    if (!score && ns == 1 && !a.raw) return;  // written by the attention launch
    const uint32_t kvh = score ? (blockIdx.x - a.q_heads) / a.chunks : blockIdx.x / G;
    const uint64_t part = ((uint64_t)row * a.p.kv_heads + kvh) * a.splits;
    const GH_GLOBAL float2* ml = gh_gp<float2>(a.part_ml) + part * G;
    const uint32_t h0 = score ? 0 : blockIdx.x % G, h1 = score ? G : h0 + 1;
    for (uint32_t h = h0 + wave; h < h1; h += 4) {
        float M = -__builtin_inff(), L = 0.0f;
        for (uint32_t s = lane; s < ns; s += 64) M = fmaxf(M, ml[(uint64_t)s * G + h].x);
        M = gh_wave_max(M);
        for (uint32_t s = lane; s < ns; s += 64) {
            const float2 x = ml[(uint64_t)s * G + h];
            L += share(x.x, M) * x.y;
        }
        L = gh_wave_sum(L);
        if (lane == 0) {
            sm[h] = M;
            sl[h] = L;
        }
    }
    __syncthreads();
    if (!score) {
        const uint32_t h = h0, grp = tid >> 5, d4 = tid & 31u;
        const float M = sm[h];
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const GH_GLOBAL float4* acc = gh_gp<float4>(a.part_acc) + (part * G + h) * 32 + d4;
#pragma unroll 4
        for (uint32_t s = grp; s < ns; s += 8) {
            const float e = share(ml[(uint64_t)s * G + h].x, M);
            const float4 x = acc[(uint64_t)s * G * 32];
            o.x += e * x.x;
            o.y += e * x.y;
            o.z += e * x.z;
            o.w += e * x.w;
        }
        red[grp][d4] = o;
        __syncthreads();
        if (tid < 32) {
            for (uint32_t i = 1; i < 8; ++i) {
                const float4 x = red[i][tid];
                o.x += x.x;
                o.y += x.y;
                o.z += x.z;
                o.w += x.w;
            }
            const float L = sl[h];
            gh_gpw<uint2>(a.out)[((uint64_t)row * a.q_heads + blockIdx.x) * 32 + tid] =
                make_uint2((uint32_t)gh_f2h(o.x / L) | (uint32_t)gh_f2h(o.y / L) << 16,
                           (uint32_t)gh_f2h(o.z / L) | (uint32_t)gh_f2h(o.w / L) << 16);
        }
        return;
    }
    const uint64_t raw = a.raw + ((uint64_t)row * a.p.kv_heads + kvh) * G * a.raw_len * 4;
    const uint64_t to = a.p.score + ((uint64_t)row * a.p.kv_heads + kvh) * (a.p.width << a.p.shift) * 4;
    for (uint32_t c = (blockIdx.x - a.q_heads) % a.chunks; c * 1024 < len; c += a.chunks) {
        const uint32_t pos = c * 1024 + 4 * tid;
        if (pos >= len) continue;
        float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t h = 0; h < G; ++h) {
            const float4 s = *gh_gp<float4>(raw + ((uint64_t)h * a.raw_len + pos) * 4);
            const float up = kUp - sm[h], inv = 1.0f / sl[h];
            w.x += __builtin_amdgcn_exp2f(s.x + up) * inv;
            w.y += __builtin_amdgcn_exp2f(s.y + up) * inv;
            w.z += __builtin_amdgcn_exp2f(s.z + up) * inv;
            w.w += __builtin_amdgcn_exp2f(s.w + up) * inv;
        }
        // positions past the row keep their bits
        GH_GLOBAL float* p = gh_gpw<float>(to) + pos;
        const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            if (pos + j < len) p[j] += v[j];
    }
}

// ---- eviction -----------------------------------------------------------------------------------
// Two launches. gh_paged_select, grid (kv heads, rows, layers), 512 threads: the budget - recent largest
// scores of the older positions by a radix select over the scores' order as 32-bit keys (11, 11 and 10 bits
// per pass, counted in LDS), then one pass in ascending order that writes the kept positions and moves
// their scores; equal keys are taken from the front. gh_paged_move, grid (16-slot blocks of the budget,
// rows, layers), 256 threads: 16 lanes per 256-byte vector, consecutive groups of lanes the heads of one
// slot, so that writes are contiguous; bound by memory.
namespace {
// f32 total order as unsigned order
__device__ __forceinline__ uint32_t order_key(uint32_t bits) { return bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u); }

// Inclusive sum over the wave (two 16-bit counts per word).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    return v;
}
}  // namespace

GH_KERNEL __launch_bounds__(512) void gh_paged_select(GhPagedEvictArgs a) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t sums[8], pick[2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t kvh = blockIdx.x, row = blockIdx.y, layer = blockIdx.z;
    const uint32_t n = row_length(a.src, row, a.src.width << a.src.shift, kvh == 0 && layer == 0);
    const bool act = n > a.budget;
    if (kvh == 0 && layer == 0 && tid == 0) gh_gpw<uint32_t>(a.act)[row] = act;
    if (!act) return;
    const uint64_t list = ((uint64_t)layer * a.rows + row) * a.src.kv_heads + kvh;
    const GH_GLOBAL uint32_t* from = gh_gp<uint32_t>(a.src.score) + list * (a.src.width << a.src.shift);
    GH_GLOBAL uint32_t* to = gh_gpw<uint32_t>(a.dst.score) + list * (a.dst.width << a.dst.shift);
    GH_GLOBAL uint32_t* kept = gh_gpw<uint32_t>(a.kept) + list * a.budget;
    const uint32_t older = n - a.recent;  // > budget - recent
    uint32_t room = a.budget - a.recent;  // of keys equal to `least`, once that is known
    uint32_t least = 0xFFFFFFFFu;
    if (room) {
        uint32_t prefix = 0;
        for (uint32_t pass = 0; pass < 3; ++pass) {
            const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (uint32_t i = tid; i < 2048; i += 512) hist[i] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < older; i += 512) {
                const uint32_t k = order_key(from[i]);
                if (pass == 0 || k >> (shift + bits) == prefix) atomicAdd(&hist[k >> shift & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            // thread t counts bins 2047 - 4 t down to 2044 - 4 t
            uint32_t c[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) c[j] = hist[2047 - 4 * tid - j];
            const uint32_t own = c[0] + c[1] + c[2] + c[3];
            uint32_t upto = wave_scan(own);
            if (lane == 63) sums[wave] = upto;
            __syncthreads();
            for (uint32_t w = 0; w < wave; ++w) upto += sums[w];
            uint32_t above = upto - own;
            if (above < room && room <= upto) {  // one thread
                uint32_t j = 0;
                while (above + c[j] < room) above += c[j++];
                pick[0] = 2047 - 4 * tid - j;
                pick[1] = room - above;
            }
            __syncthreads();
            prefix = prefix << bits | pick[0];
            room = pick[1];
        }
        least = prefix;
    }
    // ascending: 4 positions per thread and step; counts of larger keys (low half) and equal ones (high half)
    uint32_t larger = 0, equal = 0;
    for (uint32_t c0 = 0; c0 < n; c0 += 2048) {
        const uint32_t p0 = c0 + 4 * tid;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (p0 < n) x = *(const GH_GLOBAL uint4*)(from + p0);
        const uint32_t v[4] = {x.x, x.y, x.z, x.w};
        uint32_t own = 0, flag[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t k = order_key(v[j]);
            const bool stays = p0 + j < n && (p0 + j >= older || k > least);
            const bool even = p0 + j < older && k == least;
            flag[j] = (stays ? 1u : 0u) | (even ? 0x10000u : 0u);
            own += flag[j];
        }
        uint32_t upto = wave_scan(own);
        __syncthreads();  // the last step's sums are read
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        uint32_t all = 0;
        for (uint32_t w = 0; w < 8; ++w) {
            if (w < wave) upto += sums[w];
            all += sums[w];
        }
        uint32_t g = larger + ((upto - own) & 0xFFFFu), e = equal + ((upto - own) >> 16);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const bool even = flag[j] >> 16;
            if ((flag[j] & 1u) || (even && e < room)) {
                const uint32_t at = g + min(e, room);
                kept[at] = p0 + j;
                to[at] = v[j];
            }
            g += flag[j] & 1u;
            e += even;
        }
        larger += all & 0xFFFFu;
        equal += all >> 16;
    }
}

GH_KERNEL __launch_bounds__(256) void gh_paged_move(GhPagedEvictArgs a) {
    const uint32_t row = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
    if (!gh_gp<uint32_t>(a.act)[row]) return;
    if (blockIdx.x == 0 && layer == 0 && tid == 0) gh_gpw<uint32_t>(a.dst.lengths)[row] = a.budget;
    const uint32_t heads = a.src.kv_heads, part = 16 * (tid & 15u);
    const uint64_t list = ((uint64_t)layer * a.rows + row) * heads;
    const uint32_t first = 16 * blockIdx.x, items = min(16u, a.budget - first) * heads;
#pragma unroll 4
    for (uint32_t i = tid >> 4; i < items; i += 16) {
        const uint32_t j = first + i / heads, h = i % heads;
        const uint32_t pos = gh_gp<uint32_t>(a.kept)[(list + h) * a.budget + j];
        const uint32_t s = slot_of(a.src, row, pos), d = slot_of(a.dst, row, j);
        if (s == kBad || d == kBad) continue;
        const uint64_t in = layer * a.src_layer + ((uint64_t)s * heads + h) * 256 + part;
        const uint64_t to = layer * a.dst_layer + ((uint64_t)d * heads + h) * 256 + part;
        const uint4 k = *gh_gp<uint4>(a.src.kc + in), v = *gh_gp<uint4>(a.src.vc + in);
        *gh_gpw<uint4>(a.dst.kc + to) = k;
        *gh_gpw<uint4>(a.dst.vc + to) = v;
    }
}
