// A batch of sequences over paged caches in 4 bits (gh_kv_paged with GH_KV_Q4): append, with norms and RoPE, read-back,
// decode attention, eviction. The append with norms and the read-back are here for FP16 pools too.
//
// A vector of 128 values takes 80 bytes: 64 of codes, dims 2 i and 2 i + 1 in the low and high nibble of byte i, then
// per 32 dims a step d and a minimum m in FP16 (d in the low half of a dword). Code c stands for f16(m + d c), one
// rounding. What the device cannot trust (lengths, pages, positions) is checked as in paged.hip.
#include "gh_head.h"
#include "gh_paged.h"

namespace {
constexpr uint32_t kVector = 80;  // bytes
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t as_u(ph2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ ph2 as_h(uint32_t v) { return __builtin_bit_cast(ph2, v); }

// The codes in the low nibbles of both halves of w, and in the second nibbles, as FP16: a nibble in the low bits of
// 1024's mantissa is 1024 + c, in the next ones 1024 + 16 c, and both ways back are exact.
__device__ __forceinline__ ph2 codes_low(uint32_t w) {
    return as_h((w & 0x000F000Fu) | 0x64006400u) - ph2{(_Float16)1024.0f, (_Float16)1024.0f};
}
__device__ __forceinline__ ph2 codes_high(uint32_t w) {
    const ph2 x = as_h((w & 0x00F000F0u) | 0x64006400u);
    return __builtin_elementwise_fma(x, ph2{(_Float16)0.0625f, (_Float16)0.0625f}, ph2{(_Float16)-64.0f, (_Float16)-64.0f});
}
// The low halves of two dwords, and the high ones.
__device__ __forceinline__ uint32_t lows(uint32_t x0, uint32_t x1) { return __builtin_amdgcn_perm(x1, x0, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t x0, uint32_t x1) { return __builtin_amdgcn_perm(x1, x0, 0x07060302u); }
// Eight codes as values, in the order (0, 4), (1, 5), (2, 6), (3, 7); dm: step and minimum.
__device__ __forceinline__ uint4 eight(uint32_t w, uint32_t dm) {
    const ph2 d = as_h(lows(dm, dm)), m = as_h(highs(dm, dm));
    const uint32_t w8 = w >> 8;
    return make_uint4(as_u(__builtin_elementwise_fma(codes_low(w), d, m)), as_u(__builtin_elementwise_fma(codes_high(w), d, m)),
                      as_u(__builtin_elementwise_fma(codes_low(w8), d, m)), as_u(__builtin_elementwise_fma(codes_high(w8), d, m)));
}
}  // namespace

// ---- append ----------------------------------------------------------------------------------
// As gh_paged_write: thread = 8 values of one head of one token, query heads first; a head is 16 lanes, a DPP row, and
// 32 dims are a quad of them. With norms, queries and keys are divided by the root of their mean square over the head
// and multiplied by the weight, in FP32, before the rotation, and rounded once at the end.
namespace {
__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, GH_DPP(v, 0xB1, 0xF));
    return fminf(v, GH_DPP(v, 0x4E, 0xF));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, GH_DPP(v, 0xB1, 0xF));
    return fmaxf(v, GH_DPP(v, 0x4E, 0xF));
}

// The lane's 8 of 32 values as codes; returns them, step and minimum in *dm. The step is cut off to FP16, so that
// m + 15 d stays in the values' range. (x - m) / d is a true quotient: FP16 values lie on ties that a product
// with 1 / d would miss. Values that are not finite make the group NaN.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], uint32_t* dm) {
    float lo = x[0], hi = x[0], odd = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        odd += x[i] * 0.0f;
    }
    lo = quad_min(lo);
    hi = quad_max(hi);
    odd = gh_quad_sum(odd);
    const uint32_t m16 = gh_f2h(lo);
    const uint32_t d16 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz((hi - lo) / 15.0f, 0.0f)) & 0xFFFFu;
    if (odd != 0.0f) {  // a NaN
        *dm = 0x7E007E00u;
        return 0u;
    }
    *dm = d16 | m16 << 16;
    const float m = gh_h2f(m16), d = gh_h2f(d16);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = d > 0.0f ? __builtin_rintf((x[i] - m) / d) : 0.0f;
        w |= (uint32_t)fminf(fmaxf(c, 0.0f), 15.0f) << (4 * i);
    }
    return w;
}

template <bool NORM, bool Q4>
__device__ __forceinline__ void paged_append(const GhPagedWriteArgs& a) {
    const uint32_t token = blockIdx.x / a.groups, row = token / a.tokens, t = token % a.tokens;
    const uint32_t item = (blockIdx.x % a.groups) * 256 + threadIdx.x;
    const uint32_t head = item >> 4, part = item & 15u;  // 8 dims each
    if (head >= a.q_heads + 2 * a.p.kv_heads) return;
    const bool query = head < a.q_heads, value = head >= a.q_heads + a.p.kv_heads;
    const uint32_t h = query ? head : head - a.q_heads - (value ? a.p.kv_heads : 0u);
    const uint32_t heads = query ? a.q_heads : a.p.kv_heads;
    const uint64_t in = ((uint64_t)token * heads + h) * 256 + 16 * part;
    const uint4 raw = *gh_gp<uint4>((query ? a.q : value ? a.v : a.k) + in);
    uint4 weight = make_uint4(0u, 0u, 0u, 0u);
    if (NORM) weight = *gh_gp<uint4>((query ? a.q_norm : a.k_norm) + 16 * part);
    const uint32_t from = a.positions ? gh_gp<uint32_t>(a.positions)[row] : 0u;
    const uint32_t n = row_length(a.p, row, a.p.width << a.p.shift, blockIdx.x % a.groups == 0);
    if (n + t < a.tokens) return;  // a free row, or before its first position
    const uint32_t at = n - a.tokens + t, pos = from + t;
    if (a.positions && (from > a.max_pos || t > a.max_pos - from)) {
        if (item == 0) fault(a.p, GH_PAGED_POSITION);
        return;
    }
    float x[8];
    gh_unpack8(raw, x);
    if (NORM && !value) gh_head_norm(x, weight, 128, a.eps, 16);
    if (a.positions && !value && 4 * part < a.pairs)
        gh_turn4(x, gh_gp<float2>(a.table) + (uint64_t)pos * a.pairs, 4 * part, a.pairs, query ? gh_gp<float>(a.post)[pos] : 1.0f);
    if (query) {
        *gh_gpw<uint4>(a.q_out + in) = gh_pack8(x);
        return;
    }
    const uint32_t slot = slot_of(a.p, row, at);
    if (slot == kBad) return;
    const uint64_t cache = value ? a.p.vc : a.p.kc;
    if constexpr (Q4) {
        uint32_t dm;
        const uint32_t w = codes_of(x, &dm);
        const uint64_t to = cache + ((uint64_t)slot * a.p.kv_heads + h) * kVector;
        *gh_gpw<uint32_t>(to + 4 * part) = w;
        if ((part & 3u) == 0) *gh_gpw<uint32_t>(to + 64 + part) = dm;
    } else {
        *gh_gpw<uint4>(cache + ((uint64_t)slot * a.p.kv_heads + h) * 256 + 16 * part) = gh_pack8(x);
    }
    if (a.p.score && !value && part == 0)
        gh_gpw<float>(a.p.score)[((uint64_t)row * a.p.kv_heads + h) * (a.p.width << a.p.shift) + at] = 0.0f;
}
}  // namespace
GH_KERNEL __launch_bounds__(256) void gh_paged4_write(GhPagedWriteArgs a) { paged_append<false, true>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged4_norm_write(GhPagedWriteArgs a) { paged_append<true, true>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged_norm_write(GhPagedWriteArgs a) { paged_append<true, false>(a); }

// ---- read-back ---------------------------------------------------------------------------------
// Thread = 8 values of one head of one position, key heads first.
namespace {
template <bool Q4>
__device__ __forceinline__ void paged_read(const GhPagedReadArgs& a) {
    const uint32_t token = blockIdx.x / a.groups, row = token / a.tokens, t = token % a.tokens;
    const uint32_t item = (blockIdx.x % a.groups) * 256 + threadIdx.x;
    const uint32_t head = item >> 4, part = item & 15u;
    if (head >= 2 * a.p.kv_heads) return;
    const bool value = head >= a.p.kv_heads;
    const uint32_t h = head - (value ? a.p.kv_heads : 0u);
    const uint32_t n = row_length(a.p, row, a.p.width << a.p.shift, blockIdx.x % a.groups == 0);
    if (n + t < a.tokens) return;
    const uint32_t slot = slot_of(a.p, row, n - a.tokens + t);
    if (slot == kBad) return;
    const uint64_t vector = (uint64_t)slot * a.p.kv_heads + h, cache = value ? a.p.vc : a.p.kc;
    uint4 x;
    if constexpr (Q4) {
        const uint64_t from = cache + vector * kVector;
        const uint32_t w = *gh_gp<uint32_t>(from + 4 * part), dm = *gh_gp<uint32_t>(from + 64 + (part & ~3u));
        const uint4 y = eight(w, dm);  // (0, 4), (1, 5), (2, 6), (3, 7)
        x = make_uint4(lows(y.x, y.y), lows(y.z, y.w), highs(y.x, y.y), highs(y.z, y.w));
    } else {
        x = *gh_gp<uint4>(cache + vector * 256 + 16 * part);
    }
    *gh_gpw<uint4>((value ? a.v : a.k) + ((uint64_t)token * a.p.kv_heads + h) * 256 + 16 * part) = x;
}
}  // namespace
GH_KERNEL __launch_bounds__(256) void gh_paged4_read(GhPagedReadArgs a) { paged_read<true>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged_read(GhPagedReadArgs a) { paged_read<false>(a); }

// ---- decode attention ---------------------------------------------------------------------------
// The plan of paged.hip: a wave takes the G <= 16 query heads of one kv head over tiles, here of 32 positions in two
// halves of 16, each within one page and so at one address. Per half:
//   S^T = K·Q^T     4 x v_mfma_f32_16x16x32_f16: a lane's 32 k-slots are the 32 dims 32 (l / 16) .. + 32 of position
//                   l % 16, which is 16 bytes of codes in one load with one step and one minimum (the query's fragments
//                   are in the order in which the codes come out of their dwords);
// and per tile
//   O^T += V^T·P^T  per 8-dim tile t one v_mfma_f32_16x16x32_f16 over the 32 positions: a lane has dims 8 (l % 16) ..
//                   + 8, a dword of codes, of 4 (l / 16) + i of both halves. Bytes of two positions are gathered
//                   in one dword before they become values, so that steps and minima apply to pairs of positions.
// Values are f16(m + d c), as a read-back gives them. Weights are 2^(s - m + 15) in FP16, nearest: 2^-11 of each and
// 2^-39 of the largest; next to the output's own 2^-11 this is half an FP16 cache's MFMAs and none of its splitting (a V
// here is finite or NaN, so a weight of 0 hides nothing). A maximum that stays leaves the sums unscaled.
namespace {
struct Tile4 {
    uint4 k[2];                // position l % 16 of each half, dims 32 (l / 16) .. + 32
    uint32_t kd[2];
    uint32_t v[8], vd[8];      // [4 half + i]: position 4 (l / 16) + i, dims 8 (l % 16) .. + 8
};

// K and V of one head from the slot of a half's first position, `count` positions long (0: nothing is read).
struct Half {
    __amdgpu_buffer_rsrc_t k, v;
};
__device__ __forceinline__ Half half_at(const GhPages& p, uint32_t slot, uint32_t count, uint32_t kvh) {
    const uint32_t row_bytes = p.kv_heads * kVector;
    const uint64_t at = (uint64_t)slot * row_bytes + kvh * kVector;
    const int range = count ? (int)((count - 1) * row_bytes + kVector) : 0;
    return {__builtin_amdgcn_make_buffer_rsrc((void*)(p.kc + at), 0, range, kBufWord3),
            __builtin_amdgcn_make_buffer_rsrc((void*)(p.vc + at), 0, range, kBufWord3)};
}
struct Where {
    Half half[2];
};
__device__ __forceinline__ Where tile_at(const GhPages& p, uint32_t slot0, uint32_t slot1, uint32_t count, uint32_t kvh) {
    return {{half_at(p, slot0, min(count, 16u), kvh), half_at(p, slot1, max(count, 16u) - 16u, kvh)}};
}
template <int CACHE>
__device__ __forceinline__ void load_k(const Where& w, uint32_t row_bytes, Tile4& r) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        r.k[u] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(w.half[u].k, n * row_bytes + 16 * g, 0, CACHE));
        r.kd[u] = __builtin_amdgcn_raw_buffer_load_b32(w.half[u].k, n * row_bytes + 64 + 4 * g, 0, CACHE);
    }
}
template <int CACHE>
__device__ __forceinline__ void load_v(const Where& w, uint32_t row_bytes, Tile4& r) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r.v[i] = __builtin_amdgcn_raw_buffer_load_b32(w.half[i >> 2].v, (4 * g + (i & 3)) * row_bytes + 4 * n, 0, CACHE);
        r.vd[i] = __builtin_amdgcn_raw_buffer_load_b32(w.half[i >> 2].v, (4 * g + (i & 3)) * row_bytes + 64 + (n & ~3u), 0, CACHE);
    }
}

// B fragments of the G queries of a kv head: head n = l % 16 (zero past G), dims 32 (l / 16) + 8 s .. + 8 in the
// order of eight().
__device__ __forceinline__ void load_q4(const GhPagedAttnArgs& a, uint32_t row, uint32_t kvh, ph8 (&qf)[4]) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const GH_GLOBAL uint4* qp = gh_gp<uint4>(a.q + (((uint64_t)row * a.q_heads + kvh * G + min(n, G - 1)) * 128 + 32 * g) * 2);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint4 x = qp[s];
        const uint4 y = make_uint4(lows(x.x, x.z), highs(x.x, x.z), lows(x.y, x.w), highs(x.y, x.w));
        qf[s] = __builtin_bit_cast(ph8, n < G ? y : make_uint4(0u, 0u, 0u, 0u));
    }
}

__device__ __forceinline__ pf4 half_products(const uint4& k, uint32_t dm, const ph8 (&qf)[4]) {
    const uint32_t w[4] = {k.x, k.y, k.z, k.w};
    pf4 st = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s) st = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, eight(w[s], dm)), qf[s], st, 0, 0, 0);
    return st;
}
// -inf past the tile's positions
__device__ __forceinline__ void hide(pf4 (&st)[2], uint32_t count) {
    if (count >= 32) return;
    const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (16 * (i >> 2) + 4 * g + (i & 3) >= count) st[i >> 2][i & 3] = -__builtin_inff();
}
// st: products, which times `scale` are scores in base 2
__device__ __forceinline__ void tile_add(Sums& x, const pf4 (&st)[2], float scale, const Tile4& r) {
    float top = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])), fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
    const float mx = fmaxf(x.m, lanes4_max(top) * scale);
    if (__builtin_amdgcn_ballot_w64(mx != x.m)) {
        const float f = share(x.m, mx);
        x.m = mx;
        x.l *= f;
#pragma unroll
        for (int t = 0; t < 8; ++t) x.acc[t] *= f;
    }
    // nothing but -inf so far: every weight 0
    const float up = mx == -__builtin_inff() ? 0.0f : kUp - mx;
    float p[8];
    uint32_t ph[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i >> 2][i & 3], scale, up));
    x.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int i = 0; i < 4; ++i) ph[i] = as_u(ph2{(_Float16)p[2 * i], (_Float16)p[2 * i + 1]});
    const ph8 pv = __builtin_bit_cast(ph8, make_uint4(ph[0], ph[1], ph[2], ph[3]));
    ph2 d[4], m[4];  // of two positions
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        d[i] = as_h(lows(r.vd[2 * i], r.vd[2 * i + 1]));
        m[i] = as_h(highs(r.vd[2 * i], r.vd[2 * i + 1]));
    }
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // byte b of both positions, in the low bytes of the halves
            const uint32_t w = __builtin_amdgcn_perm(r.v[2 * i + 1], r.v[2 * i], 0x0C000C00u | (4 + b) << 16 | b);
            lo[i] = as_u(__builtin_elementwise_fma(codes_low(w), d[i], m[i]));
            hi[i] = as_u(__builtin_elementwise_fma(codes_high(w), d[i], m[i]));
        }
        x.acc[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, make_uint4(lo[0], lo[1], lo[2], lo[3])), pv, x.acc[2 * b], 0, 0, 0);
        x.acc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, make_uint4(hi[0], hi[1], hi[2], hi[3])), pv, x.acc[2 * b + 1], 0, 0, 0);
    }
}
// The scores of the lane's head at positions `pos` and on of a row, past its length too (raw_len is whole tiles).
__device__ __forceinline__ void keep_scores(uint64_t raw, uint32_t pos, const pf4 (&st)[2], float scale) {
    const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
        const pf4 s = st[u] * scale;
        *gh_gpw<float4>(raw + (uint64_t)(pos + 16 * u + 4 * g) * 4) = make_float4(s[0], s[1], s[2], s[3]);
    }
}

// The slots of the two halves of a tile whose first position is `pos`, `count` positions long; false where a page is
// beyond the pool.
__device__ __forceinline__ bool tile_slots(const GhPages& p, uint32_t row, uint32_t pos, uint32_t count, uint32_t* slot0, uint32_t* slot1) {
    const GH_GLOBAL uint32_t* table = gh_gp<uint32_t>(p.table) + (uint64_t)row * p.width;
    const uint32_t pos1 = count > 16 ? pos + 16 : pos, mask = (1u << p.shift) - 1;
    const uint32_t page0 = table[pos >> p.shift], page1 = table[pos1 >> p.shift];
    const bool good = page0 < p.pages && page1 < p.pages;
    if (!good) fault(p, GH_PAGED_PAGE);
    *slot0 = good ? (page0 << p.shift) + (pos & mask) : 0u;
    *slot1 = good ? (page1 << p.shift) + (pos1 & mask) : 0u;
    return good;
}

// One chunk of the rows' tiles for one kv head by one wave.
template <bool SCORED, int CACHE>
__device__ __forceinline__ void paged4_chunk(const GhPagedAttnArgs& a, const RowsLds& sh, uint32_t behind, uint32_t total,
                                             uint32_t per, uint32_t chunk, uint32_t kvh) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, G = a.group;
    const uint32_t begin = chunk * per, tiles = min(per, total - begin), row_bytes = a.p.kv_heads * kVector;

    // lane i: slots, first position, and row | positions << 16 of tile i of the current 64
    uint32_t t_slot0 = 0, t_slot1 = 0, t_pos = 0, t_row = 0;
    auto look_up = [&](uint32_t from) __attribute__((always_inline)) {
        const uint32_t t = begin + from + lane;
        t_slot0 = t_slot1 = t_pos = t_row = 0;
        uint32_t lo = 0;  // the row with first[lo] <= t < first[lo + 1]
        if (a.rows <= 64) lo = (uint32_t)__popcll(__ballot(behind <= begin + from));  // of the first tile
        if (from + lane >= tiles) return;
        if (a.rows > 64) {
            uint32_t hi = a.rows;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (sh.first[mid] <= t) lo = mid;
                else hi = mid;
            }
        }
        while (sh.first[lo + 1] <= t) ++lo;
        t_pos = (t - sh.first[lo]) * 32;
        const uint32_t count = min(sh.len[lo] - t_pos, 32u);
        t_row = lo | (tile_slots(a.p, lo, t_pos, count, &t_slot0, &t_slot1) ? count << 16 : 0u);
    };
    look_up(0);
    auto where = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t count = i < tiles ? __builtin_amdgcn_readlane(t_row, i & 63u) >> 16 : 0u;
        return tile_at(a.p, __builtin_amdgcn_readlane(t_slot0, i & 63u), __builtin_amdgcn_readlane(t_slot1, i & 63u), count, kvh);
    };

    ph8 qf[4];
    Sums x;
    uint32_t row, since;  // the row at hand and the tile it began with
    uint64_t raw = 0;
    // the row's sums up to tile i: its output if they are whole, else a partial
    auto flush = [&](uint32_t i) __attribute__((always_inline)) {
        const float L = lanes4_sum(x.l);
        if (n >= G) return;
        if (!SCORED && begin + since == sh.first[row] && begin + i == sh.first[row + 1]) store_out(a, row, kvh, x, L);
        else store_partial(a, ((uint64_t)(chunk + row) * a.p.kv_heads + kvh) * G + n, x, L);
    };
    auto start = [&](uint32_t info, uint32_t i) __attribute__((always_inline)) {
        row = info & 0xFFFFu;
        since = i;
        x.clear();
        load_q4(a, row, kvh, qf);
        if (SCORED) raw = a.raw + (((uint64_t)row * a.p.kv_heads + kvh) * G + n) * a.raw_len * 4;
    };
    start(__builtin_amdgcn_readlane(t_row, 0), 0);

    // K of the next tile is asked for as soon as this one's products are made, V behind its last use
    Tile4 r;
    Where w = where(0);
    load_k<CACHE>(w, row_bytes, r);
    load_v<CACHE>(w, row_bytes, r);
    for (uint32_t i = 0; i < tiles; ++i) {
        const uint32_t info = __builtin_amdgcn_readlane(t_row, i & 63u);
        const uint32_t pos = SCORED ? __builtin_amdgcn_readlane(t_pos, i & 63u) : 0u;
        if ((info & 0xFFFFu) != row) {
            flush(i);
            start(info, i);
        }
        pf4 st[2] = {half_products(r.k[0], r.kd[0], qf), half_products(r.k[1], r.kd[1], qf)};
        if ((i & 63u) == 63) look_up(i + 1);
        w = where(i + 1);
        load_k<CACHE>(w, row_bytes, r);
        hide(st, info >> 16);
        if (SCORED && n < G) keep_scores(raw, pos, st, a.scale);
        tile_add(x, st, a.scale, r);
        load_v<CACHE>(w, row_bytes, r);
    }
    flush(tiles);
}

// All rows' tiles in equal chunks, as gh_paged_attn.
template <bool SCORED>
__device__ __forceinline__ void paged4_attn(const GhPagedAttnArgs& a) {
    __shared__ RowsLds sh;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunk = unit / a.p.kv_heads, kvh = unit % a.p.kv_heads;
    const uint32_t behind = lay_out_rows<5>(a, sh, blockIdx.x == 0);
    const uint32_t total = sh.first[a.rows];
    const uint32_t half = (2 * total + a.chunks - 1) / a.chunks;
    const uint32_t per = max(a.least, half <= a.solo ? half : (total + a.chunks - 1) / a.chunks);
    if (blockIdx.x == 0) {  // for the join
        for (uint32_t r = threadIdx.x; r <= a.rows; r += 256) gh_gpw<uint32_t>(a.layout)[1 + r] = sh.first[r];
        if (threadIdx.x == 0) gh_gpw<uint32_t>(a.layout)[0] = per;
    }
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x)
        if (sh.len[r] == 0)
            for (uint32_t i = threadIdx.x; i < a.q_heads * 64; i += 256)
                gh_gpw<uint32_t>(a.out)[(uint64_t)r * a.q_heads * 64 + i] = 0u;
    if (chunk >= a.chunks || chunk * per >= total) return;
    if ((uint64_t)total * a.p.kv_heads * (64 * kVector) >= a.stream) paged4_chunk<SCORED, kStream>(a, sh, behind, total, per, chunk, kvh);
    else paged4_chunk<SCORED, 0>(a, sh, behind, total, per, chunk, kvh);
}

// Each row in spans, as gh_paged_split: of a.least / 2 tiles, of which wave w takes w, w + 4, ...
template <bool SCORED>
__device__ __forceinline__ void paged4_split(const GhPagedAttnArgs& a) {
    extern __shared__ __align__(16) float dyn[];  // per wave and head: 132 floats of acc, then m and l
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, G = a.group;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, row = blockIdx.z;
    const uint32_t span = a.least * 16, begin = split * span;  // < max_len
    // the wave's tile i covers positions begin + 128 i + 32 wave .. + 32
    const uint32_t first = begin + 32 * wave, mine = first + 128 * lane;
    const uint32_t len = row_length(a.p, row, a.max_len, kvh == 0 && split == 0);
    if (len == 0) {
        if (split == 0)
            for (uint32_t i = tid; i < G * 64; i += 256) gh_gpw<uint32_t>(a.out + ((uint64_t)row * a.q_heads + kvh * G) * 256)[i] = 0u;
        return;
    }
    if (begin >= len) return;
    ph8 qf[4];
    load_q4(a, row, kvh, qf);
    const uint32_t end = min(len, begin + span);
    uint32_t t_slot0 = 0, t_slot1 = 0, t_count = 0;
    if (mine < end) {
        const uint32_t count = min(end - mine, 32u);
        if (tile_slots(a.p, row, mine, count, &t_slot0, &t_slot1)) t_count = count;
    }
    const uint32_t tiles = first < end ? (end - first + 127) / 128 : 0u, row_bytes = a.p.kv_heads * kVector;
    auto where = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t count = i < tiles ? __builtin_amdgcn_readlane(t_count, i & 63u) : 0u;
        return tile_at(a.p, __builtin_amdgcn_readlane(t_slot0, i & 63u), __builtin_amdgcn_readlane(t_slot1, i & 63u), count, kvh);
    };
    const uint64_t raw = a.raw + (((uint64_t)row * a.p.kv_heads + kvh) * G + n) * a.raw_len * 4;
    Sums x;
    x.clear();
    if (tiles) {
        Tile4 r;
        Where w = where(0);
        load_k<0>(w, row_bytes, r);
        load_v<0>(w, row_bytes, r);
        for (uint32_t i = 0; i < tiles; ++i) {
            pf4 st[2] = {half_products(r.k[0], r.kd[0], qf), half_products(r.k[1], r.kd[1], qf)};
            w = where(i + 1);
            load_k<0>(w, row_bytes, r);
            hide(st, __builtin_amdgcn_readlane(t_count, i & 63u));
            if (SCORED && n < G) keep_scores(raw, first + 128 * i, st, a.scale);
            tile_add(x, st, a.scale, r);
            load_v<0>(w, row_bytes, r);
        }
    }
    split_finish<SCORED>(a, x, dyn, row, kvh, split, span, len);
}
}  // namespace
GH_KERNEL __launch_bounds__(256, 4) void gh_paged4_attn(GhPagedAttnArgs a) { paged4_attn<false>(a); }
GH_KERNEL __launch_bounds__(256, 4) void gh_paged4_attn_s(GhPagedAttnArgs a) { paged4_attn<true>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged4_split(GhPagedAttnArgs a) { paged4_split<false>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged4_split_s(GhPagedAttnArgs a) { paged4_split<true>(a); }

// ---- eviction -----------------------------------------------------------------------------------
// The move of gh_paged_move for vectors of five 16-byte pieces, a thread each. Same grid.
GH_KERNEL __launch_bounds__(256) void gh_paged4_move(GhPagedEvictArgs a) {
    const uint32_t row = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
    if (!gh_gp<uint32_t>(a.act)[row]) return;
    if (blockIdx.x == 0 && layer == 0 && tid == 0) gh_gpw<uint32_t>(a.dst.lengths)[row] = a.budget;
    const uint32_t heads = a.src.kv_heads, pieces = heads * 5;
    const uint64_t list = ((uint64_t)layer * a.rows + row) * heads;
    const uint32_t first = 16 * blockIdx.x, items = min(16u, a.budget - first) * pieces;
#pragma unroll 4
    for (uint32_t i = tid; i < items; i += 256) {
        const uint32_t j = first + i / pieces, h = i % pieces / 5, part = 16 * (i % 5);
        const uint32_t pos = gh_gp<uint32_t>(a.kept)[(list + h) * a.budget + j];
        const uint32_t s = slot_of(a.src, row, pos), d = slot_of(a.dst, row, j);
        if (s == kBad || d == kBad) continue;
        const uint64_t in = layer * a.src_layer + ((uint64_t)s * heads + h) * kVector + part;
        const uint64_t to = layer * a.dst_layer + ((uint64_t)d * heads + h) * kVector + part;
        typedef uint32_t u4v __attribute__((ext_vector_type(4)));
        const u4v k = *gh_gp<u4v>(a.src.kc + in), v = *gh_gp<u4v>(a.src.vc + in);
        __builtin_nontemporal_store(k, gh_gpw<u4v>(a.dst.kc + to));
        __builtin_nontemporal_store(v, gh_gpw<u4v>(a.dst.vc + to));
    }
}
