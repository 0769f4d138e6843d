// A batch of sequences over paged caches in 4 bits (gh_kv_paged with GH_KV_Q4): append, with norms and RoPE, read-back,
// decode attention, eviction. The append with norms and the read-back are here for FP16 pools too.
//
// A vector of 128 values takes 80 bytes: 64 of codes, dims 2 i and 2 i + 1 in the low and high nibble of byte i, then
// per 32 dims a step d and a minimum m in FP16 (d in the low half of a dword). Code c stands for m + d c.
// What the device cannot trust (lengths, pages, positions) is checked as in paged.hip.
#include "gh_head.h"
#include "gh_paged.h"

namespace {
constexpr uint32_t kVector = 80;  // bytes
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
typedef _Float16 ph4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint32_t as_u(ph2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ ph2 as_h(uint32_t v) { return __builtin_bit_cast(ph2, v); }

// The codes in the low nibbles of both halves of w, and in the second nibbles, as FP16: a nibble in the low bits of
// 1024's mantissa is 1024 + c, in the next ones 1024 + 16 c, and both ways back are exact. The constants are held in registers
// (opaque to the compiler), so that mask and exponent are one v_and_or_b32.
struct Masks {
    uint32_t low, high, up;
    __device__ __forceinline__ Masks() : low(0x000F000Fu), high(0x00F000F0u), up(0x64006400u) {
        asm("" : "+s"(low));
        asm("" : "+s"(high));
        asm("" : "+v"(up));
    }
};
__device__ __forceinline__ ph2 codes_low(uint32_t w, const Masks& c) {
    return as_h((w & c.low) | c.up) - ph2{(_Float16)1024.0f, (_Float16)1024.0f};
}
__device__ __forceinline__ ph2 codes_high(uint32_t w, const Masks& c) {
    return __builtin_elementwise_fma(as_h((w & c.high) | c.up), ph2{(_Float16)0.0625f, (_Float16)0.0625f}, ph2{(_Float16)-64.0f, (_Float16)-64.0f});
}
// The low halves of two dwords, and the high ones.
__device__ __forceinline__ uint32_t lows(uint32_t x0, uint32_t x1) { return __builtin_amdgcn_perm(x1, x0, 0x05040100u); }
__device__ __forceinline__ uint32_t highs(uint32_t x0, uint32_t x1) { return __builtin_amdgcn_perm(x1, x0, 0x07060302u); }
}  // namespace

// ---- append ----------------------------------------------------------------------------------
// As gh_paged_write: thread = 8 values of one head of one token, query heads first; a head is 16 lanes, a DPP row, and
// 32 dims are a quad of them. With norms, queries and keys are divided by the root of their mean square over the head
// and multiplied by the weight, in FP32, before the rotation, and rounded once at the end. All loads but the table's are asked for
// at once: with few tokens a launch is a chain of their latencies. 32 query and 8 kv heads with norms, 1 / 256 rows: 3.1 / 4.4 us (6 MB), with
// the rotation alone 3.0 / 4.2, with norms into FP16 pools 2.9 / 4.2; a prompt of 2000, 11 MB, without either: 5.6.
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
// m + 15 d stays in the values' range where m is the minimum itself. Keys that were turned or normed have one between FP16 numbers,
// and m may lie above it by half an FP16 step: where m + 15 d would reach 65520, which FP16 rounds to infinity, the step is
// a fifteenth of what is left above m. (x - m) / d is a true quotient (a product with 1 / d, corrected by what it leaves):
// FP16 values lie on ties that the product alone would miss. Values that FP16 does not hold as finite make the group NaN.
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
    uint32_t d16 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz((hi - lo) / 15.0f, 0.0f)) & 0xFFFFu;
    if (__builtin_fmaf(15.0f, gh_h2f(d16), gh_h2f(m16)) >= 65520.0f)
        d16 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz((hi - gh_h2f(m16)) / 15.0f, 0.0f)) & 0xFFFFu;
    if (odd != 0.0f || fmaxf(-lo, hi) >= 65520.0f) {  // (odd: a NaN)
        *dm = 0x7E007E00u;
        return 0u;
    }
    *dm = d16 | m16 << 16;
    const float m = gh_h2f(m16), d = gh_h2f(d16), r = d > 0.0f ? __builtin_amdgcn_rcpf(d) : 0.0f;
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float y = x[i] - m, t = y * r, c = __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-t, d, y), r, t));
        w |= (uint32_t)__builtin_amdgcn_fmed3f(c, 0.0f, 15.0f) << (4 * i);
    }
    return w;
}

template <bool NORM, bool Q4, bool WIDE>
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
    if (!value) {
        if (NORM) gh_head_norm(x, weight, 1.0f / 128, a.eps, 16);
        if (a.positions) {
            float2 c[4];
            gh_load_turns<WIDE>(gh_gp<float2>(a.table) + (uint64_t)pos * a.pairs, 4 * part, a.pairs, c);
            gh_turn4(x, c, 4 * part, a.pairs, query ? gh_gp<float>(a.post)[pos] : 1.0f, a.pairs == 64);
        }
    }
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
GH_KERNEL __launch_bounds__(256) void gh_paged4_write(GhPagedWriteArgs a) {
    if (a.pairs % 4 == 0) paged_append<false, true, true>(a);
    else paged_append<false, true, false>(a);
}
GH_KERNEL __launch_bounds__(256) void gh_paged4_norm_write(GhPagedWriteArgs a) {
    if (a.pairs % 4 == 0) paged_append<true, true, true>(a);
    else paged_append<true, true, false>(a);
}
GH_KERNEL __launch_bounds__(256) void gh_paged_norm_write(GhPagedWriteArgs a) {
    if (a.pairs % 4 == 0) paged_append<true, false, true>(a);
    else paged_append<true, false, false>(a);
}

// ---- read-back ---------------------------------------------------------------------------------
// Thread = 8 values of one head of one position, key heads first: 8 bytes in (the step and minimum are read by four), 16 out.
// 8 heads, 1 / 256 rows of one position 1.8 / 2.8 us, 2000 positions (11 MB) 4.4; of FP16 pools 1.7 / 2.7 and, 16 MB, 4.8.
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
        const ph2 d = as_h(lows(dm, dm)), m = as_h(highs(dm, dm));
        const Masks c;
        uint32_t y[4];  // codes 0 and 4, 1 and 5, 2 and 6, 3 and 7
#pragma unroll
        for (int i = 0; i < 4; ++i)
            y[i] = as_u(__builtin_elementwise_fma(i & 1 ? codes_high(w >> (8 * (i >> 1)), c) : codes_low(w >> (8 * (i >> 1)), c), d, m));
        x = make_uint4(lows(y[0], y[1]), lows(y[2], y[3]), highs(y[0], y[1]), highs(y[2], y[3]));
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
// halves of 16, each within one page and so at one address. Vectors of 80 bytes fill no lines, but those of adjacent heads lie
// in a row: the four waves of a workgroup take up to four heads of the same positions and bring their bytes to LDS together, five
// 16-byte loads a lane, asked for a tile ahead. (64 rows of 8192, 671 MB: fragments loaded straight from memory, 20 loads of 64 to 1024
// bytes, 282 us; each wave its own head through LDS 204; so 131, of which the loads alone take 114 and all but them 104.)
// Per half, S^T = K·Q^T with the codes as they are: a nibble in the low bits of an FP16 number is c 2^-24, in the next ones
// c 2^-20, and the matrix cores take subnormals, so that a mask is all it needs. v_mfma_f32_16x16x32_f16 s (0..3) covers dims
// 32 s .. + 32, one step and minimum a position: lane l has dims 32 s + 8 (l / 16) .. + 8 of position l % 16, which
// four row swaps make of the 16 bytes in a row that it reads. The sums are those of exact products in FP32 (Query says what is held
// of a query); steps come to
// the lanes that need them by a product with a unit vector, and the minima's part is one product with the sums of the query over
// its groups, in FP16 hi + lo. So no key is rounded, for less than the conversion of its codes to FP16 takes.
// O^T += V^T·P^T per tile: per 8-dim tile t products over the 32 positions: a lane has dims 8 (l % 16) .. + 8, a dword of
// codes, of positions 4 (l / 16) + i of both halves. Bytes of two positions are gathered in one dword before they
// become f16(m + d c), so that steps and minima apply to pairs of positions. Weights are 2^(s - m + 15), FP16 hi + lo
// each in a product of its own: 22 bits, and 2^-39 of the largest weight. V here is finite or NaN, so a weight of 0 hides
// nothing. A maximum that stays leaves the sums unscaled.
namespace {
struct Tile4 {
    uint4 x[5];  // 16-byte pieces l of each half's K and of each half's V, then the 64 H + l % 16 H-th of the (l / 16 H)-th
};
constexpr uint32_t kHalfBytes = 16 * kVector, kTileBytes = 4 * kHalfBytes;
constexpr uint32_t kStageBytes = kTileBytes + kVector;  // of a head, so that a team's pieces meet no bank twice

// A tile's slots of its first and 17th position and their number of positions (0: nothing is read).
struct Where {
    uint32_t slot0, slot1, count;
};
// A team of H waves takes H heads of the same tiles, and its 64 H lanes their bytes: 16 positions of H heads are 80 H pieces
// of 16 bytes, in a row if these are all heads. What a lane keeps of its pieces (first: the team's first head, l: the lane
// in the team):
struct Pieces {
    uint64_t base, k, v;    // of the fifth piece, and of K and V of the team's heads
    uint32_t at, row, off;  // of the first four; the fifth's position, and where it is in its row
    uint32_t row_bytes, range;
    uint32_t to, to5;       // places in LDS
    // There are `have` of the H heads (fewer in the last group): the places of others are read from these.
    __device__ __forceinline__ Pieces(const GhPages& p, uint32_t first, uint32_t heads, uint32_t l, uint32_t have) {
        const uint32_t per = 5 * heads;  // pieces of a position
        row_bytes = p.kv_heads * kVector;
        range = have * kVector;
        k = p.kc + first * kVector;
        v = p.vc + first * kVector;
        const uint32_t q = l / per, r = l % per;
        at = q * row_bytes + r % (5 * have) * 16;
        to = r / 5 * kStageBytes + q * kVector + r % 5 * 16;
        const uint32_t block = l / (16 * heads), piece = 64 * heads + l % (16 * heads), r5 = piece % per;
        row = piece / per;
        off = r5 % (5 * have) * 16;
        to5 = r5 / 5 * kStageBytes + block * kHalfBytes + row * kVector + r5 % 5 * 16;
        base = (block < 2 ? k : v) + off;
        second = block & 1;
    }
    bool second;            // the fifth is of the second half
};
template <int CACHE>
__device__ __forceinline__ void load_tile(const Where w, const Pieces& p, Tile4& r) {
    if (w.count == 0) return;
    const uint32_t c0 = min(w.count, 16u), c1 = w.count - c0, s0 = w.slot0, s1 = w.slot1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint64_t at = (i < 2 ? p.k : p.v) + (uint64_t)(i & 1 ? s1 : s0) * p.row_bytes;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)at, 0, (i & 1 ? c1 : c0) ? (int)(((i & 1 ? c1 : c0) - 1) * p.row_bytes + p.range) : 0, kBufWord3);
        r.x[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, p.at, 0, CACHE));
    }
    // past the half's positions: the last one again, which has another's weight, and hides nothing that is not seen there
    uint32_t row = p.row;
    if (w.count < 32) row = min(row, max(p.second ? c1 : c0, 1u) - 1);
    typedef uint32_t u4v __attribute__((ext_vector_type(4)));
    const GH_GLOBAL u4v* from = gh_gp<u4v>(p.base + (uint64_t)((p.second ? s1 : s0) + row) * p.row_bytes);
    r.x[4] = __builtin_bit_cast(uint4, CACHE ? __builtin_nontemporal_load(from) : *from);
}
// The lane's pieces into the team's part of LDS.
__device__ __forceinline__ void store_tile(const Tile4& r, const Pieces& p, char* lds) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *(uint4*)(lds + i * kHalfBytes + p.to) = r.x[i];
    *(uint4*)(lds + p.to5) = r.x[4];
}
// A wave's own stores and reads of LDS stay in order.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// B fragments of the G queries of a kv head: head n = l % 16 (zero past G), times the power of two that brings its largest value
// to 2^15 or more, so that what follows loses bits of FP16's least steps only far below that. x: dims 32 s + 8 (l / 16) .. + 8 in
// the order (0, 4), (1, 5), (2, 6), (3, 7), those that meet codes of 2^-20 times 2^-4: exact to 2^-36 of the largest. sums: 2^-9 of
// the sum over the dims of group l / 16, hi and lo, in the places of the minima: to 2^-22 of it, or 2^-31 of the largest. step: 2^15
// in the place of the step of group s. scale: what makes products scores in base 2, this power taken out again.
struct Query {
    ph8 x[4];
    ph4 sums, step[4];
    float scale;
};
struct RawQuery {
    uint4 x[4];
};
__device__ __forceinline__ void ask_q4(const GhPagedAttnArgs& a, uint32_t row, uint32_t kvh, RawQuery& r) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const GH_GLOBAL uint4* qp = gh_gp<uint4>(a.q + (((uint64_t)row * a.q_heads + kvh * G + min(n, G - 1)) * 128 + 8 * g) * 2);
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s) r.x[s] = qp[4 * s];
}
__device__ __forceinline__ void make_q4(const GhPagedAttnArgs& a, const RawQuery& r, Query& q) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const ph2 down = {(_Float16)0.0625f, (_Float16)0.0625f};
    pu2 top = {0, 0};  // the largest magnitude, as bits
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s)
#pragma unroll
        for (uint32_t w : {r.x[s].x, r.x[s].y, r.x[s].z, r.x[s].w})
            top = __builtin_elementwise_max(top, __builtin_bit_cast(pu2, w & 0x7FFF7FFFu));
    uint32_t largest = top.x > top.y ? top.x : top.y;
    const auto a16 = __builtin_amdgcn_permlane16_swap(largest, largest, false, false);
    largest = max(a16[0], a16[1]);
    const auto a32 = __builtin_amdgcn_permlane32_swap(largest, largest, false, false);
    largest = max(a32[0], a32[1]);
    // its exponent, 15 for none: zeros, and infinities and NaN as they are
    const uint32_t e = largest && largest < 0x7C00u ? __float_as_uint(gh_h2f(largest)) >> 23 : 127u + 15;
    const float up = __uint_as_float((127u + 127 + 15 - e) << 23);
    q.scale = a.scale * 512.0f * __uint_as_float((e - 15) << 23);
    float mine = 0.0f;
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s) {
        uint4 x = r.x[s];
        if (n >= G) x = make_uint4(0u, 0u, 0u, 0u);
        float v[8];
        gh_unpack8(x, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= up;
        const float sum = lanes4_sum(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])));
        if (s == g) mine = sum;
        uint32_t w[4];  // exact
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(v[i], v[i + 4]));
        q.x[s] = __builtin_bit_cast(ph8, make_uint4(w[0], as_u(as_h(w[1]) * down), w[2], as_u(as_h(w[3]) * down)));
        const uint32_t one = s == g ? 0x7800u : 0u;
        q.step[s] = __builtin_bit_cast(ph4, make_uint2(one, 0u));
    }
    mine *= 0x1p-9f;
    const uint32_t hi = gh_f2h(mine), lo = gh_f2h(mine - gh_h2f(hi));
    q.sums = __builtin_bit_cast(ph4, make_uint2(hi << 16, lo << 16));
}

// Products of a half, times 2^-9, from its K in LDS.
__device__ __forceinline__ pf4 half_products(const char* lds, const Query& q) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
    const uint4 k = *(const uint4*)(lds + n * kVector + 16 * g);
    const uint32_t dm = *(const uint32_t*)(lds + n * kVector + 64 + 4 * g);
    // lane g has dwords 4 g + j; it takes 4 s + g: row j and lane group g change places
    const auto a = __builtin_amdgcn_permlane32_swap(k.x, k.z, false, false), b = __builtin_amdgcn_permlane32_swap(k.y, k.w, false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    const uint32_t w[4] = {c[0], c[1], d[0], d[1]};
    const ph4 dms = __builtin_bit_cast(ph4, make_uint2(dm, dm));
    const pf4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    pf4 sum = __builtin_amdgcn_mfma_f32_16x16x16f16(dms, q.sums, zero, 0, 0, 0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint32_t w8 = w[s] >> 8;
        const ph8 codes = __builtin_bit_cast(ph8, make_uint4(w[s] & 0x000F000Fu, w[s] & 0x00F000F0u, w8 & 0x000F000Fu, w8 & 0x00F000F0u));
        const pf4 st = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q.x[s], zero, 0, 0, 0);
        const pf4 step = __builtin_amdgcn_mfma_f32_16x16x16f16(dms, q.step[s], zero, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(step[i], st[i], sum[i]);
    }
    return sum;
}
// -inf past the tile's positions
__device__ __forceinline__ void hide(pf4 (&st)[2], uint32_t count) {
    if (count >= 32) return;
    const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (16 * (i >> 2) + 4 * g + (i & 3) >= count) st[i >> 2][i & 3] = -__builtin_inff();
}
// The largest of two and of three, without the instructions by which fmaxf quiets its inputs first. (Ordinary vector results
// go in: none of a matrix instruction, which would need waits of their own.)
__device__ __forceinline__ float larger(float x, float y) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
    return r;
}
__device__ __forceinline__ float largest(float x, float y, float z) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
    return r;
}
__device__ __forceinline__ float lanes4_larger(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = larger(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return larger(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// A lane's V of a tile: dwords and steps with minima [4 half + i] of position 4 (l / 16) + i, dims 8 (l % 16) .. + 8.
struct Values {
    uint32_t v[8], dm[8];
};
__device__ __forceinline__ void load_v(const char* lds, Values& y) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const char* at = lds + (i >> 2) * kHalfBytes + (4 * g + (i & 3)) * kVector;
        y.v[i] = *(const uint32_t*)(at + 4 * n);
        y.dm[i] = *(const uint32_t*)(at + 64 + (n & ~3u));
    }
}
// st: products, which times the query's `scale` are scores in base 2
__device__ __forceinline__ void tile_add(Sums& x, const pf4 (&st)[2], float scale, const Masks& c, const Values& y) {
    const float top = largest(largest(st[0][0], st[0][1], st[0][2]), largest(st[0][3], st[1][0], st[1][1]), larger(st[1][2], st[1][3]));
    const float mx = larger(x.m, lanes4_larger(top) * scale);
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
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i >> 2][i & 3], scale, up));
    x.l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const ph2 h = __builtin_bit_cast(ph2, __builtin_amdgcn_cvt_pkrtz(p[2 * i], p[2 * i + 1]));
        hi[i] = as_u(h);
        lo[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h.x, -1.0f, p[2 * i]), __builtin_fmaf((float)h.y, -1.0f, p[2 * i + 1])));
    }
    const ph8 p0 = __builtin_bit_cast(ph8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
    const ph8 p1 = __builtin_bit_cast(ph8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
    ph2 d[4], m[4];  // of two positions
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        d[i] = as_h(lows(y.dm[2 * i], y.dm[2 * i + 1]));
        m[i] = as_h(highs(y.dm[2 * i], y.dm[2 * i + 1]));
    }
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
        uint32_t v0[4], v1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // byte b of both positions, in the low bytes of the halves
            const uint32_t w = __builtin_amdgcn_perm(y.v[2 * i + 1], y.v[2 * i], 0x0C000C00u | (4 + b) << 16 | b);
            v0[i] = as_u(__builtin_elementwise_fma(codes_low(w, c), d[i], m[i]));
            v1[i] = as_u(__builtin_elementwise_fma(codes_high(w, c), d[i], m[i]));
        }
        const ph8 a0 = __builtin_bit_cast(ph8, make_uint4(v0[0], v0[1], v0[2], v0[3]));
        const ph8 a1 = __builtin_bit_cast(ph8, make_uint4(v1[0], v1[1], v1[2], v1[3]));
        x.acc[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, p0, x.acc[2 * b], 0, 0, 0);
        x.acc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, p0, x.acc[2 * b + 1], 0, 0, 0);
        x.acc[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, p1, x.acc[2 * b], 0, 0, 0);
        x.acc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, p1, x.acc[2 * b + 1], 0, 0, 0);
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

// One chunk of the rows' tiles, `tiles` from `begin`, for a team's heads. All teams of the workgroup go through `rounds` tiles, where
// their chunks have fewer with nothing in the last. lds: the team's, mine0: the wave's, in the first of two buffers; kvh: the wave's head,
// if `there` is one.
template <bool SCORED, int CACHE>
__device__ __forceinline__ void paged4_chunk(const GhPagedAttnArgs& a, const RowsLds& sh, uint32_t behind, uint32_t begin, uint32_t tiles,
                                             uint32_t chunk, uint32_t rounds, uint32_t kvh, bool there, bool idle, const Pieces& pieces,
                                             char* lds, const char* mine0) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, G = a.group;
    const Masks masks;

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
        return Where{(uint32_t)__builtin_amdgcn_readlane(t_slot0, i & 63u), (uint32_t)__builtin_amdgcn_readlane(t_slot1, i & 63u), count};
    };

    Query q;
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
        RawQuery rq;
        ask_q4(a, row, kvh, rq);
        make_q4(a, rq, q);
        if (SCORED) raw = a.raw + (((uint64_t)row * a.p.kv_heads + kvh) * G + n) * a.raw_len * 4;
    };
    Tile4 r;
    load_tile<CACHE>(where(0), pieces, r);
    if (there && tiles) start(__builtin_amdgcn_readlane(t_row, 0), 0);
    for (uint32_t i = 0; i < rounds; ++i) {
        const uint32_t info = __builtin_amdgcn_readlane(t_row, i & 63u);
        const uint32_t pos = SCORED ? __builtin_amdgcn_readlane(t_pos, i & 63u) : 0u;
        char* buf = lds + (i & 1) * (4 * kStageBytes);
        const char* mine = mine0 + (i & 1) * (4 * kStageBytes);
        // two buffers in turn: behind the barrier all have read the tile before
        if (!idle) store_tile(r, pieces, buf);
        gh_lds_barrier();
        if ((i & 63u) == 63) look_up(i + 1);
        load_tile<CACHE>(where(i + 1), pieces, r);
        if (!there || i >= tiles) continue;
        if ((info & 0xFFFFu) != row) {
            flush(i);
            start(info, i);
        }
        pf4 st[2] = {half_products(mine, q), half_products(mine + kHalfBytes, q)};
        hide(st, info >> 16);
        if (SCORED && n < G) keep_scores(raw, pos, st, q.scale);
        Values y;
        load_v(mine + 2 * kHalfBytes, y);
        tile_add(x, st, q.scale, masks, y);
    }
    if (there && tiles) flush(tiles);
}

// All rows' tiles in chunks, as gh_paged_attn, with a team per chunk. The tiles are shared out to one each: the first `more` chunks
// have one tile more than the others (in chunks of the same number of tiles, of which the last ones are empty, 32 rows of up to
// 4000 took 29.9 us instead of 29.0, 40 of up to 2000 27.5 instead of 24.0). For the join, which takes chunks of `per` tiles, a
// tile has the number it would have if all chunks had `per`.
template <bool SCORED>
__device__ __forceinline__ void paged4_attn(const GhPaged4AttnArgs& t) {
    __shared__ RowsLds sh;
    __shared__ __align__(16) char stage[8 * kStageBytes];
    const GhPagedAttnArgs& a = t.a;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = wave / t.heads, member = wave % t.heads;
    const uint32_t set = blockIdx.x / (8 * t.groups) * 8 + blockIdx.x % 8, first = set * t.teams, chunk = first + team;
    const uint32_t head = blockIdx.x / 8 % t.groups * t.heads, kvh = head + member;
    const uint32_t behind = lay_out_rows<5>(a, sh, blockIdx.x == 0);
    const uint32_t total = sh.first[a.rows];
    const uint32_t chunks = max(1u, min(a.chunks, total / a.least)), least = total / chunks, more = total % chunks, per = least + (more ? 1u : 0u);
    auto start_of = [&](uint32_t c) __attribute__((always_inline)) { return c * least + min(c, more); };
    if (blockIdx.x == 0) {  // for the join
        for (uint32_t r = threadIdx.x; r <= a.rows; r += 256) {
            const uint32_t t = sh.first[r];
            uint32_t c = 0;
            if (t) c = t < more * per ? t / per : more + (t - more * per) / least;
            gh_gpw<uint32_t>(a.layout)[1 + r] = c * per + (t - start_of(c));
        }
        if (threadIdx.x == 0) gh_gpw<uint32_t>(a.layout)[0] = max(per, 1u);
    }
    for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x)
        if (sh.len[r] == 0)
            for (uint32_t i = threadIdx.x; i < a.q_heads * 64; i += 256)
                gh_gpw<uint32_t>(a.out)[(uint64_t)r * a.q_heads * 64 + i] = 0u;
    if (first >= chunks || total == 0) return;  // the whole workgroup
    const uint32_t rounds = least + (first < more ? 1u : 0u), heads = min(t.heads, a.p.kv_heads - head);
    const bool idle = team >= t.teams || chunk >= chunks, there = !idle && member < heads;  // three heads leave a wave without a team
    const uint32_t begin = start_of(min(chunk, chunks)), tiles = idle ? 0u : least + (chunk < more ? 1u : 0u);
    const Pieces pieces(a.p, head, t.heads, threadIdx.x - team * t.heads * 64, heads);
    char* lds = stage + team * t.heads * kStageBytes;
    const char* mine = lds + member * kStageBytes;
    if ((uint64_t)total * a.p.kv_heads * (64 * kVector) >= a.stream)
        paged4_chunk<SCORED, kStream>(a, sh, behind, begin, tiles, chunk, rounds, kvh, there, idle, pieces, lds, mine);
    else
        paged4_chunk<SCORED, 0>(a, sh, behind, begin, tiles, chunk, rounds, kvh, there, idle, pieces, lds, mine);
}

// Each row in spans, as gh_paged_split: of a.least / 2 tiles, of which wave w takes w, w + 4, ... Grid (8 kv heads, spans / 8): the
// heads of a span, whose vectors share lines, on one XCD, where workgroups go by their number mod 8, and so from one L2 (us of a call, so /
// with adjacent heads on adjacent XCDs: 100 rows of up to 1000 36.4 / 45.0, 256 of up to 300 33.2 / 36.9, 1 of 9000 23.3 / 26.0,
// 1 of 500 19.0 / 19.2).
template <bool SCORED>
__device__ __forceinline__ void paged4_split(const GhPagedAttnArgs& a) {
    extern __shared__ __align__(16) float dyn[];  // per wave and head: 132 floats of acc, then m and l
    __shared__ __align__(16) char stage[4][kTileBytes];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, G = a.group;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t spot = blockIdx.y * 8 + blockIdx.x % 8, kvh = blockIdx.x / 8;
    if (spot >= a.chunks * a.rows) return;
    const uint32_t row = spot / a.chunks, split = spot % a.chunks;
    const uint32_t span = a.least * 16, begin = split * span;  // < max_len
    // the wave's tile i covers positions begin + 128 i + 32 wave .. + 32
    const uint32_t first = begin + 32 * wave, mine = first + 128 * lane;
    RawQuery rq;
    ask_q4(a, row, kvh, rq);
    const uint32_t len = row_length(a.p, row, a.max_len, kvh == 0 && split == 0);
    if (len == 0) {
        if (split == 0)
            for (uint32_t i = tid; i < G * 64; i += 256) gh_gpw<uint32_t>(a.out + ((uint64_t)row * a.q_heads + kvh * G) * 256)[i] = 0u;
        return;
    }
    if (begin >= len) return;
    const uint32_t end = min(len, begin + span);
    uint32_t t_slot0 = 0, t_slot1 = 0, t_count = 0;
    if (mine < end) {
        const uint32_t count = min(end - mine, 32u);
        if (tile_slots(a.p, row, mine, count, &t_slot0, &t_slot1)) t_count = count;
    }
    const uint32_t tiles = first < end ? (end - first + 127) / 128 : 0u;
    const Pieces pieces(a.p, kvh, 1, lane, 1);
    const Masks masks;
    auto where = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t count = i < tiles ? __builtin_amdgcn_readlane(t_count, i & 63u) : 0u;
        return Where{(uint32_t)__builtin_amdgcn_readlane(t_slot0, i & 63u), (uint32_t)__builtin_amdgcn_readlane(t_slot1, i & 63u), count};
    };
    const uint64_t raw = a.raw + (((uint64_t)row * a.p.kv_heads + kvh) * G + n) * a.raw_len * 4;
    Sums x;
    x.clear();
    if (tiles) {
        char* lds = stage[wave];
        Tile4 r;
        load_tile<0>(where(0), pieces, r);
        Query q;
        make_q4(a, rq, q);
        for (uint32_t i = 0; i < tiles; ++i) {
            wave_order();
            store_tile(r, pieces, lds);
            wave_order();
            load_tile<0>(where(i + 1), pieces, r);
            pf4 st[2] = {half_products(lds, q), half_products(lds + kHalfBytes, q)};
            hide(st, __builtin_amdgcn_readlane(t_count, i & 63u));
            if (SCORED && n < G) keep_scores(raw, first + 128 * i, st, q.scale);
            Values y;
            load_v(lds + 2 * kHalfBytes, y);
            tile_add(x, st, q.scale, masks, y);
        }
    }
    split_finish<SCORED>(a, x, dyn, row, kvh, split, span, len);
}
}  // namespace
GH_KERNEL __launch_bounds__(256, 3) void gh_paged4_attn(GhPaged4AttnArgs a) { paged4_attn<false>(a); }
GH_KERNEL __launch_bounds__(256, 3) void gh_paged4_attn_s(GhPaged4AttnArgs a) { paged4_attn<true>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged4_split(GhPagedAttnArgs a) { paged4_split<false>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged4_split_s(GhPagedAttnArgs a) { paged4_split<true>(a); }

// ---- eviction -----------------------------------------------------------------------------------
// The move of gh_paged_move for vectors of five 16-byte pieces, a thread each. Same grid. 84 MB read and written in 20 us, 2.7 GB in
// 702 (3.8 TB/s: each head keeps positions of its own, and lines hold parts of two heads); loads past the caches, which lose
// the lines' other parts, 26 and 845, stores past them the same.
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
        *gh_gpw<u4v>(a.dst.kc + to) = k;
        *gh_gpw<u4v>(a.dst.vc + to) = v;
    }
}
