// A batch of sequences over paged FP16 caches (gh_kv_paged): append with RoPE, decode attention, eviction.
//
// The pool is a cache [layer][slot][kv_heads][128]; position j of row r lives at slot
// (table[r][j >> shift] << shift) + (j & page_size - 1). Lengths, page numbers and positions are device data
// that the host has not seen: every kernel checks them before it forms an address, skips what does not fit
// and leaves a word in pinned host memory, which gh_submit reports.
#include "gh_paged.h"

// ---- append ----------------------------------------------------------------------------------
// Thread = 8 values (16 bytes) of one head of one token: the token's query heads, then its key and value
// heads; a.groups workgroups per token. Rotation as in gh_rope: adjacent pairs turned by the (position, pair)
// table's (cos, sin) in FP32, queries times the post-scale, one rounding. Bound by launch latency at decode
// sizes (256 tokens of 32 + 8 heads 4.1 us traced) and by memory at prompt sizes (2000 tokens of 8 heads, 16 MB, 4.9 us);
// the vector, the row's length and its position are asked for at once.
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
    if (head >= a.q_heads + 2 * a.p.kv_heads) return;
    const bool query = head < a.q_heads, value = head >= a.q_heads + a.p.kv_heads;
    const uint32_t h = query ? head : head - a.q_heads - (value ? a.p.kv_heads : 0u);
    const uint32_t heads = query ? a.q_heads : a.p.kv_heads;
    const uint64_t in = ((uint64_t)token * heads + h) * 256 + 16 * part;
    uint4 x = *gh_gp<uint4>((query ? a.q : value ? a.v : a.k) + in);
    const uint32_t from = a.positions ? gh_gp<uint32_t>(a.positions)[row] : 0u;
    const uint32_t n = row_length(a.p, row, a.p.width << a.p.shift, blockIdx.x % a.groups == 0);
    if (n + t < a.tokens) return;  // a free row, or before its first position
    const uint32_t at = n - a.tokens + t, pos = from + t;
    if (a.positions && (from > a.max_pos || t > a.max_pos - from)) {
        if (item == 0) fault(a.p, GH_PAGED_POSITION);
        return;
    }
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
// Bound by the read of K and V. A wave takes the G <= 16 query heads of one kv head over tiles of 16 positions, each
// within one page (page_size >= 16) and so at one address: lanes hold the next 64 tiles' slots, looked up
// together, and a tile's is a readlane away. Per tile, with FP32 accumulators and scores in base 2:
//   S^T = K·Q^T     4 x v_mfma_f32_16x16x32_f16: A = 16 K rows straight from memory (lane l: position l % 16,
//                   dims 32 s + 8 (l / 16) .. + 8), B = the query, column n = l % 16 is head n (zero
//                   past G); lane l receives head n's scores of positions 4 (l / 16) + i;
//   O^T += V^T·P^T  per 8-dim tile t one v_mfma_f32_16x16x32_f16 whose 32 k-slots are the 16 positions
//                   twice: a lane's weights split into FP16 hi + lo (truncated, so both are positive), so
//                   that P·V keeps 22 bits of each weight. Output row m stands for value dim 8 m + t.
// Weights are 2^(s - m + 15), m the running maximum: hi + lo then reach 2^-39 of the largest weight. Both
// parts are at least 2^-24, so that an infinite V gives an infinity and not infinity times 0, but those of a score
// of -inf are 0: an infinite V gives NaN there, and a row of nothing else 0 / 0.
// K and V are read through buffer resources whose range ends at the row's last position: what a page holds
// past it reads as zero, without a memory access, and has weight 0. The next tile's K is asked for as soon as
// this one's products are made, its V behind the last use of this one's: one set of registers, 125 to 154
// VGPRs. (Two sets: 64 rows of 8192 330 / 333 us with the wait for the call, with half the waves per CU 394 / 403.)
// Other times of attention here are of calls back to back, both launches.
// Two divisions of the work over waves, paged_attn and paged_split (the host's rule says when), then
// gh_paged_join where a row is in several parts.
namespace {
struct Tile {
    uint4 k[4];  // position l % 16, dims 32 s + 8 (l / 16) .. + 8
    uint4 v[4];  // position 4 (l / 16) + i, dims 8 (l % 16) .. + 8
};

// element t of the 16-byte slices of four positions, twice (the hi and the lo slots)
__device__ __forceinline__ ph8 v_column(const uint4 (&v)[4], int t) {
    auto word = [&](int i) __attribute__((always_inline)) {
        return (t >> 1) == 0 ? v[i].x : (t >> 1) == 1 ? v[i].y : (t >> 1) == 2 ? v[i].z : v[i].w;
    };
    const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;  // the high or the low halves of two words
    const uint32_t d0 = __builtin_amdgcn_perm(word(1), word(0), sel), d1 = __builtin_amdgcn_perm(word(3), word(2), sel);
    return __builtin_bit_cast(ph8, make_uint4(d0, d1, d0, d1));
}

// two weights' FP16 hi parts in *hi, lo parts in *lo; s0, s1: their scores
__device__ __forceinline__ void weight_parts(float p0, float p1, float s0, float s1, uint32_t* hi, uint32_t* lo) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const float none = -__builtin_inff();
    const pu2 least = {(uint16_t)(s0 != none), (uint16_t)(s1 != none)};
    const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0, p1));
    const h2 hv = __builtin_bit_cast(h2, h);
    const uint32_t l = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p0 - (float)hv.x, p1 - (float)hv.y));
    *hi = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pu2, h), least));
    *lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pu2, l), least));
}

// A tile's addresses: K and V of one head from the slot of the tile's first position, `count` positions long
// (0: no range, and nothing is read). The widest row, 65535 heads, keeps offsets below 2^28.
struct Where {
    __amdgpu_buffer_rsrc_t k, v;
};
__device__ __forceinline__ Where tile_at(const GhPages& p, uint32_t slot, uint32_t count, uint32_t kvh) {
    const uint32_t row_bytes = p.kv_heads * 256;
    const uint64_t at = (uint64_t)slot * row_bytes + kvh * 256;
    const int range = count ? (int)((count - 1) * row_bytes + 256) : 0;
    return {__builtin_amdgcn_make_buffer_rsrc((void*)(p.kc + at), 0, range, kBufWord3),
            __builtin_amdgcn_make_buffer_rsrc((void*)(p.vc + at), 0, range, kBufWord3)};
}
template <int CACHE>
__device__ __forceinline__ void load_k(const Where& w, uint32_t row_bytes, Tile& r) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int s = 0; s < 4; ++s)
        r.k[s] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(w.k, n * row_bytes + 16 * g + 64 * s, 0, CACHE));
}
template <int CACHE>
__device__ __forceinline__ void load_v(const Where& w, uint32_t row_bytes, Tile& r) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        r.v[j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(w.v, (4 * g + j) * row_bytes + 16 * n, 0, CACHE));
}

// B fragments of the G queries of a kv head: head n = l % 16 (zero past G), dims 32 s + 8 (l / 16) .. + 8.
__device__ __forceinline__ void load_q(const GhPagedAttnArgs& a, uint32_t row, uint32_t kvh, ph8 (&qf)[4]) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const GH_GLOBAL uint4* qp = gh_gp<uint4>(a.q + (((uint64_t)row * a.q_heads + kvh * G + min(n, G - 1)) * 128 + 8 * g) * 2);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint4 x = qp[4 * s];
        qf[s] = __builtin_bit_cast(ph8, n < G ? x : make_uint4(0u, 0u, 0u, 0u));
    }
}

__device__ __forceinline__ pf4 tile_products(const Tile& r, const ph8 (&qf)[4]) {
    pf4 st = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s)
        st = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, r.k[s]), qf[s], st, 0, 0, 0);
    return st;
}
// products -> scores in base 2, -inf past the tile's positions
__device__ __forceinline__ pf4 tile_scores(pf4 st, uint32_t count, float scale) {
    const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) st[j] = 4 * g + (uint32_t)j < count ? st[j] * scale : -__builtin_inff();
    return st;
}
__device__ __forceinline__ void tile_add(Sums& x, pf4 st, const Tile& r) {
    const float mx = fmaxf(x.m, lanes4_max(fmaxf(fmaxf(st[0], st[1]), fmaxf(st[2], st[3]))));
    const float f = share(x.m, mx);
    // nothing but -inf so far: every weight 0
    const float up = mx == -__builtin_inff() ? 0.0f : kUp - mx;
    x.m = mx;
    float p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = __builtin_amdgcn_exp2f(st[j] + up);
    x.l = x.l * f + ((p[0] + p[1]) + (p[2] + p[3]));
    uint32_t h0, h1, l0, l1;
    weight_parts(p[0], p[1], st[0], st[1], &h0, &l0);
    weight_parts(p[2], p[3], st[2], st[3], &h1, &l1);
    const ph8 pv = __builtin_bit_cast(ph8, make_uint4(h0, h1, l0, l1));
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        x.acc[t] *= f;
        x.acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_column(r.v, t), pv, x.acc[t], 0, 0, 0);
    }
}

// One chunk of the rows' tiles for one kv head by one wave.
template <bool SCORED, int CACHE>
__device__ __forceinline__ void paged_chunk(const GhPagedAttnArgs& a, const RowsLds& sh, uint32_t behind, uint32_t total,
                                            uint32_t per, uint32_t chunk, uint32_t kvh) {
    const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const uint32_t begin = chunk * per, tiles = min(per, total - begin), row_bytes = a.p.kv_heads * 256;

    // lane i: slot, first position, and row | positions << 16 of tile i of the current 64
    uint32_t t_slot = 0, t_pos = 0, t_row = 0;
    auto look_up = [&](uint32_t from) __attribute__((always_inline)) {
        const uint32_t t = begin + from + lane;
        t_slot = t_pos = t_row = 0;
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
        t_pos = (t - sh.first[lo]) * 16;
        const uint32_t page = gh_gp<uint32_t>(a.p.table)[(uint64_t)lo * a.p.width + (t_pos >> a.p.shift)];
        const bool bad = page >= a.p.pages;
        if (bad) fault(a.p, GH_PAGED_PAGE);
        t_slot = bad ? 0u : (page << a.p.shift) + (t_pos & ((1u << a.p.shift) - 1));
        t_row = lo | (bad ? 0u : min(sh.len[lo] - t_pos, 16u) << 16);
    };
    look_up(0);
    auto where = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t count = i < tiles ? __builtin_amdgcn_readlane(t_row, i & 63u) >> 16 : 0u;
        return tile_at(a.p, __builtin_amdgcn_readlane(t_slot, i & 63u), count, kvh);
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
        load_q(a, row, kvh, qf);
        if (SCORED) raw = a.raw + (((uint64_t)row * a.p.kv_heads + kvh) * G + n) * a.raw_len * 4;
    };
    start(__builtin_amdgcn_readlane(t_row, 0), 0);

    // K of the next tile is asked for as soon as this one's products are made, V behind its last use
    Tile r;
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
        pf4 st = tile_products(r, qf);
        if ((i & 63u) == 63) look_up(i + 1);
        w = where(i + 1);
        load_k<CACHE>(w, row_bytes, r);
        st = tile_scores(st, info >> 16, a.scale);
        if (SCORED && n < G)
            *gh_gpw<float4>(raw + (uint64_t)(pos + 4 * g) * 4) = make_float4(st[0], st[1], st[2], st[3]);
        tile_add(x, st, r);
        load_v<CACHE>(w, row_bytes, r);
    }
    flush(tiles);
}

// All rows' tiles in equal chunks. Grid: a wave per (chunk, kv head), heads first, 256 threads. A workgroup's
// four waves read four heads of the same positions, 1 KiB in a row per position (four chunks of one head
// instead: 64 rows of 8192 324 -> 376 us, 32 up to 4000 52.7 -> 57.4). The number of tiles is known on the device alone: every workgroup
// adds up the rows' lengths, workgroup 0 leaves the result for the join.
template <bool SCORED>
__device__ __forceinline__ void paged_attn(const GhPagedAttnArgs& a) {
    __shared__ RowsLds sh;
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunk = unit / a.p.kv_heads, kvh = unit % a.p.kv_heads;
    const uint32_t behind = lay_out_rows<4>(a, sh, blockIdx.x == 0);
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
    if ((uint64_t)total * a.p.kv_heads * 8192 >= a.stream) paged_chunk<SCORED, kStream>(a, sh, behind, total, per, chunk, kvh);
    else paged_chunk<SCORED, 0>(a, sh, behind, total, per, chunk, kvh);
}
}  // namespace

GH_KERNEL __launch_bounds__(256, 3) void gh_paged_attn(GhPagedAttnArgs a) { paged_attn<false>(a); }
GH_KERNEL __launch_bounds__(256, 3) void gh_paged_attn_s(GhPagedAttnArgs a) { paged_attn<true>(a); }

namespace {
// Each row in spans. Grid (kv heads, spans, rows), 256 threads: wave w takes tiles w, w + 4, ... of the span, then
// the four waves' sums are joined in LDS. A row of one span is finished here, scores included.
template <bool SCORED>
__device__ __forceinline__ void paged_split(const GhPagedAttnArgs& a) {
    extern __shared__ __align__(16) float dyn[];  // per wave and head: 132 floats of acc, then m and l
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, g = lane >> 4, G = a.group;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, row = blockIdx.z;
    const uint32_t span = a.least * 16, begin = split * span;  // < max_len
    // the wave's tile i covers positions begin + 64 i + 16 wave .. + 16
    const uint32_t first = begin + 16 * wave, mine = first + 64 * lane;
    uint32_t entry = 0;
    if (64 * lane + 16 * wave < span && mine < a.max_len)
        entry = gh_gp<uint32_t>(a.p.table)[(uint64_t)row * a.p.width + (mine >> a.p.shift)];
    const uint32_t len = row_length(a.p, row, a.max_len, kvh == 0 && split == 0);
    const uint64_t out = a.out + ((uint64_t)row * a.q_heads + kvh * G) * 256;
    if (len == 0) {
        if (split == 0)
            for (uint32_t i = tid; i < G * 64; i += 256) gh_gpw<uint32_t>(out)[i] = 0u;
        return;
    }
    if (begin >= len) return;
    ph8 qf[4];
    load_q(a, row, kvh, qf);
    const uint32_t end = min(len, begin + span);
    const bool bad = mine < end && entry >= a.p.pages;
    if (bad) fault(a.p, GH_PAGED_PAGE);
    const uint32_t t_count = mine < end && !bad ? min(end - mine, 16u) : 0u;
    const uint32_t t_slot = bad ? 0u : (entry << a.p.shift) + (mine & ((1u << a.p.shift) - 1));
    const uint32_t tiles = first < end ? (end - first + 63) / 64 : 0u, row_bytes = a.p.kv_heads * 256;
    auto where = [&](uint32_t i) __attribute__((always_inline)) {
        const uint32_t count = i < tiles ? __builtin_amdgcn_readlane(t_count, i & 63u) : 0u;
        return tile_at(a.p, __builtin_amdgcn_readlane(t_slot, i & 63u), count, kvh);
    };
    const uint64_t raw0 = a.raw + ((uint64_t)row * a.p.kv_heads + kvh) * G * a.raw_len * 4;
    Sums x;
    x.clear();
    if (tiles) {
        Tile r;
        Where w = where(0);
        load_k<0>(w, row_bytes, r);
        load_v<0>(w, row_bytes, r);
        for (uint32_t i = 0; i < tiles; ++i) {
            pf4 st = tile_products(r, qf);
            w = where(i + 1);
            load_k<0>(w, row_bytes, r);
            st = tile_scores(st, __builtin_amdgcn_readlane(t_count, i & 63u), a.scale);
            if (SCORED && n < G)
                *gh_gpw<float4>(raw0 + ((uint64_t)n * a.raw_len + first + 64 * i + 4 * g) * 4) =
                    make_float4(st[0], st[1], st[2], st[3]);
            tile_add(x, st, r);
            load_v<0>(w, row_bytes, r);
        }
    }
    split_finish<SCORED>(a, x, dyn, row, kvh, split, span, len);
}
}  // namespace
GH_KERNEL __launch_bounds__(256) void gh_paged_split(GhPagedAttnArgs a) { paged_split<false>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged_split_s(GhPagedAttnArgs a) { paged_split<true>(a); }

// The parts of a row joined. Grid (q_heads + kv_heads·blocks, rows, HALVES), 256 threads.
// x < q_heads: 128 / HALVES dims of the output of one query head: M = max m_s, out = Σ 2^(m_s - M) acc_s /
// Σ 2^(m_s - M) l_s; 8·HALVES groups of threads take every so many-th partial, four dims per thread, each with a
// running maximum, and add up in group order. Bound by its chain of loads; two halves where few rows have many
// partials each (1 row of 32768, 256 partials: attention and join 33.2 us with one, 31.7 with two), one where many rows have
// few (32 up to 4000 52.7 with one, 53.3 with two).
// Else: the scores of a kv head, every blocks-th 1024 positions (add_scores).
namespace {
template <uint32_t HALVES>
__device__ __forceinline__ void paged_join(const GhPagedAttnArgs& a) {
    constexpr uint32_t kGroups = 8 * HALVES, kLanes = 32 / HALVES;
    __shared__ float sm[16], sl[16];
    __shared__ pf4 red[kGroups][kLanes];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, row = blockIdx.y, G = a.group;
    const bool score = blockIdx.x >= a.q_heads;
    if (score && blockIdx.z) return;
    const uint32_t len = row_length(a.p, row, a.max_len, false);
    const uint32_t kvh = score ? (blockIdx.x - a.q_heads) / a.blocks : blockIdx.x / G;
    const uint32_t pos = score ? 1024 * ((blockIdx.x - a.q_heads) % a.blocks) + 4 * tid : 0u;
    pf4 raw[4];
    if (score && pos < len) load_raw(a, row, kvh, 0, pos, raw);  // on their way while M and L are found
    // the row's first partial and their number
    uint32_t p0, ns;
    if (a.layout) {
        const GH_GLOBAL uint32_t* lay = gh_gp<uint32_t>(a.layout);
        const uint32_t per = lay[0], t0 = lay[1 + row], t1 = lay[2 + row];
        if (t0 == t1) return;
        p0 = t0 / per + row;
        ns = (t1 - 1) / per - t0 / per + 1;
        if (!score && ns == 1 && !a.raw) return;  // written by the attention launch
    } else {
        p0 = row * a.chunks;
        ns = (len + 16 * a.least - 1) / (16 * a.least);
        if (ns <= 1) return;  // likewise, with its scores
    }
    const uint32_t step = a.p.kv_heads * G;  // partials of a chunk or span
    const uint64_t part = (uint64_t)p0 * step + kvh * G;
    if (!score) {
        // what is asked past the row's last partial is not read (at most 2048 + 65535 partials of 512 bytes)
        const uint32_t h = blockIdx.x % G, grp = tid / kLanes, d4 = kLanes * blockIdx.z + tid % kLanes;
        const uint32_t most = (ns - 1) * step + 1;
        const __amdgpu_buffer_rsrc_t ra =
            __builtin_amdgcn_make_buffer_rsrc((void*)(a.part_acc + (part + h) * 512), 0, (int)(most * 512), kBufWord3);
        const __amdgpu_buffer_rsrc_t rm =
            __builtin_amdgcn_make_buffer_rsrc((void*)(a.part_ml + (part + h) * 8), 0, (int)(most * 8), kBufWord3);
        float M = -__builtin_inff(), L = 0.0f;
        pf4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t s0 = grp; s0 < ns; s0 += 8 * kGroups) {
            float2 x[8];
            pf4 v[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t at = (s0 + kGroups * i) * step;
                x[i] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rm, at * 8, 0, 0));
                v[i] = __builtin_bit_cast(pf4, __builtin_amdgcn_raw_buffer_load_b128(ra, at * 512 + 16 * d4, 0, 0));
            }
            float top = M;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                if (s0 + kGroups * i >= ns) x[i].x = -__builtin_inff();
                top = fmaxf(top, x[i].x);
            }
            const float f = share(M, top);
            M = top;
            L *= f;
            o *= f;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const float e = share(x[i].x, M);
                L += e * x[i].y;
                o += e * v[i];
            }
        }
        red[grp][tid % kLanes] = o;
        if (tid % kLanes == 0) {
            sm[grp] = M;
            sl[grp] = L;
        }
        __syncthreads();
        if (tid < kLanes) {
            M = sm[0];
#pragma unroll
            for (uint32_t i = 1; i < kGroups; ++i) M = fmaxf(M, sm[i]);
            L = 0.0f;
            o = pf4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t i = 0; i < kGroups; ++i) {
                const float e = share(sm[i], M);
                L += e * sl[i];
                o += e * red[i][tid];
            }
            const float inv = 1.0f / L;
            gh_gpw<uint2>(a.out)[((uint64_t)row * a.q_heads + blockIdx.x) * 32 + d4] =
                make_uint2(out2(o.x, o.y, inv), out2(o.z, o.w, inv));
        }
        return;
    }
    const GH_GLOBAL float2* ml = gh_gp<float2>(a.part_ml) + part;
    for (uint32_t h = wave; h < G; h += 4) {
        float M = -__builtin_inff(), L = 0.0f;
        for (uint32_t s = lane; s < ns; s += 64) {
            const float2 x = ml[(uint64_t)s * step + h];
            const float top = fmaxf(M, x.x);
            L = L * share(M, top) + share(x.x, top) * x.y;
            M = top;
        }
        const float top = gh_wave_max(M);
        L = gh_wave_sum(L * share(M, top));
        if (lane == 0) {
            sm[h] = top;
            sl[h] = L;
        }
    }
    __syncthreads();
    add_scores(a, row, kvh, sm, sl, pos, 1024 * a.blocks, len, raw);
}
}  // namespace
GH_KERNEL __launch_bounds__(256) void gh_paged_join(GhPagedAttnArgs a) { paged_join<1>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged_join2(GhPagedAttnArgs a) { paged_join<2>(a); }

// ---- eviction -----------------------------------------------------------------------------------
// Two launches. gh_paged_select, grid (kv heads, rows, layers), 512 threads: the budget - recent largest
// scores of the older positions by a radix select over the scores' order as 32-bit keys (11, 11 and 10 bits
// per pass, counted in LDS, until a whole bin stays), then one pass in ascending order that writes the kept
// positions and moves their scores; equal keys are taken from the front. Bound by its barriers and LDS atomics:
// 272 lists of 4096 in 9.8 us (16.5 with the scores read in every pass and shuffles through LDS). In place:
// a step's scores are read before a barrier and written after it, at or before where they came from.
// gh_paged_move, grid (16-slot blocks of the budget, rows, layers), 256 threads: 16 lanes per 256-byte vector,
// consecutive groups of lanes the heads of one slot, so that writes are contiguous; bound by memory, 570 MB
// in and out at 5.1 TB/s.
namespace {
// f32 total order as unsigned order
__device__ __forceinline__ uint32_t order_key(uint32_t bits) { return bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u); }

constexpr uint32_t kHeld = 4;  // steps of 2048 scores that a workgroup keeps in registers

// One (kv head, row, layer)'s kept positions, ascending, and their scores. HELD: n <= 2048 kHeld, the scores are
// read once; else once per pass.
template <bool HELD>
__device__ __forceinline__ void select_kept(const GhPagedEvictArgs& a, uint32_t n, const GH_GLOBAL uint32_t* from,
                                            GH_GLOBAL uint32_t* to, GH_GLOBAL uint32_t* kept) {
    __shared__ __align__(16) uint32_t hist[3][2048];
    __shared__ uint32_t sums[8], pick[3];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t older = n - a.recent;  // > budget - recent
    // thread: positions 2048 c + 4 tid .. + 4 of step c
    auto at = [&](uint32_t c) __attribute__((always_inline)) {
        const uint32_t p = 2048 * c + 4 * tid;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (p < n) x = *(const GH_GLOBAL uint4*)(from + p);
        return x;
    };
    uint4 held[HELD ? kHeld : 1];
    if (HELD)
#pragma unroll
        for (uint32_t c = 0; c < kHeld; ++c) held[c] = at(c);
    auto each = [&](auto body) __attribute__((always_inline)) {
        if constexpr (HELD) {
#pragma unroll
            for (uint32_t c = 0; c < kHeld; ++c)
                if (2048 * c < n) body(c, held[c]);
        } else {
            for (uint32_t c = 0; 2048 * c < n; ++c) body(c, at(c));
        }
    };
    // keys above `least` stay, and the first `room` of those equal to it
    uint32_t least = 0xFFFFFFFFu, room = a.budget - a.recent;
    if (room) {
        for (uint32_t i = tid; i < 3 * 2048 / 4; i += 512) ((uint4*)hist)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        uint32_t prefix = 0;
        for (uint32_t pass = 0; pass < 3; ++pass) {
            const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            each([&](uint32_t c, const uint4& x) __attribute__((always_inline)) {
                const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    const uint32_t k = order_key(v[j]);
                    if (2048 * c + 4 * tid + j < older && (pass == 0 || k >> (shift + bits) == prefix))
                        atomicAdd(&hist[pass][k >> shift & ((1u << bits) - 1)], 1u);
                }
            });
            __syncthreads();
            // thread t counts bins 2047 - 4 t down to 2044 - 4 t
            const uint4 q = *(const uint4*)&hist[pass][2044 - 4 * tid];
            const uint32_t bin[4] = {q.w, q.z, q.y, q.x}, own = q.x + q.y + q.z + q.w;
            uint32_t upto = wave_scan(own);
            if (lane == 63) sums[wave] = upto;
            __syncthreads();
            for (uint32_t w = 0; w < wave; ++w) upto += sums[w];
            uint32_t above = upto - own;
            if (above < room && room <= upto) {  // one thread
                uint32_t j = 0;
                while (above + bin[j] < room) above += bin[j++];
                pick[0] = 2047 - 4 * tid - j;
                pick[1] = room - above;
                pick[2] = bin[j];
            }
            __syncthreads();
            prefix = prefix << bits | pick[0];
            room = pick[1];
            if (pick[2] == room && prefix) {  // the whole bin stays: no need to tell its keys apart
                least = (prefix << shift) - 1;
                room = 0;
                break;
            }
            least = prefix;
        }
    }
    uint32_t larger = 0, equal = 0;  // counts so far: larger keys, and keys equal to `least`
    each([&](uint32_t c, const uint4& x) __attribute__((always_inline)) {
        const uint32_t v[4] = {x.x, x.y, x.z, x.w}, p0 = 2048 * c + 4 * tid;
        uint32_t own = 0, flag[4];  // larger ones in the low half, equal ones in the high half
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t k = order_key(v[j]);
            flag[j] = p0 + j < n && (p0 + j >= older || k > least) ? 1u : p0 + j < older && k == least ? 0x10000u : 0u;
            own += flag[j];
        }
        uint32_t upto = wave_scan(own);
        __syncthreads();  // the last step's sums are read
        if (lane == 63) sums[wave] = upto;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (uint32_t w = 0; w < 8; ++w) {
            const uint32_t y = sums[w];
            upto += w < wave ? y : 0u;
            all += y;
        }
        uint32_t g = larger + ((upto - own) & 0xFFFFu), e = equal + ((upto - own) >> 16);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (flag[j] == 1 || (flag[j] && e < room)) {
                const uint32_t i = g + min(e, room);
                kept[i] = p0 + j;
                to[i] = v[j];
            }
            g += flag[j] & 1u;
            e += flag[j] >> 16;
        }
        larger += all & 0xFFFFu;
        equal += all >> 16;
    });
}
}  // namespace

GH_KERNEL __launch_bounds__(512) void gh_paged_select(GhPagedEvictArgs a) {
    const uint32_t kvh = blockIdx.x, row = blockIdx.y, layer = blockIdx.z;
    const uint32_t n = row_length(a.src, row, a.src.width << a.src.shift, kvh == 0 && layer == 0);
    const bool act = n > a.budget;
    if (kvh == 0 && layer == 0 && threadIdx.x == 0) gh_gpw<uint32_t>(a.act)[row] = act;
    if (!act) return;
    const uint64_t list = ((uint64_t)layer * a.rows + row) * a.src.kv_heads + kvh;
    const GH_GLOBAL uint32_t* from = gh_gp<uint32_t>(a.src.score) + list * (a.src.width << a.src.shift);
    GH_GLOBAL uint32_t* to = gh_gpw<uint32_t>(a.dst.score) + list * (a.dst.width << a.dst.shift);
    GH_GLOBAL uint32_t* kept = gh_gpw<uint32_t>(a.kept) + list * a.budget;
    if (n <= 2048 * kHeld) select_kept<true>(a, n, from, to, kept);
    else select_kept<false>(a, n, from, to, kept);
}

namespace {
template <bool STREAM>
__device__ __forceinline__ void paged_move(const GhPagedEvictArgs& a) {
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
        // stored past the caches, as what is moved is not wanted again soon, and where much is moved (the host's
        // rule) read past them too: 34 layers of 2048 slots 131.9, 124.6 and 122.5 us with the selection; 2 layers
        // of 4 rows of 560, whose source is still in cache, 18.1, 17.5 and 22.5
        typedef uint32_t u4v __attribute__((ext_vector_type(4)));
        const GH_GLOBAL u4v *kp = gh_gp<u4v>(a.src.kc + in), *vp = gh_gp<u4v>(a.src.vc + in);
        const u4v k = STREAM ? __builtin_nontemporal_load(kp) : *kp, v = STREAM ? __builtin_nontemporal_load(vp) : *vp;
        __builtin_nontemporal_store(k, gh_gpw<u4v>(a.dst.kc + to));
        __builtin_nontemporal_store(v, gh_gpw<u4v>(a.dst.vc + to));
    }
}
}  // namespace
GH_KERNEL __launch_bounds__(256) void gh_paged_move(GhPagedEvictArgs a) { paged_move<false>(a); }
GH_KERNEL __launch_bounds__(256) void gh_paged_move_s(GhPagedEvictArgs a) { paged_move<true>(a); }
