// Operators over paged KV caches (gh_kv_paged): checks, launch plans and scratch. The kernels are in
// kernels/paged.hip.
#include <algorithm>
#include <cmath>
#include <new>

#include "internal.h"

using namespace gh;

namespace {

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

bool fits(const gh_buf* buf, uint64_t bytes, uint64_t align) {
    return buf && buf->addr && buf->bytes >= bytes && buf->addr % align == 0;
}

// the bytes at a and b overlap
bool meet(const gh_buf* a, uint64_t a_bytes, const gh_buf* b, uint64_t b_bytes) {
    return a->addr < b->addr + b_bytes && b->addr < a->addr + a_bytes;
}

// The bytes of a buffer that a call uses.
struct Span {
    uint64_t at = 0, bytes = 0;
};
bool meet(const Span& a, const Span& b) { return a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes; }

constexpr uint32_t kPagedRows = 512;  // rows that one attention launch lays out
constexpr uint64_t kStreamBytes = 128ull << 20;  // half the last-level cache
constexpr uint32_t kSpanTiles = 32;   // tiles of a gh_paged_split workgroup at most (its waves hold 64 each)

uint64_t capacity(const gh_kv_paged* kv) { return (uint64_t)kv->table_width * kv->page_size; }

// What a handle uses of its buffers. Operators write all but the table.
enum { CACHE_K, CACHE_V, SCORE, LENGTHS, TABLE, PARTS };
struct Parts {
    Span part[PARTS];
    explicit Parts(const gh_kv_paged* p) {
        const gh_kv& kv = p->kv;
        part[CACHE_K].bytes = part[CACHE_V].bytes = (uint64_t)kv.block_count * kv.context * kv.kv_heads * 256;
        part[CACHE_K].at = kv.k.addr;
        part[CACHE_V].at = kv.v.addr;
        if (p->score.addr) part[SCORE] = {p->score.addr, (uint64_t)kv.block_count * p->rows * kv.kv_heads * capacity(p) * 4};
        part[LENGTHS] = {p->lengths.addr, (uint64_t)p->rows * 4};
        part[TABLE] = {p->table.addr, (uint64_t)p->rows * p->table_width * 4};
    }
    bool met(const Span& x) const {
        return std::any_of(part, part + PARTS, [&](const Span& y) { return meet(x, y); });
    }
};

// Everything about the handle that the host can see. `layer`: the one the call uses.
int check_paged(gh_backend* b, const gh_kv_paged* p, uint32_t layer, const char* what) {
    auto no = [&](int code, const char* why) { return fail(b, code, std::string(what) + ": " + why); };
    if (!p) return no(GH_E_INVALID, "null");
    const gh_kv& kv = p->kv;
    if (kv.scheme != GH_KV_F16) return no(GH_E_UNSUPPORTED, "only the f16 KV scheme");
    if (kv.head_dim != 128 || kv.value_dim != 128) return no(GH_E_UNSUPPORTED, "head_dim 128 only");
    if (kv.kv_heads == 0 || kv.kv_heads > 0xFFFFu) return no(GH_E_INVALID, "kv_heads");
    if (p->page_size < 16 || p->page_size > 32768 || (p->page_size & (p->page_size - 1)))
        return no(GH_E_INVALID, "page_size must be a power of two, 16..32768");
    if (kv.context == 0 || kv.context % p->page_size) return no(GH_E_INVALID, "the pool is not whole pages");
    if (p->rows == 0 || p->rows > 0xFFFFu) return no(GH_E_INVALID, "1 to 65535 rows");
    if (p->table_width == 0 || capacity(p) > 0x7FFFFFFFull) return no(GH_E_INVALID, "table_width");
    if (layer >= kv.block_count) return no(GH_E_RANGE, "layer beyond the pool");
    const unsigned __int128 cache = (unsigned __int128)kv.block_count * kv.context * kv.kv_heads * 256;
    const unsigned __int128 score = (unsigned __int128)kv.block_count * p->rows * kv.kv_heads * capacity(p) * 4;
    if ((cache | score) >> 63) return no(GH_E_RANGE, "cache too small");
    if (!fits(&kv.k, (uint64_t)cache, 16) || !fits(&kv.v, (uint64_t)cache, 16))
        return no(GH_E_RANGE, "cache too small or not on 16 bytes");
    if (!fits(&p->table, (uint64_t)p->rows * p->table_width * 4, 4) || !fits(&p->lengths, (uint64_t)p->rows * 4, 4))
        return no(GH_E_RANGE, "table or lengths too small");
    if (p->score.addr && !fits(&p->score, (uint64_t)score, 16))
        return no(GH_E_RANGE, "scores too small or not on 16 bytes");
    // the workgroups of a launch read lengths and pages each for itself, while others write
    const Parts own(p);
    for (int i = 0; i < PARTS; ++i)
        for (int j = 0; j < i; ++j)
            if (meet(own.part[i], own.part[j])) return no(GH_E_INVALID, "the handle's buffers overlap");
    return GH_OK;
}

GhPages pages(gh_backend* b, const gh_kv_paged* p, uint32_t layer) {
    const gh_kv& kv = p->kv;
    const uint64_t at = (uint64_t)layer * kv.context * kv.kv_heads * 256;
    GhPages g{};
    g.kc = kv.k.addr + at;
    g.vc = kv.v.addr + at;
    g.table = p->table.addr;
    g.lengths = p->lengths.addr;
    g.score = p->score.addr ? p->score.addr + (uint64_t)layer * p->rows * kv.kv_heads * capacity(p) * 4 : 0;
    g.fault = (uint64_t)b->paged_fault;
    g.width = p->table_width;
    g.shift = (uint32_t)__builtin_ctz(p->page_size);
    g.pages = kv.context / p->page_size;
    g.kv_heads = kv.kv_heads;
    return g;
}

// The calls allocate scratch and a rotation table: on the backend's device, whatever the thread's is.
struct OnDevice {
    int before = 0;
    bool moved = false;
    explicit OnDevice(const gh_backend* b) {
        moved = hipGetDevice(&before) == hipSuccess && before != b->device && hipSetDevice(b->device) == hipSuccess;
    }
    ~OnDevice() {
        if (moved) (void)hipSetDevice(before);
    }
};

// An entry point's body: the encoder checked, errors latched, no exception let out.
template <class F>
int entry(gh_backend* b, gh_encoder* enc, F body) {
    int rc = check_enc(b, enc);
    if (rc) return rc;
    try {
        OnDevice on(b);
        rc = body();
    } catch (const std::bad_alloc&) {
        rc = GH_E_OOM;
    } catch (...) {
        rc = GH_E_INVALID;
    }
    return latch(enc, rc);
}

// `bytes` of the workspace. It grows by half (at most 64 MiB) more than asked where there is memory for that: sizes
// that follow the longest row rise every 16 tokens, and a growth waits for the stream and moves what recorded graphs hold.
int scratch(gh_backend* b, uint64_t bytes, char** at) {
    auto ask = [&](uint64_t n) {
        const bool grows = n > workspace_room(b);
        const int rc = workspace_at(b, n, at);
        if (rc == GH_E_OOM) b->ws_short = b->ws_short ? std::min(b->ws_short, n) : n;
        else if (!rc && grows && n >= b->ws_short) b->ws_short = 0;
        return rc;
    };
    const uint64_t more = bytes + std::min<uint64_t>(bytes / 2, 64ull << 20);
    if (bytes > workspace_room(b) && (!b->ws_short || more < b->ws_short)) {
        const int rc = ask(more);
        if (rc != GH_E_OOM) return rc;
        b->err.clear();
    }
    return ask(bytes);
}

int write(gh_backend* b, const gh_kv_paged* kv, const gh_buf* k, const gh_buf* v, uint32_t tokens, uint32_t layer,
          GhPagedWriteArgs a, const char* what) {
    const uint64_t n = (uint64_t)kv->rows * tokens, bytes = n * kv->kv.kv_heads * 256;
    if (tokens == 0 || n > 0x7FFFFFFFull) return fail(b, GH_E_INVALID, std::string(what) + ": tokens");
    if (!fits(k, bytes, 16) || !fits(v, bytes, 16))
        return fail(b, GH_E_RANGE, std::string(what) + ": vectors too small or not on 16 bytes");
    const Span score = Parts(kv).part[SCORE];
    if (meet(score, {k->addr, bytes}) || meet(score, {v->addr, bytes}))
        return fail(b, GH_E_INVALID, std::string(what) + ": k or v overlaps the scores");
    a.p = pages(b, kv, layer);
    a.k = k->addr;
    a.v = v->addr;
    a.tokens = tokens;
    a.groups = ceil_div((uint64_t)(a.q_heads + 2 * kv->kv.kv_heads) * 16, 256);
    if (n * a.groups > 0xFFFFFFull) return fail(b, GH_E_RANGE, std::string(what) + ": too many vectors");
    return launch(b, K_PAGED_WRITE, (uint32_t)(n * a.groups), 1, 1, 256, &a);
}

int attention(gh_backend* b, const gh_buf* out, const gh_buf* q, const gh_kv_paged* kv, uint32_t q_heads,
              uint32_t max_len, uint32_t layer) {
    const uint32_t hk = kv->kv.kv_heads;
    if (q_heads == 0 || q_heads % hk) return fail(b, GH_E_INVALID, "attention_decode_paged: q_heads not a multiple of kv_heads");
    const uint32_t group = q_heads / hk;
    if (q_heads > 0xFFFFu) return fail(b, GH_E_UNSUPPORTED, "attention_decode_paged: more than 65535 heads");
    if (group > 16) return fail(b, GH_E_UNSUPPORTED, "attention_decode_paged: at most 16 query heads per kv head");
    const uint64_t bytes = (uint64_t)kv->rows * q_heads * 256;
    if (!fits(q, bytes, 16) || !fits(out, bytes, 16))
        return fail(b, GH_E_RANGE, "attention_decode_paged: buffer too small or not on 16 bytes");
    if (out->addr != q->addr && meet(out, bytes, q, bytes)) return fail(b, GH_E_INVALID, "attention_decode_paged: out overlaps q");
    const Parts own(kv);
    if (own.met({out->addr, bytes}) || meet(own.part[SCORE], {q->addr, bytes}))
        return fail(b, GH_E_INVALID, "attention_decode_paged: out overlaps a buffer of the handle, or q its scores");
    if (max_len > capacity(kv)) return fail(b, GH_E_RANGE, "attention_decode_paged: max_len beyond the table");
    if (max_len == 0) max_len = (uint32_t)capacity(kv);

    GhPagedAttnArgs a{};
    a.p = pages(b, kv, layer);
    a.q_heads = q_heads;
    a.group = group;
    a.max_len = max_len;
    a.scale = 1.4426950408889634f / std::sqrt(128.0f);
    const bool scored = kv->score.addr != 0;
    a.raw_len = (max_len + 15) / 16 * 16;
    a.blocks = scored ? std::min(ceil_div(max_len, 1024), 64u) : 0;
    // Tiles of 16 positions and kv heads (8 KiB of K and V) that the rows can hold. Rows of one span, or few
    // tiles in all: each row by itself in fixed spans (gh_paged_split), which start sooner (no row needs the
    // others' lengths) and need no join where a row has one span; else all rows together in equal chunks
    // (gh_paged_attn), which balances ragged rows. us back to back, spans / chunks: 1 row of 500 9.4 / 11.9, 3 of
    // 3000 14.0 / 15.4, 256 of up to 300 40.4 / 48.0, 12 of up to 1000 15.2 / 14.4, 64 of up to 600 28.5 / 22.9, 8 of
    // up to 8192 45.9 / 33.4, 32 of up to 4000 69.3 / 52.0.
    const uint32_t tiles1 = ceil_div(max_len, 16);
    const uint64_t most = (uint64_t)kv->rows * hk * tiles1;
    const bool split = tiles1 <= kSpanTiles || most < 6144;
    if (split) {
        // about two workgroups per CU, each wave at most 8 tiles (1 row of 9000, in spans of 4 / 12 / 32 / 64 tiles:
        // 16.5 / 14.3 / 16.7 / 23.8 us)
        a.least = std::min(std::max(ceil_div(most, 8ull * b->cus) * 4, 4u), kSpanTiles);
        a.chunks = ceil_div(tiles1, a.least);
    } else {
        // eight waves per CU, all of them at once: with more, the rows' streams disturb each other (64 rows of
        // 8192 with 4 / 6 / 8 / 10 / 12 waves per CU: 389 / 376 / 324 / 378 / 342 us). Half of them where that
        // gives a wave at most 12 tiles: a second workgroup on some CUs would only make those the last
        // (16 rows of up to 2500: 29.2 / 26.5 us).
        a.least = 4;
        a.chunks = std::max(1u, 8 * b->cus / hk);
        a.solo = 12;
    }
    // From half the last-level cache on, the next call will not find this one's K and V there, and reads past
    // it are faster (64 rows of 8192 362 / 324 us, 1 of 32768 33.8 / 31.6; 16 of up to 2500, 83 MB: 26.2 / 32.3).
    a.stream = kStreamBytes;
    // scratch of a row: its partials, and with scores each query head's
    const uint64_t acc = (uint64_t)q_heads * 512, ml = acc / 64, raw = scored ? (uint64_t)q_heads * a.raw_len * 4 : 0;
    // rows in groups that the kernel lays out at once and whose scratch fits 512 MiB, or what memory there is
    const uint64_t per = (acc + ml) * (split ? a.chunks : 1) + raw, layout = (kPagedRows + 4) * 4;
    const uint64_t room = std::min<uint64_t>((512ull << 20) / per, (1u << 30) / tiles1);  // tiles count in 32 bits
    uint32_t step = (uint32_t)std::min<uint64_t>(std::min(kv->rows, kPagedRows), std::max<uint64_t>(1, room));
    auto parts = [&] { return split ? (uint64_t)a.chunks * step : (uint64_t)a.chunks + step; };
    auto need = [&] { return layout + (acc + ml) * parts() + raw * step; };
    // Where memory was short (ws_short), the scratch that there is holds half or more of what could be had then, and rows take
    // turns in it: a refusal costs two allocations, two frees and a wait. Every 256th such call asks for all again, as others
    // may have freed memory. Where it holds not one row, as many are tried as were not refused.
    if (b->ws_short && need() > workspace_room(b)) {
        const uint64_t fixed = layout + (split ? 0 : (acc + ml) * a.chunks);
        auto rows_in = [&](uint64_t bytes) { return bytes > fixed ? (uint32_t)std::min<uint64_t>((bytes - fixed) / per, step) : 0; };
        const uint32_t now = rows_in(workspace_room(b)), untried = rows_in(b->ws_short - 1);
        if (++b->ws_did_with_less % 256 == 0) b->ws_short = 0;
        else if (now || untried) step = now ? now : untried;
    }
    char* ws = nullptr;
    int rc = GH_OK;
    while ((rc = scratch(b, need(), &ws)) == GH_E_OOM && step > 1) {
        step = (step + 1) / 2;
        b->err.clear();
    }
    if (rc) return b->ws_short = 0, rc;
    a.layout = split ? 0 : (uint64_t)ws;
    a.part_acc = (uint64_t)ws + layout;
    a.raw = scored ? a.part_acc + acc * parts() : 0;
    a.part_ml = a.part_acc + acc * parts() + raw * step;
    const GhPages p0 = a.p;
    for (uint32_t r = 0; r < kv->rows; r += step) {
        a.rows = std::min(step, kv->rows - r);
        a.p.table = p0.table + (uint64_t)r * p0.width * 4;
        a.p.lengths = p0.lengths + (uint64_t)r * 4;
        a.p.score = scored ? p0.score + (uint64_t)r * hk * capacity(kv) * 4 : 0;
        a.q = q->addr + (uint64_t)r * q_heads * 256;
        a.out = out->addr + (uint64_t)r * q_heads * 256;
        if (split) {
            rc = launch(b, scored ? K_PAGED_SPLIT_S : K_PAGED_SPLIT, hk, a.chunks, a.rows, 256, &a, 4 * group * 134 * 4);
        } else {
            // no more chunks than the rows' tiles can fill
            const uint64_t chunks = std::min<uint64_t>(a.chunks, ceil_div((uint64_t)a.rows * tiles1, a.least));
            rc = launch(b, scored ? K_PAGED_ATTN_S : K_PAGED_ATTN, ceil_div(hk * chunks, 4), 1, 1, 256, &a);
        }
        // the halves of the heads apart where a row may have more partials than one round of the join takes (64)
        const uint32_t halves = a.chunks > 64 * a.rows ? 2 : 1;
        if (!rc && (!split || a.chunks > 1))
            rc = launch(b, halves == 2 ? K_PAGED_JOIN2 : K_PAGED_JOIN, q_heads + hk * a.blocks, a.rows, halves, 256, &a);
        if (rc) return rc;
    }
    return GH_OK;
}

int evict(gh_backend* b, const gh_kv_paged* dst, const gh_kv_paged* src, const gh_buf* kept, uint32_t budget,
          uint32_t recent) {
    const gh_kv &s = src->kv, &d = dst->kv;
    if (d.block_count != s.block_count || d.kv_heads != s.kv_heads || dst->page_size != src->page_size || dst->rows != src->rows)
        return fail(b, GH_E_INVALID, "kv_evict_paged: dst and src differ in rows, page_size, block_count or heads");
    if (!src->score.addr || !dst->score.addr) return fail(b, GH_E_INVALID, "kv_evict_paged: no scores kept");
    if (budget == 0 || recent > budget) return fail(b, GH_E_INVALID, "kv_evict_paged: recent > budget, or budget 0");
    if (budget > capacity(dst)) return fail(b, GH_E_RANGE, "kv_evict_paged: budget beyond dst's table");
    if (budget > (1u << 27)) return fail(b, GH_E_UNSUPPORTED, "kv_evict_paged: budget beyond 2^27");
    if (s.block_count > 0xFFFFu) return fail(b, GH_E_UNSUPPORTED, "kv_evict_paged: more than 65535 layers");
    const uint64_t list = (uint64_t)s.block_count * src->rows * s.kv_heads;
    if (list > (1ull << 40)) return fail(b, GH_E_RANGE, "kv_evict_paged: too many rows");
    if (kept && !fits(kept, list * budget * 4, 4)) return fail(b, GH_E_RANGE, "kv_evict_paged: kept too small");
    // Workgroups read while others write, and the kept positions are indexes of src's table when they are read again:
    // what is written lies in nothing that is read but its own counterpart.
    const Parts from(src), to(dst);
    const bool same = dst->score.addr == src->score.addr;
    if (same ? dst->table_width != src->table_width : meet(to.part[SCORE], from.part[SCORE]))
        return fail(b, GH_E_INVALID, "kv_evict_paged: scores overlap");
    if (dst->lengths.addr != src->lengths.addr && meet(to.part[LENGTHS], from.part[LENGTHS]))
        return fail(b, GH_E_INVALID, "kv_evict_paged: lengths overlap");
    if (kept && (from.met({kept->addr, list * budget * 4}) || to.met({kept->addr, list * budget * 4})))
        return fail(b, GH_E_INVALID, "kv_evict_paged: kept overlaps a cache, table, lengths or scores");
    for (int w = 0; w < TABLE; ++w)
        for (int r = 0; r < PARTS; ++r)
            if (w != r && meet(to.part[w], from.part[r]))
                return fail(b, GH_E_INVALID, "kv_evict_paged: a buffer of dst overlaps another one of src");
    if (to.part[TABLE].at == from.part[TABLE].at && to.part[CACHE_K].at == from.part[CACHE_K].at)
        return fail(b, GH_E_INVALID, "kv_evict_paged: dst has src's pages");
    GhPagedEvictArgs a{};
    a.src = pages(b, src, 0);
    a.dst = pages(b, dst, 0);
    a.src_layer = (uint64_t)s.context * s.kv_heads * 256;
    a.dst_layer = (uint64_t)d.context * d.kv_heads * 256;
    a.rows = src->rows;
    a.budget = budget;
    a.recent = recent;
    char* ws = nullptr;
    int rc = scratch(b, (uint64_t)src->rows * 4 + (kept ? 0 : list * budget * 4), &ws);
    if (rc) return b->ws_short = 0, rc;
    a.act = (uint64_t)ws;
    a.kept = kept ? kept->addr : (uint64_t)ws + (uint64_t)src->rows * 4;
    rc = launch(b, K_PAGED_SELECT, s.kv_heads, src->rows, s.block_count, 512, &a);
    const bool stream = list * budget * 512 >= kStreamBytes;
    if (!rc) rc = launch(b, stream ? K_PAGED_MOVE_S : K_PAGED_MOVE, ceil_div(budget, 16), src->rows, s.block_count, 256, &a);
    return rc;
}

}  // namespace

extern "C" {

int gh_kv_write_paged(gh_backend* b, gh_encoder* enc, const gh_kv_paged* kv, const gh_buf* k, const gh_buf* v,
                      uint32_t tokens, uint32_t layer) {
    return entry(b, enc, [&] {
        const int rc = check_paged(b, kv, layer, "kv_write_paged");
        return rc ? rc : write(b, kv, k, v, tokens, layer, GhPagedWriteArgs{}, "kv_write_paged");
    });
}

int gh_rope_kv_write_paged(gh_backend* b, gh_encoder* enc, const gh_kv_paged* kv, const gh_buf* q_out,
                           const gh_buf* q, const gh_buf* k, const gh_buf* v, uint32_t q_heads,
                           const gh_buf* positions, uint32_t tokens, uint32_t max_pos, const gh_yarn* yarn,
                           uint32_t layer) {
    return entry(b, enc, [&] {
        const char* what = "rope_kv_write_paged";
        int rc = check_paged(b, kv, layer, what);
        if (rc) return rc;
        if (!yarn_valid(yarn) || yarn->rope_dim > 128) return fail(b, GH_E_INVALID, "rope_kv_write_paged: invalid YaRN parameters");
        if (max_pos >= kMaxRopePositions) return fail(b, GH_E_RANGE, "rope_kv_write_paged: position beyond the table limit");
        if (q_heads == 0 || q_heads > 0xFFFFFu) return fail(b, GH_E_INVALID, "rope_kv_write_paged: q_heads");
        const uint64_t bytes = (uint64_t)kv->rows * tokens * q_heads * 256;
        if (!fits(q, bytes, 16) || !fits(q_out, bytes, 16) || !fits(positions, (uint64_t)kv->rows * 4, 4))
            return fail(b, GH_E_RANGE, "rope_kv_write_paged: buffer too small or not on 16 bytes");
        if (q->addr != q_out->addr && meet(q, bytes, q_out, bytes))
            return fail(b, GH_E_INVALID, "rope_kv_write_paged: q_out overlaps q");
        const uint64_t heads = bytes / q_heads * kv->kv.kv_heads;
        if ((k && meet(q_out, bytes, k, heads)) || (v && meet(q_out, bytes, v, heads)))
            return fail(b, GH_E_INVALID, "rope_kv_write_paged: q_out overlaps k or v");
        const Parts own(kv);
        const Span turned{q_out->addr, bytes}, at{positions->addr, (uint64_t)kv->rows * 4};
        if (own.met(turned) || meet(turned, at) || meet(own.part[SCORE], {q->addr, bytes}))
            return fail(b, GH_E_INVALID, "rope_kv_write_paged: q_out overlaps a buffer of the handle or positions, or q its scores");
        if (meet(at, own.part[CACHE_K]) || meet(at, own.part[CACHE_V]) || meet(at, own.part[SCORE]))
            return fail(b, GH_E_INVALID, "rope_kv_write_paged: positions overlap the caches or the scores");
        rc = ensure_rope(b, b->rope, yarn, max_pos + 1);
        if (rc) return rc;
        GhPagedWriteArgs a{};
        a.q = q->addr;
        a.q_out = q_out->addr;
        a.q_heads = q_heads;
        a.positions = positions->addr;
        a.table = (uint64_t)b->rope.table;
        a.post = (uint64_t)b->rope.post;
        a.pairs = yarn->rope_dim / 2;
        a.max_pos = max_pos;
        return write(b, kv, k, v, tokens, layer, a, what);
    });
}

int gh_attention_decode_paged(gh_backend* b, gh_encoder* enc, const gh_buf* out, const gh_buf* q,
                              const gh_kv_paged* kv, uint32_t q_heads, uint32_t max_len, uint32_t layer) {
    return entry(b, enc, [&] {
        const int rc = check_paged(b, kv, layer, "attention_decode_paged");
        return rc ? rc : attention(b, out, q, kv, q_heads, max_len, layer);
    });
}

int gh_kv_evict_paged(gh_backend* b, gh_encoder* enc, const gh_kv_paged* dst, const gh_kv_paged* src,
                      const gh_buf* kept, uint32_t budget, uint32_t recent) {
    return entry(b, enc, [&] {
        int rc = check_paged(b, src, 0, "kv_evict_paged");
        if (!rc) rc = check_paged(b, dst, 0, "kv_evict_paged");
        return rc ? rc : evict(b, dst, src, kept, budget, recent);
    });
}

}  // extern "C"
