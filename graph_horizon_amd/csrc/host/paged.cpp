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

bool overlap(const gh_buf& a, const gh_buf& b) { return a.addr < b.addr + b.bytes && b.addr < a.addr + a.bytes; }

uint64_t capacity(const gh_kv_paged* kv) { return (uint64_t)kv->table_width * kv->page_size; }

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

int write(gh_backend* b, const gh_kv_paged* kv, const gh_buf* k, const gh_buf* v, uint32_t tokens, uint32_t layer,
          GhPagedWriteArgs a, const char* what) {
    const uint64_t n = (uint64_t)kv->rows * tokens, bytes = n * kv->kv.kv_heads * 256;
    if (tokens == 0 || n > 0x7FFFFFFFull) return fail(b, GH_E_INVALID, std::string(what) + ": tokens");
    if (!fits(k, bytes, 16) || !fits(v, bytes, 16))
        return fail(b, GH_E_RANGE, std::string(what) + ": vectors too small or not on 16 bytes");
    a.p = pages(b, kv, layer);
    a.k = k->addr;
    a.v = v->addr;
    a.tokens = tokens;
    a.groups = ceil_div((uint64_t)(a.q_heads + 2 * kv->kv.kv_heads) * 16, 256);
    if (n * a.groups > 0x7FFFFFFFull) return fail(b, GH_E_RANGE, std::string(what) + ": too many vectors");
    return launch(b, K_PAGED_WRITE, (uint32_t)(n * a.groups), 1, 1, 256, &a);
}

// Positions per split: small enough that `rows` full rows give every CU four workgroups and that a long
// row among short ones is spread over many, large enough that the partials (520 bytes per query head and
// split) stay small beside the span's K and V (512 bytes per position).
uint32_t span_of(const gh_backend* b, uint64_t rows, uint32_t kv_heads, uint32_t max_len) {
    const uint64_t pairs = rows * kv_heads;
    const uint64_t want = std::max<uint64_t>(1, ceil_div(4ull * b->cus, pairs));
    uint64_t span = (ceil_div(max_len, want) + 63) / 64 * 64;
    span = std::min<uint64_t>(std::max<uint64_t>(span, 64), 1024);
    if (ceil_div(max_len, span) > 0xFFFFu) span = 4096;  // the grid's y
    return (uint32_t)span;
}

int attention(gh_backend* b, const gh_buf* out, const gh_buf* q, const gh_kv_paged* kv, uint32_t q_heads,
              uint32_t max_len, uint32_t layer) {
    const uint32_t hk = kv->kv.kv_heads;
    if (q_heads == 0 || q_heads % hk) return fail(b, GH_E_INVALID, "attention_decode_paged: q_heads not a multiple of kv_heads");
    const uint32_t group = q_heads / hk;
    if (group > 16) return fail(b, GH_E_UNSUPPORTED, "attention_decode_paged: at most 16 query heads per kv head");
    const uint64_t bytes = (uint64_t)kv->rows * q_heads * 256;
    if (!fits(q, bytes, 16) || !fits(out, bytes, 16))
        return fail(b, GH_E_RANGE, "attention_decode_paged: buffer too small or not on 16 bytes");
    if (max_len > capacity(kv)) return fail(b, GH_E_RANGE, "attention_decode_paged: max_len beyond the table");
    if (max_len == 0) max_len = (uint32_t)capacity(kv);

    GhPagedAttnArgs a{};
    a.p = pages(b, kv, layer);
    a.q_heads = q_heads;
    a.group = group;
    a.max_len = max_len;
    a.span = span_of(b, kv->rows, hk, max_len);
    a.splits = ceil_div(max_len, a.span);
    if (a.splits > 0xFFFFu) return fail(b, GH_E_UNSUPPORTED, "attention_decode_paged: max_len beyond 2^28");
    a.scale = 1.4426950408889634f / std::sqrt(128.0f);
    const bool scored = kv->score.addr != 0;
    a.raw_len = (max_len + 15) / 16 * 16;
    a.chunks = scored ? std::min(ceil_div(max_len, 1024), 64u) : 0;
    const bool parts = scored || a.splits > 1;
    // scratch of a row: the splits' sums, and with scores each query head's
    const uint64_t acc = parts ? (uint64_t)q_heads * a.splits * 512 : 0, ml = acc / 64;
    const uint64_t raw = scored ? (uint64_t)q_heads * a.raw_len * 4 : 0, per = acc + ml + raw;
    // rows in groups whose scratch fits 512 MiB
    const uint32_t step = per ? (uint32_t)std::min<uint64_t>(kv->rows, std::max<uint64_t>(1, (512ull << 20) / per)) : kv->rows;
    char* ws = nullptr;
    if (per) {
        const int rc = workspace_at(b, per * step, &ws);
        if (rc) return rc;
    }
    const GhKernel first = group <= 4 ? K_PAGED_ATTN_G4 : group <= 8 ? K_PAGED_ATTN_G8 : K_PAGED_ATTN_G16;
    const GhPages p0 = a.p;
    for (uint32_t r = 0; r < kv->rows; r += step) {
        const uint32_t rows = std::min(step, kv->rows - r);
        a.p.table = p0.table + (uint64_t)r * p0.width * 4;
        a.p.lengths = p0.lengths + (uint64_t)r * 4;
        a.p.score = scored ? p0.score + (uint64_t)r * hk * capacity(kv) * 4 : 0;
        a.q = q->addr + (uint64_t)r * q_heads * 256;
        a.out = out->addr + (uint64_t)r * q_heads * 256;
        a.part_acc = (uint64_t)ws;
        a.raw = scored ? (uint64_t)ws + acc * step : 0;
        a.part_ml = (uint64_t)ws + (acc + raw) * step;
        int rc = launch(b, (GhKernel)(first + (scored ? 1 : 0)), hk, a.splits, rows, 256, &a);
        if (!rc && parts) rc = launch(b, K_PAGED_JOIN, q_heads + hk * a.chunks, 1, rows, 256, &a);
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
    if (s.block_count > 0xFFFFu) return fail(b, GH_E_UNSUPPORTED, "kv_evict_paged: more than 65535 layers");
    const bool same = dst->score.addr == src->score.addr;
    if (same ? dst->table_width != src->table_width : overlap(dst->score, src->score))
        return fail(b, GH_E_INVALID, "kv_evict_paged: scores overlap");
    if (dst->lengths.addr != src->lengths.addr && overlap(dst->lengths, src->lengths))
        return fail(b, GH_E_INVALID, "kv_evict_paged: lengths overlap");
    const uint64_t list = (uint64_t)s.block_count * src->rows * s.kv_heads;
    if (list > (1ull << 40)) return fail(b, GH_E_RANGE, "kv_evict_paged: too many rows");
    if (kept && !fits(kept, list * budget * 4, 4)) return fail(b, GH_E_RANGE, "kv_evict_paged: kept too small");
    GhPagedEvictArgs a{};
    a.src = pages(b, src, 0);
    a.dst = pages(b, dst, 0);
    a.src_layer = (uint64_t)s.context * s.kv_heads * 256;
    a.dst_layer = (uint64_t)d.context * d.kv_heads * 256;
    a.rows = src->rows;
    a.budget = budget;
    a.recent = recent;
    char* ws = nullptr;
    int rc = workspace_at(b, (uint64_t)src->rows * 4 + (kept ? 0 : list * budget * 4), &ws);
    if (rc) return rc;
    a.act = (uint64_t)ws;
    a.kept = kept ? kept->addr : (uint64_t)ws + (uint64_t)src->rows * 4;
    rc = launch(b, K_PAGED_SELECT, s.kv_heads, src->rows, s.block_count, 512, &a);
    if (!rc) rc = launch(b, K_PAGED_MOVE, ceil_div(budget, 16), src->rows, s.block_count, 256, &a);
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
        const gh_buf in{q->addr, bytes, 0, 0, 0, 0}, to{q_out->addr, bytes, 0, 0, 0, 0};
        if (q->addr != q_out->addr && overlap(in, to)) return fail(b, GH_E_INVALID, "rope_kv_write_paged: q_out overlaps q");
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
