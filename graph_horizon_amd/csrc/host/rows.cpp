// Operators over rows of a batch that are not over its cache: norms of query and key heads with RoPE, and sampling. Checks,
// launch plans and scratch; the kernels are in kernels/glue.hip and kernels/sample.hip.
#include <cmath>

#include "internal.h"

using namespace gh;

namespace {

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

bool fits(const gh_buf* buf, uint64_t bytes) { return buf && buf->addr && buf->bytes >= bytes; }

// the bytes at a and b overlap
bool meet(const gh_buf* a, uint64_t a_bytes, const gh_buf* b, uint64_t b_bytes) {
    return a_bytes && b_bytes && a->addr < b->addr + b_bytes && b->addr < a->addr + a_bytes;
}

constexpr uint64_t kSampleScratch = 128ull << 20;
constexpr uint32_t kOneWord = 1u << 17;  // tokens whose weights' sums one word holds to 2^-29

}  // namespace

extern "C" {

int gh_norm_rope_batched(gh_backend* b, gh_encoder* enc, const gh_buf* q, const gh_buf* k,
                         uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t base,
                         uint32_t rows, const gh_buf* q_norm, const gh_buf* k_norm, float eps,
                         const gh_yarn* yarn) {
    return entry(b, enc, [&] {
        auto no = [&](int code, const char* why) { return fail(b, code, std::string("norm_rope_batched: ") + why); };
        if (rows == 0) return no(GH_E_INVALID, "empty batch");
        if (head_dim == 0 || head_dim % 8 || head_dim > 512) return no(GH_E_UNSUPPORTED, "head_dim must be a multiple of 8 up to 512");
        if (q_heads > 0xFFFFu || kv_heads > 0xFFFFu) return no(GH_E_UNSUPPORTED, "more than 65535 heads");
        if (!yarn_valid(yarn) || yarn->rope_dim > head_dim) return no(GH_E_INVALID, "invalid YaRN parameters");
        if (!(eps >= 0.0f) || std::isinf(eps)) return no(GH_E_INVALID, "eps");
        if ((uint64_t)base + rows > 0xFFFFFFFFull) return no(GH_E_RANGE, "position overflow");
        const uint64_t wb = (uint64_t)head_dim * 2, qb = (uint64_t)rows * q_heads * wb, kb = (uint64_t)rows * kv_heads * wb;
        if (!fits(q, qb) || !fits(k, kb) || !fits(q_norm, wb) || !fits(k_norm, wb)) return no(GH_E_RANGE, "buffer too small");
        if ((q->addr | k->addr | q_norm->addr | k_norm->addr) % 16) return no(GH_E_RANGE, "buffer not on 16 bytes");
        if (meet(q, qb, k, kb)) return no(GH_E_INVALID, "q overlaps k");
        for (const gh_buf* w : {q_norm, k_norm})
            if (meet(q, qb, w, wb) || meet(k, kb, w, wb)) return no(GH_E_INVALID, "q or k overlaps the weights");
        GhNormRopeArgs a{};
        while (8u << a.shift < head_dim) ++a.shift;
        a.share = 1.0f / (float)head_dim;
        a.groups = ceil_div((uint64_t)(q_heads + kv_heads) << a.shift, 256);
        if ((uint64_t)rows * a.groups > 0xFFFFFFull) return no(GH_E_RANGE, "too many vectors");
        const int rc = ensure_rope(b, b->rope, yarn, base + rows);
        if (rc || a.groups == 0) return rc;
        a.q = q->addr;
        a.k = k->addr;
        a.q_norm = q_norm->addr;
        a.k_norm = k_norm->addr;
        a.table = (uint64_t)b->rope.table;
        a.post = (uint64_t)b->rope.post;
        a.heads = q_heads;
        a.kheads = kv_heads;
        a.head_dim = head_dim;
        a.pairs = yarn->rope_dim / 2;
        a.base = base;
        a.rows = rows;
        a.eps = norm_eps(eps);
        return launch(b, K_NORM_ROPE, rows * a.groups, 1, 1, 256, &a);
    });
}

int gh_sample_rows(gh_backend* b, gh_encoder* enc, const gh_buf* tokens, const gh_buf* probs, const gh_buf* logits,
                   uint32_t rows, uint32_t vocab, uint32_t stride, const gh_buf* params, const gh_buf* uniform) {
    return entry(b, enc, [&] {
        auto no = [&](int code, const char* why) { return fail(b, code, std::string("sample_rows: ") + why); };
        if (rows == 0 || rows > 0xFFFFu) return no(GH_E_INVALID, "1 to 65535 rows");
        if (vocab == 0 || stride < vocab) return no(GH_E_INVALID, "vocab, or stride below it");
        if (vocab > (1u << 24)) return no(GH_E_UNSUPPORTED, "more than 2^24 tokens");
        const uint64_t lb = ((uint64_t)(rows - 1) * stride + vocab) * 4, tb = (uint64_t)rows * 4;
        if (!fits(tokens, tb) || (probs && !fits(probs, tb)) || !fits(logits, lb) || !fits(params, 4 * tb) || !fits(uniform, tb))
            return no(GH_E_RANGE, "buffer too small");
        if ((tokens->addr | (probs ? probs->addr : 0) | logits->addr | uniform->addr) % 4 || params->addr % 16)
            return no(GH_E_RANGE, "params not on 16 bytes, or another buffer not on 4");
        for (const gh_buf* out : {tokens, probs})
            if (out && (meet(out, tb, logits, lb) || meet(out, tb, params, 4 * tb) || meet(out, tb, uniform, tb)))
                return no(GH_E_INVALID, "tokens or probs overlap an input");
        if (probs && meet(tokens, tb, probs, tb)) return no(GH_E_INVALID, "tokens overlap probs");
        GhSampleArgs a{};
        a.vocab = vocab;
        a.stride = stride;
        a.wide = logits->addr % 16 == 0 && stride % 4 == 0;
        a.scale = 1.0;
        for (a.shift = 0; a.shift < 51 && a.scale * 2 * vocab <= 0x1p62; ++a.shift) a.scale *= 2;
        // Bins without a second word lie closer: 12304 bytes apart, not 16400, whose rows' same bins share memory channels (bins and pick of
        // 8 rows 10.2 and 13.5 us, instead of 6.9 and 12.4).
        a.bin_bytes = GH_SAMPLE_BIN_BYTES - 4 * GH_SAMPLE_BINS;
        // past kOneWord tokens a second word holds a count up to vocab and, above it, further parts of all tokens but the largest,
        // each up to 2^fine
        if (vocab > kOneWord) {
            a.bin_bytes = GH_SAMPLE_BIN_BYTES;
            for (a.count_bits = 1; vocab >> a.count_bits; ++a.count_bits) {}
            for (a.fine = 0; a.fine < 40 && ((uint64_t)(vocab - 1) << (a.fine + 1)) >> (64 - a.count_bits) == 0; ++a.fine) {}
        }
        uint32_t step = std::min<uint32_t>(rows, kSampleScratch / GH_SAMPLE_ROW_BYTES);
        char* ws = nullptr;
        int rc = scratch_for_rows(b, 0, GH_SAMPLE_ROW_BYTES, &step, &ws);
        if (rc) return rc;
        // about four workgroups per CU; a chunk is a whole number of a workgroup's rounds of 2048
        const uint32_t rounds = ceil_div(vocab, 2048);
        a.chunks = std::min({std::max(1u, 4 * b->cus / step), rounds, 64u});
        a.per = ceil_div(rounds, a.chunks) * 2048;
        a.chunks = ceil_div(vocab, a.per);
        a.part = (uint64_t)ws;
        a.list = a.part + (uint64_t)step * 64 * 16;
        a.bins = a.list + (uint64_t)step * GH_SAMPLE_LIST * 8;
        for (uint32_t r = 0; r < rows; r += step) {
            const uint32_t n = std::min(step, rows - r);
            a.logits = logits->addr + (uint64_t)r * stride * 4;
            a.params = params->addr + (uint64_t)r * 16;
            a.uniform = uniform->addr + (uint64_t)r * 4;
            a.tokens = tokens->addr + (uint64_t)r * 4;
            a.probs = probs ? probs->addr + (uint64_t)r * 4 : 0;
            rc = launch(b, K_SAMPLE_MAX, a.chunks, n, 1, 256, &a);
            if (!rc) rc = launch(b, K_SAMPLE_BINS, a.chunks, n, 1, 256, &a);
            if (!rc) rc = launch(b, K_SAMPLE_COLLECT, a.chunks, n, 1, 256, &a);
            if (!rc) rc = launch(b, K_SAMPLE_PICK, n, 1, 1, GH_SAMPLE_PICK, &a);
            if (rc) return rc;
        }
        return rc;
    });
}

}  // extern "C"
