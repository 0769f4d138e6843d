// The host's checks and launch plans of the operators over 4-bit pools, norms and sampling, without a device: host/paged.cpp
// and host/rows.cpp with launches recorded instead of made and scratch handed out as an address range.
#include <algorithm>

#include "../graph_horizon_amd/csrc/host/internal.h"

namespace {
struct Launch {
    uint32_t kernel, gx, gy, gz, block;
    unsigned char args[512];
};
std::vector<Launch> launches;
uint64_t scratch_bytes = 0, scratch_limit = 0;
size_t args_size(GhKernel k) {
    switch (k) {
        case K_NORM_ROPE: return sizeof(GhNormRopeArgs);
        case K_SAMPLE_MAX: case K_SAMPLE_BINS: case K_SAMPLE_COLLECT: case K_SAMPLE_PICK: return sizeof(GhSampleArgs);
        case K_PAGED_READ: case K_PAGED4_READ: return sizeof(GhPagedReadArgs);
        case K_PAGED_WRITE: case K_PAGED_NORM_WRITE: case K_PAGED4_WRITE: case K_PAGED4_NORM_WRITE: return sizeof(GhPagedWriteArgs);
        case K_PAGED_SELECT: case K_PAGED_MOVE: case K_PAGED_MOVE_S: case K_PAGED4_MOVE: return sizeof(GhPagedEvictArgs);
        default: return sizeof(GhPagedAttnArgs);
    }
}
}  // namespace

extern "C" hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }

namespace gh {
int fail(gh_backend* b, int code, const std::string& msg) { return b->err = msg, code; }
int check_enc(gh_backend* b, gh_encoder* enc) { return b && enc == &b->enc ? GH_OK : GH_E_STATE; }
int latch(gh_encoder* enc, int rc) { return rc && !enc->latched ? enc->latched = rc : rc; }
int launch(gh_backend*, GhKernel k, uint32_t gx, uint32_t gy, uint32_t gz, uint32_t bx, const void* args, uint32_t) {
    Launch l{(uint32_t)k, gx, gy, gz, bx, {}};
    std::memcpy(l.args, args, args_size(k));
    launches.push_back(l);
    return GH_OK;
}
int workspace_at(gh_backend* b, size_t bytes, char** at) {
    if (scratch_limit && bytes > scratch_limit) return fail(b, GH_E_OOM, "scratch");
    scratch_bytes = bytes;
    *at = (char*)(1ull << 50);
    return GH_OK;
}
bool yarn_valid(const gh_yarn* y) { return y && y->rope_dim && y->rope_dim % 2 == 0; }
int ensure_rope(gh_backend* b, GhRopeTable& t, const gh_yarn*, uint32_t positions) {
    if (positions > kMaxRopePositions) return fail(b, GH_E_RANGE, "rope");
    return t.positions = positions, GH_OK;
}
}  // namespace gh

extern "C" {
gh_backend* host_backend(uint32_t cus) {
    auto* b = new gh_backend();
    b->cus = cus;
    b->paged_fault = new uint32_t[16]();
    return b;
}
gh_encoder* host_encoder(gh_backend* b) { return &b->enc; }
const char* host_error(gh_backend* b) { return b->err.c_str(); }
int host_latched(gh_backend* b) { return b->enc.latched; }
void host_reset(gh_backend* b, uint64_t limit) { launches.clear(), scratch_bytes = 0, scratch_limit = limit, b->enc.latched = 0; }
uint64_t host_scratch(void) { return scratch_bytes; }
uint32_t host_launches(void) { return (uint32_t)launches.size(); }
const void* host_launch(uint32_t i) { return &launches[i]; }
const char* host_kernel(uint32_t k) {
    switch (k) {
        case K_NORM_ROPE: return "norm_rope";
        case K_SAMPLE_MAX: return "sample_max";
        case K_SAMPLE_BINS: return "sample_bins";
        case K_SAMPLE_COLLECT: return "sample_collect";
        case K_SAMPLE_PICK: return "sample_pick";
        case K_PAGED_READ: return "read";
        case K_PAGED4_READ: return "read4";
        case K_PAGED_NORM_WRITE: return "norm_write";
        case K_PAGED4_WRITE: return "write4";
        case K_PAGED4_NORM_WRITE: return "norm_write4";
        case K_PAGED4_ATTN: case K_PAGED4_ATTN_S: return "attn4";
        case K_PAGED4_SPLIT: case K_PAGED4_SPLIT_S: return "split4";
        case K_PAGED_JOIN: case K_PAGED_JOIN2: return "join";
        case K_PAGED_SELECT: return "select";
        case K_PAGED4_MOVE: return "move4";
        default: return "other";
    }
}
}

// offsets of what the tests read
#include <cstddef>
extern "C" {
uint32_t host_offset(const char* name) {
#define FIELD(type, name_) if (!std::strcmp(name, #type "." #name_)) return (uint32_t)offsetof(type, name_);
    FIELD(GhSampleArgs, logits) FIELD(GhSampleArgs, params) FIELD(GhSampleArgs, uniform) FIELD(GhSampleArgs, tokens)
    FIELD(GhSampleArgs, probs) FIELD(GhSampleArgs, part) FIELD(GhSampleArgs, bins) FIELD(GhSampleArgs, list)
    FIELD(GhSampleArgs, scale) FIELD(GhSampleArgs, chunks) FIELD(GhSampleArgs, per) FIELD(GhSampleArgs, wide) FIELD(GhSampleArgs, shift)
    FIELD(GhPagedAttnArgs, q) FIELD(GhPagedAttnArgs, part_acc) FIELD(GhPagedAttnArgs, part_ml) FIELD(GhPagedAttnArgs, raw)
    FIELD(GhPagedAttnArgs, layout) FIELD(GhPagedAttnArgs, rows) FIELD(GhPagedAttnArgs, chunks) FIELD(GhPagedAttnArgs, least)
    FIELD(GhPagedAttnArgs, raw_len) FIELD(GhPagedAttnArgs, max_len) FIELD(GhPagedEvictArgs, src_layer) FIELD(GhPagedEvictArgs, dst_layer)
    return 0xFFFFFFFFu;
}
uint32_t host_sample_bytes(uint32_t what) { return what == 0 ? GH_SAMPLE_ROW_BYTES : what == 1 ? GH_SAMPLE_BIN_BYTES : GH_SAMPLE_LIST * 8; }
}
