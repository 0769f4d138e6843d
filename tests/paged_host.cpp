// host/paged.cpp without a device, for the tests of its checks and launch plans: the backend's helpers that
// it calls, with launches recorded instead of made and scratch handed out as an address range.
#include <algorithm>

#include "../graph_horizon_amd/csrc/host/internal.h"

namespace {
struct Launch {
    uint32_t kernel, gx, gy, gz, block;
    unsigned char args[512];
};
std::vector<Launch> launches;
uint64_t scratch_bytes = 0, scratch_limit = 0;
constexpr uint64_t kScratchAt = 1ull << 50;
bool keeps_scratch = false;         // as the backend does: only a request beyond what there is asks for memory
std::vector<uint64_t> asked;        // those requests, refused ones too
size_t args_size(GhKernel k) {
    return k == K_PAGED_WRITE ? sizeof(GhPagedWriteArgs) : k >= K_PAGED_SELECT ? sizeof(GhPagedEvictArgs) : sizeof(GhPagedAttnArgs);
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
    if (keeps_scratch) {
        *at = (char*)kScratchAt;
        if (bytes <= workspace_room(b)) return GH_OK;
        asked.push_back(bytes);
        if (scratch_limit && bytes > scratch_limit) return fail(b, GH_E_OOM, "scratch");
        b->ws_bytes = bytes + kArgmaxBytes;
        return GH_OK;
    }
    if (scratch_limit && bytes > scratch_limit) return fail(b, GH_E_OOM, "scratch");
    scratch_bytes = bytes;
    *at = (char*)kScratchAt;
    return GH_OK;
}
bool yarn_valid(const gh_yarn* y) { return y && y->rope_dim && y->rope_dim % 2 == 0; }
int ensure_rope(gh_backend*, GhRopeTable& t, const gh_yarn*, uint32_t positions) { return t.positions = positions, GH_OK; }
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
uint32_t host_rope_positions(gh_backend* b) { return b->rope.positions; }
void host_reset(gh_backend* b, uint64_t limit) { launches.clear(), scratch_bytes = 0, scratch_limit = limit, b->enc.latched = 0, b->rope.positions = 0; }
// from here on the scratch of one call is there for the next; returns how many requests there were so far
uint32_t host_keep_scratch(void) { return keeps_scratch = true, (uint32_t)asked.size(); }
void host_drop_scratch(gh_backend* b) { keeps_scratch = false, asked.clear(), b->ws_bytes = 0; }
uint64_t host_asked(uint32_t i) { return asked[i]; }
uint64_t host_scratch(void) { return scratch_bytes; }
uint32_t host_launches(void) { return (uint32_t)launches.size(); }
const void* host_launch(uint32_t i) { return &launches[i]; }
// kernel ids: write, the first attention, join, select, move, join in halves
void host_kernels(uint32_t* k) { k[0] = K_PAGED_WRITE, k[1] = K_PAGED_ATTN, k[2] = K_PAGED_JOIN, k[3] = K_PAGED_SELECT, k[4] = K_PAGED_MOVE, k[5] = K_PAGED_JOIN2; }
}

// sizes and offsets of what the tests read through their own declarations
#include <cstddef>
extern "C" {
struct HostField {
    const char* name;
    uint32_t offset, size;
};
#define FIELD(type, name) {#name, (uint32_t)offsetof(type, name), (uint32_t)sizeof(((type*)nullptr)->name)}
const HostField* host_pages_fields(void) {
    static const HostField f[] = {FIELD(GhPages, kc), FIELD(GhPages, vc), FIELD(GhPages, table), FIELD(GhPages, lengths),
                                  FIELD(GhPages, score), FIELD(GhPages, fault), FIELD(GhPages, width), FIELD(GhPages, shift),
                                  FIELD(GhPages, pages), FIELD(GhPages, kv_heads), {nullptr, sizeof(GhPages), 0}};
    return f;
}
const HostField* host_attn_fields(void) {
    static const HostField f[] = {FIELD(GhPagedAttnArgs, p), FIELD(GhPagedAttnArgs, q), FIELD(GhPagedAttnArgs, out),
                                  FIELD(GhPagedAttnArgs, part_acc), FIELD(GhPagedAttnArgs, part_ml), FIELD(GhPagedAttnArgs, raw),
                                  FIELD(GhPagedAttnArgs, stream), FIELD(GhPagedAttnArgs, layout), FIELD(GhPagedAttnArgs, q_heads),
                                  FIELD(GhPagedAttnArgs, group), FIELD(GhPagedAttnArgs, rows), FIELD(GhPagedAttnArgs, max_len),
                                  FIELD(GhPagedAttnArgs, chunks), FIELD(GhPagedAttnArgs, least), FIELD(GhPagedAttnArgs, solo),
                                  FIELD(GhPagedAttnArgs, raw_len), FIELD(GhPagedAttnArgs, scale), FIELD(GhPagedAttnArgs, blocks),
                                  {nullptr, sizeof(GhPagedAttnArgs), 0}};
    return f;
}
static_assert(K_PAGED_ATTN_S == K_PAGED_ATTN + 1 && K_PAGED_SPLIT == K_PAGED_ATTN + 2 && K_PAGED_SPLIT_S == K_PAGED_ATTN + 3,
              "the tests tell the attention kernels apart by their distance from the first");
static_assert(K_PAGED_WRITE < K_PAGED_SELECT && K_PAGED_JOIN2 < K_PAGED_SELECT && K_PAGED_MOVE_S + 1 == K_COUNT,
              "args_size takes every kernel from the selection on for one of the eviction");
}
