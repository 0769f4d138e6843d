// gh_sample_rows (host/rows.cpp) with its launches run on the CPU (sample_kernels.cpp): buffers are host memory.
#include <cstdlib>

#include "../../graph_horizon_amd/csrc/host/internal.h"

extern "C" const char* wave_run(const char* kernel, uint32_t gx, uint32_t gy, uint32_t threads, const void* args, uint32_t order);
extern "C" hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
extern "C" hipError_t hipSetDevice(int) { return hipSuccess; }

namespace {
uint32_t order = 0, growths = 0;
uint64_t limit = 0;
}

namespace gh {
int fail(gh_backend* b, int code, const std::string& msg) { return b->err = msg, code; }
int check_enc(gh_backend* b, gh_encoder* enc) { return b && enc == &b->enc ? GH_OK : GH_E_STATE; }
int latch(gh_encoder*, int rc) { return rc; }
int launch(gh_backend* b, GhKernel k, uint32_t gx, uint32_t gy, uint32_t, uint32_t threads, const void* args, uint32_t) {
    if (order == ~0u) return GH_OK;  // plans alone
    const char* name = k == K_SAMPLE_MAX ? "max" : k == K_SAMPLE_BINS ? "bins" : k == K_SAMPLE_COLLECT ? "collect" : "pick";
    const char* error = wave_run(name, gx, gy, threads, args, order);
    return error ? fail(b, GH_E_HIP, std::string(name) + ": " + error) : GH_OK;
}
int workspace_at(gh_backend* b, size_t bytes, char** at) {
    if (workspace_room(b) < bytes) {
        ++growths;
        if (limit && bytes > limit) return fail(b, GH_E_OOM, "scratch");
        std::free(b->ws);
        b->ws_bytes = (bytes + kArgmaxBytes + 4095) / 4096 * 4096;
        b->ws = std::aligned_alloc(4096, b->ws_bytes);
        std::memset(b->ws, 0xA5, b->ws_bytes);
    }
    *at = (char*)b->ws + kArgmaxBytes;
    return GH_OK;
}
bool yarn_valid(const gh_yarn*) { return false; }
int ensure_rope(gh_backend*, GhRopeTable&, const gh_yarn*, uint32_t) { return GH_E_STATE; }
}  // namespace gh

extern "C" {
gh_backend* wave_backend(uint32_t cus) {
    auto* b = new gh_backend();
    b->cus = cus;
    return b;
}
gh_encoder* wave_encoder(gh_backend* b) { return &b->enc; }
const char* wave_error(gh_backend* b) { return b->err.c_str(); }
void wave_order(uint32_t o) { order = o; }
// Scratch past `bytes` cannot be had from now on (0: any); how often more was asked for than there was, since the last call of this.
uint32_t wave_limit(uint64_t bytes) {
    const uint32_t n = growths;
    return limit = bytes, growths = 0, n;
}
}
