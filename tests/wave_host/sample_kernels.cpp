// The sampling kernels (kernels/sample.hip) compiled for the CPU, a workgroup at a time: see hip/hip_runtime.h beside this file.
#include <sys/mman.h>
#include <ucontext.h>

#include <cstdio>
#include <functional>
#include <string>
#include <vector>

#include "../../graph_horizon_amd/csrc/kernels/sample.hip"

namespace {
enum State { READY, AT_OPERATION, AT_BARRIER, DONE };
constexpr size_t kStack = 128 << 10;

struct Thread {
    ucontext_t at;
    State state;
    uint32_t operation, met;  // where it waits; operations so far
    int line, value;
};
struct Wave {
    uint64_t slot[2][64];
};
struct Group {
    std::vector<Thread> threads;
    std::vector<Wave> waves;
    std::function<void()> body;
    ucontext_t out;
    uint32_t now = 0;
    dim3 block{}, grid{};
    int any = 0;
    std::string error;
} g;
char* stacks;

void start() {
    g.body();
    g.threads[g.now].state = DONE;
    swapcontext(&g.threads[g.now].at, &g.out);
}
void leave(State s) {
    Thread& t = g.threads[g.now];
    t.state = s;
    swapcontext(&t.at, &g.out);
}

// Runs a wave up to its next barrier or its end; true where it left off before (`stop` says when, at operations).
template <class F>
bool run_wave(uint32_t w, F stop) {
    for (;;) {
        uint32_t at[4] = {};
        Thread* t0 = &g.threads[64 * w];
        for (uint32_t l = 64; l-- > 0;) {  // lane 0, which writes for its wave, behind the others, which read in the same step
            g.now = 64 * w + l;
            if (t0[l].state == READY) swapcontext(&g.out, &t0[l].at);
            ++at[t0[l].state];
        }
        if (at[AT_OPERATION] == 0) return false;
        for (uint32_t l = 0; l < 64; ++l)
            if (t0[l].state != AT_OPERATION || t0[l].operation != t0->operation) {
                g.error = "lanes of a wave part at an operation";
                return false;
            }
        for (uint32_t l = 0; l < 64; ++l) t0[l].state = READY;
        if (stop()) return true;
    }
}

// order: 0 the first wave ahead of all others between barriers, 1 the last one, else waves in turns by this seed.
bool run_group(uint32_t order) {
    const uint32_t waves = (uint32_t)g.waves.size();
    uint64_t random = order * 0x9E3779B97F4A7C15ull + 1;
    auto next = [&] { return random ^= random << 13, random ^= random >> 7, random ^= random << 17, (uint32_t)(random >> 20); };
    std::vector<uint32_t> left(waves);
    for (;;) {
        left.clear();
        for (uint32_t w = 0; w < waves; ++w) left.push_back(order == 1 ? w : waves - 1 - w);
        while (!left.empty()) {
            const size_t i = order < 2 ? left.size() - 1 : next() % left.size();
            const uint32_t w = left[i];
            if (!run_wave(w, [&] { return order >= 2 && next() % 4 == 0; })) left.erase(left.begin() + (long)i);
            if (!g.error.empty()) return false;
        }
        int line = 0, any = 0;
        for (Thread& t : g.threads) {
            if (t.state == DONE) continue;
            if (line && t.line != line) {
                g.error = "threads meet at the barriers of lines " + std::to_string(line) + " and " + std::to_string(t.line);
                return false;
            }
            line = t.line;
            any |= t.value;
        }
        if (!line) return true;
        g.any = any;
        for (Thread& t : g.threads)
            if (t.state == AT_BARRIER) t.state = READY;
    }
}
}  // namespace

namespace wave_host {
dim3 thread() { return {g.now, 0, 0}; }
dim3 block() { return g.block; }
dim3 grid() { return g.grid; }
uint32_t lane() { return g.now & 63u; }
void barrier(int line) { barrier_or(line, 0); }
int barrier_or(int line, int value) {
    g.threads[g.now].line = line;
    g.threads[g.now].value = value;
    leave(AT_BARRIER);
    return g.any;
}
const uint64_t* meet(uint32_t operation, uint64_t value) {
    Thread& t = g.threads[g.now];
    uint64_t* slot = g.waves[g.now >> 6].slot[t.met++ & 1u];  // a lane is at most one operation ahead of another
    slot[g.now & 63u] = value;
    t.operation = operation;
    leave(AT_OPERATION);
    return slot;
}
}  // namespace wave_host

extern "C" {
// Runs the kernel's workgroups one after the other; NULL, or what went wrong.
const char* wave_run(const char* kernel, uint32_t gx, uint32_t gy, uint32_t threads, const void* args, uint32_t order) {
    GhSampleArgs a;
    std::memcpy(&a, args, sizeof a);
    const std::string name = kernel;
    void (*f)(GhSampleArgs) = name == "max" ? gh_sample_max : name == "bins" ? gh_sample_bins : name == "collect" ? gh_sample_collect : gh_sample_pick;
    if (!stacks) stacks = (char*)mmap(nullptr, 1024 * kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
    g.error.clear();
    g.body = [&] { f(a); };
    for (uint32_t y = 0; y < gy; ++y)
        for (uint32_t x = 0; x < gx; ++x) {
            g.block = {x, y, 0};
            g.grid = {gx, gy, 1};
            g.threads.resize(threads);
            g.waves.resize(threads / 64);
            for (uint32_t i = 0; i < threads; ++i) {
                Thread& t = g.threads[i];
                t.state = READY;
                t.met = 0;
                getcontext(&t.at);
                t.at.uc_stack.ss_sp = stacks + i * kStack;
                t.at.uc_stack.ss_size = kStack;
                t.at.uc_link = nullptr;
                makecontext(&t.at, start, 0);
            }
            if (!run_group(order)) return g.error.c_str();
        }
    return nullptr;
}
}
