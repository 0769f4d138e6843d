// Stands in for the HIP runtime's header where a kernel's source is compiled for the CPU: one workgroup at a time, each thread
// a context of its own. A wave's lanes meet at every cross-lane operation, the workgroup's threads at its barriers; between
// those the waves run one after the other in an order that the test chooses, so that an access to LDS that no
// barrier orders against another wave's gives another result in some order. Threads that meet at different
// barriers, or lanes at different operations, are an error.
#ifndef WAVE_HOST_H
#define WAVE_HOST_H
#include <stdint.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstring>

#define __device__
#define __host__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)
#define address_space(n)
using std::fmaxf;
using std::fminf;

struct dim3 { uint32_t x, y, z; };
struct uint2 { uint32_t x, y; };
struct float2 { float x, y; };
struct alignas(16) uint4 { uint32_t x, y, z, w; };
struct alignas(16) float4 { float x, y, z, w; };
struct alignas(16) ulonglong2 { unsigned long long x, y; };
inline uint2 make_uint2(uint32_t x, uint32_t y) { return {x, y}; }
inline float2 make_float2(float x, float y) { return {x, y}; }
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
inline ulonglong2 make_ulonglong2(unsigned long long x, unsigned long long y) { return {x, y}; }

namespace wave_host {
dim3 thread();
dim3 block();
dim3 grid();
uint32_t lane();
void barrier(int line);
int barrier_or(int line, int value);
// The values of all lanes of the wave at one operation.
const uint64_t* meet(uint32_t operation, uint64_t value);
}  // namespace wave_host
#define threadIdx (wave_host::thread())
#define blockIdx (wave_host::block())
#define gridDim (wave_host::grid())
#define __syncthreads() wave_host::barrier(__LINE__)
#define __syncthreads_or(x) wave_host::barrier_or(__LINE__, (int)(x))

template <class T>
inline T min(T a, T b) { return b < a ? b : a; }
template <class T>
inline T max(T a, T b) { return a < b ? b : a; }
inline uint64_t min(unsigned long long a, uint64_t b) { return b < a ? b : a; }
inline uint32_t __float_as_uint(float x) { return __builtin_bit_cast(uint32_t, x); }
inline int __float_as_int(float x) { return __builtin_bit_cast(int, x); }
inline float __uint_as_float(uint32_t x) { return __builtin_bit_cast(float, x); }
inline float __int_as_float(int x) { return __builtin_bit_cast(float, x); }
inline int __popc(uint32_t x) { return __builtin_popcount(x); }
inline int __popcll(unsigned long long x) { return __builtin_popcountll(x); }
inline int __clzll(long long x) { return x ? __builtin_clzll((unsigned long long)x) : 64; }
template <class T>
inline T atomicAdd(T* p, T v) {
    const T old = *p;
    *p = old + v;
    return old;
}

enum : uint32_t { kOpBallot = 1, kOpShfl, kOpShflUp, kOpLane, kOpSwap16, kOpSwap32, kOpDpp = 0x10000 };
inline uint64_t __ballot(bool is) {
    const uint64_t* all = wave_host::meet(kOpBallot, is);
    uint64_t mask = 0;
    for (int i = 0; i < 64; ++i) mask |= (uint64_t)(all[i] & 1) << i;
    return mask;
}
template <class T>
inline T __shfl(T v, int from, int) { return (T)wave_host::meet(kOpShfl, (uint64_t)v)[from & 63]; }
inline int __shfl_up(int v, uint32_t by, int) {
    const uint64_t* all = wave_host::meet(kOpShflUp, (uint32_t)v);
    const uint32_t l = wave_host::lane();
    return (int)(uint32_t)all[l < by ? l : l - by];
}
inline int wave_host_readlane(int v, uint32_t from) { return (int)(uint32_t)wave_host::meet(kOpLane, (uint32_t)v)[from & 63u]; }
// Of two vectors of four rows of 16 lanes: the first's odd rows and the second's even ones change places; and of two halves.
inline std::array<uint32_t, 2> wave_host_swap16(uint32_t a, uint32_t b, bool, bool) {
    const uint64_t* all = wave_host::meet(kOpSwap16, (uint64_t)b << 32 | a);
    const uint32_t l = wave_host::lane();
    if (l & 16u) return {(uint32_t)(all[l - 16] >> 32), b};
    return {a, (uint32_t)all[l + 16]};
}
inline std::array<uint32_t, 2> wave_host_swap32(uint32_t a, uint32_t b, bool, bool) {
    const uint64_t* all = wave_host::meet(kOpSwap32, (uint64_t)b << 32 | a);
    const uint32_t l = wave_host::lane();
    if (l & 32u) return {(uint32_t)(all[l - 32] >> 32), b};
    return {a, (uint32_t)all[l + 32]};
}
// The DPP controls that the kernels use, by their published definitions.
inline int wave_host_dpp(int old, int v, int ctrl, int rows, int, bool zero) {
    const uint64_t* all = wave_host::meet(kOpDpp + ctrl, (uint32_t)v);
    const uint32_t l = wave_host::lane(), row = l & ~15u, in = l & 15u;
    if (!(rows >> (l >> 4) & 1)) return old;
    int from = -1;
    if (ctrl < 0x100) from = (int)((l & ~3u) + (ctrl >> 2 * (l & 3u) & 3));       // quad_perm
    else if (ctrl > 0x110 && ctrl < 0x120) from = in >= (uint32_t)(ctrl & 15) ? (int)(l - (ctrl & 15)) : -1;  // row_shr
    else if (ctrl > 0x120 && ctrl < 0x130) from = (int)(row + ((in - (ctrl & 15)) & 15u));  // row_ror
    else if (ctrl == 0x140) from = (int)(row + 15 - in);                          // row_mirror
    else if (ctrl == 0x141) from = (int)((l & ~7u) + 7 - (l & 7u));               // row_half_mirror
    else if (ctrl == 0x142) from = l >= 16 ? (int)(row - 1) : -1;                 // row_bcast:15
    else if (ctrl == 0x143) from = l >= 32 ? 31 : -1;                             // row_bcast:31
    else __builtin_trap();
    return from < 0 ? (zero ? 0 : old) : (int)(uint32_t)all[from];
}
#define __builtin_amdgcn_update_dpp wave_host_dpp
#define __builtin_amdgcn_readlane wave_host_readlane
#define __builtin_amdgcn_permlane16_swap wave_host_swap16
#define __builtin_amdgcn_permlane32_swap wave_host_swap32
#define __builtin_amdgcn_fence(...) ((void)0)
#define __builtin_amdgcn_s_barrier() __builtin_trap()
template <class H>
inline float wave_host_dot2(H a, H b, float c, bool) { return (float)a.x * (float)b.x + (float)a.y * (float)b.y + c; }
#define __builtin_amdgcn_fdot2 wave_host_dot2
#endif
