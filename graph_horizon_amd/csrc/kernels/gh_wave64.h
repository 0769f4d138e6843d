// 64-bit values across the lanes of a wave: exchanges for sorting, running sums.
#ifndef GH_WAVE64_H
#define GH_WAVE64_H
#include "gh_common.h"

// The smaller (keep_min) or larger of x and lane ^ stride's x: DPP moves within 16 lanes (xor 4 as
// xor 7 then xor 3), row swaps beyond, which leave the lane's own and its partner's value in the two
// registers (through ds_bpermute: partial 13.5 us, final 13.9 at k = 40).
template <int CTRL>
__device__ __forceinline__ uint64_t gh_dpp64(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, 0xF, 0xF, false);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t gh_exchange64(uint64_t x, uint32_t stride, bool keep_min) {
    uint64_t y;
    if (stride >= 16) {
        const uint32_t l = (uint32_t)x, h = (uint32_t)(x >> 32);
        const auto a = stride == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false)
                                    : __builtin_amdgcn_permlane32_swap(l, l, false, false);
        const auto b = stride == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false)
                                    : __builtin_amdgcn_permlane32_swap(h, h, false, false);
        x = ((uint64_t)b[0] << 32) | a[0];
        y = ((uint64_t)b[1] << 32) | a[1];
    } else if (stride == 8) {
        y = gh_dpp64<0x128>(x);  // row_ror:8
    } else if (stride == 4) {
        y = gh_dpp64<0x1B>(gh_dpp64<0x141>(x));  // row_half_mirror, quad_perm [3,2,1,0]
    } else {
        y = stride == 2 ? gh_dpp64<0x4E>(x) : gh_dpp64<0xB1>(x);  // quad_perm [2,3,0,1], [1,0,3,2]
    }
    return ((x > y) == keep_min) ? y : x;
}

// Ascending over the lanes.
__device__ __forceinline__ uint64_t gh_sort64(uint64_t x) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (uint32_t s = size >> 1; s > 0; s >>= 1) x = gh_exchange64(x, s, ((lane & s) == 0) == ((lane & size) == 0));
    return x;
}

// Inclusive running sum: within rows of 16 lanes, then the rows' totals onward.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t gh_scan64_step(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xF, true);
    return x + (((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ uint64_t gh_scan64(uint64_t x) {
    x = gh_scan64_step<0x111, 0xF>(x);     // row_shr:1
    x = gh_scan64_step<0x112, 0xF>(x);     // row_shr:2
    x = gh_scan64_step<0x114, 0xF>(x);     // row_shr:4
    x = gh_scan64_step<0x118, 0xF>(x);     // row_shr:8
    x = gh_scan64_step<0x142, 0xA>(x);     // row_bcast:15 into rows 1 and 3
    return gh_scan64_step<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ uint64_t gh_lane64(uint64_t x, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(x >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)x, lane);
}

// Largest over the wave.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t gh_max64_step(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)x, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp((int)(x >> 32), (int)(x >> 32), CTRL, ROWS, 0xF, false);
    const uint64_t y = ((uint64_t)hi << 32) | lo;
    return x > y ? x : y;
}
__device__ __forceinline__ uint64_t gh_max64(uint64_t x) {
    x = gh_max64_step<0xB1, 0xF>(x);
    x = gh_max64_step<0x4E, 0xF>(x);
    x = gh_max64_step<0x141, 0xF>(x);
    x = gh_max64_step<0x140, 0xF>(x);
    x = gh_max64_step<0x142, 0xA>(x);
    x = gh_max64_step<0x143, 0xC>(x);
    return gh_lane64(x, 63);
}

#endif
