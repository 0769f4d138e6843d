// A head's vector over lanes, 8 values each: FP16 in and out, norm and rotation in FP32 between them.
#ifndef GH_HEAD_H
#define GH_HEAD_H
#include "gh_common.h"

__device__ __forceinline__ void gh_unpack8(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = gh_h2f(w[i] & 0xFFFFu);
        x[2 * i + 1] = gh_h2f(w[i] >> 16);
    }
}
__device__ __forceinline__ uint4 gh_pack8(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)gh_f2h(x[2 * i]) | (uint32_t)gh_f2h(x[2 * i + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sum over aligned quads of lanes, in each of them; and over groups of 1, 2, 4, .. 64.
__device__ __forceinline__ float gh_quad_sum(float v) {
    v += GH_DPP(v, 0xB1, 0xF);        // quad_perm [1,0,3,2]
    return v + GH_DPP(v, 0x4E, 0xF);  // quad_perm [2,3,0,1]
}
__device__ __forceinline__ float gh_group_sum(float v, uint32_t lanes) {
    if (lanes > 1) v += GH_DPP(v, 0xB1, 0xF);
    if (lanes > 2) v += GH_DPP(v, 0x4E, 0xF);
    if (lanes > 4) v += GH_DPP(v, 0x141, 0xF);  // row_half_mirror
    if (lanes > 8) v += GH_DPP(v, 0x140, 0xF);  // row_mirror
    if (lanes > 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if (lanes > 32) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return v;
}

// x over the root of the mean square of the head's values in `lanes` lanes, times the weight; share: 1 / their number.
__device__ __forceinline__ void gh_head_norm(float (&x)[8], const uint4& weight, float share, float eps, uint32_t lanes) {
    float s = 0.0f, w[8];
    gh_unpack8(weight, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i] * x[i];
    const float inv = __builtin_amdgcn_rsqf(gh_group_sum(s, lanes) * share + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
}

// (cos, sin) of the lane's adjacent pairs first .. first + 3 of one position; those at or past `pairs` are of others. WIDE:
// `pairs` is a multiple of four, so that these are 32 bytes on 16. (A template, not a branch: the compiler makes one path of the
// two, with eight loads of a dword, and 2000 rows of 40 heads took 24.7 us.)
template <bool WIDE>
__device__ __forceinline__ void gh_load_turns(const GH_GLOBAL float2* cs, uint32_t first, uint32_t pairs, float2 (&c)[4]) {
    if (WIDE) {
        const GH_GLOBAL float4* c4 = (const GH_GLOBAL float4*)(cs + min(first, pairs - 4));
        const float4 c0 = c4[0], c1 = c4[1];
        c[0] = make_float2(c0.x, c0.y), c[1] = make_float2(c0.z, c0.w);
        c[2] = make_float2(c1.x, c1.y), c[3] = make_float2(c1.z, c1.w);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) c[i] = cs[min(first + i, pairs - 1)];
    }
}
// Those pairs below `pairs` turned and scaled, in gh_rope's operations. all: they are all of the head's.
__device__ __forceinline__ void gh_turn4(float (&x)[8], const float2 (&c)[4], uint32_t first, uint32_t pairs, float scale, bool all) {
#pragma clang fp contract(off)
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[2 * i] = (x[2 * i] * c[i].x - x[2 * i + 1] * c[i].y) * scale;
        y[2 * i + 1] = (x[2 * i] * c[i].y + x[2 * i + 1] * c[i].x) * scale;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = all || first + i / 2 < pairs ? y[i] : x[i];
}

#endif
