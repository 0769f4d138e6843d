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

// x over the root of the mean square of the head's `dim` values in `lanes` lanes, times the weight.
__device__ __forceinline__ void gh_head_norm(float (&x)[8], const uint4& weight, uint32_t dim, float eps, uint32_t lanes) {
    float s = 0.0f, w[8];
    gh_unpack8(weight, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i] * x[i];
    const float inv = 1.0f / __builtin_sqrtf(gh_group_sum(s, lanes) / (float)dim + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
}

// The lane's adjacent pairs first .. first + 3, those below `pairs`, turned by (cos, sin) at cs[first ..] and scaled.
__device__ __forceinline__ void gh_turn(float (&x)[8], int i, float c, float s, float scale) {
#pragma clang fp contract(off)
    const float x0 = x[2 * i], x1 = x[2 * i + 1];
    x[2 * i] = (x0 * c - x1 * s) * scale;
    x[2 * i + 1] = (x0 * s + x1 * c) * scale;
}
__device__ __forceinline__ void gh_turn4(float (&x)[8], const GH_GLOBAL float2* cs, uint32_t first, uint32_t pairs, float scale) {
    if ((pairs & 3u) == 0) {  // whole lanes, on 16 bytes
        const GH_GLOBAL float4* c4 = (const GH_GLOBAL float4*)(cs + first);
        const float4 c0 = c4[0], c1 = c4[1];
        gh_turn(x, 0, c0.x, c0.y, scale);
        gh_turn(x, 1, c0.z, c0.w, scale);
        gh_turn(x, 2, c1.x, c1.y, scale);
        gh_turn(x, 3, c1.z, c1.w, scale);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (first + i < pairs) {
            const float2 c = cs[first + i];
            gh_turn(x, i, c.x, c.y, scale);
        }
}

#endif
