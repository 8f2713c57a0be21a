// Quantisation to e4m3 with one scale for each row and block of 128, shared by the kernel that writes codes to memory and
// the one that keeps them in shared memory:
//
//   a0 = max(max |x| over the block, 448 * 2^-126),  q = e4m3(x * (448 / a0)),  scale = a0 / 448
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace ftm {

constexpr int kFp8Block = 128;                       // k of one scale
constexpr float kFp8Max = 448.0f;                    // largest e4m3 value
constexpr float kFp8Least = 0x1.cp-118f;             // 448 * 2^-126: 448 / a0 and a0 / 448 stay normal

// eight elements of a row; elements from `valid` on are zero and not read.  vec: the rows start on 16-byte boundaries.
template <typename T>
__device__ __forceinline__ void fp8_load8(const T* p, bool vec, int valid, float (&f)[8]) {
    if (vec && valid >= 8) {
        if constexpr (sizeof(T) == 2) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 q = bf16x2_to_f32(w[j]);
                f[2 * j] = q.x, f[2 * j + 1] = q.y;
            }
        } else {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = j < valid ? (float)p[j] : 0.f;
    }
}

// The codes of this lane's eight elements of a block that sixteen neighbouring lanes hold, and the block's scale.  Rounds to
// nearest even, saturates; a NaN stays one and does not count as a magnitude.
__device__ __forceinline__ uint2 fp8_encode8(const float (&f)[8], float& scale) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(f[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    most = fmaxf(most, kFp8Least);
    const float inv = __fdiv_rn(kFp8Max, most);
    scale = __fdiv_rn(most, kFp8Max);
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
        c[j] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * j] * inv, f[2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

inline bool fp8_rows_aligned(const void* x, int x_dtype, long long stride) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * (x_dtype == 0 ? 2 : 4) % 16 == 0;
}

}  // namespace ftm
