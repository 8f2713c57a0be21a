// Quantisation to e4m3 with one scale for each row and block of 128, shared by the kernel that writes codes to memory and
// the one that keeps them in shared memory:
//
//   a0 = max(max |x| over the block, 448 * 2^-126),  q = e4m3(x * (448 / a0)),  scale = a0 / 448
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"
#include "umma.cuh"

namespace ftm {

constexpr int kFp8Block = 128;                       // k of one scale
constexpr float kFp8Max = 448.0f;                    // largest e4m3 value
constexpr float kFp8Least = 0x1.cp-118f;             // 448 * 2^-126: 448 / a0 and a0 / 448 stay normal

// Eight elements of a row as they are in memory.
template <typename T>
struct Fp8Eight;
template <>
struct Fp8Eight<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
    __device__ __forceinline__ void gather(const __nv_bfloat16* p, int valid) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __nv_bfloat162 v = __halves2bfloat162(2 * j < valid ? p[2 * j] : __float2bfloat16(0.f), 2 * j + 1 < valid ? p[2 * j + 1] : __float2bfloat16(0.f));
            w[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    // the largest magnitude (a NaN does not count), two at a time
    __device__ __forceinline__ float most() const {
        auto mag = [&](int j) { return __habs2(*reinterpret_cast<const __nv_bfloat162*>(w + j)); };
        const __nv_bfloat162 m = __hmax2(__hmax2(mag(0), mag(1)), __hmax2(mag(2), mag(3)));
        return fmaxf(__low2float(m), __high2float(m));
    }
    __device__ __forceinline__ float2 two(int j) const { return bf16x2_to_f32(w[j]); }
};
template <>
struct Fp8Eight<float> {
    float f[8];
    __device__ __forceinline__ void load(const float* p) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
    __device__ __forceinline__ void gather(const float* p, int valid) {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = j < valid ? p[j] : 0.f;
    }
    __device__ __forceinline__ float most() const {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) m = fmaxf(m, fabsf(f[j]));
        return m;
    }
    __device__ __forceinline__ float2 two(int j) const { return make_float2(f[2 * j], f[2 * j + 1]); }
};
// elements from `valid` on are zero and not read.  vec: the rows start on 16-byte boundaries.
template <typename T>
__device__ __forceinline__ void fp8_load8(const T* p, bool vec, int valid, Fp8Eight<T>& f) {
    if (vec && valid >= 8) f.load(p);
    else f.gather(p, valid);
}

// Codes and scales of U blocks at once, each held by sixteen neighbouring lanes, eight elements per lane.  Rounds to nearest even,
// saturates; a NaN stays one and does not count as a magnitude.  The 2 U quotients of a group are one division, of lane j < 2 U.
template <int U, typename T>
__device__ __forceinline__ void fp8_encode(const Fp8Eight<T> (&f)[U], uint2 (&codes)[U], float (&scale)[U]) {
    static_assert(U <= 8, "a lane for each quotient");
    const int lane = threadIdx.x % 16, group = threadIdx.x % 32 - lane;
    float num = 1.f, den = 1.f;
#pragma unroll
    for (int u = 0; u < U; u++) {
        float most = f[u].most();
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        most = fmaxf(most, kFp8Least);
        if (lane == 2 * u) num = kFp8Max, den = most;
        if (lane == 2 * u + 1) num = most, den = kFp8Max;
    }
    const float quotient = __fdiv_rn(num, den);
#pragma unroll
    for (int u = 0; u < U; u++) {
        const float inv = __shfl_sync(0xffffffffu, quotient, group + 2 * u);
        scale[u] = __shfl_sync(0xffffffffu, quotient, group + 2 * u + 1);
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 v = f[u].two(j);
            c[j] = __nv_cvt_float2_to_fp8x2(make_float2(v.x * inv, v.y * inv), __NV_SATFINITE, __NV_E4M3);
        }
        codes[u] = make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    }
}

// A CTA in which a wait gave up stays for about a millisecond: its copies and products still in flight take microseconds.
__device__ __forceinline__ void fp8_settle(const volatile int* gave_up) {
    if (!*gave_up) return;
    const long long from = clock64();
    while (clock64() - from < 2000000) {}
}

inline bool fp8_rows_aligned(const void* x, int x_dtype, long long stride) {
    return reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * (x_dtype == 0 ? 2 : 4) % 16 == 0;
}

// codes [rows, K] row-major, box = one block of 128 k by box_rows rows, 128-byte swizzle
inline bool fp8_codes_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int box_rows) {
    umma::EncodeTiledFn fn = umma::encode_tiled();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)K};
    cuuint32_t box[2] = {(cuuint32_t)kFp8Block, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// fp8_pair.cu: pairs of SMs on tiles of 256 x 256; a negative result is a CUDA error code
int launch_fp8_pair(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, int M, int N, int K, void* out, int out_dtype,
                    long long ldc, int sm_count, int32_t* err, cudaStream_t s);

}  // namespace ftm
