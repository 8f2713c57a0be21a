// Products in 8-bit floating point with a scale for each block of 128, and the quantisation of their activations.
//
//   quantise   a0 = max(max |x| over a row's block of 128, 448 * 2^-126),  q = e4m3(x * (448 / a0)),  scale = a0 / 448
//   product    c[t, n] = sum_b a_scale[b, t] * w_scale[n / 128, b] * (sum over k in block b of a[t, k] * w[n, k])
//
// Two factors of e4m3 have an exact product in f32.  A block's sum is taken in f32, scaled and added in f32: the scales differ
// from block to block, so they cannot wait for the end of the sum over k.
#include <cuda_fp8.h>

#include "kernels.cuh"

namespace ftm {

namespace {

constexpr int kBlock = 128;                      // k of one scale
constexpr float kMax = 448.0f;                   // largest e4m3 value
constexpr float kSmallest = 0x1.cp-118f;         // 448 * 2^-126: 448 / a0 and a0 / 448 stay normal

// ---- quantisation ------------------------------------------------------------------------------
// Memory bound: one read of x, one write of the codes.  Sixteen lanes own a block, eight elements each, so the block's maximum
// is four shuffles and x stays in registers.  The eight warps of a CTA take eight rows of the same blocks: the scales of
// neighbouring rows are neighbours in memory.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int valid, float (&f)[8]) {
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

// codes of eight values: round to nearest even, saturating (a NaN stays one)
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float inv) {
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; j++)
        c[j] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * j] * inv, f[2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

template <typename T>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const T* __restrict__ x, long long stride, int rows, int K, int vec, uint8_t* __restrict__ q, float* __restrict__ scale) {
    const int lane = threadIdx.x % 32, blocks = (K + kBlock - 1) / kBlock;
    const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    if (row >= rows) return;
    for (int b = blockIdx.y * 2 + lane / 16; b - lane / 16 < blocks; b += gridDim.y * 2) {
        const int k = b * kBlock + (lane % 16) * 8;
        float f[8];
        load8(x + row * stride + k, vec, b < blocks ? K - k : 0, f);
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(f[j]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        most = fmaxf(most, kSmallest);
        const float inv = __fdiv_rn(kMax, most);
        if (b < blocks && k < K) *reinterpret_cast<uint2*>(q + row * K + k) = encode8(f, inv);
        if (b < blocks && lane % 16 == 0) scale[(long long)b * rows + row] = __fdiv_rn(most, kMax);
    }
}

// ---- product, plain form: any shape ---------------------------------------------------------------
constexpr int kTile = 64;
template <typename OUT>
__global__ void __launch_bounds__(256)
fp8_gemm_plain_kernel(const uint8_t* __restrict__ a, const float* __restrict__ a_scale, const uint8_t* __restrict__ w,
                      const float* __restrict__ w_scale, int M, int N, int K, OUT* __restrict__ c, long long ldc) {
    __shared__ float as[32][kTile + 1], ws[32][kTile + 1];
    const int t0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int blocks = (K + kBlock - 1) / kBlock;
    float acc[4][4] = {};
    for (int b = 0; b < blocks; b++) {
        float part[4][4] = {};
        for (int k0 = b * kBlock; k0 < min(K, (b + 1) * kBlock); k0 += 32) {
            __syncthreads();
            for (int i = threadIdx.x; i < 32 * kTile; i += 256) {
                const int k = i % 32, r = i / 32;
                as[k][r] = t0 + r < M && k0 + k < K ? e4m3_to_f32(a[(size_t)(t0 + r) * K + k0 + k]) : 0.f;
                ws[k][r] = n0 + r < N && k0 + k < K ? e4m3_to_f32(w[(size_t)(n0 + r) * K + k0 + k]) : 0.f;
            }
            __syncthreads();
            for (int k = 0; k < 32; k++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) part[i][j] += as[k][ty * 4 + i] * ws[k][tx + 16 * j];
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = t0 + ty * 4 + i, n = n0 + tx + 16 * j;
                if (t < M && n < N) acc[i][j] += a_scale[(size_t)b * M + t] * w_scale[(size_t)(n / kBlock) * blocks + b] * part[i][j];
            }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = t0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (t < M && n < N) c[t * ldc + n] = (OUT)acc[i][j];
        }
}

}  // namespace

int launch_fp8_quantize(const void* x, int x_dtype, int rows, int K, long long stride, uint8_t* q, float* scale, const Ctx& c) {
    const int blocks = (K + kBlock - 1) / kBlock;
    const size_t es = x_dtype == 0 ? 2 : 4;
    const int vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (stride * es) % 16 == 0;
    const dim3 grid(((unsigned)rows + 7) / 8, min((blocks + 1) / 2, 65535));
    c.begin(K_FP8_QUANTIZE);
    if (x_dtype == 0)
        fp8_quantize_kernel<<<grid, 256, 0, c.s>>>((const __nv_bfloat16*)x, stride, rows, K, vec, q, scale);
    else
        fp8_quantize_kernel<<<grid, 256, 0, c.s>>>((const float*)x, stride, rows, K, vec, q, scale);
    c.end();
    return 1;
}

int launch_fp8_gemm(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, int M, int N, int K, void* out,
                    int out_dtype, long long ldc, const Ctx& c) {
    const dim3 grid((M + kTile - 1) / kTile, (N + kTile - 1) / kTile);
    c.begin(K_FP8_GEMM);
    if (out_dtype == 0)
        fp8_gemm_plain_kernel<<<grid, 256, 0, c.s>>>(a, a_scale, w, w_scale, M, N, K, (__nv_bfloat16*)out, ldc);
    else
        fp8_gemm_plain_kernel<<<grid, 256, 0, c.s>>>(a, a_scale, w, w_scale, M, N, K, (float*)out, ldc);
    c.end();
    return 1;
}

}  // namespace ftm
