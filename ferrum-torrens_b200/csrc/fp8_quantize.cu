// Activations to e4m3 with one scale for each row and block of 128 (the formula is in fp8.cuh).
//
// Memory bound: one read of x, one write of the codes.  Sixteen lanes own a block, eight elements each, so the block's maximum
// is four shuffles and x stays in registers.  The eight warps of a CTA take eight rows of the same blocks: the scales of
// neighbouring rows are neighbours in memory.
#include "fp8.cuh"
#include "kernels.cuh"

namespace ftm {

namespace {

constexpr int kAtOnce = 2;      // blocks a group of lanes holds at a time

template <typename T>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const T* x, long long stride, int rows, int K, bool vec, uint8_t* q, float* scale) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x % 32, blocks = (K + kFp8Block - 1) / kFp8Block;
    const long long row = (long long)blockIdx.x * 8 + threadIdx.x / 32;
    if (row >= rows) return;
    for (int b0 = blockIdx.y * 2 * kAtOnce; b0 < blocks; b0 += gridDim.y * 2 * kAtOnce) {
        float f[kAtOnce][8], sc[kAtOnce];
        uint2 codes[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int b = b0 + 2 * u + lane / 16, k = b * kFp8Block + (lane % 16) * 8;
            fp8_load8(x + row * stride + k, vec, b < blocks ? K - k : 0, f[u]);
        }
        fp8_encode(f, codes, sc);
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int b = b0 + 2 * u + lane / 16, k = b * kFp8Block + (lane % 16) * 8;
            if (b < blocks && k < K) *reinterpret_cast<uint2*>(q + row * K + k) = codes[u];
            if (b < blocks && lane % 16 == 0) scale[(long long)b * rows + row] = sc[u];
        }
    }
}

}  // namespace

int launch_fp8_quantize(const void* x, int x_dtype, int rows, int K, long long stride, uint8_t* q, float* scale, const Ctx& c) {
    const int blocks = (K + kFp8Block - 1) / kFp8Block;
    const bool vec = fp8_rows_aligned(x, x_dtype, stride);
    const dim3 grid(((unsigned)rows + 7) / 8, min((blocks + 2 * kAtOnce - 1) / (2 * kAtOnce), 65535));
    c.begin(K_FP8_QUANTIZE);
    const cudaError_t e =
        x_dtype == 0 ? launch_pdl(fp8_quantize_kernel<__nv_bfloat16>, grid, dim3(256), 0, c.s, (const __nv_bfloat16*)x, stride, rows, K, vec, q, scale)
                     : launch_pdl(fp8_quantize_kernel<float>, grid, dim3(256), 0, c.s, (const float*)x, stride, rows, K, vec, q, scale);
    c.end();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace ftm
