// Activations to e4m3 with one scale for each row and block of 128 (the formula is in fp8.cuh).
//
// Memory bound: one read of x, one write of the codes.  Sixteen lanes own a block, eight elements each, so the block's maximum
// is four shuffles and x stays in registers.  The eight warps of a CTA take eight rows of the same blocks: the scales of
// neighbouring rows are neighbours in memory.  Large inputs: a few CTAs per SM walk over them, the next blocks on their way
// while these are encoded.
#include "fp8.cuh"
#include "kernels.cuh"

namespace ftm {

namespace {

// Blocks a group of lanes holds at a time, and as many more on their way; CTAs of an SM.  8192 x 4096 bf16: 17.6 us (0.90 of measured
// HBM) with four blocks and four CTAs, 20.3 with two and five, 22.9 with one and eight; 26.6 without blocks ahead.
template <typename T>
constexpr int kBlocksAtOnce = 8 / (int)sizeof(T);
constexpr int kPerSm = 4;

template <typename T>
__global__ void __launch_bounds__(256, kPerSm)
fp8_quantize_kernel(const T* x, long long stride, int rows, int K, bool vec, uint8_t* q, float* scale, int k_steps, long long steps) {
    constexpr int kAtOnce = kBlocksAtOnce<T>;
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, blocks = (K + kFp8Block - 1) / kFp8Block;
    // A step is eight rows by 2 * kAtOnce blocks, along the rows first; a CTA's steps are the grid's size apart.
    const int far_k = (int)(gridDim.x % (unsigned)k_steps);
    const long long far_row = gridDim.x / (unsigned)k_steps * 8;
    int k_step = (int)(blockIdx.x % (unsigned)k_steps);
    long long row = blockIdx.x / (unsigned)k_steps * 8 + warp;
    Fp8Eight<T> next[kAtOnce];
    auto fetch = [&](long long row, int k0) {
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int k = k0 + u * 2 * kFp8Block;
            fp8_load8(x + row * stride + k, vec, row < rows ? K - k : 0, next[u]);
        }
    };
    auto start_of = [&](int k_step) { return k_step * (2 * kAtOnce * kFp8Block) + lane * 8; };
    fetch(row, start_of(k_step));
    for (long long step = blockIdx.x; step < steps; step += gridDim.x) {
        const long long this_row = row;
        const int k0 = start_of(k_step);
        row += far_row;
        k_step += far_k;
        if (k_step >= k_steps) k_step -= k_steps, row += 8;
        Fp8Eight<T> f[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) f[u] = next[u];
        fetch(row, start_of(k_step));
        uint2 codes[kAtOnce];
        float sc[kAtOnce];
        fp8_encode(f, codes, sc);
        if (this_row >= rows) continue;
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            const int k = k0 + u * 2 * kFp8Block;
            if (k < K) *reinterpret_cast<uint2*>(q + this_row * K + k) = codes[u];
            if (k / kFp8Block < blocks && lane % 16 == 0) scale[(long long)(k / kFp8Block) * rows + this_row] = sc[u];
        }
    }
}

}  // namespace

int launch_fp8_quantize(const void* x, int x_dtype, int rows, int K, long long stride, uint8_t* q, float* scale, int sm_count, const Ctx& c) {
    const int blocks = (K + kFp8Block - 1) / kFp8Block;
    const bool vec = fp8_rows_aligned(x, x_dtype, stride);
    const int wide = 2 * (x_dtype == 0 ? kBlocksAtOnce<__nv_bfloat16> : kBlocksAtOnce<float>), k_steps = (blocks + wide - 1) / wide;
    const long long steps = ((long long)rows + 7) / 8 * k_steps;
    const dim3 grid((unsigned)min(steps, (long long)kPerSm * sm_count));
    c.begin(K_FP8_QUANTIZE);
    const cudaError_t e =
        x_dtype == 0 ? launch_pdl(fp8_quantize_kernel<__nv_bfloat16>, grid, dim3(256), 0, c.s, (const __nv_bfloat16*)x, stride, rows, K, vec, q, scale, k_steps, steps)
                     : launch_pdl(fp8_quantize_kernel<float>, grid, dim3(256), 0, c.s, (const float*)x, stride, rows, K, vec, q, scale, k_steps, steps);
    c.end();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace ftm
