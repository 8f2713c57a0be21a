// Block-scaled 8-bit products of many rows: pairs of SMs on tiles of 256 tokens by 256 weight rows.
//
//   c[t, n] = sum_b (a_scale[b, t] * w_scale[n / 128, b]) * (sum over k in block b of a[t, k] * w[n, k])
//
// Bound by the tensor cores, then by what the SMs can fetch from L2: a lone SM on 128 x 256 would ask for 96 bytes per clock, the
// two of a pair, each with 128 tokens and half of the weight rows, for 64.  A block of 128 k is four tcgen05.mma of
// 256 x 256 x 32 by the first CTA into one of two accumulators that fill the tensor memory of both (512 cycles at the full rate).
// As the scales change with the block, the epilogue warps read every accumulator back (128 lanes, one per token; two warps of
// a quarter share its 256 columns, so each has one block of weight scales), multiply by one number per lane and add to 128
// sums in registers while the other accumulator is filled.
//   warp 0      TMA: this CTA's 128 token rows and 128 weight rows of a block; both CTAs' bytes count on the first one's barrier
//   warps 1, 3  first CTA: issue the products of a block in turn and hand the stage and the accumulator over in both CTAs
//   warp 2      fetches the scales of every block ahead of the epilogue
//   warps 4..11 epilogue
// 8192 x 8192 x 4096 bf16 out: 249 us, 2210 TFLOP/s, at the power limit (operands of one constant 219); 4096 x 4096 x 2048 40 us;
// 1000 x 4100 x 2000 14.4 us, of which the products take 7.  What bounds a tile is the epilogue: 210 us of the 219 without the products.
// Persistent, one pair per two SMs.  Every wait is bounded; a wait that gives up raises the error flag and the CTA drains.
#include "fp8.cuh"
#include "kernels.cuh"
#include "umma.cuh"

namespace ftm {

namespace {

using namespace umma;

constexpr int kM = 256, kN = 256;                // tokens and weight rows of a pair's tile
constexpr int kHalfBytes = 128 * kFp8Block;      // 128 rows of a block: 16 KiB
constexpr int kStage = 2 * kHalfBytes;           // of one CTA
constexpr int kStages = 5;
constexpr int kEpi = 8;
constexpr int kThreads = 128 + 32 * kEpi;
// registers: 384 threads are launched with 168 each, 64512; 128 x 64 + 256 x 216 = 63488
constexpr int kFewRegs = 64, kManyRegs = 216;
constexpr int kOutBytes = 32 * 256;              // one epilogue warp's output rows on their way out: 256 bytes of 32 tokens
constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + kEpi * kOutBytes + 2 * (128 + 2) * 4 + 256;
static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
// e4m3 x e4m3 -> f32, both operands K-major
constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kN >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);

struct PairArgs {
    const float* a_scale;        // [blocks, M]
    const float* w_scale;        // [ceil(N / 128), blocks]
    int M, N, blocks;
    int m_tiles, tiles;
    void* c;
    int c_dtype;
    bool c_by_tma, c_by_8;       // every row of c starts and ends on 16 bytes, starts on 8
    long long ldc;
    int32_t* err;
};

__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(kIdesc), "r"(accumulate)
        : "memory");
}
// arrives at the barrier of this offset in both CTAs when the products issued so far are done
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
}
// a box into this CTA's shared memory, its bytes counted on a barrier of the pair's first CTA
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]),
          "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]),
          "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]),
          "=f"(v[31])
        : "r"(taddr));
}

// One warp's 32 tokens from t0 on by 256 bytes of output from weight row n0 on, from its (swizzled) place in shared memory to c.
__device__ __forceinline__ void send_out(const PairArgs& a, const CUtensorMap* map, uint8_t* from, int t0, int n0, int elem, int lane) {
    const int cols = 128 / elem;      // of a box
    if (a.c_by_tma) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
            for (int b = 0; b < 2; b++)
                if (n0 + b * cols < a.N)
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(n0 + b * cols), "r"(t0),
                                 "r"(smem_u32(from + b * 4096))
                                 : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        return;
    }
    // Other rows: a lane has 8 bytes of each.  Where not all rows start on 8 bytes, these are moved up by the neighbour's so that they do in
    // memory.  What is left at the rows' two ends then goes out in pieces of 2, a row to a lane.
    __syncwarp();
    const int rows = min(32, a.M - t0), bytes = min(256, (a.N - n0) * elem);
    const long long next = a.ldc * elem;
    uint8_t* const first = reinterpret_cast<uint8_t*>(a.c) + ((long long)t0 * a.ldc + n0) * elem;
    auto at = [&](int row, int byte) { return from + (byte >> 7) * 4096 + row * 128 + ((((byte >> 4) & 7) ^ (row & 7)) << 4) + (byte & 15); };
    if (a.c_by_8) {
        if (8 * lane + 8 <= bytes)
#pragma unroll 8
            for (int row = 0; row < rows; row++) *reinterpret_cast<uint64_t*>(first + row * next + 8 * lane) = *reinterpret_cast<const uint64_t*>(at(row, 8 * lane));
    } else {
#pragma unroll 8
        for (int row = 0; row < rows; row++) {
            uint8_t* const to = first + row * next;
            const uint64_t cur = *reinterpret_cast<const uint64_t*>(at(row, 8 * lane)), before = __shfl_up_sync(0xffffffffu, cur, 1);
            const int off = (int)(reinterpret_cast<uintptr_t>(to) & 7), byte = 8 * lane - off;
            if (byte >= 0 && byte + 8 <= bytes) *reinterpret_cast<uint64_t*>(to + byte) = off ? cur << (8 * off) | before >> (64 - 8 * off) : cur;
        }
    }
    if (lane < rows) {
        uint8_t* const to = first + lane * next;
        const int ahead = min((int)(-reinterpret_cast<uintptr_t>(to) & 7), bytes), behind = ahead + ((bytes - ahead) & ~7);
#pragma unroll
        for (int q = 0; q < 6; q += 2) {
            if (q < ahead) *reinterpret_cast<uint16_t*>(to + q) = *reinterpret_cast<const uint16_t*>(at(lane, q));
            if (behind + q < bytes) *reinterpret_cast<uint16_t*>(to + behind + q) = *reinterpret_cast<const uint16_t*>(at(lane, behind + q));
        }
    }
    __syncwarp();
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                const __grid_constant__ CUtensorMap tmap_c, const PairArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* const out = ring + (size_t)kStages * kStage;                                // [epilogue warp][two boxes of 32 x 128 bytes, swizzled]
    float* const slots = reinterpret_cast<float*>(out + kEpi * kOutBytes);               // [accumulator][128 tokens, 2 halves of the weight rows]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(slots + 2 * (128 + 2));
    const uint32_t bar0 = smem_u32(bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto ACC_FULL = [&](int p) { return bar0 + 8u * (2 * kStages + p); };
    auto ACC_EMPTY = [&](int p) { return bar0 + 8u * (2 * kStages + 2 + p); };
    auto SLOT_EMPTY = [&](int p) { return bar0 + 8u * (2 * kStages + 4 + p); };
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 6);
    volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = blockIdx.x & 1;
    if (warp == 0) {
        if (lane < kStages) mbar_init(FULL(lane), 1), mbar_init(EMPTY(lane), 1);
        if (lane < 2) mbar_init(ACC_FULL(lane), 2), mbar_init(ACC_EMPTY(lane), 2 * kEpi), mbar_init(SLOT_EMPTY(lane), kEpi);
        if (lane == 0) *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();      // (no tensor memory is held while the kernel before may still want some)
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // both CTAs run and have their barriers
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    pdl_launch_dependents();
    const uint32_t tmem_base = *s_tmem;
    const int first = blockIdx.x / 2, step = gridDim.x / 2;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        if (warp == 0) {
            int st = 0;
            uint32_t round = 0;
            bool ok = true;
            for (int tile = first; tile < a.tiles && ok; tile += step) {
                const int t0 = tile % a.m_tiles * kM + rank * 128, n0 = tile / a.m_tiles * kN + rank * 128;
                for (int kb = 0; kb < a.blocks; kb++) {
                    ok = mbar_wait_warp(EMPTY(st), round ^ 1, s_abort, a.err);
                    if (!ok) break;
                    if (elect_one()) {
                        const uint32_t dst = smem_u32(ring + st * kStage), bar = in_first_cta(FULL(st));
                        // the bytes of both CTAs; what a box reads past the matrix is zero and counts all the same
                        if (rank == 0) mbar_expect_tx(FULL(st), 2 * kStage);
                        tma_load_pair(dst, &tmap_a, kb * kFp8Block, t0, bar);
                        tma_load_pair(dst + kHalfBytes, &tmap_w, kb * kFp8Block, n0, bar);
                    }
                    __syncwarp();
                    if (++st == kStages) st = 0, round ^= 1;
                }
            }
        } else if (warp == 1 || warp == 3) {
            // two issuers: the wait and the issue of one block take one warp longer than the products themselves
            if (rank == 0) {
                int st = 0, p = 0;
                uint32_t round = 0, p_round = 0;
                bool ok = true, my_turn = warp == 1;
                for (int tile = first; tile < a.tiles && ok; tile += step) {
                    for (int kb = 0; kb < a.blocks; kb++, my_turn = !my_turn) {
                        if (my_turn) {
                            ok = mbar_wait_warp(FULL(st), round, s_abort, a.err) && mbar_wait_warp(ACC_EMPTY(p), p_round ^ 1, s_abort, a.err);
                            if (!ok) break;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint32_t base = smem_u32(ring + st * kStage);
                            const uint64_t adesc = umma_desc(base), wdesc = umma_desc(base + kHalfBytes);
                            if (elect_one()) {
#pragma unroll
                                for (int kk = 0; kk < 4; kk++) umma_f8_pair(tmem_base + p * kN, adesc + kk * 2, wdesc + kk * 2, kk > 0);
                                commit_pair(ACC_FULL(p));
                                commit_pair(EMPTY(st));
                            }
                            __syncwarp();
                        }
                        if (++st == kStages) st = 0, round ^= 1;
                        if (++p == 2) p = 0, p_round ^= 1;
                    }
                }
            }
        } else {
            // two blocks' scales are asked for at a time, and the next two before these are handed out
            int p = 0;
            uint32_t p_round = 0;
            bool ok = true;
            float now[2][4], next[2][4], now_w[2][2], next_w[2][2];
            for (int tile = first; tile < a.tiles && ok; tile += step) {
                const int t0 = tile % a.m_tiles * kM + rank * 128 + lane, nb = tile / a.m_tiles * 2;
                const bool second = (nb + 1) * kFp8Block < a.N;
                const float* const sw = a.w_scale + (size_t)nb * a.blocks;
                auto ask = [&](int kb0, float (&v)[2][4], float (&w)[2][2]) {
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const int kb = kb0 + q;
                        w[q][0] = kb < a.blocks ? __ldg(sw + kb) : 0.f;
                        w[q][1] = kb < a.blocks && second ? __ldg(sw + a.blocks + kb) : 0.f;
#pragma unroll
                        for (int j = 0; j < 4; j++) v[q][j] = kb < a.blocks && t0 + 32 * j < a.M ? __ldcg(a.a_scale + (size_t)kb * a.M + t0 + 32 * j) : 0.f;
                    }
                };
                ask(0, now, now_w);
                for (int kb0 = 0; kb0 < a.blocks && ok; kb0 += 2) {
                    ask(kb0 + 2, next, next_w);
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        if (kb0 + q >= a.blocks || !ok) continue;
                        ok = mbar_wait_warp(SLOT_EMPTY(p), p_round ^ 1, s_abort, a.err);
                        if (!ok) continue;
#pragma unroll
                        for (int j = 0; j < 4; j++) slots[p * 130 + lane + 32 * j] = now[q][j];
                        if (lane < 2) slots[p * 130 + 128 + lane] = lane ? now_w[q][1] : now_w[q][0];
                        mbar_arrive_warp(ACC_FULL(p));
                        if (++p == 2) p = 0, p_round ^= 1;
                    }
#pragma unroll
                    for (int q = 0; q < 2; q++) {
#pragma unroll
                        for (int j = 0; j < 4; j++) now[q][j] = next[q][j];
                        now_w[q][0] = next_w[q][0], now_w[q][1] = next_w[q][1];
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
        const int quarter = warp & 3, half = (warp - 4) / 4;
        uint8_t* const mine = out + (warp - 4) * kOutBytes;
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 128;
        const uint32_t release[2] = {in_first_cta(ACC_EMPTY(0)), in_first_cta(ACC_EMPTY(1))};
        int p = 0;
        uint32_t p_round = 0;
        bool ok = true;
        for (int tile = first; tile < a.tiles && ok; tile += step) {
            const int t0 = tile % a.m_tiles * kM + rank * 128 + quarter * 32, n0 = tile / a.m_tiles * kN + half * 128;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; j++) acc[j] = 0.f;
            // 32 columns at a time: one of the two warps of an SM's quarter loads while the other adds (a second buffer and loads ahead
            // of the sums, 64 columns, two sums per instruction, sixteen warps of 64 columns and giving the accumulator back before
            // the last sums were all slower: 262, 424, 305, 275 and 254 us against 243 at 8192 x 8192 x 4096).
            for (int kb = 0; kb < a.blocks; kb++) {
                ok = mbar_wait_warp(ACC_FULL(p), p_round, s_abort, a.err);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float scale = slots[p * 130 + quarter * 32 + lane] * slots[p * 130 + 128 + half];
                float d[32];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    tmem_ld32(taddr + p * kN + c * 32, d);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j++) asm volatile("" : "+f"(d[j]));      // not read in front of the wait
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[c * 32 + j] = fmaf(d[j], scale, acc[c * 32 + j]);
                }
                // (relaxed: what it orders is in tensor memory; a release at cluster scope takes some hundred cycles)
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(release[p]) : "memory");
                    mbar_arrive(SLOT_EMPTY(p));
                }
                if (++p == 2) p = 0, p_round ^= 1;
            }
            if (!ok) break;
            if (t0 >= a.M || n0 >= a.N) continue;
            // Out through shared memory, 256 bytes of every token at a time: lanes hold a token each, rows in memory want neighbours.
            // 16-byte pieces are placed by the 128-byte swizzle, which keeps the lanes on different banks.
            auto piece = [&](int row, int j) { return reinterpret_cast<uint4*>(mine + (j >> 3) * 4096 + row * 128 + (((j & 7) ^ (row & 7)) << 4)); };
            auto wait_read = [&]() {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
            };
            if (a.c_dtype == 0) {
                wait_read();
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(acc[8 * j + 2 * q], acc[8 * j + 2 * q + 1]);
                        w[q] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    *piece(lane, j) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                send_out(a, &tmap_c, mine, t0, n0, 2, lane);
            } else {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    wait_read();
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        *piece(lane, j) = make_uint4(__float_as_uint(acc[64 * r + 4 * j]), __float_as_uint(acc[64 * r + 4 * j + 1]),
                                                     __float_as_uint(acc[64 * r + 4 * j + 2]), __float_as_uint(acc[64 * r + 4 * j + 3]));
                    send_out(a, &tmap_c, mine, t0, n0 + 64 * r, 4, lane);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    // neither CTA leaves while the other's products may read its operands or its barriers be arrived at
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    fp8_settle(s_abort);
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
}

// c [M, N] with rows ldc apart, box = 32 tokens by 128 bytes, 128-byte swizzle
bool out_map(CUtensorMap* map, void* c, int dtype, int M, int N, long long ldc) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const int elem = dtype == 0 ? 2 : 4;
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    cuuint64_t strides[1] = {(cuuint64_t)ldc * elem};
    cuuint32_t box[2] = {(cuuint32_t)(128 / elem), 32};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, c, dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

int launch_fp8_pair(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, int M, int N, int K, void* out, int out_dtype,
                    long long ldc, int sm_count, int32_t* err, cudaStream_t s) {
    PairArgs g{};
    g.a_scale = a_scale; g.w_scale = w_scale; g.M = M; g.N = N; g.blocks = (K + kFp8Block - 1) / kFp8Block;
    g.m_tiles = (M + kM - 1) / kM;
    g.tiles = g.m_tiles * ((N + kN - 1) / kN);
    g.c = out; g.c_dtype = out_dtype; g.ldc = ldc; g.err = err;
    const int elem = out_dtype == 0 ? 2 : 4;
    const uint64_t starts = reinterpret_cast<uintptr_t>(out) | (uint64_t)(ldc * elem);
    // (a row that ends within 16 bytes: the copy would write them whole, though the map ends with the row)
    g.c_by_tma = starts % 16 == 0 && (int64_t)N * elem % 16 == 0;
    g.c_by_8 = starts % 8 == 0;
    CUtensorMap map_a, map_w, map_c{};
    if (!fp8_codes_map(&map_a, a, M, K, 128) || !fp8_codes_map(&map_w, w, N, K, 128)) return -(int)cudaErrorInvalidValue;
    if (g.c_by_tma && !out_map(&map_c, out, out_dtype, M, N, ldc)) return -(int)cudaErrorInvalidValue;
    static PerDeviceOnce once;
    cudaError_t e = allow_dyn_smem(once, fp8_pair_kernel, kSmem);
    if (e != cudaSuccess) return -(int)e;
    e = launch_pdl(fp8_pair_kernel, dim3(2 * max(1, min(g.tiles, sm_count / 2))), dim3(kThreads), kSmem, s, map_a, map_w, map_c, g);
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace ftm
