// Block-scaled 8-bit products on the tcgen05 tensor cores.
//
//   c[t, n] = sum_b (a_scale[b, t] * w_scale[n / 128, b]) * (sum over k in block b of a[t, k] * w[n, k])
//
// A tile is 128 weight rows (one block of weight scales, the tensor memory's lanes) by NT tokens (its columns).  A block of 128 k is one
// 128-byte swizzle atom of either operand and four tcgen05.mma (kind::f8f6f4, exact products, f32 sums) into an accumulator of its own;
// the epilogue warps read it, multiply every column by its scale and add it to sums in registers.  The scales differ from block to
// block, so a sum over all of k cannot stay in tensor memory; with four accumulators the next blocks are multiplied meanwhile.
//   warp 0      TMA: weight box [128 rows x 128 k], token box [NT x 128 k]
//   warps 1, 3  issue the products, a block each in turn
//   warp 2      allocates the tensor memory; multiplies the two scales of every (block, token) ahead of the epilogue
//   warps 4..   epilogue: four warps for NT <= 32, eight for 64, sixteen for 128, each four with their share of the columns (eight and
//               two accumulators for NT = 128: 39.5 us against 34.0 at 128 x 65536 x 2048; sixteen for 64: no difference)
// Few tiles: the blocks of k are split over the CTAs of a cluster.  Every CTA stores its sums of the tokens that CTA r finishes into r's
// shared memory, which adds them in the order of the ranks, so the same inputs give the same bits and no scratch in
// global memory is needed.
// FUSED (at most 16 tokens): the rows are still bf16 or f32.  The epilogue warps and four more first quantise the CTA's share of
// them into the swizzled operand layout, while the first weight boxes are on their way; they stay there for all tiles.
// Bound by HBM where the weight is large (8 x 248320 x 2048, f32 out: 84 us, 0.95 of measured HBM), by the rate at which an SM
// fetches both operands from L2 with many tokens (about 42 bytes per clock: 128 x 65536 x 2048 34 us; that is why fp8_pair.cu takes
// over), and by launch and set-up, about 4.5 us, in small calls: 1 x 8192 x 2048 7.2 us, 13 x 2048 x 4096 f32 7.4, 64 x 10240 x 2048 8.2.
// Every wait is bounded; a wait that gives up raises the error flag and the CTA drains.
#include <atomic>
#include <climits>
#include <type_traits>

#include "fp8.cuh"
#include "kernels.cuh"
#include "umma.cuh"

namespace ftm {

namespace {

using namespace umma;

constexpr int kRows = 128;                       // weight rows of a tile
constexpr int kWBytes = kRows * kFp8Block;       // a weight box
constexpr int kMaxStages = 12, kMaxAcc = 4, kMaxSplit = 8;
// The issuers take the blocks in turn.  One that waits for block b has to know that the box a ring before has come, or it may take that
// one's phase of the barrier for its own.  It knows of what the epilogue has finished, which is all up to b - 4.
constexpr int kMinStages = 4;
static_assert(kMinStages >= kMaxAcc, "an issuer knows of the box a ring before");
constexpr size_t kWholeSm = 227 * 1024;          // what one CTA can have
constexpr int kMostFused = 64;                   // blocks of k that a CTA keeps codes of
constexpr int kBarBytes = 512;

__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// address of the same shared memory in another CTA of the cluster
__device__ __forceinline__ uint32_t map_shared_to(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// a store into another CTA's shared memory that counts its bytes on a barrier there: no fence, and who waits sees the values
__device__ __forceinline__ void remote_store(uint32_t addr, const float* v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "r"(__float_as_uint(v[0])),
                 "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_join() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ bool cluster_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
    for (uint32_t i = 0; i < kSpin; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
    }
    *abort_flag = 1;
    atomicExch(err, 3);
    return false;
}

// a place in a ring of n and the parity of the round
struct Ring {
    int n, i = 0;
    uint32_t round = 0;
    __device__ __forceinline__ explicit Ring(int size) : n(size) {}
    __device__ __forceinline__ void next() {
        if (++i == n) i = 0, round ^= 1;
    }
};

struct Fp8Args {
    const void* x;               // FUSED: the rows
    long long x_stride;
    int x_dtype, x_vec;
    const float* a_scale;        // [blocks, M]
    const float* w_scale;        // [ceil(N / 128), blocks]
    int M, N, K, blocks;
    int t_tiles, tiles;          // tiles = t_tiles * ceil(N / 128)
    int stages;
    void* c;
    int c_dtype;
    long long ldc;
    int32_t* err;
};

template <int NT, bool FUSED>
struct Shape {
    static constexpr int kEpi = NT >= 128 ? 16 : NT >= 64 ? 8 : 4;      // epilogue warps
    static constexpr int kHelp = FUSED ? 4 : 0;                  // more warps that quantise
    static constexpr int kThreads = 128 + 32 * (kEpi + kHelp);
    static constexpr int kCols = NT * 4 / kEpi;                  // columns of one epilogue warp
    static constexpr int kAcc = 4;                               // accumulators (and slots of scales)
    static constexpr int kTmem = NT * kAcc < 32 ? 32 : NT * kAcc;
    static constexpr int kABytes = NT * kFp8Block;               // a token box
    static constexpr int kPerSm = NT <= 32 ? 2 : 1;              // CTAs of an SM
    static constexpr size_t kSmem = kPerSm == 2 ? 113 * 1024 : kWholeSm;
    static constexpr int kStage = kWBytes + (FUSED ? 0 : kABytes);
    // (after the ring: FUSED codes; sums from the cluster's CTAs [ranks][groups of tokens][128] x 4; slots of scales; FUSED scales)
    // groups of four tokens that one CTA of a cluster finishes, and what they take of its shared memory
    static constexpr __host__ __device__ int share(int split) { return (NT / 4 + split - 1) / split; }
    static constexpr __host__ __device__ int sum_floats(int split) { return share(split) * split * 4 * kRows; }
    static constexpr size_t bytes(int stages, int split, int fused_blocks) {
        return 1024 + (size_t)stages * kStage + (FUSED ? (size_t)fused_blocks * (kABytes + NT * 4) : 0) + (split > 1 ? (size_t)sum_floats(split) * 4 : 0) +
               kAcc * NT * 4 + kBarBytes;
    }
    // What a CTA gets that multiplies `mine` blocks of k: as long a ring as there is room for beside a second CTA, or, where that
    // would be too short (FUSED with many blocks' codes to keep), with the SM to itself.
    struct Fit {
        int stages, per_sm;
    };
    static constexpr Fit fit(int split, int mine) {
        const int fused_blocks = FUSED ? mine : 0;
        const bool shared = bytes(kMinStages, split, fused_blocks) <= kSmem;
        int stages = kMaxStages;
        while (stages > kMinStages && bytes(stages, split, fused_blocks) > (shared ? kSmem : kWholeSm)) stages--;
        return {stages, shared ? kPerSm : 1};
    }
    static constexpr bool always_fits() {
        for (int split = 1; split <= kMaxSplit; split++)
            for (int mine = 1; mine <= (kMostFused + split - 1) / split; mine++)
                if (bytes(fit(split, mine).stages, split, FUSED ? mine : 0) > kWholeSm) return false;
        return true;
    }
};
static_assert(Shape<16, true>::always_fits() && Shape<16, false>::always_fits() && Shape<32, false>::always_fits() && Shape<64, false>::always_fits() &&
                  Shape<128, false>::always_fits(),
              "the shortest ring fits beside everything else");

template <int NT, bool FUSED>
__global__ void __launch_bounds__(Shape<NT, FUSED>::kThreads, (Shape<NT, FUSED>::kPerSm))
fp8_umma_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a, const Fp8Args a, const int split) {
    using S = Shape<NT, FUSED>;
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);   // e4m3 x e4m3 -> f32
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int rank = split > 1 ? (int)cluster_rank() : 0;
    const int kb0 = a.blocks * rank / split, kb1 = a.blocks * (rank + 1) / split, nkb = kb1 - kb0;
    const int max_nkb = (a.blocks + split - 1) / split;
    uint8_t* const codes = ring + (size_t)a.stages * S::kStage;                          // FUSED [max_nkb][NT x 128]
    float* const sums = reinterpret_cast<float*>(codes + (FUSED ? (size_t)max_nkb * S::kABytes : 0));
    float* const slots = sums + (split > 1 ? S::sum_floats(split) : 0);                            // [kAcc][NT]
    float* const row_scales = slots + S::kAcc * NT;                                      // FUSED [max_nkb][NT]
    uint64_t* const bars = reinterpret_cast<uint64_t*>(row_scales + (FUSED ? max_nkb * NT : 0));
    const uint32_t bar0 = smem_u32(bars);
    auto FULL = [&](int s) { return bar0 + 8u * s; };
    auto EMPTY = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
    auto ACC_FULL = [&](int p) { return bar0 + 8u * (2 * kMaxStages + p); };
    auto ACC_EMPTY = [&](int p) { return bar0 + 8u * (2 * kMaxStages + kMaxAcc + p); };
    const uint32_t SUM_FULL = bar0 + 8u * (2 * kMaxStages + 2 * kMaxAcc);
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 2 * kMaxAcc + 4);
    volatile int* const s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int first = blockIdx.x / split, step = gridDim.x / split;
    auto load = [&](int st, int tile, int kb) {
        const uint32_t dst = smem_u32(ring + st * S::kStage);
        mbar_expect_tx(FULL(st), S::kStage);      // what a box reads past the matrix is zero and counts all the same
        tma_load_2d(dst, &tmap_w, kb * kFp8Block, tile / a.t_tiles * kRows, FULL(st));
        if (!FUSED) tma_load_2d(dst + kWBytes, &tmap_a, kb * kFp8Block, tile % a.t_tiles * NT, FULL(st));
    };
    const int early = min(2, nkb);         // blocks of the first tile that are asked for before the CTA is set up
    if (warp == 0) {
        if (lane < a.stages) mbar_init(FULL(lane), 1), mbar_init(EMPTY(lane), 1);
        if (lane < S::kAcc) mbar_init(ACC_FULL(lane), 2), mbar_init(ACC_EMPTY(lane), S::kEpi);
        if (lane == 0) {
            mbar_init(SUM_FULL, 1);
            *s_abort = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
        pdl_wait();
        if (elect_one())
            for (int i = 0; i < early; i++) load(i, first, kb0 + i);
        __syncwarp();
    }
    if (warp != 0) pdl_wait();      // (no tensor memory is held while the kernel before may still want some)
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_tmem)), "n"(S::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (FUSED && warp >= 4) {
        const int etid = threadIdx.x - 128;
        // sixteen lanes quantise one block of one row, eight elements each, into its place of the swizzled operand; all of a
        // pass's rows are asked for before the first is used
        constexpr int kGroups = 2 * (S::kEpi + S::kHelp), kAtOnce = 4;
        const int piece = lane % 16, units = nkb * a.M;
        const uint32_t by_m = 65536u / a.M + 1;      // (w * by_m) >> 16 = w / M for w < 65536 / M
        auto quantise = [&](auto* x) {
            using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
            for (int w0 = etid / 32 * 2; w0 < units; w0 += kGroups * kAtOnce) {
                Fp8Eight<T> f[kAtOnce];
                float sc[kAtOnce];
                uint2 q[kAtOnce];
                int at[kAtOnce], row[kAtOnce];
#pragma unroll
                for (int u = 0; u < kAtOnce; u++) {
                    const int w = w0 + lane / 16 + u * kGroups, i = (w * by_m) >> 16, r = w - i * a.M, k = (kb0 + i) * kFp8Block + piece * 8;
                    at[u] = i, row[u] = r;
                    fp8_load8(x + r * a.x_stride + k, a.x_vec, w < units ? a.K - k : 0, f[u]);
                }
                fp8_encode(f, q, sc);
#pragma unroll
                for (int u = 0; u < kAtOnce; u++) {
                    if (w0 + lane / 16 + u * kGroups >= units) continue;
                    *reinterpret_cast<uint2*>(codes + at[u] * S::kABytes + row[u] * 128 + (((piece >> 1) ^ (row[u] & 7)) << 4) + (piece & 1) * 8) = q[u];
                    if (piece == 0) row_scales[at[u] * NT + row[u]] = sc[u];
                }
            }
        };
        if (a.x_dtype == 0) quantise(reinterpret_cast<const __nv_bfloat16*>(a.x));
        else quantise(reinterpret_cast<const float*>(a.x));
        // rows past M are zero
        for (int w = etid; w < nkb * (NT * 8); w += 32 * (S::kEpi + S::kHelp))
            if (w / 8 % NT >= a.M) *reinterpret_cast<uint4*>(codes + w * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the tensor core reads these bytes
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // Two barriers of the cluster.  The first: every CTA runs and has its barriers before another one reaches into its shared
    // memory (waited for before the first sums are sent).  The second: none leaves while another may still reach into it.
    if (split > 1) cluster_arrive();
    pdl_launch_dependents();
    const uint32_t tmem_base = *s_tmem;
    bool joined = split == 1, left = split == 1;      // this thread has waited for the first, has arrived at the second

    if (warp == 0) {
        Ring st(a.stages);
        bool ok = true;
        uint32_t asked = 0;
        for (int tile = first; tile < a.tiles && ok; tile += step) {
            for (int kb = kb0; kb < kb1; kb++, st.next(), asked++) {
                if (asked < (uint32_t)early) continue;
                ok = mbar_wait_warp(EMPTY(st.i), st.round ^ 1, s_abort, a.err);
                if (!ok) break;
                if (elect_one()) load(st.i, tile, kb);
                __syncwarp();
            }
        }
    } else if (warp == 1 || warp == 3) {
        // two issuers take the blocks in turn: what a wait and the issue cost one of them passes while the other issues
        Ring st(a.stages), p(S::kAcc);
        bool ok = true, my_turn = warp == 1;
        for (int tile = first; tile < a.tiles && ok; tile += step) {
            for (int i = 0; i < nkb; i++, st.next(), p.next(), my_turn = !my_turn) {
                if (!my_turn) continue;
                ok = mbar_wait_warp(ACC_EMPTY(p.i), p.round ^ 1, s_abort, a.err) && mbar_wait_warp(FULL(st.i), st.round, s_abort, a.err);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t wsm = smem_u32(ring + st.i * S::kStage);
                const uint64_t wdesc = umma_desc(wsm), adesc = umma_desc(FUSED ? smem_u32(codes + i * S::kABytes) : wsm + kWBytes);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) umma_f8_ss(tmem_base + p.i * NT, wdesc + kk * 2, adesc + kk * 2, kIdesc, kk > 0);
                    umma_commit(EMPTY(st.i));
                    umma_commit(ACC_FULL(p.i));
                }
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        // slots of scales, four blocks asked for at a time and the next four before these are handed out
        constexpr int kPer = (NT + 31) / 32, kAhead = 4;
        Ring p(S::kAcc);
        bool ok = true;
        float now[kAhead][kPer], next[kAhead][kPer];
        for (int tile = first; tile < a.tiles && ok; tile += step) {
            const int nb = tile / a.t_tiles, t0 = tile % a.t_tiles * NT;
            auto ask = [&](int i0, float (&v)[kAhead][kPer]) {
#pragma unroll
                for (int q = 0; q < kAhead; q++) {
                    const int i = i0 + q;
                    const float ws = i < nkb ? __ldg(a.w_scale + (size_t)nb * a.blocks + kb0 + i) : 0.f;
#pragma unroll
                    for (int j = 0; j < kPer; j++) {
                        const int col = lane + 32 * j, t = t0 + col;
                        float s = 0.f;
                        if (i < nkb && col < NT && t < a.M) s = FUSED ? row_scales[i * NT + col] : __ldcg(a.a_scale + (size_t)(kb0 + i) * a.M + t);
                        v[q][j] = s * ws;
                    }
                }
            };
            ask(0, now);
            for (int i0 = 0; i0 < nkb && ok; i0 += kAhead) {
                ask(i0 + kAhead, next);
#pragma unroll
                for (int q = 0; q < kAhead; q++) {
                    if (i0 + q >= nkb || !ok) continue;
                    ok = mbar_wait_warp(ACC_EMPTY(p.i), p.round ^ 1, s_abort, a.err);
                    if (!ok) continue;
#pragma unroll
                    for (int j = 0; j < kPer; j++)
                        if (lane + 32 * j < NT) slots[p.i * NT + lane + 32 * j] = now[q][j];
                    mbar_arrive_warp(ACC_FULL(p.i));
                    p.next();
                }
#pragma unroll
                for (int q = 0; q < kAhead; q++)
#pragma unroll
                    for (int j = 0; j < kPer; j++) now[q][j] = next[q][j];
            }
        }
    } else if (warp >= 4) {
        const int etid = threadIdx.x - 128, quarter = warp & 3, col0 = (warp - 4) / 4 * S::kCols;
        Ring p(S::kAcc);
        bool ok = true;
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + col0;
        const int row = quarter * 32 + lane;
        for (int tile = first; tile < a.tiles && ok && warp < 4 + S::kEpi; tile += step) {
            const int n0 = tile / a.t_tiles * kRows, t0 = tile % a.t_tiles * NT;
            float acc[S::kCols];
#pragma unroll
            for (int j = 0; j < S::kCols; j++) acc[j] = 0.f;
            for (int i = 0; i < nkb; i++, p.next()) {
                ok = mbar_wait_warp(ACC_FULL(p.i), p.round, s_abort, a.err);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                float d[S::kCols / 16][16];
#pragma unroll
                for (int q = 0; q < S::kCols / 16; q++) tmem_ld16(taddr + p.i * NT + q * 16, d[q]);
                tmem_ld_wait();
                const float4* const sl = reinterpret_cast<const float4*>(slots + p.i * NT + col0);
#pragma unroll
                for (int q = 0; q < S::kCols / 4; q++) {
                    const float4 s = sl[q];
                    const float* const dd = &d[q / 4][q % 4 * 4];
                    acc[4 * q] = fmaf(dd[0], s.x, acc[4 * q]);
                    acc[4 * q + 1] = fmaf(dd[1], s.y, acc[4 * q + 1]);
                    acc[4 * q + 2] = fmaf(dd[2], s.z, acc[4 * q + 2]);
                    acc[4 * q + 3] = fmaf(dd[3], s.w, acc[4 * q + 3]);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                mbar_arrive_warp(ACC_EMPTY(p.i));
            }
            if (!ok) break;
            if (split == 1) {
                // a warp's lanes are neighbouring weight rows: one store is 64 or 128 contiguous bytes of a token's output
                const int cols = n0 + row < a.N ? min(S::kCols, a.M - t0 - col0) : 0;
                const long long base = (long long)(t0 + col0) * a.ldc + n0 + row;
                if (a.c_dtype == 0) {
                    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.c) + base;
#pragma unroll
                    for (int j = 0; j < S::kCols; j++, o += a.ldc)
                        if (j < cols) *o = __float2bfloat16_rn(acc[j]);
                } else {
                    float* o = reinterpret_cast<float*>(a.c) + base;
#pragma unroll
                    for (int j = 0; j < S::kCols; j++, o += a.ldc)
                        if (j < cols) *o = acc[j];
                }
                continue;
            }
            // the cluster's sums (a cluster has one tile): the group of tokens 4 g .. 4 g + 3 belongs to the CTA g / share.  A lane is a
            // weight row, so its four sums of a group are one store of 16 bytes, beside its neighbours'.
            const int share = S::share(split), groups = (min(NT, a.M - t0) + 3) / 4, mine = min(share, groups - rank * share);
            if (etid == 0 && mine > 0) mbar_expect_tx(SUM_FULL, split * mine * kRows * 16);
            cluster_join();
            joined = true;
            const uint32_t my_sums = smem_u32(sums + (rank * share * kRows + row) * 4);
            uint32_t to_sums = 0, to_bar = 0;
            int to = col0 / 4 / share, in_share = col0 / 4 - to * share;
#pragma unroll
            for (int j = 0; j < S::kCols / 4; j++) {
                if (col0 / 4 + j >= groups) break;
                if (j == 0 || in_share == 0) to_sums = map_shared_to(my_sums, to), to_bar = map_shared_to(SUM_FULL, to);
                remote_store(to_sums + in_share * kRows * 16, acc + 4 * j, to_bar);
                if (++in_share == share) in_share = 0, to++;
            }
            __syncwarp();
            cluster_arrive();      // nothing of this warp's goes to another CTA from here on
            left = true;
            if (mine > 0) {
                ok = __all_sync(0xffffffffu, cluster_wait(SUM_FULL, 0, s_abort, a.err));
                if (!ok) break;
                for (int q = etid; q < mine * kRows; q += 32 * S::kEpi) {
                    const int g = q / kRows, n = q % kRows, t = t0 + (rank * share + g) * 4;
                    float4 v[kMaxSplit], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int r = 0; r < kMaxSplit; r++)
                        v[r] = r < split ? reinterpret_cast<const float4*>(sums)[(r * share + g) * kRows + n] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int r = 0; r < kMaxSplit; r++) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
                    if (n0 + n < a.N) {
                        const float out[4] = {sum.x, sum.y, sum.z, sum.w};
                        const size_t at = (size_t)t * a.ldc + n0 + n;
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            if (t + j < a.M) store_act(a.c, a.c_dtype, at + j * a.ldc, out[j]);
                    }
                }
            }
        }
    }
    if (!joined) cluster_join();
    if (!left) cluster_arrive();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (split > 1) cluster_join();
    if (warp == 2) {
        fp8_settle(s_abort);
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "n"(S::kTmem) : "memory");
    }
}

template <int NT, bool FUSED>
cudaError_t prepare() {
    static PerDeviceOnce once;
    return allow_dyn_smem(once, fp8_umma_kernel<NT, FUSED>, kWholeSm);
}

// Clusters of q CTAs that the device holds at a time (SMs are grouped, so eights and sevens leave some of them empty)
template <int NT>
int clusters_at_once(int dev, int q) {
    static std::atomic<int> known[64][kMaxSplit + 1];
    if (dev < 0 || dev >= 64) return 0;
    int n = known[dev][q].load(std::memory_order_relaxed);
    if (n) return n;
    if (prepare<NT, false>() != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(q);
    cfg.blockDim = dim3(Shape<NT, false>::kThreads);
    cfg.dynamicSmemBytes = Shape<NT, false>::kSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = q;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, fp8_umma_kernel<NT, false>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 1;
    }
    known[dev][q].store(max(n, 1), std::memory_order_relaxed);
    return max(n, 1);
}

// CTAs that share a tile's blocks, and what the call then takes by measurement, in ns: its start, the blocks of the busiest SM (of a
// CTA alone there or of several) and the join of a cluster's sums.  (Joins of 6 or 12 blocks of time in the place of 9 for NT = 128: no
// difference over 26 sizes.)
struct Plan {
    int split;
    long long ns;
};
struct Costs {
    int start, alone, several, join, second;      // second: what a second CTA on an SM adds once
};
template <int NT>
constexpr Costs kCosts = NT == 16   ? Costs{2200, 300, 300, 1800, 0}
                         : NT == 32 ? Costs{2200, 325, 210, 1900, 1000}
                         : NT == 64 ? Costs{2660, 345, 345, 2070, 0}
                                    : Costs{3400, 410, 410, 3000, 0};
// One plan for a size, whether the rows are quantised in the kernel or before it: the bits go by the split.
template <int NT>
Plan plan_for(int M, int N, int blocks, int sm_count) {
    using S = Shape<NT, false>;
    constexpr Costs c = kCosts<NT>;
    const long long tiles = (long long)((M + NT - 1) / NT) * ((N + kRows - 1) / kRows);
    Plan best{1, 0};
    int dev = -1;
    if (tiles * 2 <= S::kPerSm * sm_count && cudaGetDevice(&dev) != cudaSuccess) dev = -1;
    for (int q = 1; q <= kMaxSplit && q <= blocks && (q == 1 || tiles * q <= S::kPerSm * sm_count); q++) {
        if (q > 1 && tiles > clusters_at_once<NT>(dev, q)) continue;
        const long long each = (tiles * q + sm_count - 1) / sm_count, mine = (blocks + q - 1) / q;
        const long long ns = c.start + mine * (each > 1 ? c.several * each : c.alone) + (q > 1 ? c.join : 0) + (each > 1 ? c.second : 0);
        if (q == 1 || ns < best.ns) best = {q, ns};
    }
    return best;
}

// The same for pairs of SMs on tiles of 256 x 256, each of which takes `turns` of them.
constexpr long long pair_ns(int blocks, long long turns) { return 6000 + 480ll * blocks * turns; }
static_assert(pair_ns((1 << 30) / kFp8Block, 1) > 4000000000ll, "the most blocks there are");

template <int NT, bool FUSED>
int launch(const uint8_t* codes, const uint8_t* w, Fp8Args a, int sm_count, cudaStream_t s) {
    using S = Shape<NT, FUSED>;
    a.blocks = (a.K + kFp8Block - 1) / kFp8Block;
    a.t_tiles = (a.M + NT - 1) / NT;
    a.tiles = a.t_tiles * ((a.N + kRows - 1) / kRows);
    cudaError_t e = prepare<NT, FUSED>();
    if (e != cudaSuccess) return -(int)e;
    const Plan plan = plan_for<NT>(a.M, a.N, a.blocks, sm_count);
    const int split = plan.split;
    const int mine = (a.blocks + split - 1) / split;
    const typename S::Fit fit = S::fit(split, mine);
    a.stages = fit.stages;
    const size_t smem = S::bytes(a.stages, split, FUSED ? mine : 0);
    CUtensorMap map_w, map_a;
    if (!fp8_codes_map(&map_w, w, a.N, a.K, kRows) || (!FUSED && !fp8_codes_map(&map_a, codes, a.M, a.K, NT))) return -(int)cudaErrorInvalidValue;
    if (FUSED) map_a = map_w;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(split > 1 ? split * a.tiles : min(a.tiles, fit.per_sm * sm_count));
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = split;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = split > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, fp8_umma_kernel<NT, FUSED>, map_w, map_a, a, split);
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace

// FUSED keeps the codes of sixteen rows in shared memory beside the weight ring
bool fp8_fused_supported(int M, int K) { return M <= 16 && K <= kMostFused * kFp8Block; }

// In one kernel every CTA quantises all that it multiplies before its first product and keeps the codes; in two that is done once,
// and the rings are longer.  The second launch costs the host 2.5 us, so two kernels are for where they save the GPU about that:
// more than 160 blocks of one row to quantise, or more than 16 blocks of codes to a CTA (the shortest ring beside them, or the SM to itself) unless
// it has a dozen tiles to spread their quantisation over.
// Rows x weight rows x k, us in one and in two kernels of a graph: one is taken for 1 x 248320 x 2048 79.6, 83.5; 8 x 2048 x 4096
// 6.3, 6.4; 13 x 2048 x 4096 7.4, 6.6; 16 x 2048 x 8192 10.2, 8.2; 1 x 248320 x 4096 154, 162; 8 x 248320 x 2560 100, 105; 1 x 262144 x 2560 98, 107
// (lost: 2 x 230000 x 6144 223, 215); two for 16 x 248320 x 2048 87.7, 84.9; 8 x 248320 x 4096 161, 159; 1 x 151936 x 4096 99, 100; 1 x 40000 x 4096
// 37.0, 35.8; 3 x 40000 x 4096 37.7, 35.2; 1 x 60000 x 8176 96, 79; 16 x 60000 x 2048 29.4, 24.9; 2 x 20000 x 8192 51, 32.
bool fp8_fused_faster(int M, int N, int K, int sm_count) {
    const int blocks = (K + kFp8Block - 1) / kFp8Block, split = plan_for<16>(M, N, blocks, sm_count).split, mine = (blocks + split - 1) / split;
    return mine * M <= 160 && (mine <= 16 || (N + kRows - 1) / kRows >= 12 * sm_count);
}

int launch_fp8_gemm(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, int M, int N, int K, void* out,
                    int out_dtype, long long ldc, int sm_count, int32_t* err, const Ctx& c) {
    Fp8Args g{};
    g.a_scale = a_scale; g.w_scale = w_scale; g.M = M; g.N = N; g.K = K; g.c = out; g.c_dtype = out_dtype; g.ldc = ldc; g.err = err;
    c.begin(K_FP8_GEMM);
    int n;
    const int blocks = (K + kFp8Block - 1) / kFp8Block;
    if (M <= 16) n = launch<16, false>(a, w, g, sm_count, c.s);
    else if (M <= 32) n = launch<32, false>(a, w, g, sm_count, c.s);
    else {
        // Tiles of 32, 64 or 128 tokens, or pairs of SMs on 256, whichever takes the least time: narrow tiles keep more SMs at work on
        // small problems, wide ones fetch less.  Us with 32, 64, 128 and pairs: 64 x 512 x 2048 3.9, 4.6, -, -; 512 x 512 x 512 3.6, 3.8, 4.7, -;
        // 100 x 8192 x 2048 9.5, 8.2, 9.8, -; 512 x 2048 x 2048 9.5, 8.2, 9.7, -; 200 x 8192 x 8192 52.5, 46.9, 29.9, 34.5; 256 x 8192 x 2048
        // 15.8, 14.1, 9.9, 12.8; 700 x 2048 x 4096 -, -, 16.6, 19.3; 400 x 5000 x 2048 -, -, 16.9, 13.0; 1000 x 8192 x 8192 177, 158, -, 68.
        const long long pair_tiles = (long long)((M + 255) / 256) * ((N + 255) / 256), pairs = sm_count / 2;
        const long long ns32 = plan_for<32>(M, N, blocks, sm_count).ns, ns64 = plan_for<64>(M, N, blocks, sm_count).ns;
        const long long ns128 = M > 64 ? plan_for<128>(M, N, blocks, sm_count).ns : LLONG_MAX;
        const long long ns_pair = M > 128 && pairs > 0 ? pair_ns(blocks, (pair_tiles + pairs - 1) / pairs) : LLONG_MAX;
        const long long least = min(min(ns32, ns64), min(ns128, ns_pair));
        n = least == ns_pair ? launch_fp8_pair(a, a_scale, w, w_scale, M, N, K, out, out_dtype, ldc, sm_count, err, c.s)
            : least == ns128 ? launch<128, false>(a, w, g, sm_count, c.s)
            : least == ns64  ? launch<64, false>(a, w, g, sm_count, c.s)
                             : launch<32, false>(a, w, g, sm_count, c.s);
    }
    c.end();
    return n;
}

int launch_fp8_linear(const void* x, int x_dtype, long long x_stride, const uint8_t* w, const float* w_scale, int M, int N, int K, void* out,
                      int out_dtype, long long ldc, int sm_count, int32_t* err, const Ctx& c) {
    Fp8Args g{};
    g.x = x; g.x_stride = x_stride; g.x_dtype = x_dtype; g.x_vec = fp8_rows_aligned(x, x_dtype, x_stride);
    g.w_scale = w_scale; g.M = M; g.N = N; g.K = K; g.c = out; g.c_dtype = out_dtype; g.ldc = ldc; g.err = err;
    c.begin(K_FP8_GEMM);
    const int n = launch<16, true>(nullptr, w, g, sm_count, c.s);
    c.end();
    return n;
}

}  // namespace ftm
