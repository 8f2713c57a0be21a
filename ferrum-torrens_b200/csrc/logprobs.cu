// Log probabilities read off rows of logits: of a given token, with its rank, the row's entropy and the most probable
// alternatives.  One pass over the logits.
//
//   m = max x,  d = x - m,  s = sum e^d,  t = sum e^d d
//   logprob = d_id - log s,   entropy = log s - t / s,
//   rank = #{v : x_v > x_id, or x_v = x_id and v < id},   alternatives in the order (value descending, index ascending)
//
// Every thread keeps s and t of what it has read in f32 (pairs of elements in one instruction), and rescales them when its warp's
// maximum rises (t gains s * (old - new)); the partial sums are joined over the warp, the CTA and the cluster.
// Differences are clamped: an element of -inf adds e^d = 0 times a finite d; a NaN makes s a NaN.
//
// Alternatives (n <= 32).  The pass itself only notes the maximum of every warp's part of every tile.  The lanes' maxima, some
// taken together, give 64 values, and the n-th largest of these is a bound: n elements reach it, so what is below
// cannot belong to the answer.  The tiles whose maximum reaches it are read again (from L2 mostly), the elements that reach it
// are collected and placed by counting the better ones.  Where ties make them too many, every warp keeps its n best as
// a sorted list over its lanes instead.
//
// Rank: a lane counts in a tile only if its maximum there reaches the token's value; bf16 pairs are compared as they are.
//
// Rows of small batches are split over the CTAs of a cluster, so that every SM loads; results are sent to the first CTA's shared
// memory, so no workspace in global memory is needed and calls on several streams share nothing.
//
// Bound by instruction issue and the exponentials' unit where there are rows for all SMs (999 x 248320 bf16, one alternative: 104 us,
// 4760 GB/s, 0.74 of measured HBM; 512 x 248320 f32 5600 GB/s; 4096 x 32003 bf16, 20 alternatives: 81 us), by the passage from the last
// load to the results, about 5 us, in single waves (64 x 248320 f32, 5 alternatives: 18 us; one row, 20 alternatives: 10 us).  Through
// a ring in shared memory filled by bulk copies the same rows took 176 and 109 us.
#include <cfloat>
#include <climits>

#include "kernels.cuh"

namespace ftm {

namespace {

constexpr int kMaxCluster = 16;      // more than 8 CTAs need the opt-in of launch_logprobs
constexpr int kVecs = 4;             // 128-bit words of a lane per tile
constexpr int kWarpVecs = 32 * kVecs;        // 128-bit words of a warp per tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();
constexpr float kFar = -1e20f;       // differences below this have exponential 0; clamped there, sums of them stay finite
constexpr float kLarge = 4e6f;       // maxima below this in magnitude: products with log2(e) are below 2^23, so f32 has the whole number next to them
constexpr int kCandidates = 512;
constexpr int kNotes = 64;           // noted maxima of a warp; longer parts note several tiles together
constexpr uint32_t kSpin = 1u << 24; // looks at a barrier before a wait is given up (a part full of ties takes some ms longer than the others)

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// the larger one, or a NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// two floats in one register pair, added and multiplied together
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// whole numbers in the order of the floats
__device__ __forceinline__ int ordered(float f) {
    const int i = __float_as_int(f);
    return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// One 32-bit word of a row: one f32 or two bf16.
template <typename T>
struct Word;
template <>
struct Word<float> {
    static constexpr int kElems = 1;
    static constexpr uint32_t kLowest = 0xff800000u;      // -inf
    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    __device__ __forceinline__ static float largest(uint32_t w) { return __uint_as_float(w); }
    __device__ __forceinline__ static uint32_t all(float v) { return __float_as_uint(v); }
    __device__ __forceinline__ static bool any_reaches(uint32_t w, uint32_t v) { return __uint_as_float(w) >= __uint_as_float(v); }
    // one bit for each element of four words that is v or more
    __device__ __forceinline__ static uint32_t reaching(const uint4& w, uint32_t v) {
        return any_reaches(w.x, v) | any_reaches(w.y, v) << 1 | any_reaches(w.z, v) << 2 | any_reaches(w.w, v) << 3;
    }
    // elements of a word that are v become -inf and are counted, in each half of `taken`
    __device__ __forceinline__ static void take_out(uint32_t& w, uint32_t v, uint32_t& taken) {
        if (__uint_as_float(w) == __uint_as_float(v)) w = kLowest, taken++;
    }
    using Count = uint64_t;
    __device__ __forceinline__ static float above(uint32_t w, float v) {
        float r;
        asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(w)), "f"(v));
        return r;
    }
    // how many elements of four words are above v, added to a tile's counts of even and odd elements
    __device__ __forceinline__ static void count_above(const uint4& w, uint32_t v, uint64_t& count) {
        const float f = __uint_as_float(v);
        count = add2(count, add2(pair(above(w.x, f), above(w.y, f)), pair(above(w.z, f), above(w.w, f))));
    }
    __device__ __forceinline__ static uint64_t none() { return 0; }
    __device__ __forceinline__ static int total(uint64_t count) {
        const float2 c = unpair(count);
        return (int)(c.x + c.y);
    }
    // the largest value below v (not -inf): what is above it is v or more
    __device__ __forceinline__ static float below(float v) { return nextafterf(v, -kInf); }
};
template <>
struct Word<__nv_bfloat16> {
    static constexpr int kElems = 2;
    static constexpr uint32_t kLowest = 0xff80ff80u;
    __device__ __forceinline__ static __nv_bfloat162 as2(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hmax2(as2(a), as2(b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ static float largest(uint32_t w) {
        const float2 f = bf16x2_to_f32(w);
        return fmaxf(f.x, f.y);
    }
    __device__ __forceinline__ static uint32_t all(float v) { return (__float_as_uint(v) >> 16) * 0x10001u; }      // (v is a bf16 value)
    __device__ __forceinline__ static bool any_reaches(uint32_t w, uint32_t v) { return __hge2_mask(as2(w), as2(v)) != 0; }
    __device__ __forceinline__ static uint32_t reaching(const uint4& w, uint32_t v) {
        const uint32_t a = __hge2_mask(as2(w.x), as2(v)) & 0x00020001u, b = __hge2_mask(as2(w.y), as2(v)) & 0x00080004u;
        const uint32_t c = __hge2_mask(as2(w.z), as2(v)) & 0x00200010u, d = __hge2_mask(as2(w.w), as2(v)) & 0x00800040u;
        const uint32_t m = a | b | c | d;
        return (m | m >> 16) & 0xffu;
    }
    __device__ __forceinline__ static uint64_t both(uint32_t w) { return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    // the larger of each, or a NaN where w is one
    __device__ __forceinline__ static uint32_t at_least(uint32_t w, uint32_t v) {
        const __nv_bfloat162 r = __hmax2_nan(as2(w), as2(v));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    __device__ __forceinline__ static void take_out(uint32_t& w, uint32_t v, uint32_t& taken) {
        const uint32_t same = __heq2_mask(as2(w), as2(v));
        w = (w & ~same) | (kLowest & same);
        taken += same & 0x10001u;
    }
    using Count = __nv_bfloat162;      // (a tile's counts of even and odd elements are whole numbers that a bf16 holds)
    __device__ __forceinline__ static void count_above(const uint4& w, uint32_t v, __nv_bfloat162& count) {
        count = __hadd2(count, __hadd2(__hadd2(__hgt2(as2(w.x), as2(v)), __hgt2(as2(w.y), as2(v))), __hadd2(__hgt2(as2(w.z), as2(v)), __hgt2(as2(w.w), as2(v)))));
    }
    __device__ __forceinline__ static __nv_bfloat162 none() { return __floats2bfloat162_rn(0.f, 0.f); }
    __device__ __forceinline__ static int total(__nv_bfloat162 count) { return (int)__low2float(count) + (int)__high2float(count); }
    __device__ __forceinline__ static float below(float v) {
        const uint32_t b = __float_as_uint(v) >> 16;
        return bf16_bits_to_f32(b == 0 || b == 0x8000u ? 0x8001u : b & 0x8000u ? b + 1 : b - 1);
    }
};

// Softmax statistics of what was read: the maximum m, the sum of the exponentials and that of e^d d, in powers of two:
//   z = x log2(e) - c,  s = sum 2^z,  t = sum 2^z z      c = m log2(e) rounded to a whole number
// so that z is one multiply-add, and a tile whose maximum rises less than that changes nothing.  (Where m is so large that c, the rounded
// product, would be far from m log2(e), z is (x - m) log2(e).)  The elements that made the maximum rise are counted in `ones` and left out of s: beside them a small s would lose its
// last places, and the logarithm of a sum close to one element (a token that is all but certain) with them.
struct Stats {
    float m = -kInf, s = 0.f, t = 0.f;
    int ones = 0;

    __device__ __forceinline__ bool near() const { return fabsf(m) < kLarge; }
    __device__ __forceinline__ float whole() const { return rintf(m * kLog2e); }
    // z of the maximum
    __device__ __forceinline__ float own() const { return near() ? fmaf(m, kLog2e, -whole()) : 0.f; }
    // the maximum rises to mx (the lanes of a warp share theirs)
    __device__ __forceinline__ void rise(float mx) {
        const float from = m, z = own(), e = (float)ones * ex2(z), all = s + e;
        m = mx;
        const float d = (from == -kInf ? 0.f : max_nan((from - mx) * kLog2e, kFar)) + (own() - z), f = ex2(d);
        t = f * (fmaf(e, z, t) + all * d);
        s = f * all;
        ones = 0;
    }
    __device__ __forceinline__ static void add_two(uint64_t z, uint64_t& s2, uint64_t& t2) {
        const float2 v = unpair(z);
        const uint64_t e = pair(ex2(v.x), ex2(v.y));
        s2 = add2(s2, e);
        t2 = fma2(e, z, t2);
    }
    __device__ __forceinline__ static uint64_t clamped(uint64_t z) {
        const float2 v = unpair(z);
        return pair(max_nan(v.x, kFar), max_nan(v.y, kFar));
    }
    // the elements of one tile
    template <typename T>
    __device__ __forceinline__ void add(const uint4 (&r)[kVecs]) {
        using W = Word<T>;
        uint64_t s2 = 0, t2 = 0;
        if (near()) {
            const uint64_t c = pair(-whole(), -whole()), by = pair(kLog2e, kLog2e);
            // what is this far below m has exponential 0 (and -inf times 0 would be a NaN)
            const uint32_t lowest = W::all(m - fmaxf(200.f, fabsf(m) * 0.03125f));
#pragma unroll
            for (int u = 0; u < kVecs; u++) {
                const uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
#pragma unroll
                for (int j = 0; j < 4; j += 2 / W::kElems) {
                    if constexpr (W::kElems == 2) add_two(fma2(W::both(W::at_least(w[j], lowest)), by, c), s2, t2);
                    else add_two(clamped(fma2(pair(__uint_as_float(w[j]), __uint_as_float(w[j + 1])), by, c)), s2, t2);
                }
            }
        } else {
            const float from = m == -kInf ? 0.f : -m;
#pragma unroll
            for (int u = 0; u < kVecs; u++) {
                const uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
#pragma unroll
                for (int j = 0; j < 4; j += 2 / W::kElems) {
                    uint64_t x;
                    if constexpr (W::kElems == 2) x = W::both(w[j]);
                    else x = pair(__uint_as_float(w[j]), __uint_as_float(w[j + 1]));
                    add_two(mul2(clamped(add2(x, pair(from, from))), pair(kLog2e, kLog2e)), s2, t2);
                }
            }
        }
        const float2 a = unpair(s2), b = unpair(t2);
        s += a.x + a.y;
        t += b.x + b.y;
    }
    __device__ __forceinline__ void add_one(float x) {
        const float z = max_nan(near() ? fmaf(x, kLog2e, -whole()) : (x - (m == -kInf ? 0.f : m)) * kLog2e, kFar), e = ex2(z);
        s += e;
        t = fmaf(e, z, t);
    }
    // the lanes' statistics joined, in every lane
    __device__ __forceinline__ void join_warp() {
        const float top = from_ordered(__reduce_max_sync(0xffffffffu, ordered(m)));
        if (!(m == top)) rise(top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
        }
        ones = __reduce_add_sync(0xffffffffu, ones);
    }
};

// An element as one whole number, larger for what comes first: the value in the order of the floats (the two zeros as one),
// then the lower index.  0 is no element.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    return (uint64_t)((uint32_t)ordered(v + 0.f) ^ 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t k) { return from_ordered((int)((uint32_t)(k >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

// A warp's n best elements, sorted, one per lane (0: none yet).
struct TopList {
    uint64_t k = 0, last = 0;      // last: the n-th entry, in every lane

    // offers one element per lane (0: none)
    __device__ __forceinline__ void offer(uint64_t e, int n, int lane) {
        unsigned todo = __ballot_sync(0xffffffffu, e > last);
        while (todo) {
            const uint64_t x = __shfl_sync(0xffffffffu, e, __ffs(todo) - 1);
            const int pos = __popc(__ballot_sync(0xffffffffu, k > x));
            const uint64_t up = __shfl_up_sync(0xffffffffu, k, 1);
            if (lane > pos) k = up;
            if (lane == pos) k = x;
            last = __shfl_sync(0xffffffffu, k, n - 1);
            todo &= todo - 1;
            todo &= __ballot_sync(0xffffffffu, e > last);
        }
    }
};

// how many of `count` different keys are larger than k; `keys` has room for one key more and is aligned to 16 bytes
__device__ __forceinline__ int larger_than(const uint64_t* keys, int count, uint64_t k) {
    int place = 0;
#pragma unroll 4
    for (int o = 0; o < count; o += 2) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(keys + o);
        place += (v.x > k) + (int)((v.y > k) & (o + 1 < count));
    }
    return place;
}

// The best n <= 32 of up to 32 sorted lists (0 ends one), by one warp, which gets them in its lanes: n times the best of the heads.
// (Code that runs once per row is kept short: what it takes to fetch its instructions is most of its time.)
__device__ __forceinline__ uint64_t merge_lists(const uint64_t (*list)[32], int lists, int n, int lane) {
    int at = 0;
    uint64_t head = lane < lists ? list[lane][0] : 0, mine = 0;
#pragma unroll 1
    for (int q = 0; q < n; q++) {
        const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32));
        const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(head >> 32) == high ? (uint32_t)head : 0u);
        const uint64_t best = (uint64_t)high << 32 | low;
        if (lane == q) mine = best;
        if (head == best) {
            at++;
            head = at < n && lane < lists ? list[lane][at] : 0;
        }
    }
    return mine;
}

// ---- sending results to the first CTA of the cluster -------------------------------------------
__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
// a store into another CTA's shared memory that counts its bytes on a barrier there
__device__ __forceinline__ void send(uint32_t to, uint32_t v, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to), "r"(v), "r"(bar) : "memory");
}

// bounded wait for a phase of a barrier in this CTA's shared memory
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpin; i++) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

struct LogprobArgs {
    const void* logits;
    long long stride;
    int vocab;
    const void* ids;
    int ids_dtype;
    int top_n;
    float* logprob;
    float* entropy;
    int32_t* rank;
    int32_t* top_ids;
    float* top_logprobs;
    int32_t* bad_flag;
    int32_t* err;
};

template <typename T, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 32 / kWarps)
logprobs_kernel(LogprobArgs a, int parts) {
    using W = Word<T>;
    constexpr int kPer = 4 * W::kElems;           // elements of a 128-bit word
    constexpr int kThreads = kWarps * 32, kTileVecs = kWarps * kWarpVecs;
    const long long row = blockIdx.x / parts;
    const int part = blockIdx.x - (int)row * parts;        // (a cluster is one row's CTAs, in their order)
    const T* const x = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, n = a.top_n;

    __shared__ __align__(8) uint64_t arrived;     // first CTA: counts the bytes the others send
    __shared__ uint64_t lists[kMaxCluster][32];   // first CTA: the best of every CTA of the cluster
    __shared__ uint32_t c_all[kMaxCluster][5];    // first CTA: m, s, t, rank and ones of every CTA
    __shared__ uint64_t best[32];                 // this CTA's best
    __shared__ __align__(16) uint64_t found[kCandidates];  // elements that reached the bound
    __shared__ int c_count, s_bound;
    __shared__ float p_stat[kWarps][3];           // m, s, t
    __shared__ int p_rank[kWarps], p_ones[kWarps];
    __shared__ int note[kWarps][kNotes];          // (ordered) maxima of a warp's part of one or more tiles
    __shared__ int lane_max[kThreads];            // (ordered)

    // whole 128-bit words of the row, and the elements in front of and behind them
    const int head = min((int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)), a.vocab);
    const int vecs = (a.vocab - head) / kPer, tail = a.vocab - head - vecs * kPer;
    const int each = vecs / parts, more = vecs - each * parts, v0 = part * each + min(part, more), v1 = v0 + each + (part < more);
    const uint4* const xv = reinterpret_cast<const uint4*>(x + head);
    // tiles of this CTA, and how many are noted together
    const int tiles = (v1 - v0 + kTileVecs - 1) / kTileVecs;
    int together = 0;
    while ((tiles - 1) >> together >= kNotes) together++;

    // this warp's share of a tile: words first_of(tile) .. + kWarpVecs, as far as the part goes
    auto first_of = [&](int tile) { return v0 + tile * kTileVecs + warp * kWarpVecs; };
    uint4 next[kVecs];
    auto fetch = [&](int tile) {
        const int first = first_of(tile) + lane;
#pragma unroll
        for (int u = 0; u < kVecs; u++) next[u] = first + u * 32 < v1 ? __ldg(xv + first + u * 32) : make_uint4(W::kLowest, W::kLowest, W::kLowest, W::kLowest);
    };
    fetch(0);      // on its way while the token is looked up
    if (parts > 1) {
        if (tid == 0) {
            const uint32_t bar = shared_addr(&arrived);
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar));
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            if (part == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((parts - 1) * (5 + 2 * n) * 4) : "memory");
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }

    // the given token: a negative id asks for nothing, one past the vocabulary is an error
    long long id = -1;
    if (a.ids) id = a.ids_dtype == 3 ? reinterpret_cast<const long long*>(a.ids)[row] : (long long)reinterpret_cast<const int32_t*>(a.ids)[row];
    const bool wrong = id >= a.vocab, asked = id >= 0 && !wrong;
    const int want = asked ? (int)id : -1;
    const float x_id = asked ? load_logit(x + want) : kInf;
    const bool low_id = asked && !(x_id > -kInf);                 // -inf and NaN count as equals, by index
    // in front of the token an element counts from x_id on, behind it above x_id only
    const float x_id_below = x_id > -kInf ? W::below(x_id) : -kInf;

    for (int q = lane; q < kNotes; q += 32) note[warp][q] = ordered(-kInf);
    if (tid == 0) c_count = 0;
    if (tid < 32) best[tid] = 0;
    Stats st;
    int ahead = 0;
    bool room = true;      // for another candidate (where there is none, this lane stops collecting)
    auto collect = [&](float v, int at, float bound) {
        if (v >= bound && v > -kInf) {
            const int place = atomicAdd(&c_count, 1);
            room = place < kCandidates;
            if (room) found[place] = key_of(v, at);
        }
    };
    // the elements outside whole words: one per lane of the first CTA's first warp
    const bool extra = part == 0 && warp == 0 && lane < head + tail;
    const int extra_at = lane < head ? lane : a.vocab - tail + (lane - head);
    const float extra_x = extra ? load_logit(x + extra_at) : -kInf;
    float lane_m = fmaxf(extra_x, -kInf);      // (a NaN is not a maximum)
    if (extra && asked && !low_id) ahead += extra_x > (extra_at < want ? x_id_below : x_id);
    if (part == 0 && warp == 0) {
        st.m = from_ordered(__reduce_max_sync(0xffffffffu, ordered(lane_m)));
        if (extra && extra_x == st.m && st.m > -kInf) st.ones = 1;
        else if (extra) st.add_one(extra_x);
    }
    __syncwarp();

    const uint32_t id_word = W::all(low_id ? kInf : x_id), below_word = W::all(low_id ? kInf : x_id_below);
    const float look = asked && !low_id ? x_id : kInf;
    for (int tile = 0; tile < tiles; tile++) {
        uint4 r[kVecs];
#pragma unroll
        for (int u = 0; u < kVecs; u++) r[u] = next[u];
        fetch(tile + 1);
        uint32_t top = W::kLowest;
#pragma unroll
        for (int u = 0; u < kVecs; u++) top = W::larger(top, W::larger(W::larger(r[u].x, r[u].y), W::larger(r[u].z, r[u].w)));
        const float mx = W::largest(top);
        lane_m = fmaxf(lane_m, mx);
        const int warp_mx = __reduce_max_sync(0xffffffffu, ordered(mx));
        if (lane == 0) note[warp][tile >> together] = together ? max(note[warp][tile >> together], warp_mx) : warp_mx;
        if (mx >= look) {
            typename W::Count count = W::none();
#pragma unroll
            for (int u = 0; u < kVecs; u++) W::count_above(r[u], head + (first_of(tile) + lane + u * 32) * kPer < want ? below_word : id_word, count);
            ahead += W::total(count);
        }
        const float risen = from_ordered(warp_mx);
        if (risen > st.m) {
            st.rise(risen);
            const uint32_t out = W::all(risen);
            uint32_t taken = 0;
#pragma unroll
            for (int u = 0; u < kVecs; u++) W::take_out(r[u].x, out, taken), W::take_out(r[u].y, out, taken), W::take_out(r[u].z, out, taken), W::take_out(r[u].w, out, taken);
            st.ones = (int)((taken & 0xffffu) + (taken >> 16));
        }
        st.template add<T>(r);
    }
    if (asked) {
        const int id_vec = want >= head && want < head + vecs * kPer ? (want - head) / kPer : -1;
        if (low_id) {
            // -inf and NaN come behind everything else, by index
            const uint32_t finite = W::all(-FLT_MAX);
            for (int vi = v0 + tid; vi < v1; vi += kThreads)
                ahead += __popc(W::reaching(__ldg(xv + vi), finite) | ((1u << min(max(want - head - vi * kPer, 0), kPer)) - 1));
            if (extra) ahead += extra_x > -kInf || extra_at < want;
        } else if (id_vec >= v0 && id_vec < v1 && tid == 0 && head + id_vec * kPer < want) {
            // the token's own word was counted as in front of it: the token and its equals behind it do not count
            for (int at = want; at < head + (id_vec + 1) * kPer; at++) ahead -= load_logit(x + at) == x_id;
        }
    }

    // ---- the CTA's results --------------------------------------------------------------------------
    lane_max[tid] = ordered(lane_m);
    st.join_warp();
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (lane == 0) p_stat[warp][0] = st.m, p_stat[warp][1] = st.s, p_stat[warp][2] = st.t, p_rank[warp] = ahead, p_ones[warp] = st.ones;
    __syncthreads();
    if (warp == kWarps - 1) {
        Stats all;
        int sum = 0;
        if (lane < kWarps) all.m = p_stat[lane][0], all.s = p_stat[lane][1], all.t = p_stat[lane][2], all.ones = p_ones[lane], sum = p_rank[lane];
        all.join_warp();
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) {
            c_all[part][0] = __float_as_uint(all.m), c_all[part][1] = __float_as_uint(all.s), c_all[part][2] = __float_as_uint(all.t);
            c_all[part][3] = (uint32_t)sum, c_all[part][4] = (uint32_t)all.ones;
        }
    }
    if (n > 0) {
        if (warp == 0) {
            // the n-th largest of 64 values, each the largest of some lanes' maxima (of every 64th lane: in a short row one warp may have
            // all the elements), two to a lane here
            int u = INT_MIN, w = INT_MIN;
#pragma unroll
            for (int q = 0; q < kThreads; q += 64) {
                u = max(u, lane_max[q + lane]);
                w = max(w, lane_max[q + 32 + lane]);
            }
            int best = INT_MIN;
#pragma unroll 1
            for (int q = 0; q < n; q++) {
                best = __reduce_max_sync(0xffffffffu, max(u, w));
                if (lane == __ffs(__ballot_sync(0xffffffffu, max(u, w) == best)) - 1) {
                    if (u == best) u = INT_MIN;
                    else w = INT_MIN;
                }
            }
            if (lane == 0) s_bound = best;
        }
        __syncthreads();
        const float bound = from_ordered(s_bound);
        const uint32_t bound_word = W::all(bound);
        for (int g = 0; tiles > 0 && g <= (tiles - 1) >> together && room; g++) {
            // (compared as floats: a tile of -0 reaches a bound of 0, one noted as a NaN is read as well)
            const float most = from_ordered(note[warp][g]);
            if (most < bound || most == -kInf) continue;
            for (int tile = g << together; tile < min(tiles, (g + 1) << together); tile++) {
                fetch(tile);
                uint32_t hit = 0;      // 128-bit words with an element that reaches the bound
#pragma unroll
                for (int u = 0; u < kVecs; u++)
                    hit |= W::any_reaches(W::larger(W::larger(next[u].x, next[u].y), W::larger(next[u].z, next[u].w)), bound_word) ? 1u << u : 0u;
                for (; hit && room; hit &= hit - 1) {
                    const int vi = first_of(tile) + lane + (__ffs(hit) - 1) * 32, at = head + vi * kPer;
                    if (vi >= v1) continue;      // (the fill behind the part's last word reaches a bound of -inf)
                    const uint4 r = __ldg(xv + vi);
                    for (uint32_t m = W::reaching(r, bound_word); m && room; m &= m - 1) {
                        const int e = __ffs(m) - 1;
                        collect(load_logit(x + at + e), at + e, bound);
                    }
                }
            }
        }
        collect(extra_x, extra_at, bound);
        __syncthreads();
        const int count = c_count;
        if (count <= kCandidates) {
            // an element's place is the number of better ones
            for (int q = tid; q < count; q += kThreads) {
                const uint64_t k = found[q];
                const int place = larger_than(found, count, k);
                if (place < n) best[place] = k;
            }
        } else {
            // Ties: every warp keeps its best as a list.  Its tiles come by index, so once the list is full only what is above its
            // last entry can enter, and a tile whose maximum is not is left out unread.
            TopList top;
            float least = -kInf;      // the list's last value once it is full
            for (int g = 0; tiles > 0 && g <= (tiles - 1) >> together; g++) {
                const float most = from_ordered(note[warp][g]);
                if (most < bound || most <= least) continue;
                for (int tile = g << together; tile < min(tiles, (g + 1) << together); tile++) {
                    fetch(tile);
                    uint32_t hit = 0;      // 128-bit words that any lane has something in
#pragma unroll
                    for (int u = 0; u < kVecs; u++) {
                        const float v = W::largest(W::larger(W::larger(next[u].x, next[u].y), W::larger(next[u].z, next[u].w)));
                        hit |= v > least && v >= bound ? 1u << u : 0u;
                    }
                    for (hit = __reduce_or_sync(0xffffffffu, hit); hit; hit &= hit - 1) {
                        const int vi = first_of(tile) + lane + (__ffs(hit) - 1) * 32;
#pragma unroll 1
                        for (int e = 0; e < kPer; e++) {
                            const int at = head + vi * kPer + e;
                            const float v = vi < v1 ? load_logit(x + at) : -kInf;
                            top.offer(v >= bound && v > -kInf ? key_of(v, at) : 0, n, lane);
                        }
                        if (top.last != 0) least = key_value(top.last);
                    }
                }
            }
            top.offer(extra_x >= bound && extra_x > -kInf ? key_of(extra_x, extra_at) : 0, n, lane);
            // (in the place of the candidates; kWarps lists of 32)
            found[tid] = top.k;
            __syncthreads();
            if (lane < n) {
                int place = 0;
                for (int o = 0; o < kWarps; o++)
                    for (int q = 0; q < n; q++) place += found[o * 32 + q] > top.k;
                if (top.k != 0 && place < n) best[place] = top.k;
            }
        }
    }
    __syncthreads();
    if (parts > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");      // the first CTA runs and has its barrier
    if (warp != 0) return;
    if (parts > 1) {
        const uint32_t bar = shared_addr(&arrived);
        if (part != 0) {
            const uint32_t to = in_first_cta(bar);
            if (lane < 5) send(in_first_cta(shared_addr(&c_all[part][lane])), c_all[part][lane], to);
            if (lane < n) {
                const uint32_t at = in_first_cta(shared_addr(&lists[part][lane]));
                send(at, (uint32_t)best[lane], to);
                send(at + 4, (uint32_t)(best[lane] >> 32), to);
            }
            return;
        }
        lists[0][lane] = best[lane];
        if (!__all_sync(0xffffffffu, wait_for(bar, 0))) {
            // Others may still be storing into this CTA: it stays until they have left the kernel (who has does not hold up the barrier;
            // they wait for nothing any more) and, for about a millisecond, for what is on its way from them.
            asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            const long long from = clock64();
            while (clock64() - from < 2000000) {}
            if (lane == 0) atomicExch(a.err, 3);
            return;
        }
        __syncwarp();      // the list of every lane, before one lane reads it
    }
    uint64_t mine = best[lane];
    if (parts > 1 && n > 0) mine = merge_lists(lists, parts, n, lane);
    Stats all;
    int rank = 0;
    if (lane < parts) {
        all.m = __uint_as_float(c_all[lane][0]), all.s = __uint_as_float(c_all[lane][1]), all.t = __uint_as_float(c_all[lane][2]);
        rank = (int)c_all[lane][3], all.ones = (int)c_all[lane][4];
    }
    all.join_warp();
    rank = __reduce_add_sync(0xffffffffu, rank);

    // ---- results ------------------------------------------------------------------------------------
    // in units of the maximum's own exponential, and of e
    const float m = all.m, z = all.own(), unit = ex2(-z), sum = all.s * unit, t = (all.t - z * all.s) * unit * kLn2;
    const float rest = sum + (float)(all.ones - 1), total = sum + (float)all.ones;
    const bool broken = total != total || m == kInf, empty = !broken && m == -kInf;
    const float log_s = empty ? 0.f : log1pf(rest);
    const float nan = __int_as_float(0x7fffffff);
    auto prob = [&](float v) { return broken ? nan : empty ? -kInf : (v - m) - log_s; };
    if (lane == 0) {
        if (wrong) atomicExch(a.bad_flag, 1);
        if (a.logprob) a.logprob[row] = wrong ? nan : asked ? prob(x_id) : 0.f;
        const float h = log_s - t / total;
        if (a.entropy) a.entropy[row] = broken ? nan : empty || h < 0.f ? 0.f : h;
        if (a.rank) a.rank[row] = asked ? rank : -1;
    }
    if (n > 0) {
        const bool real = lane < n && mine != 0;
        const float v = real ? key_value(mine) : -kInf;
        int i = real ? key_index(mine) : INT_MAX;
        // fewer than n elements above -inf: the lowest indices of the others follow.  They are within the first 64.
        const int have = __popc(__ballot_sync(0xffffffffu, real));
        int filled = have;
        for (int base = 0; base < a.vocab && filled < n; base += 32) {
            const int at = base + lane;
            const unsigned low = __ballot_sync(0xffffffffu, at < a.vocab && !(load_logit(x + min(at, a.vocab - 1)) > -kInf));
            const int k = lane - filled;      // this lane takes the k-th of them
            if (k >= 0 && k < __popc(low)) i = base + __fns(low, 0, k + 1);
            filled += __popc(low);
        }
        if (lane < n) {
            const bool none = i == INT_MAX;      // the vocabulary is smaller than n
            a.top_ids[row * n + lane] = none ? -1 : i;
            a.top_logprobs[row * n + lane] = none ? -kInf : prob(v);
        }
    }
}

template <typename T, int kWarps>
cudaError_t launch(const LogprobArgs& a, int rows, int parts, cudaStream_t s) {
    static PerDeviceOnce once_large;
    cudaError_t e;
    if (parts > 8) {
        int dev = 0;
        e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(once_large.mask.load(std::memory_order_acquire) & bit)) {
            e = cudaFuncSetAttribute(logprobs_kernel<T, kWarps>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            once_large.mask.fetch_or(bit, std::memory_order_release);
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)rows * parts);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, kWarps>, a, parts);
}

}  // namespace

int launch_logprobs(const void* logits, int dtype, int rows, int vocab, long long stride, const void* ids, int ids_dtype, int top_n,
                    float* logprob, float* entropy, int32_t* rank, int32_t* top_ids, float* top_logprobs, int sm_count,
                    int32_t* bad_flag, int32_t* err, const Ctx& c) {
    LogprobArgs a{logits, stride, vocab, ids, ids_dtype, top_n, logprob, entropy, rank, top_ids, top_logprobs, bad_flag, err};
    const int elem = dtype == 0 ? 2 : 4;
    // Eight warps to a CTA; four where there are many rows that are short, for more of them at a time and less to join (4096 rows of
    // 32003 bf16: 79 us against 89; 999 rows of 248320 bf16: 117 against 109, both before small sums kept their places)
    const bool narrow = rows > 4 * sm_count && (long long)vocab * elem <= 8 * 8 * kWarpVecs * 16;
    // CTAs per row: as many as keep every SM at 32 warps (clusters of more than eight CTAs do not pack that well: up to one per SM), each
    // with two tiles of its own at least, or with one where it has its SM alone and few alternatives to find.  One row of 248320 f32 with 1, 4,
    // 8 and 16 CTAs: 34.5, 13.3, 9.5, 7.5 us; 64 of them with 2, 4, 8, 12: 29, 21, 20, 27; 300 of 32003 bf16 with 1, 2, 4: 12, 14, 17.
    // Parts of one tile in the place of two: 1 x 17000 f32, 8 alternatives, 5.8 us against 7.3; 32 alternatives of 17000 bf16 9.9, 9.4;
    // 100 x 9000 f32 6.5, 5.9.
    const int tile_bytes = (narrow ? 4 : 8) * kWarpVecs * 16;
    const long long tiles = ((long long)vocab * elem + tile_bytes - 1) / tile_bytes;
    int parts = 1;
    for (int next = 2; next <= kMaxCluster; next++) {
        const long long ctas = (long long)rows * next;
        if (ctas > (next <= 8 ? (narrow ? 8 : 4) * sm_count : sm_count) || tiles < next * (top_n <= 16 && ctas <= sm_count ? 1 : 2)) break;
        parts = next;
    }
    c.begin(K_LOGPROBS);
    const cudaError_t e = dtype == 0 ? (narrow ? launch<__nv_bfloat16, 4>(a, rows, parts, c.s) : launch<__nv_bfloat16, 8>(a, rows, parts, c.s))
                                     : (narrow ? launch<float, 4>(a, rows, parts, c.s) : launch<float, 8>(a, rows, parts, c.s));
    c.end();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace ftm
