// Log probabilities read off rows of logits: of a given token, with its rank, the row's entropy and the most probable
// alternatives.  One pass over the logits.
//
//   m = max x,  d = x - m,  s = sum e^d,  t = sum e^d d
//   logprob = d_id - log s,   entropy = log s - t / s,
//   rank = #{v : x_v > x_id, or x_v = x_id and v < id},   alternatives in the order (value descending, index ascending)
//
// Every thread keeps m, s and t of what it has read in f32 (pairs of elements in one instruction) and rescales s and t when its
// maximum rises (t gains s * (old - new)); the partial triples are joined over the warp, the CTA and the cluster.
// Differences are clamped at -1e20: an element of -inf adds e^d = 0 times a finite d; NaN and +inf make s a NaN.
//
// Alternatives (n <= 32).  The pass itself only notes the maximum of every warp's part of every tile.  Then every warp publishes
// the largest of its lanes' maxima over the whole row, k of them with 8 k >= n, and the n-th largest of what is published is a
// bound: n elements reach it, so what is below cannot belong to the answer.  The few tiles whose maximum reaches it are read again
// (from L2), the elements that reach it are collected and placed by counting the better ones.  Where ties make them too
// many, every warp keeps its n best as a sorted list over its lanes instead.
//
// Rank: a lane counts in a tile only if its maximum there reaches the token's value; bf16 pairs are compared as they are.
//
// A row is split over the CTAs of a cluster when there are few rows; results meet in the first CTA's shared memory, so
// no workspace in global memory is needed and calls on several streams share nothing.
#include <climits>
#include <cooperative_groups.h>

#include "kernels.cuh"

namespace ftm {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 16;      // more than 8 CTAs need the opt-in of launch_logprobs
constexpr int kVecs = 4;             // 128-bit loads of a thread per tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();
constexpr float kFar = -1e20f;       // differences below this have exponential 0; clamped there, sums of them stay finite
constexpr int kCandidates = 1024;
constexpr int kNotes = 64;           // noted maxima of a warp; longer rows note several tiles together
constexpr int kPublish = 8;          // values that a warp can publish

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
    __device__ __forceinline__ static float get(uint32_t w, int) { return __uint_as_float(w); }
    // how many elements of four words are above v, added to a tile's count
    using Count = int;
    __device__ __forceinline__ static void count_above(const uint4& w, uint32_t v, int& count) {
        const float f = __uint_as_float(v);
        count += (__uint_as_float(w.x) > f) + (__uint_as_float(w.y) > f) + (__uint_as_float(w.z) > f) + (__uint_as_float(w.w) > f);
    }
    __device__ __forceinline__ static int none() { return 0; }
    __device__ __forceinline__ static int total(int count) { return count; }
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
    __device__ __forceinline__ static float get(uint32_t w, int e) { return bf16_bits_to_f32(e ? w >> 16 : w & 0xffffu); }
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

// softmax statistics of what was read: the maximum, the sum of the exponentials and that of e^d d
struct Stats {
    float m = -kInf, s = 0.f, t = 0.f;

    // distance from the maximum `top` that this one is joined under: 0 where nothing was summed (or a NaN, which stays)
    __device__ __forceinline__ float below(float top) const { return m == -kInf ? 0.f : max_nan(m - top, kFar); }
    __device__ __forceinline__ void rise(float mx) {       // the maximum may rise to mx
        if (mx > m) {
            const float d = below(mx), f = ex2(d * kLog2e);
            t = f * (t + s * d);
            s *= f;
            m = mx;
        }
    }
    // the elements of one 128-bit vector; s2 and t2 hold sums of even and odd elements until take()
    template <typename T>
    __device__ __forceinline__ void add(const uint4& v, uint64_t& s2, uint64_t& t2) const {
        const float from = m == -kInf ? 0.f : -m;
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; j += 2 / Word<T>::kElems) {
            const uint64_t x = Word<T>::kElems == 2 ? pair(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u))
                                                    : pair(__uint_as_float(w[j]), __uint_as_float(w[(j + 1) & 3]));
            const float2 y = unpair(add2(x, pair(from, from)));
            const uint64_t d = pair(max_nan(y.x, kFar), max_nan(y.y, kFar));
            const float2 z = unpair(mul2(d, pair(kLog2e, kLog2e)));
            const uint64_t e = pair(ex2(z.x), ex2(z.y));
            s2 = add2(s2, e);
            t2 = fma2(e, d, t2);
        }
    }
    __device__ __forceinline__ void take(uint64_t s2, uint64_t t2) {
        const float2 a = unpair(s2), b = unpair(t2);
        s += a.x + a.y;
        t += b.x + b.y;
    }
    __device__ __forceinline__ void add_one(float x) {
        const float d = max_nan(x - (m == -kInf ? 0.f : m), kFar), e = ex2(d * kLog2e);
        s += e;
        t = fmaf(e, d, t);
    }
    __device__ __forceinline__ void join(float m2, float s2, float t2) {
        Stats o;
        o.m = m2, o.s = s2, o.t = t2;
        const float top = fmaxf(m, m2);
        const float d1 = below(top), d2 = o.below(top);
        const float f1 = ex2(d1 * kLog2e), f2 = ex2(d2 * kLog2e);
        t = f1 * (t + s * d1) + f2 * (t2 + s2 * d2);
        s = f1 * s + f2 * s2;
        m = top;
    }
    __device__ __forceinline__ void join_warp() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o), t2 = __shfl_xor_sync(0xffffffffu, t, o);
            join(m2, s2, t2);
        }
    }
};

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// a warp's sorted list, one entry per lane; empty entries are (-inf, INT_MAX)
struct TopList {
    float v = -kInf;
    int i = INT_MAX;
    float last_v = -kInf;      // the n-th entry, in every lane: an element enters when it is better
    int last_i = -1;           // (nothing that is -inf enters an empty place: those are filled in at the end)

    __device__ __forceinline__ void insert(float x, int at, int n, int lane) {
        const int pos = __popc(__ballot_sync(0xffffffffu, better(v, i, x, at)));
        const float pv = __shfl_up_sync(0xffffffffu, v, 1);
        const int pi = __shfl_up_sync(0xffffffffu, i, 1);
        if (lane > pos) v = pv, i = pi;
        if (lane == pos) v = x, i = at;
        const float lv = __shfl_sync(0xffffffffu, v, n - 1);
        const int li = __shfl_sync(0xffffffffu, i, n - 1);
        last_v = lv;
        last_i = lv == -kInf ? -1 : li;
    }
    // offers one element per lane; below `bound` nothing can belong to the answer
    __device__ __forceinline__ void offer(float x, int at, float bound, int n, int lane) {
        unsigned todo = __ballot_sync(0xffffffffu, x >= bound && better(x, at, last_v, last_i));
        while (todo) {
            const int src = __ffs(todo) - 1;
            insert(__shfl_sync(0xffffffffu, x, src), __shfl_sync(0xffffffffu, at, src), n, lane);
            todo &= todo - 1;
            todo &= __ballot_sync(0xffffffffu, better(x, at, last_v, last_i));
        }
    }
};

// place of entry (w, p) among `lists` sorted lists of n entries
__device__ __forceinline__ int merged_place(const float (*val)[32], const int (*idx)[32], int lists, int n, int w, int p) {
    const float v = val[w][p];
    const int i = idx[w][p];
    int place = p;
    for (int q = 0; q < lists; q++) {
        if (q == w) continue;
        int lo = 0, hi = n;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (better(val[q][mid], idx[q][mid], v, i)) lo = mid + 1;
            else hi = mid;
        }
        place += lo;
    }
    return place;
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
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
logprobs_kernel(LogprobArgs a) {
    using W = Word<T>;
    constexpr int kPer = 4 * W::kElems;           // elements of a 128-bit load
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const long long row = blockIdx.x / parts;
    const T* const x = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, n = a.top_n;

    __shared__ float l_val[kMaxCluster][32];      // sorted lists to be merged: the warps', then the cluster's
    __shared__ int l_idx[kMaxCluster][32];
    __shared__ float m_val[32];                   // this CTA's best
    __shared__ int m_idx[32];
    __shared__ float c_val[kCandidates];          // elements that reached the bound
    __shared__ int c_idx[kCandidates];
    __shared__ int c_count;
    __shared__ float p_stat[kWarps][3], c_stat[3];     // m, s, t
    __shared__ int p_rank[kWarps], c_rank;
    __shared__ int note[kWarps][kNotes];          // (ordered) maxima of a warp's part of one or more tiles
    __shared__ int share[kWarps * kPublish], s_bound;
    for (int q = lane; q < kNotes; q += 32) note[warp][q] = ordered(-kInf);
    if (tid == 0) c_count = 0;
    __syncwarp();      // (a warp's notes are its own until the barrier behind the pass)

    // the given token: a negative id asks for nothing, one past the vocabulary is an error
    long long id = -1;
    if (a.ids) id = a.ids_dtype == 3 ? reinterpret_cast<const long long*>(a.ids)[row] : (long long)reinterpret_cast<const int32_t*>(a.ids)[row];
    const bool wrong = id >= a.vocab, asked = id >= 0 && !wrong;
    const int want = asked ? (int)id : -1;
    const float x_id = asked ? load_logit(x + want) : kInf;
    const bool low_id = asked && !(x_id > -kInf);                 // -inf and NaN count as equals, by index
    // in front of the token an element counts from x_id on, behind it above x_id only
    const float x_id_below = x_id > -kInf ? W::below(x_id) : -kInf;

    // whole 128-bit vectors of the row, and the elements in front of and behind them
    const int head = min((int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)), a.vocab);
    const int vecs = (a.vocab - head) / kPer, tail = a.vocab - head - vecs * kPer;
    const int v0 = (int)((long long)vecs * part / parts), v1 = (int)((long long)vecs * (part + 1) / parts);
    const uint4* const xv = reinterpret_cast<const uint4*>(x + head);

    Stats st;
    int ahead = 0;

    auto collect = [&](float v, int at, float bound) {
        if (v >= bound && v > -kInf) {
            const int place = atomicAdd(&c_count, 1);
            if (place < kCandidates) c_val[place] = v, c_idx[place] = at;
        }
    };
    // the elements outside whole vectors: one per lane of the first CTA's first warp
    const bool extra = part == 0 && warp == 0 && lane < head + tail;
    const int extra_at = lane < head ? lane : a.vocab - tail + (lane - head);
    const float extra_x = extra ? load_logit(x + extra_at) : -kInf;
    if (extra) {
        st.rise(extra_x);
        st.add_one(extra_x);
        if (asked && !low_id) ahead += extra_x > (extra_at < want ? x_id_below : x_id);
    }

    // tiles of this CTA, and how many are noted together
    constexpr int kTileVecs = kThreads * kVecs;
    const int tiles = (v1 - v0 + kTileVecs - 1) / kTileVecs;
    int together = 0;
    while ((tiles - 1) >> together >= kNotes) together++;
    const uint32_t id_word = W::all(low_id ? kInf : x_id), below_word = W::all(low_id ? kInf : x_id_below);
    const float look = asked && !low_id ? x_id : kInf;
    for (int tile = 0; tile < tiles; tile++) {
        const int first = v0 + tile * kTileVecs + tid;
        uint4 r[kVecs];
#pragma unroll
        for (int u = 0; u < kVecs; u++)
            r[u] = first + u * kThreads < v1 ? __ldg(xv + first + u * kThreads) : make_uint4(W::kLowest, W::kLowest, W::kLowest, W::kLowest);
        uint32_t top = W::kLowest;
#pragma unroll
        for (int u = 0; u < kVecs; u++) top = W::larger(top, W::larger(W::larger(r[u].x, r[u].y), W::larger(r[u].z, r[u].w)));
        const float mx = W::largest(top);
        if (n > 0) {
            const int m = __reduce_max_sync(0xffffffffu, ordered(mx));
            if (lane == 0) note[warp][tile >> together] = together ? max(note[warp][tile >> together], m) : m;
        }
        if (mx >= look) {
            typename W::Count count = W::none();
#pragma unroll
            for (int u = 0; u < kVecs; u++) W::count_above(r[u], head + (first + u * kThreads) * kPer < want ? below_word : id_word, count);
            ahead += W::total(count);
        }
        st.rise(mx);
        uint64_t s2 = 0, t2 = 0;
#pragma unroll
        for (int u = 0; u < kVecs; u++) st.template add<T>(r[u], s2, t2);
        st.take(s2, t2);
    }
    if (asked) {
        const int id_vec = want >= head && want < head + vecs * kPer ? (want - head) / kPer : -1;
        if (low_id) {
            // -inf and NaN come behind everything else, by index
            for (int vi = v0 + tid; vi < v1; vi += kThreads)
                for (int e = 0; e < kPer; e++) ahead += load_logit(x + head + vi * kPer + e) > -kInf || head + vi * kPer + e < want;
            if (extra) ahead += extra_x > -kInf || extra_at < want;
        } else if (id_vec >= v0 && id_vec < v1 && (id_vec - v0) % kThreads == tid && head + id_vec * kPer < want) {
            // the token's own vector was counted as in front of it: the token and its equals behind it do not count
            for (int at = want; at < head + (id_vec + 1) * kPer; at++) ahead -= load_logit(x + at) == x_id;
        }
    }

    // ---- warp, CTA, cluster -------------------------------------------------------------------------
    if (n > 0) {
        int u = ordered(st.m);
        const int rounds = min(kPublish, (n + kWarps - 1) / kWarps * 2);
        for (int q = 0; q < kPublish; q++) {
            int best = INT_MIN;
            if (q < rounds) {
                best = __reduce_max_sync(0xffffffffu, u);
                if (lane == __ffs(__ballot_sync(0xffffffffu, u == best)) - 1) u = INT_MIN;
            }
            if (lane == 0) share[warp * kPublish + q] = best;
        }
    }
    st.join_warp();
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (lane == 0) p_stat[warp][0] = st.m, p_stat[warp][1] = st.s, p_stat[warp][2] = st.t, p_rank[warp] = ahead;
    if (tid < 32) m_val[tid] = -kInf, m_idx[tid] = INT_MAX;
    __syncthreads();
    if (warp == kWarps - 1) {
        Stats all;
        int sum = 0;
        if (lane < kWarps) all.m = p_stat[lane][0], all.s = p_stat[lane][1], all.t = p_stat[lane][2], sum = p_rank[lane];
        all.join_warp();
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) c_stat[0] = all.m, c_stat[1] = all.s, c_stat[2] = all.t, c_rank = sum;
    }
    if (n > 0) {
        if (warp == 0) {
            // the n-th largest of the published values (two per lane)
            int u = share[lane], w = share[lane + 32], best = INT_MIN;
            for (int q = 0; q < n; q++) {
                best = __reduce_max_sync(0xffffffffu, max(u, w));
                if (lane == __ffs(__ballot_sync(0xffffffffu, u == best || w == best)) - 1) {
                    if (u == best) u = INT_MIN;
                    else w = INT_MIN;
                }
            }
            if (lane == 0) s_bound = max(best, ordered(-kInf));
        }
        __syncthreads();
        const float bound = from_ordered(s_bound);
        const uint32_t bound_word = W::all(bound);
        for (int g = 0; g <= (tiles - 1) >> together && tiles > 0; g++) {
            if (note[warp][g] < s_bound || note[warp][g] == ordered(-kInf)) continue;
            for (int tile = g << together; tile < min(tiles, (g + 1) << together); tile++)
#pragma unroll 1
                for (int vi = v0 + tile * kTileVecs + tid; vi < min(v1, v0 + (tile + 1) * kTileVecs); vi += kThreads) {
                    const uint4 r = __ldg(xv + vi);
                    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (W::any_reaches(w[j], bound_word)) {
#pragma unroll
                            for (int e = 0; e < W::kElems; e++) collect(W::get(w[j], e), head + vi * kPer + j * W::kElems + e, bound);
                        }
                }
        }
        collect(extra_x, extra_at, bound);
        __syncthreads();
        const int count = c_count;
        if (count <= kCandidates) {
            // an element's place is the number of better ones
            for (int q = tid; q < count; q += kThreads) {
                const float v = c_val[q];
                const int i = c_idx[q];
                int place = 0;
#pragma unroll 4
                for (int o = 0; o < count; o++) place += better(c_val[o], c_idx[o], v, i);
                if (place < n) m_val[place] = v, m_idx[place] = i;
            }
        } else {
            TopList top;
            for (int vi = v0 + warp * 32; vi < v1; vi += kThreads)
                for (int e = 0; e < kPer; e++) {
                    const int at = head + min(vi + lane, v1 - 1) * kPer + e;
                    top.offer(vi + lane < v1 ? load_logit(x + at) : -kInf, at, bound, n, lane);
                }
            top.offer(extra_x, extra_at, bound, n, lane);
            l_val[warp][lane] = top.v, l_idx[warp][lane] = top.i;
            __syncthreads();
            for (int q = tid; q < kWarps * n; q += kThreads) {
                const int place = merged_place(l_val, l_idx, kWarps, n, q / n, q % n);
                if (place < n) m_val[place] = l_val[q / n][q % n], m_idx[place] = l_idx[q / n][q % n];
            }
        }
    }
    if (parts > 1) {
        cluster.sync();
        if (part == 0) {
            for (int q = tid; q < parts * n; q += kThreads) {
                l_val[q / n][q % n] = cluster.map_shared_rank(m_val, q / n)[q % n];
                l_idx[q / n][q % n] = cluster.map_shared_rank(m_idx, q / n)[q % n];
            }
            if (warp == kWarps - 1) {
                Stats one;
                int sum = 0;
                if (lane < parts) {
                    const float* const o = cluster.map_shared_rank(c_stat, lane);
                    one.m = o[0], one.s = o[1], one.t = o[2];
                    sum = *cluster.map_shared_rank(&c_rank, lane);
                }
                one.join_warp();
                sum = __reduce_add_sync(0xffffffffu, sum);
                if (lane == 0) p_stat[0][0] = one.m, p_stat[0][1] = one.s, p_stat[0][2] = one.t, p_rank[0] = sum;
            }
        }
        cluster.sync();       // the others' shared memory has been read
        if (part != 0) return;
        for (int q = tid; q < parts * n; q += kThreads) {
            const int place = merged_place(l_val, l_idx, parts, n, q / n, q % n);
            if (place < n) m_val[place] = l_val[q / n][q % n], m_idx[place] = l_idx[q / n][q % n];
        }
    } else if (tid == kThreads - 32) {
        p_stat[0][0] = c_stat[0], p_stat[0][1] = c_stat[1], p_stat[0][2] = c_stat[2];
        p_rank[0] = c_rank;
    }
    __syncthreads();

    // ---- results ------------------------------------------------------------------------------------
    if (warp != 0) return;
    const float m = p_stat[0][0], total = p_stat[0][1], t = p_stat[0][2];
    const bool broken = total != total, empty = !broken && m == -kInf;
    const float log_s = empty ? 0.f : logf(total);
    const float nan = __int_as_float(0x7fffffff);
    auto prob = [&](float v) { return broken ? nan : empty ? -kInf : (v - m) - log_s; };
    if (lane == 0) {
        if (wrong) atomicExch(a.bad_flag, 1);
        if (a.logprob) a.logprob[row] = wrong ? nan : asked ? prob(x_id) : 0.f;
        const float h = log_s - t / total;
        if (a.entropy) a.entropy[row] = broken ? nan : empty || h < 0.f ? 0.f : h;
        if (a.rank) a.rank[row] = asked ? p_rank[0] : -1;
    }
    if (n > 0) {
        float v = lane < n ? m_val[lane] : -kInf;
        int i = lane < n ? m_idx[lane] : INT_MAX;
        // fewer than n elements above -inf: the lowest indices of the others follow.  They are within the first 64.
        const int have = __popc(__ballot_sync(0xffffffffu, lane < n && i != INT_MAX));
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

template <typename T>
cudaError_t launch(const LogprobArgs& a, int rows, int parts, cudaStream_t s) {
    static PerDeviceOnce once;
    if (parts > 8) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(once.mask.load(std::memory_order_acquire) & bit)) {
            e = cudaFuncSetAttribute(logprobs_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return e;
            once.mask.fetch_or(bit, std::memory_order_release);
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)rows * parts);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, a);
}

}  // namespace

int launch_logprobs(const void* logits, int dtype, int rows, int vocab, long long stride, const void* ids, int ids_dtype, int top_n,
                    float* logprob, float* entropy, int32_t* rank, int32_t* top_ids, float* top_logprobs, int sm_count,
                    int32_t* bad_flag, const Ctx& c) {
    LogprobArgs a{logits, stride, vocab, ids, ids_dtype, top_n, logprob, entropy, rank, top_ids, top_logprobs, bad_flag};
    // CTAs per row: as many as keep every SM at four, each with a tile of its own at least
    int parts = 1;
    const int tile = kThreads * kVecs * (dtype == 0 ? 8 : 4);
    while (parts < kMaxCluster && (long long)rows * parts * 2 <= 4ll * sm_count && vocab / (parts * 2) >= tile) parts *= 2;
    c.begin(K_LOGPROBS);
    const cudaError_t e = dtype == 0 ? launch<__nv_bfloat16>(a, rows, parts, c.s) : launch<float>(a, rows, parts, c.s);
    c.end();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace ftm
