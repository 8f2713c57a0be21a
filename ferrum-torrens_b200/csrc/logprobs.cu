// Log probabilities read off rows of logits: of a given token, with its rank, the row's entropy and the most probable
// alternatives.  One pass over the logits.
//
//   m = max x,  s = sum exp(x - m),  t = sum exp(x - m) (x - m)
//   logprob = (x_id - m) - log s,   entropy = log s - t / s,
//   rank = #{v : x_v > x_id, or x_v = x_id and v < id},   alternatives in the order (value descending, index ascending)
//
// Every thread keeps m, s and t of what it has read in f32 and rescales s and t when its maximum rises (t gains s * (old - new));
// the partial triples are joined over the warp, the CTA and the cluster.  A term of -inf adds nothing: its exponential is 0,
// and its difference is clamped before it multiplies that 0.  NaN and +inf make s a NaN.
//
// Alternatives.  Every warp keeps its n best as a list over its lanes (n <= 32), sorted.  An element is looked at only
// when its thread's maximum of the tile beats the warp's own n-th best and reaches a bound that the CTA's warps share:
// each publishes its ceil(n / warps)-th best, and as there are at least n elements no worse than the least of those, what
// is below it cannot belong to the answer.  Published values only rise, so a stale read is a valid bound too.  A warp whose
// tile has many hits first takes the n-th largest of its lanes' maxima as a bound.  The lists are merged by counting:
// an entry's place is its place in its own list plus the number of better entries in every other one.
//
// A row is split over the CTAs of a cluster when there are few rows; results meet in the first CTA's shared memory, so
// no workspace in global memory is needed and calls on several streams share nothing.
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

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 p = bf16x2_to_f32(w[j]);
        f[2 * j] = p.x, f[2 * j + 1] = p.y;
    }
}

// running softmax statistics of one thread
struct Stats {
    float m = -kInf, s = 0.f, t = 0.f;

    __device__ __forceinline__ void rise(float mx) {       // the maximum may rise to mx
        if (mx > m) {
            const float d = m == -kInf ? 0.f : fmaxf(m - mx, kFar);     // nothing was summed while m was -inf (or a NaN, which stays)
            const float c = ex2(d * kLog2e);
            t = c * (t + s * d);
            s *= c;
            m = mx;
        }
    }
    __device__ __forceinline__ void add(float x, float m_finite) {
        const float d = x - m_finite;
        const float e = ex2(d * kLog2e);
        s += e;
        t += e * fmaxf(d, kFar);
    }
    __device__ __forceinline__ float base() const { return m == -kInf ? 0.f : m; }
    __device__ __forceinline__ void join(float m2, float s2, float t2) {
        const float top = fmaxf(m, m2);
        const float d1 = m == -kInf ? 0.f : fmaxf(m - top, kFar), d2 = m2 == -kInf ? 0.f : fmaxf(m2 - top, kFar);
        const float c1 = ex2(d1 * kLog2e), c2 = ex2(d2 * kLog2e);
        t = c1 * (t + s * d1) + c2 * (t2 + s2 * d2);
        s = c1 * s + c2 * s2;
        m = top;
    }
};

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// a warp's sorted list, one entry per lane; empty entries are (-inf, INT_MAX)
struct TopList {
    float v = -kInf;
    int i = 0x7fffffff;
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
    constexpr int kPer = 16 / sizeof(T);          // elements of a 128-bit load
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const long long row = blockIdx.x / parts;
    const T* const x = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, n = a.top_n;

    __shared__ float l_val[kMaxCluster][32];      // lists to be merged: the warps', then the cluster's
    __shared__ int l_idx[kMaxCluster][32];
    __shared__ float m_val[32];                   // this CTA's merged list
    __shared__ int m_idx[32];
    __shared__ float p_stat[kWarps][3], c_stat[3];
    __shared__ int p_rank[kWarps], c_rank;
    __shared__ volatile float share[kWarps];      // every warp's ceil(n / kWarps)-th best
    if (tid < kWarps) share[tid] = -kInf;
    __syncthreads();

    // the given token: a negative id asks for nothing, one past the vocabulary is an error
    long long id = -1;
    if (a.ids) id = a.ids_dtype == 3 ? reinterpret_cast<const long long*>(a.ids)[row] : (long long)reinterpret_cast<const int32_t*>(a.ids)[row];
    const bool wrong = id >= a.vocab, asked = id >= 0 && !wrong;
    const int want = asked ? (int)id : -1;
    const float x_id = asked ? load_logit(x + want) : kInf;
    const bool low_id = asked && !(x_id > -kInf);                 // -inf and NaN count as equals, by index
    // in front of the token an element counts from x_id on, behind it above x_id only
    const float x_id_below = x_id > -kInf ? nextafterf(x_id, -kInf) : -kInf;

    // whole 128-bit vectors of the row, and the elements in front of and behind them
    const int head = min((int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T)), a.vocab);
    const int vecs = (a.vocab - head) / kPer, tail = a.vocab - head - vecs * kPer;
    const int v0 = (int)((long long)vecs * part / parts), v1 = (int)((long long)vecs * (part + 1) / parts);
    const uint4* const xv = reinterpret_cast<const uint4*>(x + head);

    Stats st;
    TopList top;
    int ahead = 0;
    const int share_at = (n + kWarps - 1) / kWarps - 1;

    auto bound_now = [&]() {
        float b = share[lane % kWarps];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) b = fminf(b, __shfl_xor_sync(0xffffffffu, b, o));
        return b;
    };
    auto publish = [&]() {
        const float v = __shfl_sync(0xffffffffu, top.v, share_at);
        if (lane == 0) share[warp] = v;
    };

    for (int base = v0; base < v1; base += kThreads * kVecs) {
        float f[kVecs][kPer];
        float mx = -kInf;
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
            const int vi = base + u * kThreads + tid;
            if (vi < v1) {
                unpack(__ldg(xv + vi), f[u]);
            } else {
#pragma unroll
                for (int e = 0; e < kPer; e++) f[u][e] = -kInf;
            }
        }
#pragma unroll
        for (int u = 0; u < kVecs; u++)
#pragma unroll
            for (int e = 0; e < kPer; e++) mx = fmaxf(mx, f[u][e]);

        st.rise(mx);
        const float m_finite = st.base();
#pragma unroll
        for (int u = 0; u < kVecs; u++)
#pragma unroll
            for (int e = 0; e < kPer; e++) st.add(f[u][e], m_finite);

        // rank: most tiles hold nothing that comes in front of the token
        if (asked && (low_id || mx >= x_id)) {
#pragma unroll
            for (int u = 0; u < kVecs; u++) {
                const int vi = base + u * kThreads + tid;
                const int at = head + vi * kPer;
                if (vi < v1) {
                    if (low_id) {
#pragma unroll
                        for (int e = 0; e < kPer; e++) ahead += (f[u][e] > -kInf) || at + e < want;
                    } else {
#pragma unroll
                        for (int e = 0; e < kPer; e++) ahead += f[u][e] > (at + e < want ? x_id_below : x_id);
                    }
                }
            }
        }
        // alternatives
        if (n > 0) {
            const unsigned hits = __ballot_sync(0xffffffffu, mx > top.last_v);
            if (hits) {
                float bound = bound_now();
                if (__popc(hits) > 8) {
                    int place = 0;
#pragma unroll
                    for (int o = 0; o < 32; o++) place += better(__shfl_sync(0xffffffffu, mx, o), o, mx, lane);
                    const unsigned who = __ballot_sync(0xffffffffu, place == n - 1);
                    bound = fmaxf(bound, __shfl_sync(0xffffffffu, mx, __ffs(who) - 1));
                }
                if (__any_sync(0xffffffffu, mx >= bound && mx > top.last_v)) {
#pragma unroll
                    for (int u = 0; u < kVecs; u++)
#pragma unroll
                        for (int e = 0; e < kPer; e++) top.offer(f[u][e], head + (base + u * kThreads + tid) * kPer + e, bound, n, lane);
                    publish();
                }
            }
        }
    }
    // the elements outside whole vectors: one per lane of the first CTA's first warp
    if (part == 0 && warp == 0 && head + tail > 0) {
        const bool valid = lane < head + tail;
        const int at = lane < head ? lane : a.vocab - tail + (lane - head);
        const float v = valid ? load_logit(x + at) : -kInf;
        st.rise(v);
        st.add(v, st.base());
        if (asked && valid) ahead += low_id ? (v > -kInf || at < want) : v > (at < want ? x_id_below : x_id);
        if (n > 0) top.offer(v, at, bound_now(), n, lane);
    }

    // ---- warp, CTA, cluster -------------------------------------------------------------------------
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, st.m, o), s2 = __shfl_xor_sync(0xffffffffu, st.s, o), t2 = __shfl_xor_sync(0xffffffffu, st.t, o);
        st.join(m2, s2, t2);
        ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    }
    if (lane == 0) {
        p_stat[warp][0] = st.m, p_stat[warp][1] = st.s, p_stat[warp][2] = st.t;
        p_rank[warp] = ahead;
    }
    l_val[warp][lane] = top.v, l_idx[warp][lane] = top.i;
    __syncthreads();
    if (tid == 0) {
        Stats all;
        int sum = 0;
        for (int w = 0; w < kWarps; w++) all.join(p_stat[w][0], p_stat[w][1], p_stat[w][2]), sum += p_rank[w];
        c_stat[0] = all.m, c_stat[1] = all.s, c_stat[2] = all.t;
        c_rank = sum;
    }
    for (int q = tid; q < kWarps * n; q += kThreads) {
        const int place = merged_place(l_val, l_idx, kWarps, n, q / n, q % n);
        if (place < n) m_val[place] = l_val[q / n][q % n], m_idx[place] = l_idx[q / n][q % n];
    }
    if (parts > 1) {
        cluster.sync();
        if (part == 0) {
            for (int q = tid; q < parts * n; q += kThreads) {
                l_val[q / n][q % n] = cluster.map_shared_rank(m_val, q / n)[q % n];
                l_idx[q / n][q % n] = cluster.map_shared_rank(m_idx, q / n)[q % n];
            }
            if (tid == 0) {
                Stats all;
                int sum = 0;
                for (int c = 0; c < parts; c++) {
                    const float* const o = cluster.map_shared_rank(c_stat, c);
                    all.join(o[0], o[1], o[2]);
                    sum += *cluster.map_shared_rank(&c_rank, c);
                }
                p_stat[0][0] = all.m, p_stat[0][1] = all.s, p_stat[0][2] = all.t;
                p_rank[0] = sum;
            }
        }
        cluster.sync();       // the others' shared memory has been read
        if (part != 0) return;
        for (int q = tid; q < parts * n; q += kThreads) {
            const int place = merged_place(l_val, l_idx, parts, n, q / n, q % n);
            if (place < n) m_val[place] = l_val[q / n][q % n], m_idx[place] = l_idx[q / n][q % n];
        }
    } else if (tid == 0) {
        p_stat[0][0] = c_stat[0], p_stat[0][1] = c_stat[1], p_stat[0][2] = c_stat[2];
        p_rank[0] = c_rank;
    }
    __syncthreads();

    // ---- results ------------------------------------------------------------------------------------
    if (warp != 0) return;
    const float m = p_stat[0][0], s = p_stat[0][1], t = p_stat[0][2];
    const bool broken = s != s, empty = !broken && m == -kInf;
    const float log_s = empty ? 0.f : logf(s);
    const float nan = __int_as_float(0x7fffffff);
    auto prob = [&](float v) { return broken ? nan : empty ? -kInf : (v - m) - log_s; };
    if (lane == 0) {
        if (wrong) atomicExch(a.bad_flag, 1);
        if (a.logprob) a.logprob[row] = wrong ? nan : asked ? prob(x_id) : 0.f;
        const float h = log_s - t / s;
        if (a.entropy) a.entropy[row] = broken ? nan : empty || h < 0.f ? 0.f : h;
        if (a.rank) a.rank[row] = asked ? p_rank[0] : -1;
    }
    if (n > 0) {
        float v = lane < n ? m_val[lane] : -kInf;
        int i = lane < n ? m_idx[lane] : 0x7fffffff;
        // fewer than n elements above -inf: the lowest indices of the others follow.  They are within the first 64.
        const int have = __popc(__ballot_sync(0xffffffffu, lane < n && i != 0x7fffffff));
        int filled = have;
        for (int base = 0; base < a.vocab && filled < n; base += 32) {
            const int at = base + lane;
            const unsigned low = __ballot_sync(0xffffffffu, at < a.vocab && !(load_logit(x + min(at, a.vocab - 1)) > -kInf));
            const int k = lane - filled;      // this lane takes the k-th of them
            if (k >= 0 && k < __popc(low)) i = base + __fns(low, 0, k + 1);
            filled += __popc(low);
        }
        if (lane < n) {
            const bool none = i == 0x7fffffff;      // the vocabulary is smaller than n
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
