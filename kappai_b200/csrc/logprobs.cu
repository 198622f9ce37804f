// Of each row of logits: the log probability of a given token and how many tokens have a larger logit, the row's entropy, and the `top` tokens
// with the largest logits (equal ones: the lowest index) with their log probabilities.
//
// With m = max x, S = sum e^(x - m) and W = sum e^(x - m) (x - m):  log p = (x - m) - log S,  entropy = log S - W / S.  One pass over the row
// carries (m, S, W) a thread, rescaled when the thread's maximum grows, in float32 (differences to the maximum are bounded below at -10^4, where the
// exponential is 0: a logit of -inf adds nothing, and 0 * inf does not arise).
//
// The alternatives need no second pass over the row.  A thread's values are a subset of the row; the top-th largest of the threads' maxima is a bound
// below which no alternative lies, so only the subsets whose maximum reaches it (`top` of them) are read again, from L2, and the values that reach
// the bound, few more than `top`, are put in order by counting.  Values are compared together with their index, as one 64-bit number: no two are
// equal, and equal logits do not make more candidates.  Logits that crowd in few subsets can make more than there is room for; then the
// alternatives are found one after the other.
//
// Few rows are shared out over clusters of up to 8 CTAs, which hand their sums and candidates to the first one through its shared memory.  Bound by reading the
// logits once.
#include <cooperative_groups.h>

#include "common.cuh"

namespace cg = cooperative_groups;

#define LP_THREADS 256
#define LP_MAX_TOP 32
#define LP_CAND 1024
#define LP_LEAST (-1e4f)

typedef unsigned long long u64;

struct LpArgs {
    const void* logits; long long ld; int n, V, top;
    const int* ids;
    float* logprob; float* entropy; int* rank; int* top_ids; float* top_logprobs;
};

// (value, index) as a number that orders as the value does, of equal values the lower index first; both zeros alike
__device__ __forceinline__ u64 lp_key(float x, int i) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return ((u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (unsigned)~i;
}
__device__ __forceinline__ float lp_value(u64 k) {
    const unsigned b = (unsigned)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int lp_index(u64 k) { return (int)~(unsigned)k; }

__device__ __forceinline__ float lp_max_nan(float a, float b) {      // NaN if either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

template <typename T> struct LpVec { static constexpr int N = 16 / sizeof(T); };
__device__ __forceinline__ void lp_unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void lp_unpack(const uint4& v, float (&f)[8]) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

// running sums relative to a maximum
struct LpSums {
    float m, s, w;
    __device__ __forceinline__ void to(float m2) {                   // relative to m2 >= m
        const float d = fmaxf(m - m2, LP_LEAST), c = __expf(d);
        w = (w + s * d) * c;
        s *= c;
        m = m2;
    }
    __device__ __forceinline__ void add(float x) {
        const float d = lp_max_nan(x - m, LP_LEAST), e = __expf(d);
        s += e;
        w = fmaf(e, d, w);
    }
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_logprobs_kernel(const LpArgs p) {
    kp_pdl_begin();
    constexpr int N = LpVec<T>::N;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ float red[LP_THREADS / 32];
    __shared__ float red2[2][LP_THREADS / 32];
    __shared__ int redi[LP_THREADS / 32];
    __shared__ float s_sums[3];                                      // of this CTA's part, read by the cluster's first CTA
    __shared__ int s_count;
    __shared__ u64 s_best[LP_THREADS];                               // the threads' largest
    __shared__ u64 s_cand[LP_CAND];
    __shared__ u64 s_sel[LP_MAX_TOP];                                // the part's alternatives in order (0: there are no more)
    __shared__ u64 s_bound;
    __shared__ int s_subset[LP_THREADS], s_n_subset, s_n_cand;

    const T* x = (const T*)p.logits + (long long)row * p.ld;
    const int V = p.V, id_ = p.ids ? p.ids[row] : -1;
    const int id = id_ >= 0 && id_ < V ? id_ : -1;
    const float mine = id >= 0 ? to_f32(x[id]) : INFINITY;           // (no logit is larger)
    // the row: a few values up to a 16-byte boundary, pieces of 16 bytes, a few values
    const int head = min(V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
    const int n_vec = (V - head) / N, tail0 = head + n_vec * N;
    const int v0 = (int)((long long)n_vec * part / C), v1 = (int)((long long)n_vec * (part + 1) / C);
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    int single = -1;                                                 // the value before or behind the pieces that this thread looks at
    if (part == 0) {
        if (tid < head) single = tid;
        else if (tid >= 8 && tid - 8 < V - tail0) single = tail0 + tid - 8;
    }

    LpSums a = {-3.402823466e38f, 0.f, 0.f};
    float best = -INFINITY;                                          // the thread's largest, and where it is: a piece, -2 the single value, -1 nowhere yet
    int best_at = -1, count = 0;
    auto one = [&]() {
        const float v = to_f32(x[single]);
        if (v > best) { best = v; best_at = -2; if (v > a.m) a.to(v); }
        a.add(v);
        count += v > mine;
    };
    if (single >= 0 && single < head) one();
    auto piece = [&](const uint4& q, int v) {
        float f[N];
        lp_unpack(q, f);
        float m = f[0];
#pragma unroll
        for (int j = 1; j < N; j++) m = fmaxf(m, f[j]);
        if (m > best) {
            best = m;
            best_at = v;
            if (m > a.m) a.to(m);
        }
#pragma unroll
        for (int j = 0; j < N; j++) { a.add(f[j]); count += f[j] > mine; }
    };
    int v = v0 + tid;
    for (; v + 3 * LP_THREADS < v1; v += 4 * LP_THREADS) {
        uint4 q[4];
#pragma unroll
        for (int u = 0; u < 4; u++) q[u] = __ldg(xv + v + u * LP_THREADS);
#pragma unroll
        for (int u = 0; u < 4; u++) piece(q[u], v + u * LP_THREADS);
    }
    for (; v < v1; v += LP_THREADS) piece(__ldg(xv + v), v);
    if (single >= head) one();

    // ---- the CTA's sums
    const float M = block_max(a.m, red);
    a.to(M);
    {
        const float s = warp_sum(a.s), w = warp_sum(a.w);
        const int c = __reduce_add_sync(0xffffffffu, count);
        if (lane == 0) { red2[0][warp] = s; red2[1][warp] = w; redi[warp] = c; }
    }
    if (tid == 0) { s_n_subset = 0; s_n_cand = 0; s_bound = 0; }
    const int top = p.top;
    // a thread's largest value with its index; 0 where it has none
    u64 key = 0;
    if (top) {
        if (best_at == -2) key = lp_key(best, single);
        else if (best_at >= 0 || v0 + tid < v1) {
            // (the first of the piece that is as large; where all are -inf the first of the first piece)
            const int at = best_at >= 0 ? best_at : v0 + tid;
            float f[N];
            lp_unpack(__ldg(xv + at), f);
            int j = N - 1;
#pragma unroll
            for (int i = N - 2; i >= 0; i--) if (f[i] == best) j = i;
            key = lp_key(best, head + at * N + j);
            if (best_at < 0 && single >= 0 && single < head) key = lp_key(best, single);
        } else if (single >= 0) key = lp_key(best, single);
        s_best[tid] = key;
        if (tid < LP_MAX_TOP) s_sel[tid] = 0;
    }
    __syncthreads();
    if (tid == 0) {
        float s = 0.f, w = 0.f;
        int c = 0;
#pragma unroll
        for (int i = 0; i < LP_THREADS / 32; i++) { s += red2[0][i]; w += red2[1][i]; c += redi[i]; }
        s_sums[0] = M; s_sums[1] = s; s_sums[2] = w; s_count = c;
    }
    if (top) {
        // ---- the subsets that can hold alternatives, and the bound
        int above = 0;
        const ulonglong2* b2 = reinterpret_cast<const ulonglong2*>(s_best);
#pragma unroll 8
        for (int i = 0; i < LP_THREADS / 2; i++) { const ulonglong2 b = b2[i]; above += (b.x > key) + (b.y > key); }
        const bool reaches = key && above < top;
        if (reaches) s_subset[atomicAdd(&s_n_subset, 1)] = tid;
        if (key && above == top - 1) s_bound = key;                  // (fewer maxima: no bound)
        __syncthreads();
        const u64 bound = s_bound;
        auto take = [&](float f, int i) {
            const u64 k = lp_key(f, i);
            if (k >= bound) { const int at = atomicAdd(&s_n_cand, 1); if (at < LP_CAND) s_cand[at] = k; }
        };
        if (reaches && single >= 0) take(to_f32(x[single]), single);
        const int n_sub = s_n_subset, per = (v1 - v0 + LP_THREADS - 1) / LP_THREADS;
        for (int i = tid; i < n_sub * per; i += LP_THREADS) {
            const int at = v0 + s_subset[i / per] + (i % per) * LP_THREADS;
            if (at >= v1) continue;
            float f[N];
            lp_unpack(__ldg(xv + at), f);
#pragma unroll
            for (int j = 0; j < N; j++) if (lp_key(f[j], head + at * N + j) >= bound) take(f[j], head + at * N + j);
        }
        __syncthreads();
        const int n_cand = s_n_cand;
        if (n_cand <= LP_CAND) {
            for (int i = tid; i < n_cand; i += LP_THREADS) {
                const u64 k = s_cand[i];
                int before = 0;
                for (int j = 0; j < n_cand; j++) before += s_cand[j] > k;
                if (before < top) s_sel[before] = k;
            }
        } else {
            // ---- more candidates than there is room for: one alternative after the other, the largest below the last one
            u64 last = ~0ull;
            for (int t = 0; t < top; t++) {
                u64 k = 0;
                auto look = [&](float f, int i) { const u64 c = lp_key(f, i); if (c < last && c > k) k = c; };
                if (single >= 0) look(to_f32(x[single]), single);
                for (int at = v0 + tid; at < v1; at += LP_THREADS) {
                    float f[N];
                    lp_unpack(__ldg(xv + at), f);
#pragma unroll
                    for (int j = 0; j < N; j++) look(f[j], head + at * N + j);
                }
                __syncthreads();
                s_best[tid] = k;
                __syncthreads();
                if (warp == 0) {
#pragma unroll
                    for (int i = 1; i < LP_THREADS / 32; i++) k = max(k, s_best[i * 32 + lane]);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
                    if (lane == 0) { s_sel[t] = k; s_bound = k; }
                }
                __syncthreads();
                last = s_bound;
            }
        }
    }
    __syncthreads();

    // ---- the row's, from its parts'
    if (C > 1) {
        cluster.sync();
        if (part) {
            cluster.sync();                                          // (its shared memory is read until then)
            return;
        }
    }
    LpSums z = {s_sums[0], s_sums[1], s_sums[2]};
    int rank = s_count;
    for (int i = 1; i < C; i++) {
        const float* o = cluster.map_shared_rank(s_sums, i);
        LpSums b = {o[0], o[1], o[2]};
        const float m = fmaxf(z.m, b.m);
        z.to(m);
        b.to(m);
        z.s += b.s;
        z.w += b.w;
        rank += *cluster.map_shared_rank(&s_count, i);
    }
    const float log_s = logf(z.s);
    const bool bad = !(z.s >= 0.f), none = z.s == 0.f;               // a NaN or +inf among the logits; nothing but -inf
    auto logprob = [&](float f) { return none ? -INFINITY : (f - z.m) - log_s; };
    if (tid == 0) {
        p.logprob[row] = id >= 0 ? (bad ? z.s : logprob(mine)) : 0.f;
        p.entropy[row] = none ? 0.f : log_s - z.w / z.s;
        p.rank[row] = id >= 0 ? rank : -1;
    }
    if (top) {
        const int n_all = C * top;
        auto put = [&](int place, u64 k) {
            const long long at = (long long)row * top + place;
            p.top_ids[at] = bad ? -1 : lp_index(k);
            p.top_logprobs[at] = bad ? z.s : logprob(lp_value(k));
        };
        if (C == 1) {
            if (tid < top) put(tid, s_sel[tid]);
        } else {
            for (int i = tid; i < n_all; i += LP_THREADS) s_cand[i] = *cluster.map_shared_rank(&s_sel[i % top], i / top);
            __syncthreads();
            for (int i = tid; i < n_all; i += LP_THREADS) {
                const u64 k = s_cand[i];
                int before = 0;
                for (int j = 0; j < n_all; j++) before += s_cand[j] > k;
                if (k && before < top) put(before, k);
            }
        }
    }
    if (C > 1) cluster.sync();
}

extern "C" int kp_token_logprobs(const void* logits, long long ld, const int* ids, int n, int V, int top, int parts, float* logprob, float* entropy,
                                 int* rank, int* top_ids, float* top_logprobs, int dtype, void* stream) {
    if (n < 0 || V < 1 || top < 0 || top > LP_MAX_TOP || top > V || (parts != 1 && parts != 2 && parts != 4 && parts != 8) || n > 2147483647 / 8 ||
        ((uintptr_t)logits & (dtype == KP_DTYPE_F32 ? 3 : 1)))
        return KP_ERR_BAD_ARG;
    if (!n) return 0;
    LpArgs a = {logits, ld, n, V, top, ids, logprob, entropy, rank, top_ids, top_logprobs};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n * parts);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t c;
    KP_DISPATCH_DTYPE(dtype, T, c = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a));
    return c ? (int)c : kp_launch_status();
}
