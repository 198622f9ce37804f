// Of each row of logits: the log probability of a given token and how many tokens have a larger logit, the row's entropy, and the `top` tokens
// with the largest logits (equal ones: the lowest index) with their log probabilities.
//
// With a reference r, S = sum 2^y and W = sum 2^y y, y = (x - r) log2 e:  log p = x - r - ln S,  entropy = ln S - ln 2 W / S.  One pass over the
// row carries (r, S, W) a thread in float32, y as one fma of x with r log2 e: whatever that is rounded to, it is the same for all.  r follows the thread's
// maximum in steps of at least 16: with every new maximum rescaled, some lane of a warp had one at almost every piece.  Pieces with logits so far below
// r that they have no probability (-inf, or the type's lowest value) have y bounded below: 0 * inf does not arise.  References beyond +-1e6, those of rows of
// nothing else among them, take differences x - r instead.  2048 rows of 65536 float32 logits: 85 us, 6.3 TB/s; with 5, 20 and 32 alternatives 99, 108 and 118; one row 4.6 us, 8.5 with alternatives.
//
// The alternatives need no second pass over the row.  A thread's values are a subset of the row, 64 bytes of every 16 KB.  The top-th largest of the maxima of
// four subsets each is a bound below which no alternative lies, so only the subsets that reach it (few more than `top`) are read again, of these the pieces
// that reach it a value a thread, and the values that reach it, few more than `top` again, are put in order by counting, compared together with their index as one 64-bit number: no two are
// equal.  Where many maxima equal the bound (most of the row is masked), they are compared with their indices too, so that equal logits make no more
// candidates.  Logits that crowd in few subsets can make more than there is room for; then the alternatives are found one after the other.
// (A list that logits above a bound so far were put on as they came by made the pass half as long again.)
//
// A warp of its own copies the row, 16 KB at a time, into a ring of four stages (cp.async.bulk), on into the CTA's next row while the alternatives of this one
// are put in order: loads of the threads' own stand still meanwhile.  A share of a row that the ring holds is read again from there.
//
// Few rows are shared out over clusters of up to 8 CTAs, which hand their sums and candidates to the first one through its shared memory.  Bound by reading the
// logits once.  Every mbarrier wait is bounded; one that gives up sets the status word.
#include <cooperative_groups.h>

#include <type_traits>

#include "mma.cuh"

namespace cg = cooperative_groups;

#define LP_THREADS 256                                               // that look at logits; a warp more copies them
#define LP_PIECES 4                                                  // pieces of 16 bytes a thread of a stage
#define LP_STAGE (LP_THREADS * LP_PIECES * 16)
#define LP_STAGES 4
#define LP_CTAS_SM 3                                                 // as many as shared memory allows
#define LP_SMEM_ALONE (128 * 1024)                                   // shared memory of which an SM has room for one, or two
#define LP_SMEM_TWO (96 * 1024)
#define LP_MAX_TOP 32
#define LP_CAND 512
#define LP_LEAST (-1e4f)
#define LP_SLACK 16.0f                                               // by how much a logit passes its thread's reference before that follows: terms are at most e^16

typedef unsigned long long u64;

KP_STATUS_WORD(g_logprobs_status, logprobs)            // 0 ok; 1: a bounded wait gave up

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

// two float32 operations at once
__device__ __forceinline__ float2 lp_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<u64&>(d)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
    return d;
}
__device__ __forceinline__ float2 lp_mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<u64&>(d)) : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)));
    return d;
}
__device__ __forceinline__ float2 lp_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<u64&>(d))
        : "l"(reinterpret_cast<u64&>(a)), "l"(reinterpret_cast<u64&>(b)), "l"(reinterpret_cast<u64&>(c)));
    return d;
}
__device__ __forceinline__ float lp_exp2(float x) {                 // (with subnormal results flushed: what that loses is below 2^-126 of the largest term)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

#define LP_LOG2E 1.4426950408889634f
__device__ __forceinline__ float lp_max3(float a, float b, float c) {        // the largest of three (one instruction on this architecture)
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float lp_min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A reference r: what sums are relative to is 2^(r log2 e), with r log2 e as the fma takes it, `rl`.  Beyond +-1e6 (`wild`) what that is rounded by would no longer
// be small beside the differences, and these are taken themselves instead: r is `sub`, and rl is 0.  All terms of a sum are of one kind: what rl is off by,
// up to 0.06, is put right for the sum as a whole.
struct LpRef {
    float r, sub, rl;
    __device__ __forceinline__ LpRef(float x) {
        const bool wild = !(fabsf(x) <= 1e6f);
        r = x;
        sub = wild ? x : 0.f;
        rl = wild ? 0.f : x * LP_LOG2E;
    }
    __device__ __forceinline__ bool wild() const { return sub != 0.f; }
    __device__ __forceinline__ float y(float x) const { return lp_max_nan(fmaf(x - sub, LP_LOG2E, -rl), LP_LEAST); }
    // by how much less (a power of two) sums count that were relative to `o`, o.r <= r (of either kind: one rounding, of the result)
    __device__ __forceinline__ float from(const LpRef& o) const { return fmaxf(fmaf(o.sub - sub, LP_LOG2E, o.rl - rl), LP_LEAST); }
};
// sums, and what becomes of them when their reference moves by y <= 0
__device__ __forceinline__ void lp_move(float& s, float& w, float y) {
    const float c = lp_exp2(y);
    w = (w + s * y) * c;
    s *= c;
}

__device__ __forceinline__ void lp_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// a CTA's share of a row: a few values up to a 16-byte boundary (part 0), pieces of 16 bytes, a few values (part 0)
template <typename T>
struct LpShare {
    const T* x; const uint4* xv;
    int head, tail0, v0, v1;
    __device__ __forceinline__ LpShare(const LpArgs& p, int row, int part, int C) {
        constexpr int N = LpVec<T>::N;
        x = (const T*)p.logits + (long long)row * p.ld;
        head = min(p.V, (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)));
        const int n_vec = (p.V - head) / N;
        tail0 = head + n_vec * N;
        v0 = (int)((long long)n_vec * part / C);
        v1 = (int)((long long)n_vec * (part + 1) / C);
        xv = reinterpret_cast<const uint4*>(x + head);
    }
    __device__ __forceinline__ int stages() const { return (v1 - v0 + LP_THREADS * LP_PIECES - 1) / (LP_THREADS * LP_PIECES); }
};

// C CTAs (a cluster) a row; the grid's clusters take the rows in turn
template <typename T>
__global__ void __launch_bounds__(LP_THREADS + 32, LP_CTAS_SM)
token_logprobs_kernel(const LpArgs p) {
    kp_pdl_begin();
    constexpr int N = LpVec<T>::N;
    extern __shared__ __align__(128) unsigned char ring[];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), part = (int)cluster.block_rank(), step = gridDim.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ uint64_t s_full[LP_STAGES], s_empty[LP_STAGES];
    __shared__ float red[LP_THREADS / 32];
    __shared__ float red2[2][LP_THREADS / 32];
    __shared__ int redi[LP_THREADS / 32];
    __shared__ float s_sums[3];                                      // of this CTA's part, read by the cluster's first CTA
    __shared__ int s_count;
    __shared__ u64 s_best[LP_THREADS];                               // the threads' largest; then pieces
    static_assert(LP_CAND * 4 <= sizeof(s_best), "");
    __shared__ u64 s_cand[LP_CAND];
    __shared__ u64 s_sel[LP_MAX_TOP];                                // the part's alternatives in order (0: there are no more)
    __shared__ u64 s_bound;
    __shared__ __align__(16) float s_most[LP_THREADS / 4];           // the largest of four threads
    __shared__ int s_subset[LP_THREADS], s_n_subset, s_n_hit, s_n_cand, s_reach;
    __shared__ float s_tau;

    if (tid == 0) {
        for (int i = 0; i < LP_STAGES; i++) { kp_mbar_init(&s_full[i], 1); kp_mbar_init(&s_empty[i], LP_THREADS / 32); }
        kp_mbar_init_fence();
    }
    __syncthreads();

    if (warp == LP_THREADS / 32) {
        // ---- the copies
        bool ok = true;
        int at = 0;                                                  // stages filled so far
        for (int row = blockIdx.x / C; row < p.n && ok; row += step) {
            const LpShare<T> sh(p, row, part, C);
            for (int i = 0; i < sh.stages() && ok; i++, at++) {
                const int st = at % LP_STAGES, from = sh.v0 + i * LP_THREADS * LP_PIECES, bytes = min(LP_THREADS * LP_PIECES, sh.v1 - from) * 16;
                ok = __all_sync(0xffffffffu, kp_mbar_wait_bounded(&s_empty[st], ((at / LP_STAGES) & 1) ^ 1));
                if (ok && lane == 0) {
                    kp_mbar_expect_tx(&s_full[st], bytes);
                    kp_bulk_g2s(ring + st * LP_STAGE, sh.xv + from, bytes, &s_full[st]);
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) atomicExch(&g_logprobs_status, 1);
        if (C > 1) { cluster.sync(); cluster.sync(); }               // (of a cluster every CTA has one row)
        return;
    }

    bool ok = true;
    int at0 = 0;                                                     // stages of the rows before
    for (int row = blockIdx.x / C; row < p.n; row += step) {
    const LpShare<T> sh(p, row, part, C);
    const T* x = sh.x;
    const uint4* xv = sh.xv;
    const int V = p.V, head = sh.head, tail0 = sh.tail0, v0 = sh.v0, v1 = sh.v1, n_stages = sh.stages();
    const int top = p.top;
    const bool held = top && n_stages <= LP_STAGES;                  // the ring keeps the share until the alternatives are found
    const int id_ = p.ids ? p.ids[row] : -1, id = id_ >= 0 && id_ < V ? id_ : -1;
    const float mine = id >= 0 ? to_f32(x[id]) : INFINITY;           // (no logit is larger)
    int single = -1;                                                 // the value before or behind the pieces that this thread looks at
    if (part == 0) {
        if (tid < head) single = tid;
        else if (tid >= 8 && tid - 8 < V - tail0) single = tail0 + tid - 8;
    }

    LpRef ref(-3.402823466e38f);
    float2 s2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);   // the sums, two at a time
    float best = -INFINITY;                                          // the thread's largest, and where it is: a piece, -2 the single value, -1 nowhere yet
    int best_at = -1, count = 0;
    auto refer = [&](float m) {
        if (m > ref.r + LP_SLACK) {
            const LpRef to(m);
            const float y = to.from(ref), c = lp_exp2(y);
            w2 = lp_mul2(lp_fma2(s2, make_float2(y, y), w2), make_float2(c, c));
            s2 = lp_mul2(s2, make_float2(c, c));
            ref = to;
        }
    };
    auto add = [&](float f) {
        const float y = ref.y(f), e = lp_exp2(y);
        s2.x += e;
        w2.x = fmaf(e, y, w2.x);
    };
    auto one = [&]() {
        const float f = to_f32(x[single]);
        if (f > best) { best = f; best_at = -2; }
        refer(f);
        add(f);
        count += f > mine;
    };
    if (single >= 0 && single < head) one();
    // This thread's logits of a stage: 64 bytes in a row (that a share that is read again comes in whole sectors), in an order that has the threads in
    // different banks.  One test of each kind for all of them: a test a piece kept the next piece's arithmetic waiting.
    auto piece_of = [&](int u) { return tid * LP_PIECES + ((u + (tid >> 1)) & (LP_PIECES - 1)); };
    auto pieces = [&](const uint4* q, int v, int u0, auto count_c) {
        constexpr int K = decltype(count_c)::value;
        float f[K * N];
#pragma unroll
        for (int u = 0; u < K; u++) lp_unpack(q[piece_of(u0 + u)], reinterpret_cast<float (&)[N]>(f[u * N]));
        float m = fmaxf(f[0], f[1]), least = fminf(f[0], f[1]);
#pragma unroll
        for (int j = 2; j < K * N; j += 2) { m = lp_max3(m, f[j], f[j + 1]); least = lp_min3(least, f[j], f[j + 1]); }
        best_at = m > best ? v : best_at;
        best = fmaxf(best, m);
        refer(m);
        if (m > mine)
#pragma unroll
            for (int j = 0; j < K * N; j++) count += f[j] > mine;
        if (least < ref.r + LP_LEAST || ref.wild()) {
#pragma unroll
            for (int j = 0; j < K * N; j++) add(f[j]);
        } else {
            const float2 less = make_float2(-ref.rl, -ref.rl), log2e = make_float2(LP_LOG2E, LP_LOG2E);
            float2 t2 = make_float2(0.f, 0.f), x2 = t2;
#pragma unroll
            for (int j = 0; j < K * N; j += 4) {
                const float2 y = lp_fma2(make_float2(f[j], f[j + 1]), log2e, less), e = make_float2(lp_exp2(y.x), lp_exp2(y.y));
                const float2 z = lp_fma2(make_float2(f[j + 2], f[j + 3]), log2e, less), g = make_float2(lp_exp2(z.x), lp_exp2(z.y));
                s2 = lp_add2(s2, e);
                w2 = lp_fma2(e, y, w2);
                t2 = lp_add2(t2, g);
                x2 = lp_fma2(g, z, x2);
            }
            s2 = lp_add2(s2, t2);
            w2 = lp_add2(w2, x2);
        }
    };
    for (int i = 0; i < n_stages; i++) {
        const int st = (at0 + i) % LP_STAGES, v = v0 + i * LP_THREADS * LP_PIECES;
        if (ok && !kp_mbar_wait_bounded(&s_full[st], ((at0 + i) / LP_STAGES) & 1)) ok = false;
        const uint4* q = reinterpret_cast<const uint4*>(ring + st * LP_STAGE);
        if (v + (tid + 1) * LP_PIECES <= v1) pieces(q, i, 0, std::integral_constant<int, LP_PIECES>{});
        else
#pragma unroll 1
            for (int u = 0; u < LP_PIECES; u++) if (v + piece_of(u) < v1) pieces(q, i, u, std::integral_constant<int, 1>{});
        if (!held) {
            __syncwarp();
            if (lane == 0) kp_mbar_arrive(&s_empty[st]);
        }
    }
    // a piece of this CTA's share once more
    auto again = [&](int v) {
        if (!held) return __ldg(xv + v);
        const int i = v - v0;
        return *(reinterpret_cast<const uint4*>(ring + (at0 + i / (LP_THREADS * LP_PIECES)) % LP_STAGES * LP_STAGE) + i % (LP_THREADS * LP_PIECES));
    };
    if (single >= head) one();

    // ---- the CTA's sums
    float M = warp_max(fmaxf(best, -3.402823466e38f));
    if (lane == 0) red[warp] = M;
    lp_sync();
    M = red[lane & 7];
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    {
        float s = s2.x + s2.y, w = w2.x + w2.y;
        lp_move(s, w, LpRef(M).from(ref));
        s = warp_sum(s);
        w = warp_sum(w);
        const int c = __reduce_add_sync(0xffffffffu, count);
        if (lane == 0) { red2[0][warp] = s; red2[1][warp] = w; redi[warp] = c; }
    }
    const bool some = v0 + tid * LP_PIECES < v1 || single >= 0;      // this thread has values
    if (tid == 0) { s_n_subset = 0; s_n_hit = 0; s_n_cand = 0; s_bound = 0; s_tau = -INFINITY; s_reach = 0; }
    if (top) {
        // (NaN where four threads have nothing: no comparison counts it)
        const unsigned any = __ballot_sync(0xffffffffu, some);
        float most = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (!(lane & 3)) s_most[tid >> 2] = (any >> lane) & 15 ? most : __int_as_float(0x7fffffff);
        if (tid < LP_MAX_TOP) s_sel[tid] = 0;
    }
    lp_sync();
    if (tid == 0) {
        float s = 0.f, w = 0.f;
        int c = 0;
#pragma unroll
        for (int i = 0; i < LP_THREADS / 32; i++) { s += red2[0][i]; w += red2[1][i]; c += redi[i]; }
        s_sums[0] = M; s_sums[1] = s; s_sums[2] = w; s_count = c;
    }
    if (top) {
        // ---- the bound: the top-th largest of the maxima (none: there are fewer), and how many reach it; four threads count for one maximum
        {
            const float mx = s_most[tid >> 2];
            int above = 0, reach = 0;
            const float4* q = reinterpret_cast<const float4*>(s_most) + (tid & 3) * (LP_THREADS / 64);
#pragma unroll
            for (int i = 0; i < LP_THREADS / 64; i++) {
                const float4 o = q[i];
                above += (o.x > mx) + (o.y > mx) + (o.z > mx) + (o.w > mx);
                reach += (o.x >= mx) + (o.y >= mx) + (o.z >= mx) + (o.w >= mx);
            }
            above += __shfl_xor_sync(0xffffffffu, above, 1); above += __shfl_xor_sync(0xffffffffu, above, 2);
            reach += __shfl_xor_sync(0xffffffffu, reach, 1); reach += __shfl_xor_sync(0xffffffffu, reach, 2);
            if (above < top && top <= reach) { s_tau = mx; s_reach = reach; }        // (all that write write the same)
        }
        lp_sync();
        const float tau = s_tau;
        u64 low = 0;                                                 // candidates are no less than this
        bool reaches = some && best >= tau;
        if (s_reach > LP_THREADS / 4 - 8) {
            // nearly all maxima equal the bound (a row with few tokens that are not masked, or of few values): the lowest indices of them
            u64 key = 0;                                             // the thread's largest value with its index; 0 where it has none
            if (best_at == -2) key = lp_key(best, single);
            else if (best_at >= 0 || v0 + tid * LP_PIECES < v1) {
                // (the first of a stage that is as large; where all are -inf the first of all)
                const int v = v0 + (max(best_at, 0) * LP_THREADS + tid) * LP_PIECES;
                for (int u = LP_PIECES - 1; u >= 0; u--) {
                    if (v + u >= v1) continue;
                    float f[N];
                    lp_unpack(again(v + u), f);
#pragma unroll
                    for (int i = N - 1; i >= 0; i--) if (f[i] == best) key = lp_key(best, head + (v + u) * N + i);
                }
                if (best_at < 0 && single >= 0 && single < head) key = lp_key(best, single);
            } else if (single >= 0) key = lp_key(best, single);
            s_best[tid] = key;
            lp_sync();
            int above = 0;
#pragma unroll 8
            for (int i = 0; i < LP_THREADS; i++) above += s_best[i] > key;
            reaches = key && above < top;
            if (key && above == top - 1) s_bound = key;              // (fewer maxima: no bound)
            lp_sync();
            low = s_bound;
        } else if (s_reach) low = lp_key(tau, 0x7fffffff);
        const unsigned who = __ballot_sync(0xffffffffu, reaches);
        int first = 0;
        if (lane == 0 && who) first = atomicAdd(&s_n_subset, __popc(who));
        first = __shfl_sync(0xffffffffu, first, 0);
        if (reaches) s_subset[first + __popc(who & ((1u << lane) - 1))] = tid;
        lp_sync();
        auto take = [&](float f, int i) {
            const u64 k = lp_key(f, i);
            if (k >= low) { const int at = atomicAdd(&s_n_cand, 1); if (at < LP_CAND) s_cand[at] = k; }
        };
        if (reaches && single >= 0) take(to_f32(x[single]), single);
        // the threads' shares that reach it, a piece a thread: place i of them is piece i % 4 of stage (i / 4) % n_stages of share i / 4 / n_stages
        const int n_all = s_n_subset * n_stages * LP_PIECES;
        int* s_hit = reinterpret_cast<int*>(s_best);                 // pieces that may have some
        constexpr int U = 4;                                         // pieces under way
        if (n_all) {
            const int d_sub = LP_THREADS / LP_PIECES / n_stages, d_stage = LP_THREADS / LP_PIECES - d_sub * n_stages;
            int sub = tid / LP_PIECES / n_stages, stage = tid / LP_PIECES - sub * n_stages;
            for (int i0 = tid; i0 < n_all; i0 += U * LP_THREADS) {
                uint4 q[U];
                int at[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    at[u] = i0 + u * LP_THREADS < n_all ? v0 + (stage * LP_THREADS + s_subset[sub]) * LP_PIECES + (tid & (LP_PIECES - 1)) : v1;
                    q[u] = at[u] < v1 ? again(at[u]) : make_uint4(0, 0, 0, 0);
                    sub += d_sub;
                    stage += d_stage;
                    if (stage >= n_stages) { stage -= n_stages; sub++; }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float f[N];
                    lp_unpack(q[u], f);
                    float m = f[0];
#pragma unroll
                    for (int j = 1; j < N; j++) m = fmaxf(m, f[j]);
                    // (as if the largest were the piece's first)
                    if (at[u] < v1 && lp_key(m, head + at[u] * N) >= low) { const int h = atomicAdd(&s_n_hit, 1); if (h < LP_CAND) s_hit[h] = at[u]; }
                }
            }
            lp_sync();
            // ... and those once more, a value a thread: where they were found a place for each of a thread's values made so much code that fetching it took
            // longest (592 rows of 100003 16-bit logits, 32 alternatives: 68 us, 45 so)
            const int n_hit = s_n_hit;
            if (n_hit <= LP_CAND)
#pragma unroll 1
                for (int i = tid; i < n_hit * N; i += LP_THREADS) {
                    const int v = s_hit[i / N];
                    take(to_f32(held ? *(reinterpret_cast<const T*>(ring + (at0 + (v - v0) / (LP_THREADS * LP_PIECES)) % LP_STAGES * LP_STAGE) + (v - v0) % (LP_THREADS * LP_PIECES) * N + i % N)
                                     : x[head + v * N + i % N]), head + v * N + i % N);
                }
            else if (tid == 0) s_n_cand = LP_CAND + 1;
        }
        lp_sync();
        const int n_cand = s_n_cand;
        if (n_cand <= LP_CAND) {
            for (int i = tid; i < n_cand; i += LP_THREADS) {
                const u64 k = s_cand[i];
                int before = 0;
#pragma unroll 4
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
                    lp_unpack(again(at), f);
#pragma unroll
                    for (int j = 0; j < N; j++) look(f[j], head + at * N + j);
                }
                lp_sync();
                s_best[tid] = k;
                lp_sync();
                if (warp == 0) {
#pragma unroll
                    for (int i = 1; i < LP_THREADS / 32; i++) k = max(k, s_best[i * 32 + lane]);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
                    if (lane == 0) { s_sel[t] = k; s_bound = k; }
                }
                lp_sync();
                last = s_bound;
            }
        }
    }
    lp_sync();
    if (held && lane == 0) for (int i = 0; i < n_stages; i++) kp_mbar_arrive(&s_empty[(at0 + i) % LP_STAGES]);
    at0 += n_stages;

    // ---- the row's, from its parts'
    if (C > 1) {
        cluster.sync();
        if (part) {
            cluster.sync();                                          // (its shared memory is read until then)
            break;
        }
    }
    LpRef z(s_sums[0]);
    float S = s_sums[1], W = s_sums[2];
    int rank = s_count;
    for (int i = 1; i < C; i++) {
        const float* o = cluster.map_shared_rank(s_sums, i);
        const LpRef b(o[0]), to(fmaxf(z.r, b.r));
        float s = o[1], w = o[2];
        lp_move(S, W, to.from(z));
        lp_move(s, w, to.from(b));
        S += s;
        W += w;
        z = to;
        rank += *cluster.map_shared_rank(&s_count, i);
    }
    // The last differences are taken in 64 bits, each rounded once: r, log2 e and y = x log2 e - rl as they were rounded add up to (r log2 e - rl) in y.
    const double off = z.wild() ? 0.0 : (double)z.rl - (double)z.r * (double)LP_LOG2E, log_s = log((double)S) + off * 0.6931471805599453;
    const bool bad = !(S >= 0.f), none = S == 0.f;                   // a NaN or +inf among the logits; nothing but -inf
    auto logprob = [&](float f) { return none ? -INFINITY : (float)(((double)f - (double)z.r) - log_s); };
    if (tid == 0) {
        p.logprob[row] = id >= 0 ? (bad ? S : logprob(mine)) : 0.f;
        p.entropy[row] = none ? 0.f : (float)(log_s - ((double)W / (double)S + off) / (double)LP_LOG2E);
        p.rank[row] = id >= 0 ? rank : -1;
    }
    if (top) {
        const int n_all = C * top;
        auto put = [&](int place, u64 k) {
            const long long at = (long long)row * top + place;
            p.top_ids[at] = bad ? -1 : lp_index(k);
            p.top_logprobs[at] = bad ? S : logprob(lp_value(k));
        };
        if (C == 1 || bad) {                                         // (of numbers there may be fewer than alternatives then)
            if (tid < top) put(tid, s_sel[tid]);
        } else {
            for (int i = tid; i < n_all; i += LP_THREADS) s_cand[i] = *cluster.map_shared_rank(&s_sel[i % top], i / top);
            lp_sync();
            for (int i = tid; i < n_all; i += LP_THREADS) {
                const u64 k = s_cand[i];
                int before = i % top;                                // in its own part's list; in the others', each in order:
                for (int o = 0; o < C; o++) {
                    if (o == i / top) continue;
                    int n = 0;
#pragma unroll
                    for (int b = LP_MAX_TOP; b; b >>= 1) if (n + b <= top && s_cand[o * top + n + b - 1] > k) n += b;
                    before += n;
                }
                if (k && before < top) put(before, k);
            }
        }
    }
    if (C > 1) { cluster.sync(); break; }
    lp_sync();                                                       // (what the next row writes has been read)
    }
    if (__builtin_expect(!ok, 0)) {
        atomicExch(&g_logprobs_status, 1);
        kp_linger_after_failure();
    }
}

extern "C" int kp_token_logprobs(const void* logits, long long ld, const int* ids, int n, int V, int top, int parts, float* logprob, float* entropy,
                                 int* rank, int* top_ids, float* top_logprobs, int dtype, void* stream) {
    if (n < 0 || V < 1 || top < 0 || top > LP_MAX_TOP || top > V || (parts != 1 && parts != 2 && parts != 4 && parts != 8) || n > 2147483647 / 8 ||
        ((uintptr_t)logits & (dtype == KP_DTYPE_F32 ? 3 : 1)))
        return KP_ERR_BAD_ARG;
    if (!n) return 0;
    LpArgs a = {logits, ld, n, V, top, ids, logprob, entropy, rank, top_ids, top_logprobs};
    int sms = 0, dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts > 1 ? (unsigned)n * parts : (unsigned)(n < sms * LP_CTAS_SM ? n : sms * LP_CTAS_SM));
    cfg.blockDim = dim3(LP_THREADS + 32);
    // Few CTAs ask for more shared memory than they need, so that no SM takes more of them than its share: clusters are put three on an SM
    // while others have none (148 rows of 100003 16-bit logits in two parts each 15.4 us, 13.3 so).
    const int share = ((int)cfg.gridDim.x + sms - 1) / sms;
    cfg.dynamicSmemBytes = share == 1 ? LP_SMEM_ALONE : (share == 2 ? LP_SMEM_TWO : LP_STAGES * LP_STAGE);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;                                                // (2048 rows in clusters of one 85 us, in none 89)
    cudaError_t c;
    KP_DISPATCH_DTYPE(dtype, T, {
        static std::atomic<unsigned long long> ready{0};
        const int e = kp_smem_limit(token_logprobs_kernel<T>, LP_SMEM_ALONE, ready, true);
        if (e) return e;
        c = cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T>, a);
    });
    return c ? (int)c : kp_launch_status();
}
