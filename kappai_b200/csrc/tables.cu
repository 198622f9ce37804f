// Block tables, first rows, positions and slots of a step made on the GPU from the sequences' lengths, and the pages that go with them.
//
// With b(L) = ceil(L / ps) blocks of a sequence of L tokens and a change d of its length: d >= 0 adds d rows at positions L .. L + d - 1 and
// takes b(L + d) - b(L) pages; d < 0 takes the last tokens back, not those of the first `own_from` blocks (which other sequences name too), and
// gives the pages of the blocks that no token is left in back; L + d <= 0 ends it: all of its blocks are forgotten, its own pages given back.  Pages
// that come back are put on the stack of free ones so that the first sequence's first one lies uppermost, and then pages are taken from the top in
// the same order: a step and the step that takes it back leave the stack as it was.
//
// Three exclusive sums over the sequences (rows, pages back, pages taken) say where everything goes; every CTA makes them for itself, then the
// pages and the rows are shared out over all threads, each of which finds its sequence by bisection.  CTAs are one cluster: its barrier stands between
// reading the lengths and writing them, and between putting pages on the stack and taking them.  Launch and latency bound: a chain of loads,
// the sums, the bisection and a page's load.  64 sequences with a row each 4 us, 2000 with 60000 rows 9.8.  Nothing happens, and `status` says why, where pages are short (1), a table is too
// narrow (2), the rows have no room (4) or lengths or counts make no sense (8): bits that are added up (the rows and
// pages of a sequence with 2 or 8 are not counted for the others).
#include "common.cuh"

#define PT_MAX_SEQS 8192
#define PT_MAX_ROWS 65535

struct PtArgs {
    int* table; int width; int* length; const int* delta; const int* own_from;
    int* free_pages; int n_pages; int* n_free; int ps, ps_log2, S, cap;
    int* cu_rows; int* seg_pos; int* row_seg; int* positions; int* slots; int* status;
};

__device__ __forceinline__ void pt_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Division by a page's size, in 32 bits: a shift where it is a power of two.  (In 64 bits it was a
// tenth of the time.)
struct PtPages {
    unsigned ps; int log2;
    __device__ __forceinline__ unsigned of(unsigned x) const { return log2 >= 0 ? x >> log2 : x / ps; }
    __device__ __forceinline__ int blocks(int tokens) const { return (int)of((unsigned)tokens + ps - 1); }      // (below 2^32: both are below 2^31)
};

// what a sequence of length L does with a change d
struct PtSeq { int rows, back, taken, after; bool ended, wide, bad; };
__device__ __forceinline__ PtSeq pt_seq(int L, int d, int own, const PtPages& pages, int width) {
    PtSeq q = {0, 0, 0, L, false, false, false};
    const long long most = (long long)width * pages.ps;      // (below 2^31)
    if (L < 0 || own < 0 || L > most) { q.bad = true; q.after = 0; return q; }
    const int b0 = pages.blocks(L);
    own = min(own, b0);
    long long after = (long long)L + d;
    q.ended = after <= 0;
    if (q.ended) after = 0;
    else if (d < 0) after = min((long long)L, max(after, (long long)own * pages.ps));
    if (after > most) { q.wide = true; return q; }
    const int b1 = pages.blocks((int)after);
    q.rows = min(max(d, 0), PT_MAX_ROWS + 1);               // (more have no room, and their sum stays within 32 bits)
    q.after = (int)after;
    if (b1 < b0) q.back = b0 - max(b1, own);
    else q.taken = b1 - b0;
    return q;
}

// the i with cu[i] <= x < cu[i + 1]
__device__ __forceinline__ int pt_find(const int* cu, int S, int x) {
    int lo = 0, hi = S;                                      // cu[lo] <= x < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(1024)
page_tables_kernel(const PtArgs p) {
    kp_pdl_begin();
    extern __shared__ int pt_smem[];
    const PtPages pages = {(unsigned)p.ps, p.ps_log2};
    const int S = p.S, ps = p.ps, tid = threadIdx.x, T = blockDim.x, lane = tid & 31, warp = tid >> 5;
    int* cu_r = pt_smem;                                     // [S + 1] each
    int* cu_b = cu_r + S + 1;
    int* cu_t = cu_b + S + 1;
    int* len = cu_t + S + 1;                                 // [S]: the old length, the sign for a sequence that ends
    __shared__ int wsum[3][32], s_bad;
    if (tid == 0) s_bad = 0;
    __syncthreads();

    // ---- the sums: a stretch of sequences a thread
    const int per = (S + T - 1) / T, i0 = min(tid * per, S), i1 = min(i0 + per, S);
    int r = 0, b = 0, t = 0, bad = 0;
    for (int j = i0; j < i1; j += 4) {
        int L[4], d[4], own[4];                              // (under way together)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool there = j + k < i1;
            L[k] = there ? p.length[j + k] : 0;
            d[k] = there ? p.delta[j + k] : 0;
            own[k] = there && p.own_from ? p.own_from[j + k] : 0;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int i = j + k;
            if (i >= i1) break;
            const PtSeq q = pt_seq(L[k], d[k], own[k], pages, p.width);
            cu_r[i] = r; cu_b[i] = b; cu_t[i] = t;
            len[i] = q.ended ? (int)((unsigned)L[k] | 0x80000000u) : L[k];
            r += q.rows; b += q.back; t += q.taken;
            bad |= (q.wide ? 2 : 0) | (q.bad ? 8 : 0);
        }
    }
    int xr = r, xb = b, xt = t;                              // inclusive sums over the warp's threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int yr = __shfl_up_sync(0xffffffffu, xr, o), yb = __shfl_up_sync(0xffffffffu, xb, o), yt = __shfl_up_sync(0xffffffffu, xt, o);
        if (lane >= o) { xr += yr; xb += yb; xt += yt; }
    }
    if (lane == 31) { wsum[0][warp] = xr; wsum[1][warp] = xb; wsum[2][warp] = xt; }
    if (bad) atomicOr(&s_bad, bad);
    const int n_free = p.n_free[0];
    __syncthreads();
    const int n_warps = T >> 5, wr = lane < n_warps ? wsum[0][lane] : 0, wb = lane < n_warps ? wsum[1][lane] : 0, wt = lane < n_warps ? wsum[2][lane] : 0;
    int rows = __reduce_add_sync(0xffffffffu, wr), back = __reduce_add_sync(0xffffffffu, wb), taken = __reduce_add_sync(0xffffffffu, wt);
    const int fr = xr - r + __reduce_add_sync(0xffffffffu, lane < warp ? wr : 0), fb = xb - b + __reduce_add_sync(0xffffffffu, lane < warp ? wb : 0),
              ft = xt - t + __reduce_add_sync(0xffffffffu, lane < warp ? wt : 0);
    int status = s_bad;
    // (a count that makes no sense, or more pages back than the stack has places for)
    if (n_free < 0 || n_free > p.n_pages || back > p.n_pages - n_free) status |= 8;
    else if (taken > n_free + back) status |= 1;
    if (rows > p.cap) status |= 4;
    for (int i = i0; i < i1; i++) { cu_r[i] += fr; cu_b[i] += fb; cu_t[i] += ft; }
    if (tid == 0) { cu_r[S] = rows; cu_b[S] = back; cu_t[S] = taken; }
    __syncthreads();
    if (status) rows = back = taken = 0;

    const int gt = blockIdx.x * T + tid, GT = gridDim.x * T, top = n_free + back;
    // ---- pages that come back
    for (int a = gt; a < back; a += GT) {
        const int i = pt_find(cu_b, S, a);
        const int b0 = pages.blocks(len[i] & 0x7fffffff), block = b0 - (cu_b[i + 1] - cu_b[i]) + a - cu_b[i];
        int* entry = p.table + (size_t)i * p.width + block;
        p.free_pages[top - 1 - a] = *entry;
        *entry = -1;
    }
    if (!status)
        for (int i = gt >> 5; i < S; i += GT >> 5)           // of a sequence that ends the shared blocks are forgotten too
            if (len[i] < 0) {
                const int shared = pages.blocks(len[i] & 0x7fffffff) - (cu_b[i + 1] - cu_b[i]);
                for (int block = lane; block < shared; block += 32) p.table[(size_t)i * p.width + block] = -1;
            }
    __threadfence();
    pt_cluster_sync();                                       // every CTA has read the lengths and put its pages back
    // ---- pages that are taken
    for (int k = gt; k < taken; k += GT) {
        const int i = pt_find(cu_t, S, k);
        p.table[(size_t)i * p.width + pages.blocks(len[i]) + k - cu_t[i]] = p.free_pages[top - 1 - k];
    }
    // ---- the rows
    for (int x = gt; x < p.cap; x += GT) {
        int seg = 0, pos = -1, slot = -1;
        if (x < rows) {
            seg = pt_find(cu_r, S, x);
            const int L = len[seg], b0 = pages.blocks(L);   // (a sequence with rows does not end)
            pos = L + x - cu_r[seg];
            const int block = (int)pages.of(pos);
            const int page = block < b0 ? p.table[(size_t)seg * p.width + block] : p.free_pages[top - 1 - (cu_t[seg] + block - b0)];
            slot = page * ps + pos - block * ps;
        }
        p.row_seg[x] = seg;
        p.positions[x] = pos;
        p.slots[x] = slot;
    }
    // ---- the sequences
    for (int i = gt; i < S; i += GT) {
        const int L = len[i] & 0x7fffffff;
        if (status) {
            p.cu_rows[i + 1] = 0;
            p.seg_pos[i] = p.length[i];
            continue;
        }
        const int n = cu_r[i + 1] - cu_r[i];
        const PtSeq q = pt_seq(L, p.delta[i], p.own_from ? p.own_from[i] : 0, pages, p.width);
        p.cu_rows[i + 1] = cu_r[i + 1];
        p.seg_pos[i] = n ? L : q.after;
        p.length[i] = q.after;
    }
    if (gt == 0) {
        p.cu_rows[0] = 0;
        p.status[0] = status;
        if (!status) p.n_free[0] = top - taken;
    }
}

// CTAs of the largest cluster that the GPU can have, 16 or 8
static int pt_cluster() {
    static std::atomic<int> known[64];
    int dev = 0, fit = 0;
    if (cudaGetDevice(&dev) || dev >= 64) return 8;
    if (const int k = known[dev].load(std::memory_order_relaxed)) return k;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = (size_t)(4 * PT_MAX_SEQS + 3) * 4;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(page_tables_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) || cudaOccupancyMaxActiveClusters(&fit, page_tables_kernel, &cfg)) {
        cudaGetLastError();
        fit = 0;
    }
    const int most = fit > 0 ? 16 : 8;
    known[dev].store(most, std::memory_order_relaxed);
    return most;
}

extern "C" int kp_page_tables(int* table, int width, int* length, const int* delta, const int* own_from, int* free_pages, int n_pages, int* n_free,
                              int ps, int S, int cap, int* cu_rows, int* seg_pos, int* row_seg, int* positions, int* slots, int* status, void* stream) {
    if (S < 0 || S > PT_MAX_SEQS || cap < 0 || cap > PT_MAX_ROWS || ps < 1 || width < 0 || n_pages < 0 ||
        (long long)S * width >= 2147483647LL || (long long)n_pages * ps >= 2147483648LL || (long long)width * ps >= 2147483648LL)
        return KP_ERR_BAD_ARG;
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(page_tables_kernel, (size_t)(4 * PT_MAX_SEQS + 3) * 4, ready);
    if (e) return e;
    // Measured (a step and the one that takes it back): 64 sequences with a row each, one CTA 9.5 us, four 8.0, sixteen 7.7; 2000 with 60000 rows, four, eight and
    // sixteen CTAs 30, 23 and 19.5.  More than eight are for long ones, where the GPU can have such a cluster.
    const int work = cap > S ? cap : S;
    int threads = 128, ps_log2 = -1;
    for (int i = 0; i < 31; i++) if (ps == 1 << i) ps_log2 = i;
    while (threads < 1024 && threads < work) threads *= 2;
    const int ctas = work <= 2048 ? 4 : pt_cluster();
    PtArgs a = {table, width, length, delta, own_from, free_pages, n_pages, n_free, ps, ps_log2, S, cap, cu_rows, seg_pos, row_seg, positions, slots, status};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = (size_t)(4 * S + 3) * 4;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t c = cudaLaunchKernelEx(&cfg, page_tables_kernel, a);
    return c ? (int)c : kp_launch_status();
}
