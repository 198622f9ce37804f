// Eviction from a 4-bit cache (kv4.cuh) by the weight that its keys have got.
//
// Of the n keys of a (segment, kv head) the first `first`, the last `recent` and, of those between, the ones with the most
// mass stay, `keep` in all (equal mass: the lowest index); all of them where n <= keep.  They move, in their order, to
// places 0 .. of the segment's new pages, which are other pages than the old ones: nothing is read that this pass writes.
#include "kv4.cuh"

#define KE_THREADS 1024
#define KE_BINS 2048
#define KE_STAGED 49152                                    // masses of a head that fit in shared memory beside the histogram

struct KeArgs {
    const unsigned char* pages; const float* mass; const int* table; int max_blocks;
    unsigned char* new_pages; float* new_mass; const int* new_table; int new_blocks;
    const int* n_keys; int* kept;
    int max_keys, keep, recent, first, ps, G, hd;
};

// a float's bits in an order that unsigned integers have (both zeros alike)
__device__ __forceinline__ uint32_t ke_order(float m) {
    const uint32_t b = __float_as_uint(m + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// ---- which keys stay: one CTA a (segment, kv head)
__global__ void __launch_bounds__(KE_THREADS)
kv4_select_kernel(const KeArgs p) {
    kp_pdl_begin();
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* staged = reinterpret_cast<uint32_t*>(smem);
    __shared__ int hist[KE_BINS];
    __shared__ int wsum[2][32];
    __shared__ int s_bin, s_above;
    const int seg = blockIdx.y, kvh = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = min(p.n_keys[seg], p.max_keys);
    int* kept = p.kept + ((size_t)seg * p.G + kvh) * p.keep;
    if (n <= p.keep) {
        for (int i = tid; i < p.keep; i += KE_THREADS) kept[i] = i < n ? i : -1;
        return;
    }
    const int* bt = p.table + (size_t)seg * p.max_blocks;
    const int m0 = p.first, m1 = n - p.recent, want = p.keep - p.first - p.recent;      // candidates m0 .. m1 - 1
    auto fetch = [&](int i) { return ke_order(p.mass[((size_t)bt[i / p.ps] * p.G + kvh) * p.ps + i % p.ps]); };
    const bool fits = m1 - m0 <= KE_STAGED;
    if (fits)
        for (int i = m0 + tid; i < m1; i += KE_THREADS) staged[i - m0] = fetch(i);
    __syncthreads();
    auto get = [&](int i) { return fits ? staged[i - m0] : fetch(i); };
    // the want-th largest, 11 + 11 + 10 bits at a time from the top
    uint32_t prefix = 0, mask = 0;
    int left = want;                                       // how many of those that match the prefix are still wanted
#pragma unroll 1
    for (int pass = 0; pass < 3 && want > 0; pass++) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < KE_BINS; i += KE_THREADS) hist[i] = 0;
        __syncthreads();
        for (int i = m0 + tid; i < m1; i += KE_THREADS) {
            const uint32_t v = get(i);
            if ((v & mask) == prefix) atomicAdd(&hist[(v >> shift) & ((1 << bits) - 1)], 1);
        }
        __syncthreads();
        // counts from the top: thread t owns bins 2 t, 2 t + 1 counted from the largest
        const int b0 = KE_BINS - 1 - 2 * tid, c0 = hist[b0], c1 = hist[b0 - 1];
        int run = c0 + c1;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
        if (lane == 31) wsum[0][warp] = run;
        __syncthreads();
        int before = run - c0 - c1;
        for (int w = 0; w < warp; w++) before += wsum[0][w];
        if (before < left && left <= before + c0) { s_bin = b0; s_above = before; }
        else if (before + c0 < left && left <= before + c0 + c1) { s_bin = b0 - 1; s_above = before + c0; }
        __syncthreads();
        left -= s_above;
        prefix |= (uint32_t)s_bin << shift;
        mask |= (uint32_t)((1 << bits) - 1) << shift;
        __syncthreads();
    }
    // the keys that stay, in their order: those above the bound, and the first `left` of those that equal it
    int base = 0, eq_base = 0;                             // how many were kept, and were equal, before this stretch
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += KE_THREADS) {
        const int i = i0 + tid;
        bool sure = false, eq = false;
        if (i < n) {
            if (i < m0 || i >= m1) sure = true;
            else if (want > 0) { const uint32_t v = get(i); sure = v > prefix; eq = v == prefix; }
        }
        const unsigned be = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) wsum[0][warp] = __popc(be);
        __syncthreads();
        int e = eq_base, e_all = 0;
        for (int w = 0; w < 32; w++) { const int c = wsum[0][w]; if (w < warp) e += c; e_all += c; }
        e += __popc(be & ((1u << lane) - 1));
        const bool stays = sure || (eq && e < left);
        const unsigned bs = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) wsum[1][warp] = __popc(bs);
        __syncthreads();
        int at = base, all = 0;
        for (int w = 0; w < 32; w++) { const int c = wsum[1][w]; if (w < warp) at += c; all += c; }
        if (stays) kept[at + __popc(bs & ((1u << lane) - 1))] = i;
        base += all;
        eq_base += e_all;
    }
}

// ---- moves them: a warp 16 places of a (segment, kv head)
__global__ void __launch_bounds__(128)
kv4_move_kernel(const KeArgs p) {
    kp_pdl_begin();
    const int seg = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 31;
    const int d0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * 16;
    const int stay = min(min(p.n_keys[seg], p.max_keys), p.keep);
    if (d0 >= stay) return;
    const int count = min(16, stay - d0);
    const int hd = p.hd, ng = hd / (hd % 64 == 0 ? 64 : 32), pp = hd / 32;
    const size_t rec = (size_t)kv4_page_bytes(p.ps, hd);
    const int src = lane < count ? p.kept[((size_t)seg * p.G + kvh) * p.keep + d0 + lane] : 0;
    const int page = lane < count ? p.table[(size_t)seg * p.max_blocks + src / p.ps] : 0, off = src % p.ps;
    const int to = p.new_table[(size_t)seg * p.new_blocks + d0 / p.ps], to_off = d0 % p.ps;      // (16 places never straddle a page)
    unsigned char* dst = p.new_pages + ((size_t)to * p.G + kvh) * rec;
    if (lane < count)
        p.new_mass[((size_t)to * p.G + kvh) * p.ps + to_off + lane] = p.mass[((size_t)page * p.G + kvh) * p.ps + off];
    for (int j = lane; j < ((16 * pp + 31) & ~31); j += 32) {                                    // 16-byte pieces of the code rows
        const int k = min(j / pp, 15), e = j % pp;
        const int pg = __shfl_sync(0xffffffffu, page, k), of = __shfl_sync(0xffffffffu, off, k);
        if (j / pp < count) {
            const unsigned char* s = p.pages + ((size_t)pg * p.G + kvh) * rec;
            const uint4 a = *reinterpret_cast<const uint4*>(s + (size_t)of * (hd / 2) + e * 16);
            const uint4 b = *reinterpret_cast<const uint4*>(s + (size_t)(p.ps + of) * (hd / 2) + e * 16);
            *reinterpret_cast<uint4*>(dst + (size_t)(to_off + k) * (hd / 2) + e * 16) = a;
            *reinterpret_cast<uint4*>(dst + (size_t)(p.ps + to_off + k) * (hd / 2) + e * 16) = b;
        }
    }
    for (int j = lane; j < ((16 * ng + 31) & ~31); j += 32) {                                    // and the ranges
        const int k = min(j / ng, 15), e = j % ng;
        const int pg = __shfl_sync(0xffffffffu, page, k), of = __shfl_sync(0xffffffffu, off, k);
        if (j / ng < count) {
            const uint32_t* s = reinterpret_cast<const uint32_t*>(p.pages + ((size_t)pg * p.G + kvh) * rec + (size_t)p.ps * hd);
            uint32_t* d = reinterpret_cast<uint32_t*>(dst + (size_t)p.ps * hd);
            d[(to_off + k) * ng + e] = s[of * ng + e];
            d[(p.ps + to_off + k) * ng + e] = s[(p.ps + of) * ng + e];
        }
    }
}

extern "C" int kp_kv4_evict(const void* pages, const float* mass, const int* table, int max_blocks, const int* n_keys, void* new_pages, float* new_mass,
                            const int* new_table, int new_blocks, int* kept, int n_seg, int max_keys, int keep, int recent, int first, int ps, int G,
                            int hd, void* stream) {
    if (n_seg <= 0) return 0;
    if (hd < 32 || hd % 32 || hd > 256 || ps < 16 || (ps & (ps - 1)) || G < 1 || G > 65535 || n_seg > 65535 || keep < 1 || recent < 0 || first < 0 || first + recent > keep ||
        max_keys < 1 || (((uintptr_t)pages | (uintptr_t)new_pages) & 15))
        return KP_ERR_BAD_ARG;
    KeArgs a = {(const unsigned char*)pages, mass, table, max_blocks, (unsigned char*)new_pages, new_mass, new_table, new_blocks, n_keys, kept,
                max_keys, keep, recent, first, ps, G, hd};
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(kv4_select_kernel, KE_STAGED * 4, ready);
    if (e) return e;
    const int room = max_keys < KE_STAGED ? max_keys : KE_STAGED;
    cudaError_t c = kp_launch_pdl(kv4_select_kernel, dim3(G, n_seg), dim3(KE_THREADS), (size_t)room * 4, (cudaStream_t)stream, a);
    if (c) return (int)c;
    const int stay = keep < max_keys ? keep : max_keys;
    c = kp_launch_pdl(kv4_move_kernel, dim3((stay + 63) / 64, G, n_seg), dim3(128), 0, (cudaStream_t)stream, a);
    if (c) return (int)c;
    return kp_launch_status();
}
