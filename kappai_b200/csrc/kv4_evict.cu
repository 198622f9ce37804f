// Eviction from a 4-bit cache (kv4.cuh) by the weight that its keys have got.
//
// Of the n keys of a (segment, kv head) the first `first`, the last `recent` and, of those between, the ones with the most
// mass stay, `keep` in all (equal mass: the lowest index; one that is not a number counts as the most); all of them where n <= keep.  They move, in their order, to
// places 0 .. of the segment's new pages, which are other pages than the old ones: nothing is read that this pass writes.
#include "kv4.cuh"

#define KE_THREADS 1024
#define KE_BINS 2048
#define KE_STAGED 49152                                    // masses of a head that fit in shared memory beside the histogram

struct KeArgs {
    const unsigned char* pages; const float* mass; const int* table; int max_blocks;
    unsigned char* new_pages; float* new_mass; const int* new_table; int new_blocks;
    const int* n_keys; int* kept;
    int max_keys, keep, recent, first, ps, ps_log2, G;
};

// a float's bits in an order that unsigned integers have (both zeros alike)
__device__ __forceinline__ uint32_t ke_order(float m) {
    const uint32_t b = __float_as_uint(m + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// ---- which keys stay: one CTA a (segment, kv head).  A radix selection finds the want-th largest mass, 11, 11 and 10 bits at a time,
// from masses that were brought to shared memory once (more than fit there are read again each time); then every warp has a stretch
// of the keys, counts in it and, when it knows what stands in front of it, writes down the ones that stay, in their order.  16 x 8 lists of up
// to 16,384 masses: 20 us (a CTA a list, 128 of 148 SMs: the passes over shared memory bound it, not the 8 MB).
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
    const float* mass = p.mass + (size_t)kvh * p.ps;
    auto fetch = [&](int i) { return ke_order(mass[(size_t)bt[i >> p.ps_log2] * p.G * p.ps + (i & (p.ps - 1))]); };
    const bool fits = m1 - m0 <= KE_STAGED && want > 0;
    if (fits) {
        constexpr int U = 8;                               // loads under way together: a page's number comes before a mass
        for (int i0 = m0 + tid; i0 < m1; i0 += U * KE_THREADS) {
            int page[U];
            uint32_t v[U];
#pragma unroll
            for (int u = 0; u < U; u++) page[u] = bt[min(i0 + u * KE_THREADS, m1 - 1) >> p.ps_log2];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = ke_order(mass[(size_t)page[u] * p.G * p.ps + (min(i0 + u * KE_THREADS, m1 - 1) & (p.ps - 1))]);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i0 + u * KE_THREADS < m1) staged[i0 + u * KE_THREADS - m0] = v[u];
        }
    }
    auto get = [&](int i) { return fits ? staged[i - m0] : fetch(i); };
    uint32_t prefix = 0, mask = 0;
    int left = want;                                       // how many of those that match the prefix are still wanted
#pragma unroll 1
    for (int pass = 0; pass < 3 && want > 0; pass++) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
        for (int i = tid; i < KE_BINS; i += KE_THREADS) hist[i] = 0;
        __syncthreads();
#pragma unroll 4
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
        const int before = run - c0 - c1 + __reduce_add_sync(0xffffffffu, lane < warp ? wsum[0][lane] : 0);
        if (before < left && left <= before + c0) { s_bin = b0; s_above = before; }
        else if (before + c0 < left && left <= before + c0 + c1) { s_bin = b0 - 1; s_above = before + c0; }
        __syncthreads();
        left -= s_above;
        prefix |= (uint32_t)s_bin << shift;
        mask |= (uint32_t)((1 << bits) - 1) << shift;
    }
    __syncthreads();
    // the keys that stay: those above the bound, and the first `left` of those that equal it
    const int stretch = ((n + 1023) / 1024) * 32, w0 = warp * stretch, w1 = min(n, w0 + stretch);
    auto look = [&](int i, bool& sure, bool& eq) {
        sure = eq = false;
        if (i < w1) {
            if (i < m0 || i >= m1) sure = true;
            else if (want > 0) { const uint32_t v = get(i); sure = v > prefix; eq = v == prefix; }
        }
    };
    int n_sure = 0, n_eq = 0;
#pragma unroll 4
    for (int i0 = w0; i0 < w1; i0 += 32) {
        bool sure, eq;
        look(i0 + lane, sure, eq);
        n_sure += __popc(__ballot_sync(0xffffffffu, sure));
        n_eq += __popc(__ballot_sync(0xffffffffu, eq));
    }
    if (lane == 0) { wsum[0][warp] = n_sure; wsum[1][warp] = n_eq; }
    __syncthreads();
    int eq_before = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[1][lane] : 0);
    int at = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[0][lane] : 0) + min(eq_before, left);
#pragma unroll 4
    for (int i0 = w0; i0 < w1; i0 += 32) {
        bool sure, eq;
        look(i0 + lane, sure, eq);
        const unsigned below = (1u << lane) - 1, be = __ballot_sync(0xffffffffu, eq);
        const bool stays = sure || (eq && eq_before + __popc(be & below) < left);
        const unsigned bs = __ballot_sync(0xffffffffu, stays);
        if (stays) kept[at + __popc(bs & below)] = i0 + lane;
        at += __popc(bs);
        eq_before += __popc(be);
    }
}

// ---- moves them: a warp 16 places of a (segment, kv head), all of whose loads are under way together
template <int HD>
__global__ void __launch_bounds__(128)
kv4_move_kernel(const KeArgs p) {
    using F = Kv4<HD>;
    kp_pdl_begin();
    const int seg = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 31;
    const int d0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * 16;
    const int stay = min(min(p.n_keys[seg], p.max_keys), p.keep);
    if (d0 >= stay) return;
    const int count = min(16, stay - d0), ps = p.ps;
    const size_t rec = (size_t)kv4_page_bytes(ps, HD);
    const int src = lane < count ? p.kept[((size_t)seg * p.G + kvh) * p.keep + d0 + lane] : 0;
    const int page = lane < count ? p.table[(size_t)seg * p.max_blocks + (src >> p.ps_log2)] : 0, off = src & (ps - 1);
    const int to = p.new_table[(size_t)seg * p.new_blocks + (d0 >> p.ps_log2)], to_off = d0 & (ps - 1);      // (16 places never straddle a page)
    unsigned char* dst = p.new_pages + ((size_t)to * p.G + kvh) * rec;
    constexpr int NC = (16 * F::PP + 31) / 32, NR = (16 * F::NG + 31) / 32;
    uint4 code[NC][2];
    uint32_t range[NR][2];
    float m = 0.f;
    if (lane < count) m = p.mass[((size_t)page * p.G + kvh) * ps + off];
#pragma unroll
    for (int i = 0; i < NC; i++) {                         // 16-byte pieces of the code rows
        const int j = i * 32 + lane, k = min(j / F::PP, 15), e = j % F::PP;
        const int pg = __shfl_sync(0xffffffffu, page, k), of = __shfl_sync(0xffffffffu, off, k);
        if (j / F::PP < count) {
            const uint4* s = reinterpret_cast<const uint4*>(p.pages + ((size_t)pg * p.G + kvh) * rec + (size_t)of * F::ROW) + e;
            code[i][0] = s[0];
            code[i][1] = s[(size_t)ps * F::PP];
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {                         // and the ranges
        const int j = i * 32 + lane, k = min(j / F::NG, 15), e = j % F::NG;
        const int pg = __shfl_sync(0xffffffffu, page, k), of = __shfl_sync(0xffffffffu, off, k);
        if (j / F::NG < count) {
            const uint32_t* s = reinterpret_cast<const uint32_t*>(p.pages + ((size_t)pg * p.G + kvh) * rec + (size_t)ps * HD) + of * F::NG + e;
            range[i][0] = s[0];
            range[i][1] = s[(size_t)ps * F::NG];
        }
    }
    if (lane < count) p.new_mass[((size_t)to * p.G + kvh) * ps + to_off + lane] = m;
#pragma unroll
    for (int i = 0; i < NC; i++) {
        const int j = i * 32 + lane;
        if (j / F::PP < count) {
            uint4* d = reinterpret_cast<uint4*>(dst + (size_t)to_off * F::ROW) + j;
            d[0] = code[i][0];
            d[(size_t)ps * F::PP] = code[i][1];
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int j = i * 32 + lane;
        if (j / F::NG < count) {
            uint32_t* d = reinterpret_cast<uint32_t*>(dst + (size_t)ps * HD) + to_off * F::NG + j;
            d[0] = range[i][0];
            d[(size_t)ps * F::NG] = range[i][1];
        }
    }
}

template <int HD>
static cudaError_t ke_move(const KeArgs& a, int stay, int n_seg, cudaStream_t st) {
    return kp_launch_pdl(kv4_move_kernel<HD>, dim3((stay + 63) / 64, a.G, n_seg), dim3(128), 0, st, a);
}

extern "C" int kp_kv4_evict(const void* pages, const float* mass, const int* table, int max_blocks, const int* n_keys, void* new_pages, float* new_mass,
                            const int* new_table, int new_blocks, int* kept, int n_seg, int max_keys, int keep, int recent, int first, int ps, int G,
                            int hd, void* stream) {
    if (n_seg <= 0) return 0;
    if (hd < 32 || hd % 32 || hd > 256 || ps < 16 || (ps & (ps - 1)) || G < 1 || G > 65535 || n_seg > 65535 || keep < 1 || recent < 0 || first < 0 || first + recent > keep ||
        max_keys < 1 || (((uintptr_t)pages | (uintptr_t)new_pages) & 15))
        return KP_ERR_BAD_ARG;
    int ps_log2 = 0;
    while ((1 << ps_log2) < ps) ps_log2++;
    KeArgs a = {(const unsigned char*)pages, mass, table, max_blocks, (unsigned char*)new_pages, new_mass, new_table, new_blocks, n_keys, kept,
                max_keys, keep, recent, first, ps, ps_log2, G};
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(kv4_select_kernel, KE_STAGED * 4, ready);
    if (e) return e;
    const int room = max_keys < KE_STAGED ? max_keys : KE_STAGED;
    cudaError_t c = kp_launch_pdl(kv4_select_kernel, dim3(G, n_seg), dim3(KE_THREADS), (size_t)room * 4, (cudaStream_t)stream, a);
    if (c) return (int)c;
    const int stay = keep < max_keys ? keep : max_keys;
    const cudaStream_t st = (cudaStream_t)stream;
    switch (hd) {
        case 32: c = ke_move<32>(a, stay, n_seg, st); break;
        case 64: c = ke_move<64>(a, stay, n_seg, st); break;
        case 96: c = ke_move<96>(a, stay, n_seg, st); break;
        case 128: c = ke_move<128>(a, stay, n_seg, st); break;
        case 192: c = ke_move<192>(a, stay, n_seg, st); break;
        case 256: c = ke_move<256>(a, stay, n_seg, st); break;
        default: return KP_ERR_UNSUPPORTED;
    }
    if (c) return (int)c;
    return kp_launch_status();
}
