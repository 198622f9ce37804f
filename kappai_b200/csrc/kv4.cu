// The 4-bit cache (kv4.cuh): writing rows to it, reading them back, and causal attention over it.
//
// Rows of one segment are consecutive rows of q (cu_rows); row r of segment i stands at key index p = seg_pos[i] + r and
// reads the keys max(0, p - window + 1) .. p (no window: 0 .. p).  A row with no key (p < 0) gives zeros.
#include "kv4.cuh"

// ------------------------------------------------------------------ write and read
// A thread takes 8 consecutive values of a group; the lanes of a group (8, or 4) find its range together.
__device__ __forceinline__ float kv4_min_nan(float a, float b) { float d; asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ float kv4_max_nan(float a, float b) { float d; asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ float kv4_min_nan(float a, float b, float c) { float d; asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ float kv4_max_nan(float a, float b, float c) { float d; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }

// (a call: inlined, the compiler makes its first steps where nothing is divided)
__device__ __noinline__ float kv4_divide(float a, float b) { return __fdiv_rn(a, b); }
// bfloat16(x / 15), x >= 0: the product with the reciprocal is off by a unit or two of float32's last place, which matters only where it lies next to
// a half of bfloat16's; there (and for the smallest) x is divided.
__device__ __forceinline__ bf16 kv4_fifteenth(float x) {
    float q = x * (1.0f / 15.0f);
    if (q < 1e-30f || ((__float_as_uint(q) & 0xffffu) - 0x7ffcu) < 8u) q = kv4_divide(x, 15.0f);
    return __float2bfloat16_rn(q);
}
// A group's scale, bfloat16((hi - lo) / 15).  Where hi - lo is above the largest float32 it is taken of a sixteenth of both, which rounds no differently.
__device__ __forceinline__ bf16 kv4_group_scale(float lo, float hi) {
    const float x = hi - lo;
    if (x != INFINITY) return kv4_fifteenth(x);
    return __float2bfloat16_rn(kv4_divide(hi * 0.0625f - lo * 0.0625f, 15.0f) * 16.0f);
}
// The codes round((x - z) / s) of eight values, halves to even, within 0 .. 15 (s > 0).  One Newton step on the quotient by the reciprocal (Markstein's
// method): q + (d - q s) / s with the remainder exact.  Where d / s is at a half or rounds to it the step gives that half itself, and elsewhere a
// unit of the last place changes no code.  Scales whose reciprocal is not to be had are divided by.  Adding 2^23 rounds to the even integer and
// leaves the code in the low bits, under the same 0x4b000000 for each.
__device__ __forceinline__ uint32_t kv4_eight_codes(const float (&x)[8], float s, float z) {
    float inv, q[8];
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float d = x[i] - z, t = d * inv;
        q[i] = fmaf(fmaf(-t, s, d), inv, t);
    }
    if (!(s >= 1e-30f && s <= 1e30f)) {
        const float f = s > 1.0f ? 0.0625f : 1.0f;         // (a difference of finite values may be above the largest float32)
#pragma unroll
        for (int i = 0; i < 8; i++) q[i] = kv4_divide(x[i] * f - z * f, s * f);
    }
    uint32_t w = 0u;
#pragma unroll
    for (int i = 7; i >= 0; i--) w = w * 16u + __float_as_uint(fminf(fmaxf(q[i], 0.f), 15.f) + 8388608.0f);
    return w - 0xfb000000u;                                // (0x4b000000 and 16 times it; the others have left the word)
}

template <typename T, bool VEC>
__device__ __forceinline__ void kv4_load8(float (&v)[8], const T* p) {
    if (VEC && sizeof(T) == 2) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    } else if (VEC) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(p[i]);
    }
}

// Thread idx of a launch of `n_threads`: place `idx % per_row` of the rows idx / per_row + u (n_threads / per_row), u < U.  With
// U rows a thread their loads are under way together: one row a thread leaves a CTA waiting for its slot, then for its values.
// 6,007 rows of 8 heads of 128 float32 values written: 18.9 us with one row, 16.6 with two, 15.2 with three, 15.7 with four (15.4 with three since
// ranges above float32's are looked for); 49 MB read and 7 written, 3.7 TB/s.  257 instructions a warp and row of 8 values a thread use 74 % of the
// issue slots, with 43 % of the warps there: fewer of either would help, no wall is reached.
struct Kv4Rows { int n, ps_log2, G, hd, gs; long long n_slots; };

template <typename T, bool VEC, int U>
__global__ void __launch_bounds__(256)
kv4_write_kernel(const T* __restrict__ k, long long ldk, const T* __restrict__ v, long long ldv, unsigned char* __restrict__ pages,
                 const int* __restrict__ slot_map, const Kv4Rows p) {
    kp_pdl_begin();
    const int half = p.G * p.hd / 8, per_row = 2 * half;   // threads a row: its keys, then its values
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;
    const int row0 = idx / per_row, place = idx - (unsigned)row0 * per_row, step = (p.n + U - 1) / U;
    const bool is_v = place >= half;
    const int within = is_v ? place - half : place, head = within / (p.hd / 8), d8 = within - head * (p.hd / 8);
    const int lanes = p.gs / 8, ng = p.hd / p.gs;          // lanes of a group, groups of a head
    const long long ld = is_v ? ldv : ldk, stride = step * ld;
    const T* src = (is_v ? v : k) + within * 8 + row0 * ld;
    const int ps = 1 << p.ps_log2;
    const unsigned rec = kv4_page_bytes(ps, p.hd);
    unsigned char* codes = pages + ((is_v ? ps : 0) * (p.hd / 2) + d8 * 4);       // of this head's first page, its first slot
    unsigned char* ranges = pages + (ps * p.hd + ((is_v ? ps : 0) * ng + d8 / lanes) * 4);
    int slot[U];
    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * step;
        slot[u] = row0 < step && row < p.n ? slot_map[row] : -1;
        if (slot[u] >= p.n_slots) slot[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[u][i] = 0.f;
        if (slot[u] >= 0) kv4_load8<T, VEC>(x[u], src + u * stride);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        // a range that holds a NaN, or an infinity, is none: the group reads as NaN
        float lo = kv4_min_nan(x[u][0], x[u][1]), hi = kv4_max_nan(x[u][0], x[u][1]);
#pragma unroll
        for (int i = 2; i < 8; i += 2) { lo = kv4_min_nan(lo, x[u][i], x[u][i + 1]); hi = kv4_max_nan(hi, x[u][i], x[u][i + 1]); }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
            if (d == 4 && lanes == 4) break;
            lo = kv4_min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
            hi = kv4_max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
        }
        if (slot[u] < 0) continue;
        const bf16 sb = kv4_group_scale(lo, hi), zb = __float2bfloat16_rn(lo);
        const float s = __bfloat162float(sb), z = __bfloat162float(zb);
        const uint32_t w = s > 0.f ? kv4_eight_codes(x[u], s, z) : 0u;
        const unsigned page = slot[u] >> p.ps_log2, off = slot[u] & (ps - 1);
        const size_t at = (size_t)(page * p.G + head) * rec;
        *reinterpret_cast<uint32_t*>(codes + at + off * (p.hd / 2)) = w;
        if (d8 % lanes == 0)
            *reinterpret_cast<uint32_t*>(ranges + at + off * ng * 4) = (uint32_t)__bfloat16_as_ushort(sb) | ((uint32_t)__bfloat16_as_ushort(zb) << 16);
    }
}

// A pair of lanes has values 0 .. 7 and 8 .. 15: the first lane gets 0 .. 3 and 8 .. 11, the second the others, so that an instruction that
// stores four of each writes whole sectors of 32 bytes (6,007 rows of 8 heads of 128 float32 values read back: 18.9 us without, 13.4 with;
// the same for the loads of the write, which find their other half in L1, cost 2 us more than it saved).
__device__ __forceinline__ void kv4_swap_pair(float (&v)[8], unsigned mask) {
    const bool odd = threadIdx.x & 1;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float other = __shfl_xor_sync(mask, odd ? v[i] : v[4 + i], 1);
        if (odd) v[i] = other; else v[4 + i] = other;
    }
}

template <typename T, int U>
__global__ void __launch_bounds__(256)
kv4_read_kernel(const unsigned char* __restrict__ pages, const int* __restrict__ slot_map, T* __restrict__ k, T* __restrict__ v, const Kv4Rows p) {
    kp_pdl_begin();
    const int half = p.G * p.hd / 8, per_row = 2 * half;
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;
    const int row0 = idx / per_row, place = idx - (unsigned)row0 * per_row, step = (p.n + U - 1) / U;
    if (row0 >= step) return;
    const bool is_v = place >= half;
    const int within = is_v ? place - half : place, head = within / (p.hd / 8), d8 = within - head * (p.hd / 8), ng = p.hd / p.gs, g = d8 / (p.gs / 8);
    const int ps = 1 << p.ps_log2;
    const unsigned rec = kv4_page_bytes(ps, p.hd);
    const unsigned char* codes = pages + ((is_v ? ps : 0) * (p.hd / 2) + d8 * 4);
    const unsigned char* ranges = pages + (ps * p.hd + ((is_v ? ps : 0) * ng + g) * 4);
    int slot[U];
    uint32_t w[U], r[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * step;
        slot[u] = row < p.n ? slot_map[row] : -1;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        w[u] = r[u] = 0u;                                  // a row without a slot reads as zeros
        if (slot[u] < 0 || slot[u] >= p.n_slots) continue;
        const unsigned page = slot[u] >> p.ps_log2, off = slot[u] & (ps - 1);
        const size_t at = (size_t)(page * p.G + head) * rec;
        w[u] = *reinterpret_cast<const uint32_t*>(codes + at + off * (p.hd / 2));
        r[u] = *reinterpret_cast<const uint32_t*>(ranges + at + off * ng * 4);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int row = row0 + u * step;
        if (row >= p.n) break;
        const float s = kv4_scale(r[u]), z = kv4_least(r[u]);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // 128 + c as float bits, without a conversion; s c is exact
            const uint32_t c = i < 4 ? w[u] << (16 - 4 * i) : w[u] >> (4 * i - 16);
            x[i] = fmaf(s, __uint_as_float((c & 0x000f0000u) | 0x43000000u) - 128.0f, z);
        }
        T* dst = (is_v ? v : k) + (size_t)row * p.G * p.hd + within * 8;
        if (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
        } else {
            // (the lanes of a pair have the same row, and write 32 bytes an instruction)
            kv4_swap_pair(x, 3u << (threadIdx.x & 30));
            float4* pair = reinterpret_cast<float4*>(dst) - (threadIdx.x & 1);
            pair[0] = make_float4(x[0], x[1], x[2], x[3]);
            pair[2] = make_float4(x[4], x[5], x[6], x[7]);
        }
    }
}

// ------------------------------------------------------------------ attention
struct Kv4Args {
    const void* q; long long ldq;
    void* out; long long ldo;
    const unsigned char* pages;
    const int* block_table; int max_blocks;
    const int* cu_rows; const int* seg_pos;
    float scale; int window; int ps, ps_log2; int H, G;
    // split form, [place] = [segment][row of it, of max_rows][head]: results of chunks [place][chunk][hd], (shift, sum of p)
    // [place][chunk][2]; with mass, or else null: scores [place][key], shift + log2(sum of p) [place]
    float* part_o; float* part_ml; float* scores; int ld_scores; float* lse_split;
    float* lse;                                            // tiled form with mass: shift + log2(sum of p) (base 2) [row][head], or null
    float* mass;                                           // [page][G][ps], or null
    int n_chunks, chunk;                                   // split form: chunks of `chunk` keys (from the first key of the segment's window on)
    int fused;                                             // split form: a segment's chunks are the CTAs of a cluster, which join them itself
    int max_rows;                                          // split form: segments of more rows are not its own
    int min_rows;                                          // tiled form: nor are segments of fewer rows this form's
    int n_seg;
    int split;                                             // tiled form: CTAs that share the keys of a tile of columns, or the columns of a tile of keys
};

// What a warp knows of its columns: column c of a segment stands for row c / R and head kvh R + c % R.
template <int NT>
struct Kv4Cols { int hi[NT][2], lo[NT][2]; };

template <int NT>
__device__ __forceinline__ void kv4_columns(Kv4Cols<NT>& C, int col0, int n_cols, int R, int pos0, int window, int lane) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int c = col0 + nt * 8 + 2 * (lane & 3) + i;
            const int hi = c < n_cols ? pos0 + c / R : -1;
            C.hi[nt][i] = hi;
            C.lo[nt][i] = window > 0 ? max(0, hi - window + 1) : 0;
        }
}

// ---- split form: few rows a segment (decode).  One CTA per (chunk of keys, kv head and 8 of its columns, segment).  Its tiles of KEYS
// keys come by the TMA into a ring of three stages, asked for two tiles ahead by the warps in turn; each of the four warps takes a
// quarter of a tile, with the softmax and output of its own keys, and the four are joined at the end.  A block of 16 keys takes 185 instructions
// with heads of 64 values and 333 with 128: hence the TMA and not cp.async (80 more), four CTAs an SM, and codes that are operands as they lie.
// 64 sequences of 1,000 to 2,100 keys, 32 heads over 8 of 128 values: 43 us, 2.7 TB/s; 90,001 and 131,072 keys with mass, 16 heads over 8 of 64: 61 us,
// 2.3 TB/s, 14 of them the join's.  No one thing bounds it there: 51 and 57 % of the issue slots and 31 % of memory's rate are used, by 11 to 13 of 64
// warps an SM that wait for their own products and loads; and the chunks are as long as the longest sequence's, so that CTAs with shorter ones (or none: 88
// of 592) leave SMs idle at the end.  A sequence much longer than the others of its batch pays for that most: 131,072 keys beside 63 x 500 are one
// chunk, 697 us, where 64 x 2,548, the same bytes, take 36.
KP_STATUS_WORD(g_kv4_status, kv4)                     // 0 ok; 1: a bounded wait gave up

template <int HD, int PARTS>
struct Kv4Split {
    static constexpr int TILE = HD <= 64 ? 64 : (HD <= 128 ? 32 : 16), TB = TILE / 16, STAGES = 3, NW = 4, KEYS = NW * TILE;
    static constexpr int STAGE = (Kv4<HD>::bytes(KEYS) + 1023) / 1024 * 1024;
    static constexpr size_t RING = (size_t)STAGES * STAGE, JOIN = sizeof(float) * (NW + 1) * 8 * (HD + 2);
    static constexpr size_t SMEM = 1024 + (RING > JOIN ? RING : JOIN);
};

// The first key of a segment's chunks: that of its first row's window, down to a whole tile.
__device__ __forceinline__ int kv4_chunk_base(int pos0, int window, int keys) {
    const int first = pos0 - window + 1;
    return window > 0 && first > 0 ? first / keys * keys : 0;
}
__host__ __device__ constexpr int kv4_tile_keys(int hd) { return hd <= 64 ? 256 : (hd <= 128 ? 128 : 64); }

template <int HD, int PARTS, bool KEEP, typename T>
__global__ void __launch_bounds__(128, PARTS == 1 && HD <= 128 ? 4 : 2)
kv4_split_kernel(const __grid_constant__ CUtensorMap codes, const Kv4Args p) {
    using F = Kv4<HD>;
    using S = Kv4Split<HD, PARTS>;
    constexpr bool CENTRE = KEEP || PARTS > 1;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ uint64_t full[S::STAGES], empty[S::STAGES];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // (the warp's number in a uniform register)
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; i++) { kp_mbar_init(&full[i], 1); kp_mbar_init(&empty[i], S::NW); }
        kp_mbar_init_fence();
    }
    __syncthreads();
    kp_pdl_begin();
    const int R = p.H / p.G, kvh = blockIdx.y % p.G, seg = blockIdx.z, chunk = blockIdx.x;
    const int row0 = p.cu_rows[seg], n_rows = p.cu_rows[seg + 1] - row0, pos0 = p.seg_pos[seg];
    const int col0 = (blockIdx.y / p.G) * 8, n_cols = n_rows * R;
    if (n_rows > p.max_rows || col0 >= n_cols) return;
    const int col1 = min(col0 + 8, n_cols) - 1;
    const int c_base = kv4_chunk_base(pos0, p.window, kv4_tile_keys(HD)) + chunk * p.chunk;      // the chunk's first key
    // the last key that the columns read in the chunk (and none that the block table has no page for)
    const int k_hi = min(min(pos0 + col1 / R, c_base + p.chunk - 1), p.max_blocks * p.ps - 1);
    const int k_first = p.window > 0 ? max(0, pos0 + col0 / R - p.window + 1) : 0;
    const int k_lo = max(k_first, c_base);
    const int t_lo = k_lo / S::KEYS, n_tiles = k_hi >= k_lo ? k_hi / S::KEYS - t_lo + 1 : 0;
    if (p.n_chunks > 1 && !p.fused && n_tiles == 0) return;      // (what joins chunks itself writes rows also where they read nothing)
    const int* bt = p.block_table + (size_t)seg * p.max_blocks;
    const int s_base = c_base - chunk * p.chunk;           // the key of the scores' first column

    // Lane j has piece j of a tile: the keys of one page (at most 16 pieces).
    const int piece = min(p.ps, S::KEYS);
    auto page_of = [&](int i) {                            // piece's page of tile i, or -1 if nothing of it is read
        const int key = (t_lo + i) * S::KEYS + lane * piece;
        return i < n_tiles && lane * piece < S::KEYS && key <= k_hi && key + piece - 1 >= k_lo ? bt[key >> p.ps_log2] : -1;
    };
    auto load = [&](int i, int page) {
        unsigned char* dst = smem + (i % S::STAGES) * S::STAGE;
        uint64_t* bar = &full[i % S::STAGES];
        const unsigned need = __ballot_sync(0xffffffffu, page >= 0);
        kp_mbar_expect_tx_warp(bar, (uint32_t)(__popc(need) * F::bytes(piece)));
        const int off = (t_lo + i) * S::KEYS & (p.ps - 1);
        // (piece by piece and by an elected lane, so that the copies' operands are uniform)
        for (int j = 0; j * piece < S::KEYS; j++) {
            const int rec = __shfl_sync(0xffffffffu, page, j) * p.G + kvh, at = j * piece;
            if (!(need >> j & 1)) continue;
            kp_tma_load_3d_warp(dst + at * F::ROW, &codes, 0, off, rec, bar);
            kp_tma_load_3d_warp(dst + (S::KEYS + at) * F::ROW, &codes, 0, p.ps + off, rec, bar);
            // (64 bytes of ranges a piece where pages have 16 keys: less than a tensor copy's destination is aligned to)
            const unsigned char* from = p.pages + (size_t)rec * kv4_page_bytes(p.ps, HD) + (size_t)p.ps * HD + off * 4 * F::NG;
            unsigned char* r = dst + S::KEYS * HD + at * 4 * F::NG;
            kp_bulk_g2s_warp(r, from, piece * 4 * F::NG, bar);
            kp_bulk_g2s_warp(r + S::KEYS * 4 * F::NG, from + (size_t)p.ps * 4 * F::NG, piece * 4 * F::NG, bar);
        }
    };
    // warp w asks for tiles w, w + 4, ...; the first two before anything else
    int page = page_of(warp);
    if (warp < S::STAGES - 1 && warp < n_tiles) {
        load(warp, page);
        page = page_of(warp + S::NW);
    }

    const Kv4Block<HD, S::KEYS> B(lane);
    Kv4Cols<1> C;
    kv4_columns<1>(C, col0, n_cols, R, pos0, p.window, lane);
    Kv4Q<HD, PARTS, 1> Q;
    {
        const int c = col0 + (lane >> 2);
        const T* const src[1] = {c < n_cols ? (const T*)p.q + (size_t)(row0 + c / R) * p.ldq + (size_t)(kvh * R + c % R) * HD : nullptr};
        kv4_load_q<HD, PARTS, 1, CENTRE, T>(Q, src, p.scale, lane);
    }
    float* sc[1][2] = {{nullptr, nullptr}};
    if (KEEP) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int c = col0 + 2 * (lane & 3) + i;
            if (c < n_cols) sc[0][i] = p.scores + (((size_t)seg * p.max_rows + c / R) * p.H + kvh * R + c % R) * p.ld_scores - s_base;
        }
    }
    Kv4Acc<HD, PARTS, 1> A;
    A.clear();
    // no key at all is masked between these
    const int safe_lo = p.window > 0 ? max(0, pos0 + col1 / R - p.window + 1) : 0, safe_hi = min(k_hi, pos0 + col0 / R);
    bool ok = true;
    int stage = 0, phase = 0;
#pragma unroll 1
    for (int i = 0; i < n_tiles; i++) {
        const int ahead = i + S::STAGES - 1;
        if (ahead < n_tiles && warp == ahead % S::NW) {
            // its stage is that of tile i - 1, which every warp has to be through with
            if (i > 0) ok = __all_sync(0xffffffffu, kp_mbar_wait_bounded(&empty[ahead % S::STAGES], ((ahead / S::STAGES) & 1) ^ 1));
            if (!ok) break;
            load(ahead, page);
            page = page_of(ahead + S::NW);
        }
        ok = __all_sync(0xffffffffu, kp_mbar_wait_bounded(&full[stage], phase));      // (a warp gives up as one)
        if (!ok) break;
        const int key0 = (t_lo + i) * S::KEYS + warp * S::TILE;
        const unsigned char* tile = smem + stage * S::STAGE;
        if (key0 <= k_hi && key0 + S::TILE - 1 >= k_lo) {
            if (key0 >= max(k_lo, safe_lo) && key0 + S::TILE - 1 <= safe_hi)
                kv4_tile<HD, S::KEYS, PARTS, 1, S::TB, CENTRE, false, KEEP>(A, Q, B, tile, warp * S::TILE, key0, C.hi, C.lo, k_lo, k_hi, lane, sc);
            else
                kv4_tile<HD, S::KEYS, PARTS, 1, S::TB, CENTRE, true, KEEP>(A, Q, B, tile, warp * S::TILE, key0, C.hi, C.lo, k_lo, k_hi, lane, sc);
        }
        __syncwarp();
        if (lane == 0) kp_mbar_arrive(&empty[stage]);
        if (++stage == S::STAGES) { stage = 0; phase ^= 1; }
    }
    if (__builtin_expect(!ok, 0)) {
        if (lane == 0) atomicExch(&g_kv4_status, 1);
        kp_linger_after_failure();
    }
    A.finish();
    __syncthreads();                                       // the rings are done with: the warps' results take their place
    float* jo = reinterpret_cast<float*>(smem);            // [warp][column][HD]
    float* jm = jo + S::NW * 8 * HD;                       // [warp][column]: shift
    float* jl = jm + S::NW * 8;                            // sum of p
#pragma unroll
    for (int y = 0; y < F::NG; y++)
#pragma unroll
        for (int j = 0; j < F::MT; j++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                *reinterpret_cast<float2*>(jo + (size_t)(warp * 8 + 2 * (lane & 3) + i) * HD + A.dim(y, j, lane)) = A.value(0, y, j, i);
    if (lane < 4) {
#pragma unroll
        for (int i = 0; i < 2; i++) { jm[warp * 8 + 2 * lane + i] = A.shift[0][i]; jl[warp * 8 + 2 * lane + i] = A.l[0][i]; }
    }
    __syncthreads();
    const int live = col1 - col0 + 1;
    float* co = jl + S::NW * 8;                            // the CTA's own: [column][HD], shift, sum of p
    float *cm = co + 8 * HD, *cl = cm + 8;
    auto place_of = [&](int col) { return ((size_t)seg * p.max_rows + col / R) * p.H + kvh * R + col % R; };
    auto write = [&](int c, int d, float v) {
        ((T*)p.out)[(size_t)(row0 + (col0 + c) / R) * p.ldo + (size_t)(kvh * R + (col0 + c) % R) * HD + d] = from_f32<T>(v);
    };
    for (int e = threadIdx.x; e < live * HD; e += 128) {
        const int c = e / HD, d = e - c * HD;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < S::NW; w++) M = fmaxf(M, jm[w * 8 + c]);
        float acc = 0.f, L = 0.f;
#pragma unroll
        for (int w = 0; w < S::NW; w++) {
            const float f = jm[w * 8 + c] == -INFINITY ? 0.f : kv4_exp2(jm[w * 8 + c] - M);
            if (jm[w * 8 + c] != -INFINITY) acc = fmaf(jo[(size_t)(w * 8 + c) * HD + d], f, acc);
            L = fmaf(jl[w * 8 + c], f, L);
        }
        if (p.n_chunks > 1 && p.fused) {
            co[e] = acc;
            if (d == 0) { cm[c] = M; cl[c] = L; }
        } else if (p.n_chunks == 1) {
            write(c, d, M == -INFINITY ? 0.f : acc / L);
            if (KEEP && d == 0) cm[c] = M == -INFINITY ? INFINITY : M + log2f(L);
            if (KEEP && d == 0 && !p.fused) p.lse_split[place_of(col0 + c)] = cm[c];
        } else {
            const size_t at = place_of(col0 + c) * p.n_chunks + chunk;
            p.part_o[at * HD + d] = acc;
            if (d == 0) { p.part_ml[at * 2] = M; p.part_ml[at * 2 + 1] = L; }
        }
    }
    if (!p.fused) return;
    float* lse = jm;                                       // (the warps' shifts have been read) [column]
    if (p.n_chunks > 1) {
        // the cluster's CTAs are the chunks: each joins its share of the outputs, in the order of the chunks, from all of them
        float* weight = jo;                                // (so have their results) [column][chunk of 8]
        kv4_cluster_sync();
        if (threadIdx.x < live) {
            float m[8], l[8], M = -INFINITY, L = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < p.n_chunks) { m[k] = kv4_peer(cm + threadIdx.x, k); l[k] = kv4_peer(cl + threadIdx.x, k); }
#pragma unroll
            for (int k = 0; k < 8; k++) if (k < p.n_chunks) M = fmaxf(M, m[k]);
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < p.n_chunks) { m[k] = kv4_exp2(m[k] - (M == -INFINITY ? 0.f : M)); L = fmaf(l[k], m[k], L); }
#pragma unroll
            for (int k = 0; k < 8; k++) if (k < p.n_chunks) weight[threadIdx.x * 8 + k] = M == -INFINITY ? 0.f : m[k] / L;
            if (KEEP) lse[threadIdx.x] = M == -INFINITY ? INFINITY : M + log2f(L);
        }
        __syncthreads();
        for (int e = chunk * 128 + threadIdx.x; e < live * HD; e += p.n_chunks * 128) {
            const int c = e / HD;
            float x[8], acc = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) if (k < p.n_chunks) x[k] = kv4_peer(co + e, k);
#pragma unroll
            for (int k = 0; k < 8; k++) if (k < p.n_chunks) acc = fmaf(x[k], weight[c * 8 + k], acc);
            write(c, e - c * HD, acc);
        }
    }
    if (KEEP) {
        // the weights of the chunk's keys: a thread a key, columns in order (they are all of the segment's); all loads of four keys at once
        __syncthreads();
        const float* sums = p.n_chunks > 1 ? lse : cm;
        constexpr int U = 4;
        for (int key0 = k_lo + threadIdx.x; key0 <= k_hi; key0 += 128 * U) {
            float x[U][8], *to[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int key = min(key0 + u * 128, k_hi);
                to[u] = p.mass + ((size_t)bt[key >> p.ps_log2] * p.G + kvh) * p.ps + (key & (p.ps - 1));
#pragma unroll
                for (int c = 0; c < 8; c++) if (c < live) x[u][c] = p.scores[place_of(c) * p.ld_scores + key - s_base];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                float w = 0.f;                             // (a score of -inf: the column does not read the key, whatever its sum is)
#pragma unroll
                for (int c = 0; c < 8; c++) if (c < live) w += x[u][c] == -INFINITY ? 0.f : kv4_exp2(x[u][c] - sums[c]);
                if (key0 + u * 128 <= k_hi) kv4_add_mass(to[u], w);
            }
        }
    }
    if (p.n_chunks > 1) kv4_cluster_sync();                // (nobody leaves while another reads its shared memory)
}

#define KV4_MASS_KEYS 1024                              // keys of a CTA that adds weights up
// ---- joins the chunks and adds up the mass: a warp a (segment, row, head), in the order of the chunks; behind those CTAs, where
// there is mass, a CTA a (1024 keys, kv head, segment) with a thread a key, rows and heads in order.  Both find a (row, head)'s shift and sum from
// the chunks' (at most a few dozen), so that neither waits for the other.
// Largest shift and sum of p of the chunks c_lo .. c_hi of a place; every lane gets them.
__device__ __forceinline__ float2 kv4_total(const float* ml, int c_lo, int c_hi, int lane) {
    float M = -INFINITY, L = 0.f;
    for (int c0 = c_lo; c0 <= c_hi; c0 += 32) {
        const int c = c0 + lane;
        const float2 x = c <= c_hi ? reinterpret_cast<const float2*>(ml)[c] : make_float2(-INFINITY, 0.f);
        const float top = fmaxf(M, warp_max(x.x));
        const float part = warp_sum(x.x == -INFINITY ? 0.f : x.y * kv4_exp2(x.x - top));
        L = (M == -INFINITY ? 0.f : L * kv4_exp2(M - top)) + part;
        M = top;
    }
    return make_float2(M, L);
}

template <typename T>
__global__ void __launch_bounds__(128)
kv4_join_kernel(const Kv4Args p, int hd, int n_join, int mass_blocks) {
    kp_pdl_begin();
    const int lane = threadIdx.x & 31;
    if ((int)blockIdx.x < n_join) {
        const int place = blockIdx.x * 4 + (threadIdx.x >> 5);
        const int h = place % p.H, r = (place / p.H) % p.max_rows, seg = place / p.H / p.max_rows;
        if (seg >= p.n_seg) return;
        const int row = p.cu_rows[seg] + r, n_rows = p.cu_rows[seg + 1] - p.cu_rows[seg];
        if (r >= n_rows || n_rows > p.max_rows) return;
        const int hi = p.seg_pos[seg] + r;
        const int lo = p.window > 0 ? max(0, hi - p.window + 1) : 0;
        const float* ml = p.part_ml + (size_t)place * p.n_chunks * 2;
        const float* po = p.part_o + (size_t)place * p.n_chunks * hd;
        const int base = kv4_chunk_base(p.seg_pos[seg], p.window, kv4_tile_keys(hd));
        const int c_lo = (lo - base) / p.chunk, c_hi = hi < 0 ? -1 : min((hi - base) / p.chunk, p.n_chunks - 1);
        const float2 t = kv4_total(ml, c_lo, c_hi, lane);
        const float inv = t.x == -INFINITY ? 0.f : 1.0f / t.y;
        for (int d = lane * 2; d < hd; d += 64) {
            float2 acc = make_float2(0.f, 0.f);
            for (int c0 = c_lo; c0 <= c_hi; c0 += 8) {
                float2 v[8];
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool in = c0 + e <= c_hi;
                    w[e] = in ? ml[2 * (c0 + e)] : -INFINITY;
                    v[e] = in ? *reinterpret_cast<const float2*>(po + (size_t)(c0 + e) * hd + d) : make_float2(0.f, 0.f);
                }
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (w[e] != -INFINITY) {
                        const float f = kv4_exp2(w[e] - t.x);
                        acc.x = fmaf(v[e].x, f, acc.x);
                        acc.y = fmaf(v[e].y, f, acc.y);
                    }
            }
            T* dst = (T*)p.out + (size_t)row * p.ldo + (size_t)h * hd + d;
            dst[0] = from_f32<T>(acc.x * inv);
            dst[1] = from_f32<T>(acc.y * inv);
        }
        return;
    }
    __shared__ float lse[64];                              // of 64 (row, head)s at a time
    const int b = blockIdx.x - n_join, kvh = b / mass_blocks % p.G, seg = b / mass_blocks / p.G;
    const int n_rows = p.cu_rows[seg + 1] - p.cu_rows[seg], pos0 = p.seg_pos[seg], R = p.H / p.G, n_cols = n_rows * R;
    const int base = kv4_chunk_base(pos0, p.window, kv4_tile_keys(hd)), k0 = base + (b % mass_blocks) * KV4_MASS_KEYS;
    // (in front of the first row's window nothing is read, and the pages may be somebody else's by now)
    const int first = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
    const int last = min(min(pos0 + n_rows, p.max_blocks * p.ps), base + p.ld_scores) - 1;
    if (n_rows > p.max_rows || k0 > last || k0 + KV4_MASS_KEYS - 1 < first) return;
    constexpr int U = KV4_MASS_KEYS / 128;
    // what does not wait for the chunks' sums is asked for first: where the keys' masses lie, and the scores of the first two columns
    float sum[U], *to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int key = min(max(k0 + u * 128 + (int)threadIdx.x, first), last);
        to[u] = p.mass + ((size_t)p.block_table[(size_t)seg * p.max_blocks + (key >> p.ps_log2)] * p.G + kvh) * p.ps + (key & (p.ps - 1));
        sum[u] = 0.f;
    }
    struct Two { int lo[2], hi[2]; float x[2][U]; };
    auto fetch = [&](Two& t, int c) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int r = (c + j) / R;
            t.hi[j] = c + j < n_cols ? min(pos0 + r, last) : -1;
            t.lo[j] = p.window > 0 ? max(0, pos0 + r - p.window + 1) : 0;
            const float* sc = p.scores + (((size_t)seg * p.max_rows + r) * p.H + kvh * R + (c + j) % R) * p.ld_scores - base;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int key = k0 + u * 128 + threadIdx.x;
                t.x[j][u] = key >= t.lo[j] && key <= t.hi[j] ? sc[key] : 0.f;
            }
        }
    };
    Two now;
    fetch(now, 0);
    for (int c0 = 0; c0 < n_cols; c0 += 64) {
        const int n = min(64, n_cols - c0);
        __syncthreads();
        for (int i = threadIdx.x >> 5; i < n; i += 4) {
            const int r = (c0 + i) / R, h = kvh * R + (c0 + i) % R, hi = pos0 + r;
            const size_t place = ((size_t)seg * p.max_rows + r) * p.H + h;
            float v;
            if (p.n_chunks == 1) {
                v = p.lse_split[place];
            } else {
                const int lo = p.window > 0 ? max(0, hi - p.window + 1) : 0;
                const int c_lo = (lo - base) / p.chunk, c_hi = hi < 0 ? -1 : min((hi - base) / p.chunk, p.n_chunks - 1);
                const float2 t = kv4_total(p.part_ml + place * p.n_chunks * 2, c_lo, c_hi, lane);
                v = t.x == -INFINITY ? INFINITY : t.x + log2f(t.y);
            }
            if (lane == 0) lse[i] = v;
        }
        __syncthreads();
#pragma unroll 1
        for (int i = 0; i < n; i += 2) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int key = k0 + u * 128 + threadIdx.x;
                    if (key >= now.lo[j] && key <= now.hi[j]) sum[u] += kv4_exp2(now.x[j][u] - lse[i + j]);
                }
            if (c0 + i + 2 < n_cols) fetch(now, c0 + i + 2);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int key = k0 + u * 128 + threadIdx.x;
        if (key >= first && key <= last) kv4_add_mass(to[u], sum[u]);
    }
}

// ---- tiled form: many rows a segment (portions of prompts) that the tcgen05 form does not take.  A CTA takes 32 NT columns of a kv head (8 NT a warp,
// as many as the registers of its output hold: codes become operands once for all of them) and walks
// their keys in tiles of 64 that its warps bring and share.
template <int HD, int PARTS>
struct Kv4Tiled {
    static constexpr int NT = PARTS == 1 ? (HD <= 64 ? 4 : (HD <= 128 ? 2 : 1)) : (HD <= 64 ? 2 : 1);
    static constexpr int COLS = 32 * NT, TILE = 64, STAGE = Kv4<HD>::bytes(64);
    static constexpr size_t JOIN = sizeof(float) * kv4_share_floats(COLS, HD, 8), SMEM = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
};

// The tile'th of the tiles that the segments of at least min_rows rows make of `per` columns each: its segment and first column
// (found by one warp; segment -1: there is none).
__device__ __forceinline__ void kv4_find_tile(const Kv4Args& p, int tile, int per, int R, int lane, int& seg, int& col0) {
    seg = -1;
    int before = 0;
    for (int base = 0; base < p.n_seg; base += 32) {
        const int i = base + lane;
        int rows = 0;
        if (i < p.n_seg) rows = p.cu_rows[i + 1] - p.cu_rows[i];
        const int mine = rows >= p.min_rows ? (rows * R + per - 1) / per : 0;
        int run = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < before + run);
        if (hit) {
            const int src = __ffs(hit) - 1;
            seg = base + src;
            const int all = __shfl_sync(0xffffffffu, mine, src), end = before + __shfl_sync(0xffffffffu, run, src);
            col0 = (all - 1 - (tile - (end - all))) * per;     // (the last columns of a segment, which read the most keys, first)
            return;
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    }
}

template <int HD, int PARTS, bool CENTRE, typename T>
__global__ void __launch_bounds__(128)
kv4_tiled_kernel(const Kv4Args p) {
    using F = Kv4<HD>;
    using S = Kv4Tiled<HD, PARTS>;
    constexpr int NT = S::NT;
    kp_pdl_begin();
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // (the warp's number in a uniform register)
    // (the longest tiles first, of all heads)
    const int R = p.H / p.G, rank = blockIdx.x % p.split, kvh = blockIdx.x / p.split % p.G;
    int seg, cta_col0 = 0;
    kv4_find_tile(p, blockIdx.x / p.split / p.G, S::COLS, R, lane, seg, cta_col0);
    if (seg < 0) return;
    const int row0 = p.cu_rows[seg], n_rows = p.cu_rows[seg + 1] - row0, pos0 = p.seg_pos[seg], n_cols = n_rows * R;
    const int cta_col1 = min(cta_col0 + S::COLS, n_cols) - 1;
    const int k_hi = min(pos0 + cta_col1 / R, p.max_blocks * p.ps - 1), k_lo = p.window > 0 ? max(0, pos0 + cta_col0 / R - p.window + 1) : 0;
    const int t_all = k_hi >= k_lo ? k_hi / S::TILE - k_lo / S::TILE + 1 : 0, t_skip = t_all * rank / p.split;
    const int t_lo = k_lo / S::TILE + t_skip, n_tiles = t_all * (rank + 1) / p.split - t_skip;      // this CTA's
    const int* bt = p.block_table + (size_t)seg * p.max_blocks;
    const size_t rec = (size_t)kv4_page_bytes(p.ps, HD);
    auto load = [&](int i) {                               // every warp a block of the tile
        const int key = (t_lo + i) * S::TILE + warp * 16;
        if (i < n_tiles && key <= k_hi && key + 15 >= k_lo) {
            const int page = key >> p.ps_log2;
            kv4_load_block<HD, S::TILE>(smem + (size_t)(i & 1) * S::STAGE, warp * 16, p.pages + ((size_t)bt[page] * p.G + kvh) * rec, key & (p.ps - 1), p.ps, lane);
        }
        cp_async_commit();
    };
    load(0);
    const int col0 = cta_col0 + warp * 8 * NT;
    const Kv4Block<HD, S::TILE> B(lane);
    Kv4Cols<NT> C;
    kv4_columns<NT>(C, col0, n_cols, R, pos0, p.window, lane);
    Kv4Q<HD, PARTS, NT> Q;
    const T* src[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int c = col0 + nt * 8 + (lane >> 2);
        src[nt] = c < n_cols ? (const T*)p.q + (size_t)(row0 + c / R) * p.ldq + (size_t)(kvh * R + c % R) * HD : nullptr;
    }
    kv4_load_q<HD, PARTS, NT, CENTRE, T>(Q, src, p.scale, lane);
    float* sc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) sc[nt][0] = sc[nt][1] = nullptr;
    Kv4Acc<HD, PARTS, NT> A;
    A.clear();
    const int col1 = min(col0 + 8 * NT, n_cols) - 1;       // the warp's last column (it has none where col1 < col0)
    const int w_hi = min(pos0 + col1 / R, k_hi), w_lo = p.window > 0 ? max(0, pos0 + col0 / R - p.window + 1) : 0;
    const int safe_hi = pos0 + col0 / R, safe_lo = p.window > 0 ? max(0, pos0 + col1 / R - p.window + 1) : 0;
#pragma unroll 1
    for (int i = 0; i < n_tiles; i++) {
        load(i + 1);
        cp_async_wait<1>();
        __syncthreads();
        const unsigned char* tile = smem + (size_t)(i & 1) * S::STAGE;
#pragma unroll 1
        for (int b = 0; b < 4; b++) {
            const int key0 = (t_lo + i) * S::TILE + b * 16;
            if (col1 < col0 || key0 > w_hi || key0 + 15 < w_lo) continue;
            if (key0 >= max(k_lo, safe_lo) && key0 + 15 <= safe_hi)                  // (columns that are not there read along, and are not written)
                kv4_tile<HD, S::TILE, PARTS, NT, 1, CENTRE, false, false>(A, Q, B, tile, b * 16, key0, C.hi, C.lo, k_lo, k_hi, lane, sc);
            else
                kv4_tile<HD, S::TILE, PARTS, NT, 1, CENTRE, true, false>(A, Q, B, tile, b * 16, key0, C.hi, C.lo, k_lo, k_hi, lane, sc);
        }
        __syncthreads();                                   // the next tile but one takes this one's place
    }
    cp_async_wait<0>();
    A.finish();
    if (p.split > 1) {
        float* part = reinterpret_cast<float*>(smem);      // (the last tile has been read by all)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int c = warp * 8 * NT + nt * 8 + 2 * (lane & 3) + i;
                const bool none = A.shift[nt][i] == -INFINITY;
                const float inv = none ? 0.f : 1.0f / A.l[nt][i];
#pragma unroll
                for (int y = 0; y < F::NG; y++)
#pragma unroll
                    for (int j = 0; j < F::MT; j++) {
                        const float2 o = A.value(nt, y, j, i);
                        *reinterpret_cast<float2*>(part + kv4_share_at(c, A.dim(y, j, lane), HD)) = none ? make_float2(0.f, 0.f) : make_float2(o.x * inv, o.y * inv);
                    }
                if (lane < 4) kv4_share_sums(part, S::COLS, HD, c, A.shift[nt][i], A.l[nt][i]);
            }
        kv4_cluster_sync();
        kv4_join_shares<T, HD, S::COLS, 128, false, 8>(
            part, p.split, rank, cta_col1 - cta_col0 + 1,
            [&](int col) { return (T*)p.out + (size_t)(row0 + (cta_col0 + col) / R) * p.ldo + (size_t)(kvh * R + (cta_col0 + col) % R) * HD; },
            [&](int col, float top, float sum) {
                const int c = cta_col0 + col;
                if (p.lse && c < n_cols) p.lse[(size_t)(row0 + c / R) * p.H + kvh * R + c % R] = sum == 0.f ? INFINITY : top + log2f(sum);
            });
        kv4_cluster_sync();                                // (nobody leaves while its shares are read)
        return;
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int c = col0 + nt * 8 + 2 * (lane & 3) + i;
            if (c >= n_cols) continue;
            const size_t row = row0 + c / R;
            const int h = kvh * R + c % R;
            const bool none = A.shift[nt][i] == -INFINITY;
            const float inv = none ? 0.f : 1.0f / A.l[nt][i];
            T* dst = (T*)p.out + row * p.ldo + (size_t)h * HD;
#pragma unroll
            for (int y = 0; y < F::NG; y++)
#pragma unroll
                for (int j = 0; j < F::MT; j++) {
                    float2 o = A.value(nt, y, j, i);
                    if (none) o = make_float2(0.f, 0.f);
                    dst[A.dim(y, j, lane)] = from_f32<T>(o.x * inv);
                    dst[A.dim(y, j, lane) + 1] = from_f32<T>(o.y * inv);
                }
            if (p.lse && lane < 4) p.lse[row * p.H + h] = none ? INFINITY : A.shift[nt][i] + log2f(A.l[nt][i]);
        }
}

// ---- the tiled form's mass: a cluster of CTAs per (128 keys or 64, kv head, segment), which share the columns that read the keys.  Their warps take 8 at a
// time, compute the scores again and add up 2^(score - lse); the warps' sums are added in their order, then the CTAs'.
template <int HD, int PARTS, typename T>
__global__ void __launch_bounds__(128)
kv4_mass_kernel(const Kv4Args p) {
    using F = Kv4<HD>;
    constexpr int NB = HD <= 128 ? 8 : 4, KEYS = NB * 16;
    kp_pdl_begin();
    __shared__ __align__(128) unsigned char smem[F::bytes(KEYS)];
    __shared__ float part[4][KEYS];
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;      // (the warp's number in a uniform register)
    // the first keys first, of all heads and segments: most rows read them
    const int n_ctas = p.split, rank = blockIdx.x % n_ctas, place = blockIdx.x / n_ctas;
    const int kvh = place % p.G, seg = place / p.G % p.n_seg, k0 = place / p.G / p.n_seg * KEYS, R = p.H / p.G;
    const int row0 = p.cu_rows[seg], n_rows = p.cu_rows[seg + 1] - row0, pos0 = p.seg_pos[seg];
    // keys that any row reads (in front of them the pages may be somebody else's by now)
    const int last = min(pos0 + n_rows - 1, p.max_blocks * p.ps - 1), first = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
    if (n_rows < p.min_rows || k0 > last || k0 + KEYS - 1 < first) return;
    // rows that read any of the keys
    const int r_lo = max(0, k0 - pos0), r_hi = p.window > 0 ? min(n_rows - 1, k0 - pos0 + KEYS - 2 + p.window) : n_rows - 1;
    if (r_hi < r_lo) return;
    const int* bt = p.block_table + (size_t)seg * p.max_blocks;
    for (int b = warp; b < NB; b += 4) {
        const int key = k0 + b * 16;
        if (key <= last && key + 15 >= first) {
            const int page = key >> p.ps_log2;
            kv4_load_block<HD, KEYS>(smem, b * 16, p.pages + ((size_t)bt[page] * p.G + kvh) * (size_t)kv4_page_bytes(p.ps, HD), key & (p.ps - 1), p.ps, lane);
        }
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    float sum[NB][2];
#pragma unroll
    for (int b = 0; b < NB; b++) sum[b][0] = sum[b][1] = 0.f;
    const Kv4Block<HD, KEYS> B(lane);
    const int c_end = (r_hi + 1) * R, key = F::key_of(lane >> 2);
#pragma unroll 1
    for (int col0 = r_lo * R + (rank * 4 + warp) * 8; col0 < c_end; col0 += 32 * n_ctas) {
        Kv4Q<HD, PARTS, 1> Q;
        const int cq = col0 + (lane >> 2);
        const T* const src[1] = {cq < c_end ? (const T*)p.q + (size_t)(row0 + cq / R) * p.ldq + (size_t)(kvh * R + cq % R) * HD : nullptr};
        kv4_load_q<HD, PARTS, 1, true, T>(Q, src, p.scale, lane);
        float lse[2];
        int hi[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int c = col0 + 2 * (lane & 3) + i;
            hi[i] = c < c_end ? pos0 + c / R : -1;
            lse[i] = c < c_end ? p.lse[(size_t)(row0 + c / R) * p.H + kvh * R + c % R] : 0.f;
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float s[1][4];
            kv4_scores<HD, KEYS, PARTS, 1, true>(s, smem, b * 16, B, Q);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int k = k0 + b * 16 + key + (e >> 1) * 8, h = hi[e & 1];
                const bool sees = k <= h && (p.window <= 0 || k > h - p.window);
                sum[b][e >> 1] += sees ? kv4_exp2(s[0][e] - lse[e & 1]) : 0.f;
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float v = sum[b][e];
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            if ((lane & 3) == 0) part[warp][b * 16 + key + e * 8] = v;
        }
    __syncthreads();
    const int k = threadIdx.x;
    float all = 0.f;
    if (k < KEYS) part[0][k] = all = (part[0][k] + part[1][k]) + (part[2][k] + part[3][k]);
    if (n_ctas > 1) kv4_cluster_sync();
    if (rank == 0 && k < KEYS && k0 + k <= last && k0 + k >= first) {
        for (int i = 1; i < n_ctas; i++) all += kv4_peer(part[0] + k, i);
        const int page = bt[(k0 + k) >> p.ps_log2];
        kv4_add_mass(p.mass + ((size_t)page * p.G + kvh) * p.ps + ((k0 + k) & (p.ps - 1)), all);
    }
    if (n_ctas > 1) kv4_cluster_sync();                    // (nobody leaves while its sums are read)
}

// ------------------------------------------------------------------ launchers
#define KV4_DISPATCH_HD(hd, HD, ...)                                   \
    switch (hd) {                                                      \
        case 32: { constexpr int HD = 32; __VA_ARGS__; } break;        \
        case 64: { constexpr int HD = 64; __VA_ARGS__; } break;        \
        case 96: { constexpr int HD = 96; __VA_ARGS__; } break;        \
        case 128: { constexpr int HD = 128; __VA_ARGS__; } break;      \
        case 192: { constexpr int HD = 192; __VA_ARGS__; } break;      \
        case 256: { constexpr int HD = 256; __VA_ARGS__; } break;      \
        default: return KP_ERR_UNSUPPORTED;                            \
    }

static int kv4_log2(int v) { int l = 0; while ((1 << l) < v) l++; return l; }

// CTAs of the writing and reading kernels with one row a thread, and with `rows`
#define KV4_ONE_ROW (148 * 8)                              // more CTAs than that are more than fit at once: several rows a thread
static int kv4_row_blocks(const Kv4Rows& p, int rows, unsigned (&blocks)[2]) {
    const long long per_row = 2LL * p.G * p.hd / 8;
    if (p.n * per_row >= (1LL << 32) - 256 || (p.n_slots >> p.ps_log2) * p.G >= 1LL << 32 || 2LL * p.hd << p.ps_log2 > 1LL << 30) return KP_ERR_UNSUPPORTED;
    blocks[0] = (unsigned)((p.n * per_row + 255) / 256);
    blocks[1] = (unsigned)((((long long)p.n + rows - 1) / rows * per_row + 255) / 256);
    return 0;
}

template <int HD, int PARTS, bool CENTRE, typename T>
static int kv4_run_tiled(Kv4Args a, long long tiles, long long busy, int max_context, cudaStream_t st) {
    using S = Kv4Tiled<HD, PARTS>;
    static_assert(S::SMEM <= 48 * 1024, "needs no raised limit of shared memory");
    // A tile's keys over as many CTAs, up to eight, as the GPU holds clusters of, where each has a tile of keys and there are three or more.  Measured
    // with 32 heads over 8, one CTA a tile against the rule's: float32 rows of 64 values, 64 rows behind 4000 keys 139 us against 42, behind
    // 500 26 against 17, 4 x 64 behind 2000 77 against 57; bfloat16 of 256 values 168 against 72, 32 against 22, 133 against 132.
    const int reach = a.window > 0 && a.window + S::COLS / (a.H / a.G) < max_context ? a.window + S::COLS / (a.H / a.G) : max_context;
    a.split = 1;
    for (int n = 8; n > 1 && a.split == 1; n--)
        if (busy * a.G <= kv4_fit<kv4_tiled_kernel<HD, PARTS, CENTRE, T>>(n, 128, S::SMEM) && (reach + S::TILE - 1) / S::TILE >= max(n, 3)) a.split = n;
    if (tiles * a.G * a.split > 2147483647LL) return KP_ERR_UNSUPPORTED;
    const Kv4Launch l((unsigned)(tiles * a.G), a.split, 128, S::SMEM, st);
    const cudaError_t c = cudaLaunchKernelEx(&l.cfg, kv4_tiled_kernel<HD, PARTS, CENTRE, T>, a);
    return c ? (int)c : kp_launch_status();
}

// The pages' codes as the TMA sees them: one record a (page, kv head), rows of codes (keys', then values').  A box has the keys of one page that lie
// in one tile.
template <int HD>
static int kv4_codes_map(CUtensorMap* codes, const Kv4Args& a, long long n_pages, int tile) {
    using F = Kv4<HD>;
    const KpEncodeTiledFn fn = kp_encode_tiled_fn();
    const cuuint64_t records = (cuuint64_t)n_pages * a.G, bytes = (cuuint64_t)kv4_page_bytes(a.ps, HD);
    if (!fn || n_pages < 1 || records > 2147483647ull) return KP_ERR_UNSUPPORTED;
    const cuuint32_t one[3] = {1, 1, 1}, box[3] = {F::ROW, (cuuint32_t)(a.ps < tile ? a.ps : tile), 1};
    const cuuint64_t dims[3] = {F::ROW, 2ull * a.ps, records}, strides[2] = {F::ROW, bytes};
    const CUresult r = fn(codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<unsigned char*>(a.pages), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          F::ROW == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : (F::ROW == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE),
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : KP_ERR_UNSUPPORTED;
}

template <int HD, int PARTS, bool KEEP, typename T>
static int kv4_run_split(const Kv4Args& a, long long n_pages, cudaStream_t st) {
    using S = Kv4Split<HD, PARTS>;
    static std::atomic<unsigned long long> ready{0};
    alignas(64) CUtensorMap codes;
    int e = kv4_codes_map<HD>(&codes, a, n_pages, S::KEYS);
    if (e) return e;
    if ((e = kp_smem_limit(kv4_split_kernel<HD, PARTS, KEEP, T>, S::SMEM, ready))) return e;
    static_assert(S::KEYS == kv4_tile_keys(HD), "chunks begin and end with a tile");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_chunks, a.G * ((a.max_rows * (a.H / a.G) + 7) / 8), a.n_seg);
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.n_chunks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.fused && a.n_chunks > 1 ? 2 : 1;
    const cudaError_t c = cudaLaunchKernelEx(&cfg, kv4_split_kernel<HD, PARTS, KEEP, T>, codes, a);
    return c ? (int)c : kp_launch_status();
}

template <int HD, int PARTS, typename T>
static int kv4_run(const Kv4Args& a, long long n_pages, int n_rows, int long_rows, int long_keys, cudaStream_t st) {
    using S = Kv4Tiled<HD, PARTS>;
    constexpr int KEYS = HD <= 128 ? 128 : 64;         // of the mass kernel
    const int R = a.H / a.G;
    const long long tiles = ((long long)n_rows * R + S::COLS - 1) / S::COLS + a.n_seg, places = (long long)((long_keys + KEYS - 1) / KEYS) * a.G * a.n_seg;
    if (long_rows > 0 && (tiles * a.G > 2147483647LL || (a.mass && places > 2147483647LL))) return KP_ERR_UNSUPPORTED;
    if (a.max_rows > 0) {
        const int e = a.mass ? kv4_run_split<HD, PARTS, true, T>(a, n_pages, st) : kv4_run_split<HD, PARTS, false, T>(a, n_pages, st);
        if (e) return e;
        if (!a.fused && (a.n_chunks > 1 || a.mass)) {
            const long long join = a.n_chunks > 1 ? ((long long)a.n_seg * a.max_rows * a.H + 3) / 4 : 0;
            const int mass_blocks = a.mass ? (a.n_chunks * a.chunk + KV4_MASS_KEYS - 1) / KV4_MASS_KEYS : 0;
            const long long blocks = join + (long long)mass_blocks * a.G * a.n_seg;
            if (blocks > 2147483647LL) return KP_ERR_UNSUPPORTED;
            const cudaError_t c = kp_launch_pdl(kv4_join_kernel<T>, dim3((unsigned)blocks), dim3(128), 0, st, a, HD, (int)join, mass_blocks);
            if (c) return (int)c;
        }
    }
    if (long_rows > 0) {
        // about how many tiles there are: as where each segment has the most rows
        const long long busy = max(tiles - a.n_seg, (long long)(n_rows / long_rows) * (((long long)long_rows * R + S::COLS - 1) / S::COLS));
        // (with mass the scores are those that the mass is computed from again)
        const int e = a.mass ? kv4_run_tiled<HD, PARTS, true, T>(a, tiles, busy, long_keys, st) : kv4_run_tiled<HD, PARTS, (PARTS > 1), T>(a, tiles, busy, long_keys, st);
        if (e) return e;
        if (a.mass) {
            Kv4Args m = a;
            m.split = 1;
            for (int n = 8; n > 1 && m.split == 1; n--)
                if (places <= kv4_fit<kv4_mass_kernel<HD, PARTS, T>>(n, 128, 0) && (long long)long_rows * R >= 64 * n) m.split = n;
            const Kv4Launch l((unsigned)places, m.split, 128, 0, st);
            const cudaError_t c = cudaLaunchKernelEx(&l.cfg, kv4_mass_kernel<HD, PARTS, T>, m);
            if (c) return (int)c;
        }
    }
    return kp_launch_status();
}

extern "C" {

int kp_kv4_write(const void* k, long long ldk, const void* v, long long ldv, void* pages, long long n_pages, const int* slot_map, int n, int ps,
                 int G, int hd, int dtype, void* stream) {
    if (n <= 0) return 0;
    if (hd < 32 || hd % 32 || ps < 16 || (ps & (ps - 1)) || G < 1 || ((uintptr_t)pages & 15)) return KP_ERR_BAD_ARG;
    const Kv4Rows p = {n, kv4_log2(ps), G, hd, hd % 64 == 0 ? 64 : 32, n_pages * ps};
    unsigned blocks[2];
    const int e = kv4_row_blocks(p, 3, blocks);
    if (e) return e;
    const bool many = blocks[0] > KV4_ONE_ROW;
    KP_DISPATCH_DTYPE(dtype, T, {
        const long long a = 16 / sizeof(T);
        const bool vec = !(((uintptr_t)k | (uintptr_t)v) & 15) && ldk % a == 0 && ldv % a == 0;
        auto kern = vec ? (many ? kv4_write_kernel<T, true, 3> : kv4_write_kernel<T, true, 1>) : (many ? kv4_write_kernel<T, false, 3> : kv4_write_kernel<T, false, 1>);
        const cudaError_t c = kp_launch_pdl(kern, dim3(blocks[many]), dim3(256), 0, (cudaStream_t)stream, (const T*)k, ldk, (const T*)v, ldv,
                                            (unsigned char*)pages, slot_map, p);
        if (c) return (int)c;
    });
    return kp_launch_status();
}

int kp_kv4_read(const void* pages, long long n_pages, const int* slot_map, void* k, void* v, int n, int ps, int G, int hd, int dtype, void* stream) {
    if (n <= 0) return 0;
    if (hd < 32 || hd % 32 || ps < 16 || (ps & (ps - 1)) || G < 1 || (((uintptr_t)pages | (uintptr_t)k | (uintptr_t)v) & 15)) return KP_ERR_BAD_ARG;
    const Kv4Rows p = {n, kv4_log2(ps), G, hd, hd % 64 == 0 ? 64 : 32, n_pages * ps};
    unsigned blocks[2];
    const int e = kv4_row_blocks(p, 4, blocks);
    if (e) return e;
    const bool many = blocks[0] > KV4_ONE_ROW;
    KP_DISPATCH_DTYPE(dtype, T, {
        const cudaError_t c = kp_launch_pdl(many ? kv4_read_kernel<T, 4> : kv4_read_kernel<T, 1>, dim3(blocks[many]), dim3(256), 0, (cudaStream_t)stream,
                                            (const unsigned char*)pages, slot_map, (T*)k, (T*)v, p);
        if (c) return (int)c;
    });
    return kp_launch_status();
}

// Segments of at most `short_rows` rows go to the split form (0: none), the others to the tiled form if `long_rows` is not 0.
// Scratch: see Kv4Args; lse_split and scores where there is mass and a split form, lse where there is mass and a tiled one.
int kp_kv4_attention(const void* q, long long ldq, const void* pages, long long n_pages, const int* block_table, int max_blocks, const int* cu_rows, const int* seg_pos,
                     int n_seg, void* out, long long ldo, float scale, int window, int ps, int H, int G, int hd, int n_rows, int short_rows,
                     int long_rows, int n_chunks, int chunk, int fused, int max_context, float* part_o, float* part_ml, float* scores, int ld_scores,
                     float* lse_split, float* lse, float* mass, int dtype, void* stream) {
    if (n_rows <= 0 || n_seg <= 0) return 0;
    if (G < 1 || H < 1 || H % G || ps < 16 || (ps & (ps - 1)) || window < 0 || n_chunks < 1 || chunk < 64 || chunk % 64 || n_seg > 65535 || H > 65535 ||
        ((uintptr_t)pages & 15) || (mass && ((long_rows && !lse) || (short_rows > 0 && (!scores || !lse_split)))) || (n_chunks > 1 && short_rows > 0 && !fused && (!part_o || !part_ml)) ||
        chunk % kv4_tile_keys(hd) || (fused && (n_chunks > 8 || (mass && (long long)short_rows * (H / G) > 8))))
        return KP_ERR_BAD_ARG;
    Kv4Args a = {};
    a.q = q; a.ldq = ldq; a.out = out; a.ldo = ldo; a.pages = (const unsigned char*)pages;
    a.block_table = block_table; a.max_blocks = max_blocks; a.cu_rows = cu_rows; a.seg_pos = seg_pos;
    a.scale = scale; a.window = window; a.ps = ps; a.ps_log2 = kv4_log2(ps); a.H = H; a.G = G;
    a.part_o = part_o; a.part_ml = part_ml; a.scores = mass ? scores : nullptr; a.ld_scores = ld_scores;
    a.lse_split = mass ? lse_split : nullptr; a.lse = mass ? lse : nullptr; a.mass = mass;
    a.n_chunks = n_chunks; a.chunk = chunk; a.fused = fused; a.max_rows = short_rows; a.min_rows = short_rows + 1; a.n_seg = n_seg;
    if (dtype == KP_DTYPE_BF16) {
        KV4_DISPATCH_HD(hd, HD, return (kv4_run<HD, 1, bf16>(a, n_pages, n_rows, long_rows, max_context, (cudaStream_t)stream)));
    } else if (dtype == KP_DTYPE_F32) {
        KV4_DISPATCH_HD(hd, HD, return (kv4_run<HD, 2, float>(a, n_pages, n_rows, long_rows, max_context, (cudaStream_t)stream)));
    }
    return KP_ERR_BAD_ARG;
}

}  // extern "C"
