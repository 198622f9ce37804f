// Attention of many rows (portions of prompts) over the 4-bit cache on the 5th-generation tensor cores: bfloat16 rows, heads
// of 64 or 128 values.  Formulas and bytes as in kv4.cuh.
//
// Columns.  The rows of a segment and the R query heads that share a kv head are one list of columns, c = row R + head: a tile of
// 128 columns reads the same keys once for all of them.  A CTA takes 256 columns of a kv head, two groups of 128, and walks
// their keys in tiles of 128:
//   4 warps turn the codes of a tile into fp16 operands in shared memory, a thread a key;
//   1 warp issues  S = Q K^T  and  O += P V  (tcgen05.mma, kind::f16; S and O in tensor memory);
//   2 x 4 warps have a thread a column: S from tensor memory (once for the maximum; half of it stays in registers, the other half is read
//   again), softmax, P (fp16) back to tensor memory, where it is the A operand of the second product.
// The groups run half a tile apart, so that the tensor core works for one while the other is at its exponentials.  P through shared
// memory made that memory's bandwidth the bound (a product with both operands there reads 128 bytes a cycle, all there is).  With heads
// of 128 tensor memory has no room for P beside S and O: it takes the half of S that has been read.
//
// Exactness.  K's operand is s (c - 8): an 8-bit times a 4-bit number, exact in fp16's 11 bits.  The rest, (z + 8 s) times the
// query's sum over the group, is 16 more columns of the same product: both factors in two fp16 parts.  So S is off by float32
// rounding only, and the weights added up as mass are those of the definition to 1e-6.  V's operand s (c - 8) + (z + 8 s) is
// rounded to fp16 once (by up to 2^-11 of it; the output's own rounding to bfloat16 is up to 2^-8), and so is P; further products
// for what fp16 leaves of them would be lost in the output's rounding.
// Ranges.  Queries are scaled by a power of two a column, K by one a tile of keys, V by one that only grows from tile to tile
// (O is rescaled when it does).  fp16 then holds a query's values down to 2^-24 of its largest, K's codes of groups whose scale is above 2^-24
// of the tile's largest key, 11 bits of values down to 2^-28 of the largest so far; what is smaller loses bits, also in columns that do not read the key that
// is so large.  P is taken against a reference that follows the row's maximum
// in steps of at least 2^8 (O is rescaled in tensor memory only then), P <= 2^15.
// Every mbarrier wait is bounded; one that gives up sets the status word, and the CTA frees its tensor memory and returns.
//
// Measured.  A tile (256 columns, 128 keys) takes 1.9 us with heads of 64, whose exponentials alone are 1.04 us of the SM's, and 2.4 us with heads of
// 128, whose products are 1.1: what bounds it is the chain of S, softmax, P and second product, which two groups cannot hide.  A CTA's start
// and end take 8 us and 12.  1,024 rows of 32 heads over 8 of 128 values behind 15,360 keys: 326 us on the device, 0.81 PFLOP/s.
#include "kv4.cuh"
#include "tcgen05.cuh"

KP_STATUS_WORD(g_kv4_tc_status, kv4_tc)               // 0 ok; 1: a bounded wait gave up

#define KT_ROWS 128                                    // columns a group, and keys a tile
#define KT_MOST 16                                     // most CTAs that share a tile's keys
#define KT_EXT 4096                                    // 128 rows of 16 fp16 beside a tile: the parts of the second term

struct Kv4TcArgs {
    const bf16* q; long long ldq;
    bf16* out; long long ldo;
    const unsigned char* pages;
    const int* block_table; int max_blocks;
    const int* cu_rows; const int* seg_pos;
    float scale; int window; int ps, ps_log2; int H, G;
    unsigned char* q_image; float2* col;               // with mass: the groups' Q operands and (factor, lse) of their columns
    float* mass;
    int split;                                         // CTAs that share the keys of a tile of columns
    int cluster;                                       // CTAs that share the columns of a tile of keys
    int min_rows, n_seg, n_tiles;                      // n_tiles: an upper bound of the CTAs' tiles
};

template <int HD>
struct Kt {
    static constexpr int NG = HD / 64, TILE = NG * 16384, OPER = TILE + KT_EXT, ST = 2;
    static constexpr bool ALIAS = HD == 128;           // P lies in S's columns 64..127, not in columns of its own
    static constexpr int S_COL = 0, O_COL = 256, P_COL = ALIAS ? 64 : 256 + 2 * HD, P_STEP = ALIAS ? 128 : 64;   // columns of tensor memory (of group 0)
    static constexpr size_t SMEM = 1024 + 2 * OPER + ST * OPER + ST * TILE + 512;
    static constexpr int THREADS = 416;
    // the pass that adds up the mass: one K tile, a ring of Q images; two CTAs an SM
    static constexpr int QST = HD == 64 ? 3 : 2, IMAGE = OPER + 1024;            // an image in shared memory, and (factor, lse) of its columns
    static constexpr int MASS_THREADS = 288;
    static constexpr size_t MASS_SMEM = 1024 + OPER + QST * IMAGE + 512;
};

// tcgen05 instruction descriptor with fp16 operands (the helper's are bfloat16)
__host__ __device__ constexpr uint32_t kt_idesc(int M, int N, bool b_mn) { return kp_umma_idesc(M, N, b_mn) & ~((1u << 7) | (1u << 10)); }
// K-major operand of 16 columns: rows of 32 bytes with the 32-byte swizzle, 8-row groups 256 bytes apart
__device__ __forceinline__ uint64_t kt_desc_ext(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(256 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)6 << 61;
    return d;
}
__device__ __forceinline__ int kt_ext_at(int row, int chunk) { return row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4); }
__device__ __forceinline__ int kt_at(int row, int chunk) { return (chunk >> 3) * 16384 + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }

__device__ __forceinline__ float kt_pow2(int e) { return __uint_as_float((uint32_t)(max(-126, min(127, e)) + 127) << 23); }

// eight codes as fp16 pairs (0, 4), (1, 5), (2, 6), (3, 7), times s (s16: s / 16), plus z
__device__ __forceinline__ uint4 kt_codes(uint32_t w, __half2 s, __half2 s16, __half2 z, bool add) {
    uint32_t x[4] = {w & 0x000f000fu, w & 0x00f000f0u, (w >> 8) & 0x000f000fu, (w >> 8) & 0x00f000f0u};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t y = x[i] | 0x64006400u, c = (i & 1) ? 0x64806480u : 0x64086408u;
        const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&y), *reinterpret_cast<const __half2*>(&c));
        const __half2 v = add ? __hfma2(d, (i & 1) ? s16 : s, z) : __hmul2(d, (i & 1) ? s16 : s);
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
// the power of two above a group's largest magnitude (nothing for one that is not finite)
__device__ __forceinline__ int kt_exponent(uint32_t range) {
    const float s = kv4_scale(range), z = kv4_least(range), top = fmaxf(fabsf(z), fabsf(fmaf(15.0f, s, z)));
    return top < INFINITY ? (int)(__float_as_uint(top) >> 23) - 126 : -126;
}
// What a thread of the code warps has of its key, or of its value: codes and ranges
template <int HD>
struct KtRow {
    uint4 c[HD / 32];
    uint32_t r[HD / 64];
    __device__ __forceinline__ void load(const unsigned char* rec, int off, int ps, bool there, bool value) {
        constexpr int NG = HD / 64;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) c[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int y = 0; y < NG; y++) r[y] = 0u;
        if (!there) return;                            // a key that is not there: zeros, whatever lies in its place
        const int row = value ? ps + off : off;
        const uint4* from = reinterpret_cast<const uint4*>(rec + (size_t)row * (HD / 2));
        const uint32_t* ranges = reinterpret_cast<const uint32_t*>(rec + (size_t)ps * HD) + row * NG;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) c[i] = from[i];
#pragma unroll
        for (int y = 0; y < NG; y++) r[y] = ranges[y];
    }
};
// One row of an operand of the score product: K's codes of a key
template <int HD>
__device__ __forceinline__ void kt_write_key(unsigned char* tile, int row, const KtRow<HD>& x, int e) {
    const uint4 (&codes)[HD / 32] = x.c;
    const uint32_t (&ranges)[HD / 64] = x.r;
    const float f = kt_pow2(7 - e);
    uint32_t ext[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int y = 0; y < HD / 64; y++) {
        const float s = kv4_scale(ranges[y]) * f, z = fmaf(8.0f, kv4_scale(ranges[y]), kv4_least(ranges[y])) * f;
        const __half2 s2 = __float2half2_rn(s), s16 = __float2half2_rn(s * 0.0625f);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 c = codes[2 * y + i];
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                *reinterpret_cast<uint4*>(tile + kt_at(row, y * 8 + i * 4 + j)) = kt_codes(w[j], s2, s16, s2, false);
        }
        const __half zh = __float2half_rn(z), zl = __float2half_rn(z - __half2float(zh));
        const __half2 h2 = __halves2half2(zh, zh), l2 = __halves2half2(zl, zl);
        ext[2 * y] = *reinterpret_cast<const uint32_t*>(&h2);
        ext[2 * y + 1] = *reinterpret_cast<const uint32_t*>(&l2);
    }
    *reinterpret_cast<uint4*>(tile + Kt<HD>::TILE + kt_ext_at(row, 0)) = make_uint4(ext[0], ext[1], ext[2], ext[3]);
    *reinterpret_cast<uint4*>(tile + Kt<HD>::TILE + kt_ext_at(row, 1)) = make_uint4(0u, 0u, 0u, 0u);
}
// and the queries of a warp's 32 columns, HD / 8 lanes a query (from memory whole lines at a time: a lane with a query of its own would ask for
// 32 lines an instruction).  `at`: where this lane's own query lies, in elements of q; -1: none, zeros.  Returns the factor that makes its
// scores (base 2) of the product with a tile scaled by 2^(7 - e): factor 2^(e - 7).
template <int HD>
__device__ __forceinline__ float kt_write_queries(unsigned char* tile, int row0, const bf16* q, long long at, float scale, int lane) {
    constexpr int LANES = HD / 8, STEP = 32 / LANES;
    const int chunk = lane % LANES, sub = lane / LANES;
    int mine = 0;
#pragma unroll 1
    for (int base = 0; base < 32; base += 8 * STEP) {
        uint4 raw[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long long from = __shfl_sync(0xffffffffu, at, base + i * STEP + sub);
            raw[i] = from >= 0 ? *reinterpret_cast<const uint4*>(q + from + 8 * chunk) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float x[8], top = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) { x[2 * j] = kv4_scale(w[j]); x[2 * j + 1] = kv4_least(w[j]); }
#pragma unroll
            for (int j = 0; j < 8; j += 2) top = kv4_max3(top, fabsf(x[j]), fabsf(x[j + 1]));
#pragma unroll
            for (int d = 1; d < LANES; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            // the largest value to [2^6, 2^7): a sum of 64 then fits fp16
            const int e = top > 0.f && top < INFINITY ? min(133 - (int)(__float_as_uint(top) >> 23), 100) : 0;
            const float up = kt_pow2(e);
            const int theirs = __shfl_sync(0xffffffffu, e, lane % STEP * LANES);
            if (lane / STEP == base / STEP + i) mine = theirs;
            float sum = 0.f;
            uint32_t r[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                r[j] = pack_f16(x[j] * up, x[j + 4] * up);
                const __half2 h = *reinterpret_cast<const __half2*>(&r[j]);
                sum += __low2float(h) + __high2float(h);
            }
            const int row = row0 + base + i * STEP + sub;
            *reinterpret_cast<uint4*>(tile + kt_at(row, chunk)) = make_uint4(r[0], r[1], r[2], r[3]);
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);               // of the 64 values of a group
            const __half sh = __float2half_rn(sum), sl = __float2half_rn(sum - __half2float(sh));
            const __half2 both = __halves2half2(sh, sl);
            const uint32_t first = *reinterpret_cast<const uint32_t*>(&both), second = HD == 64 ? 0u : __shfl_xor_sync(0xffffffffu, first, 8);
            if (chunk < 2)
                *reinterpret_cast<uint4*>(tile + Kt<HD>::TILE + kt_ext_at(row, chunk)) =
                    chunk == 0 ? make_uint4(first, first, second, second) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    return scale * KV4_LOG2E * kt_pow2(-mine);
}
// S of 128 x 128.  A warp in step issues it, by an elected lane: from inside a branch that one lane took, the operands would pass through general
// registers, at three times the cycles an MMA.
template <int HD>
__device__ __forceinline__ void kt_issue_s(uint32_t tmem, const unsigned char* a, const unsigned char* b) {
    constexpr uint32_t idesc = kt_idesc(128, 128, false);
#pragma unroll
    for (int y = 0; y < HD / 64; y++)
        kp_umma_bf16_box(tmem, kp_umma_desc(kp_smem_u32(a + y * 16384)), kp_umma_desc(kp_smem_u32(b + y * 16384)), idesc, y > 0);
    kp_umma_bf16_warp(tmem, kt_desc_ext(kp_smem_u32(a + Kt<HD>::TILE)), kt_desc_ext(kp_smem_u32(b + Kt<HD>::TILE)), idesc, 1u);
}
// D += A B with A in tensor memory (a lane a row, a column two consecutive elements), by an elected lane of a warp in step
__device__ __forceinline__ void kt_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
// a wait of a warp in step, which gives up as one
__device__ __forceinline__ bool kt_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, kp_mbar_wait_bounded(bar, parity)); }

// bits lo .. hi of 32 (lo may lie below, hi above them)
__device__ __forceinline__ uint32_t kt_bits(int lo, int hi) {
    const uint32_t upto = hi >= 31 ? 0xffffffffu : (hi < 0 ? 0u : (2u << hi) - 1u), from = lo <= 0 ? 0xffffffffu : (lo > 31 ? 0u : 0xffffffffu << lo);
    return upto & from;
}
// two float32 operations at once
__device__ __forceinline__ float2 kt_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 kt_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
// segment, its first row, number of rows and position, and first column, of a tile of 256 columns (kv4.cu's tiles: the last columns of a segment
// first); seg = -1: none
struct KtTile { int seg, row0, n_rows, pos0, col0; };
__device__ __forceinline__ KtTile kt_find(const Kv4TcArgs& p, int tile, int R, int lane) {
    int before = 0;
    for (int base = 0; base < p.n_seg; base += 32) {
        const int i = base + lane;
        int row0 = 0, rows = 0, pos = 0;
        if (i < p.n_seg) { row0 = p.cu_rows[i]; rows = p.cu_rows[i + 1] - row0; pos = p.seg_pos[i]; }
        const int mine = rows >= p.min_rows ? (rows * R + 255) / 256 : 0;
        int run = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
        const unsigned hit = __ballot_sync(0xffffffffu, tile < before + run);
        if (hit) {
            const int src = __ffs(hit) - 1, end = before + __shfl_sync(0xffffffffu, run, src);
            return {base + src, __shfl_sync(0xffffffffu, row0, src), __shfl_sync(0xffffffffu, rows, src), __shfl_sync(0xffffffffu, pos, src),
                    (end - 1 - tile) * 256};
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    }
    return {-1, 0, 0, 0, 0};
}
// the tile of segment `seg`'s first 256 columns (its tiles run downwards from there)
__device__ __forceinline__ int kt_first_tile(const Kv4TcArgs& p, int seg, int R, int lane) {
    int sum = 0;
    for (int i = lane; i <= seg; i += 32) {
        const int rows = p.cu_rows[i + 1] - p.cu_rows[i];
        sum += rows >= p.min_rows ? (rows * R + 255) / 256 : 0;
    }
    return __reduce_add_sync(0xffffffffu, sum) - 1;
}

// The rows of a tile from the shares of the cluster's CTAs, by 256 threads, and with mass what the pass over it needs of them.  (A call: inlined, it
// costs the loop over the keys registers.)
template <int HD>
__device__ __noinline__ void kt_join_shares(const Kv4TcArgs& p, unsigned char* sm, int rank, int kvh, int tile, int row0, int cta_col0, int n_here) {
    const int R = p.H / p.G;
    float* part = reinterpret_cast<float*>(sm);
    const float* factor = part + kv4_share_floats(256, HD, KT_MOST);
    kv4_join_shares<bf16, HD, 256, 256, true, KT_MOST>(
        part, p.split, rank, n_here,
        [&](int col) { return p.out + (size_t)(row0 + (cta_col0 + col) / R) * p.ldo + (size_t)(kvh * R + (cta_col0 + col) % R) * HD; },
        [&](int col, float top, float sum) {
            if (p.mass) p.col[((size_t)kvh * p.n_tiles + tile) * 256 + col] = make_float2(factor[col], sum == 0.f ? INFINITY : top - 7.0f + log2f(sum));
        });
}

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(Kt<HD>::THREADS, 1)
kv4_tc_kernel(const __grid_constant__ Kv4TcArgs p) {
    using S = Kt<HD>;
    constexpr int ST = S::ST;
    extern __shared__ unsigned char smem_dyn[];
    // (these at fixed addresses: a pointer to them costs the loop over the keys a register, and 10 % of its time)
    __shared__ volatile unsigned unsound[4 * S::NG * 4];      // [4 tiles][group][4]: a bit a key, whose value's group is not finite
    __shared__ volatile unsigned char struck[256];     // groups in which a column reads such a value
    unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    unsigned char* Qs = sm;                            // [2] OPER
    unsigned char* Ks = Qs + 2 * S::OPER;              // [ST] OPER
    unsigned char* Vs = Ks + ST * S::OPER;             // [ST] TILE
    uint64_t* bars = reinterpret_cast<uint64_t*>(Vs + ST * S::TILE);
    uint64_t* q_full = bars;                           // [2] each, by group or by stage
    uint64_t* k_full = bars + 2; uint64_t* k_empty = bars + 4;
    uint64_t* v_full = bars + 6; uint64_t* v_empty = bars + 8;
    uint64_t* s_full = bars + 10; uint64_t* s_free = bars + 12;
    uint64_t* p_full = bars + 14; uint64_t* o_done = bars + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* meta = abort_flag + 1;               // [K's scale, V's][4 tiles]: exponents; V's twice, plus 1 where a value is not finite
    volatile int* tops = meta + 8;                     // [2][4 warps]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    kp_pdl_begin();
    // (the longest tiles first, of all heads)
    const int n_split = SPLIT ? p.split : 1, rank = blockIdx.x % n_split, place = blockIdx.x / n_split;
    const int R = p.H / p.G, kvh = place % p.G, tile = place / p.G;
    const KtTile t = kt_find(p, tile, R, lane);
    if (t.seg < 0) return;                             // (the grid is an upper bound)
    const int seg = t.seg, cta_col0 = t.col0, row0 = t.row0, n_cols = t.n_rows * R, pos0 = t.pos0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            kp_mbar_init(&q_full[i], 128);
            kp_mbar_init(&k_full[i], 128); kp_mbar_init(&k_empty[i], 1);
            kp_mbar_init(&v_full[i], 128); kp_mbar_init(&v_empty[i], 1);
            kp_mbar_init(&s_full[i], 1); kp_mbar_init(&s_free[i], 128);
            kp_mbar_init(&p_full[i], 128); kp_mbar_init(&o_done[i], 1);
        }
        *abort_flag = 0;
        kp_mbar_init_fence();
    }
    if (warp == 12) kp_tmem_alloc(tmem_slot, 512);
    kp_tc_fence_before();
    __syncthreads();
    kp_tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;             // S of the groups: 2 x 128 columns; then O: 2 x HD

    const int n_here = min(256, n_cols - cta_col0);    // columns of this CTA
    const int k_hi = min(pos0 + (cta_col0 + n_here - 1) / R, p.max_blocks * p.ps - 1);
    const int k_lo = p.window > 0 ? max(0, pos0 + cta_col0 / R - p.window + 1) : 0;
    // tiles of keys, and this CTA's of them
    const int kt_all = k_hi >= k_lo ? k_hi / KT_ROWS - k_lo / KT_ROWS + 1 : 0;
    const int kt_skip = kt_all * rank / n_split, kt_lo = k_lo / KT_ROWS + kt_skip, n_kt = kt_all * (rank + 1) / n_split - kt_skip;

    if (warp >= 8 && warp < 12) {
        // ---- codes to operands: thread d has key d of every tile.  Keys run a tile ahead of the values: K's stage is free once both groups'
        // scores are there, V's half a tile later.
        const int d = threadIdx.x - 256;
        const int* bt = p.block_table + (size_t)seg * p.max_blocks;
        const size_t rec = (size_t)kv4_page_bytes(p.ps, HD);
        auto page_of = [&](int i) {
            const int key = (kt_lo + i) * KT_ROWS + d;
            return i < n_kt && key >= k_lo && key <= k_hi ? bt[key >> p.ps_log2] : -1;
        };
        auto fetch = [&](KtRow<HD>& x, int i, int page, bool value) {
            const int key = (kt_lo + i) * KT_ROWS + d;
            x.load(p.pages + ((size_t)max(page, 0) * p.G + kvh) * rec, key & (p.ps - 1), p.ps, page >= 0, value);
        };
        // the largest exponent of the tile's groups, of all 128 threads
        int turn = 0;
        auto exponent = [&](const KtRow<HD>& x, int e) {
#pragma unroll
            for (int y = 0; y < S::NG; y++) e = max(e, kt_exponent(x.r[y]));
            e = __reduce_max_sync(0xffffffffu, e);
            volatile int* t = tops + turn * 4;
            turn ^= 1;
            if (lane == 0) t[warp & 3] = e;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            return max(max(t[0], t[1]), max(t[2], t[3]));
        };
        bool ok = true;
        KtRow<HD> key, value;
        int key_page = page_of(1), value_page = page_of(1), ev = -100;
        fetch(key, 0, page_of(0), false);
        fetch(value, 0, page_of(0), true);
        auto do_key = [&](int i) {
            const int st = i % ST, use = i / ST, e = exponent(key, -100);
            if (ok && (*abort_flag || !kp_mbar_wait_bounded(&k_empty[st], (use & 1) ^ 1))) ok = false;
            if (d == 0) meta[i & 3] = e;
            kt_write_key<HD>(Ks + st * S::OPER, d, key, e);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            kp_mbar_arrive(&k_full[st]);
            fetch(key, i + 1, key_page, false);
            key_page = page_of(i + 2);
        };
        auto do_value = [&](int i) {
            const int st = i % ST, use = i / ST;
            // a group that is not finite is zeros in the product, and the columns that read its key are told
#pragma unroll
            for (int y = 0; y < S::NG; y++) {
                const bool fine = kv4_finite(value.r[y]);
                const unsigned bits = __ballot_sync(0xffffffffu, !fine);
                if (lane == 0) unsound[((i & 3) * S::NG + y) * 4 + (warp & 3)] = bits;
                if (!fine) value.r[y] = 0u;
            }
            ev = exponent(value, ev);
            if (ok && (*abort_flag || !kp_mbar_wait_bounded(&v_empty[st], (use & 1) ^ 1))) ok = false;
            if (d == 0) {
                unsigned any = 0u;
#pragma unroll
                for (int e = 0; e < 4 * S::NG; e++) any |= unsound[(i & 3) * 4 * S::NG + e];
                meta[4 + (i & 3)] = ev * 2 + (any ? 1 : 0);
            }
            const float f = kt_pow2(14 - ev);
#pragma unroll
            for (int y = 0; y < S::NG; y++) {
                const float s = kv4_scale(value.r[y]) * f, z = fmaf(8.0f, kv4_scale(value.r[y]), kv4_least(value.r[y])) * f;
                const __half2 s2 = __float2half2_rn(s), s16 = __float2half2_rn(s * 0.0625f), z2 = __float2half2_rn(z);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint4 c = value.c[2 * y + j];
                    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        *reinterpret_cast<uint4*>(Vs + st * S::TILE + kt_at(d, y * 8 + j * 4 + e)) = kt_codes(w[e], s2, s16, z2, true);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            kp_mbar_arrive(&v_full[st]);
            fetch(value, i + 1, value_page, true);
            value_page = page_of(i + 2);
        };
        // keys 0, keys 1, values 0, keys 2, values 1, ...: in the order in which the products free their stages
#pragma unroll 1
        for (int i = -2; i < n_kt; i++) {
            if (i + 2 < n_kt) do_key(i + 2);
            if (i + 1 >= 0 && i + 1 < n_kt) do_value(i + 1);
        }
        if (__builtin_expect(!ok, 0)) { *abort_flag = 1; atomicExch(&g_kv4_tc_status, 1); }
    } else if (warp == 12) {
        // ---- the tensor core's work
        if (n_kt > 0) {
            constexpr uint32_t idesc_pv = kt_idesc(128, HD, true);
            auto issue_s = [&](int i, int g) {
                if (!kt_wait(&k_full[i % ST], (i / ST) & 1) || (!S::ALIAS && i > 0 && !kt_wait(&s_free[g], (i - 1) & 1))) return false;
                kp_tc_fence_after();
                kt_issue_s<HD>(tmem_base + S::S_COL + 128 * g, Qs + g * S::OPER, Ks + (i % ST) * S::OPER);
                kp_umma_commit_warp(&s_full[g]);
                if (g == 1) kp_umma_commit_warp(&k_empty[i % ST]);
                return true;
            };
            auto issue_pv = [&](int i, int g) {
                if (!kt_wait(&v_full[i % ST], (i / ST) & 1) || !kt_wait(&p_full[g], i & 1)) return false;
                kp_tc_fence_after();
                const uint32_t va = kp_smem_u32(Vs + (i % ST) * S::TILE);
#pragma unroll
                for (int kk = 0; kk < KT_ROWS / 16; kk++)
                    kt_umma_ts(tmem_base + S::O_COL + HD * g, tmem_base + S::P_COL + S::P_STEP * g + 8 * kk,
                               HD == 64 ? kp_umma_desc(va + kk * 2048) : kp_umma_desc_mn(va + kk * 2048, 16384), idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
                kp_umma_commit_warp(&o_done[g]);
                if (g == 1) kp_umma_commit_warp(&v_empty[i % ST]);
                return true;
            };
            bool ok = kt_wait(&q_full[0], 0) && issue_s(0, 0) && kt_wait(&q_full[1], 0) && issue_s(0, 1);
            // (a group's products run in the order in which they are issued: where P lies in S, the next S comes behind the product that reads it)
            for (int i = 0; i < n_kt && ok; i++)
                for (int g = 0; g < 2 && ok; g++) {
                    const bool more = i + 1 < n_kt;
                    ok = S::ALIAS ? issue_pv(i, g) && (!more || issue_s(i + 1, g)) : (!more || issue_s(i + 1, g)) && issue_pv(i, g);
                }
            if (!ok && lane == 0) { *abort_flag = 1; atomicExch(&g_kv4_tc_status, 1); }
        }
    } else {
        // ---- the columns: warps 0-3 group 0, warps 4-7 group 1; thread r of a group has column r
        const int g = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane;
        const int c = cta_col0 + g * 128 + r;
        const int pos = min(pos0 + min(c, n_cols - 1) / R, k_hi);                // (a column that is not there reads what the last one does)
        // where column c's row lies in q or in out; -1: nowhere
        auto place_of = [&](int c, long long ld) { return c < n_cols ? (long long)(row0 + c / R) * ld + (kvh * R + c % R) * HD : -1LL; };
        unsigned char* Qg = Qs + g * S::OPER;
        struck[threadIdx.x] = 0;
        const float f = kt_write_queries<HD>(Qg, q4 * 32, p.q, place_of(c, p.ldq), p.scale, lane);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        kp_mbar_arrive(&q_full[g]);
        if (p.mass && rank == 0 && r == 0) {
            const size_t tile_id = ((size_t)kvh * p.n_tiles + tile) * 2 + g;
            // the pass that adds up the mass takes the same operand, as it lies
            kp_mbar_wait_bounded(&q_full[g], 0);       // (nothing that arrives there waits)
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n cp.async.bulk.commit_group;"
                         ::"l"(p.q_image + tile_id * S::OPER), "r"(kp_smem_u32(Qg)), "r"((uint32_t)S::OPER) : "memory");
        }
        const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        // keys that every column of the group reads
        const int g_first = min(cta_col0 + g * 128, n_cols - 1), g_last = min(cta_col0 + g * 128 + 127, n_cols - 1);
        const int all_hi = min(pos0 + g_first / R, k_hi);
        const int all_lo = p.window > 0 ? max(0, pos0 + g_last / R - p.window + 1) : 0;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t tmem_s = tmem_base + S::S_COL + 128 * g + lane_off, tmem_o = tmem_base + S::O_COL + HD * g + lane_off;
        const uint32_t tmem_p = tmem_base + S::P_COL + S::P_STEP * g + lane_off;
        bool ok = true;
        float m = -INFINITY, l = 0.f;
        int ev = -100;
#pragma unroll 1
        for (int i = 0; i < n_kt; i++) {
            if (ok && (*abort_flag || !kp_mbar_wait_bounded(&s_full[g], i & 1))) ok = false;
            kp_tc_fence_after();
            const int key0 = (kt_lo + i) * KT_ROWS;
            const bool masked = !(key0 + KT_ROWS - 1 <= all_hi && key0 >= all_lo);
            const float fk = fmaxf(f * kt_pow2(meta[i & 3] - 7), 1.17549435e-38f);     // (not 0: a masked score stays -inf)
            uint32_t s[2][32], w[32];
            auto load = [&](int at) {                                            // 64 scores; one that is not there: the lowest value
                kp_tmem_ld32_issue(tmem_s + at, s[0]);
                kp_tmem_ld32_issue(tmem_s + at + 32, s[1]);
                kp_tmem_ld_wait();
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const uint32_t there = kt_bits(lo - key0 - at - e * 32, pos - key0 - at - e * 32);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!(there & (1u << j))) s[e][j] = 0xff800000u;
                    }
                }
            };
            auto largest = [&] {
                float t[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    t[e] = fmaxf(__uint_as_float(s[e][0]), __uint_as_float(s[e][1]));
#pragma unroll
                    for (int j = 2; j < 32; j += 2) t[e] = kv4_max3(t[e], __uint_as_float(s[e][j]), __uint_as_float(s[e][j + 1]));
                }
                return fmaxf(t[0], t[1]);
            };
            load(0);
            float top = largest();
            load(64);
            top = fmaxf(top, largest()) * fk;
            const float m_new = top > m + 8.0f ? top : m;                        // (the first: m = -inf)
            const float corr_l = m_new == m ? 1.0f : kv4_exp2(m - m_new);
            const float sub = m_new == -INFINITY ? 0.f : m_new - 7.0f;
            const float2 fk2 = make_float2(fk, fk), sub2 = make_float2(-sub, -sub);
            float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            auto weights = [&] {                                                 // of the 64 loaded scores, packed
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float2 x = kt_fma2(make_float2(__uint_as_float(s[e][j]), __uint_as_float(s[e][j + 1])), fk2, sub2);
                        x.x = kv4_exp2(x.x);
                        x.y = kv4_exp2(x.y);
                        sums[e] = kt_add2(sums[e], x);
                        w[e * 16 + (j >> 1)] = pack_f16(x.x, x.y);
                    }
            };
            weights();
            // the product of the tile before has read P and added to O (known from S where P lies in it); this tile's values are there
            if (!S::ALIAS && i > 0 && ok && !kp_mbar_wait_bounded(&o_done[g], (i - 1) & 1)) ok = false;
            if (ok && !kp_mbar_wait_bounded(&v_full[i % ST], (i / ST) & 1)) ok = false;
            const int of_v = meta[4 + (i & 3)], ev_now = of_v >> 1;
            if (__builtin_expect(of_v & 1, 0)) {
#pragma unroll 1
                for (int e = 0; e < 4 * S::NG; e++)
                    if (unsound[(i & 3) * 4 * S::NG + e] & kt_bits(lo - key0 - (e & 3) * 32, pos - key0 - (e & 3) * 32)) struck[threadIdx.x] |= 1 << (e >> 2);
            }
            const float corr_o = corr_l * kt_pow2(ev - ev_now);
            if (i > 0 && __any_sync(0xffffffffu, corr_o != 1.0f)) {
                kp_tc_fence_after();
#pragma unroll 1
                for (int e = 0; e < HD; e += 32) {
                    uint32_t v[32];
                    kp_tmem_ld32(tmem_o + e, v);
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr_o);
                    kp_tmem_st32(tmem_o + e, v);
                }
            }
            kp_tmem_st32(tmem_p + 32, w);
            load(0);
            if (!S::ALIAS) {
                kp_tc_fence_before();
                kp_mbar_arrive(&s_free[g]);                                      // the next tile's S may be computed
            }
            weights();
            kp_tmem_st32(tmem_p, w);
            kp_tmem_st_wait();
            kp_tc_fence_before();
            kp_mbar_arrive(&p_full[g]);                                          // P, and O where it was rescaled, are written
            const float2 total = kt_add2(sums[0], sums[1]);
            l = l * corr_l + (total.x + total.y);
            m = m_new;
            ev = ev_now;
        }
        if (n_kt > 0 && ok && !kp_mbar_wait_bounded(&o_done[g], (n_kt - 1) & 1)) ok = false;
        kp_tc_fence_after();
        const bool none = m == -INFINITY && l == 0.f;                            // (not: scores that are NaN)
        const float inv = none ? 0.f : kt_pow2(ev - 14) / l;
        if (p.mass && r == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (SPLIT) {
            // this CTA's share of the rows, and what it counts for: in place of the operands, once neither group's products read them
            asm volatile("bar.sync 4, 256;" ::: "memory");
            const int col = g * 128 + r;
            float* part = reinterpret_cast<float*>(sm);
#pragma unroll 1
            for (int e = 0; e < HD; e += 32) {
                uint32_t v[32];
                if (n_kt > 0) kp_tmem_ld32(tmem_o + e, v);
                const float by = struck[threadIdx.x] >> (e / 64) & 1 ? __int_as_float(0x7fffffff) : inv;
#pragma unroll
                for (int d = 0; d < 32; d += 4) {
                    // places 0..7 hold dimensions 0, 4, 1, 5, 2, 6, 3, 7
                    float x[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = none ? 0.f : __uint_as_float(v[(d & ~7) + 2 * j + (d >> 2 & 1)]) * by;
                    *reinterpret_cast<float4*>(part + kv4_share_at(col, e + d, HD)) = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
            kv4_share_sums(part, 256, HD, col, m, l);
            part[kv4_share_floats(256, HD, KT_MOST) + col] = f;
        } else {
            if (p.mass) {
                p.col[((size_t)kvh * p.n_tiles + tile) * 256 + g * 128 + r] = make_float2(f, none ? INFINITY : m - 7.0f + log2f(l));
                asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory");
            }
            // the rows pass through the operand's place, which nothing reads any more, so that memory gets whole lines
#pragma unroll 1
            for (int e = 0; e < HD; e += 32) {
                uint32_t v[32];
                if (n_kt > 0) kp_tmem_ld32(tmem_o + e, v);
                const float by = struck[threadIdx.x] >> (e / 64) & 1 ? __int_as_float(0x7fffffff) : inv;
#pragma unroll
                for (int d = 0; d < 32; d += 8) {
                    // places 0..7 hold dimensions 0, 4, 1, 5, 2, 6, 3, 7
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) x[(j >> 1) + (j & 1) * 4] = none ? 0.f : __uint_as_float(v[d + j]) * by;
                    *reinterpret_cast<uint4*>(Qg + kt_at(r, (e + d) / 8)) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
                }
            }
            __syncwarp();
            constexpr int LANES = HD / 8, STEP = 32 / LANES;
            const long long to = ok ? place_of(c, p.ldo) : -1LL;
#pragma unroll
            for (int i = 0; i < 32; i += STEP) {
                const int of = i + lane / LANES;
                const long long at = __shfl_sync(0xffffffffu, to, of);
                if (at >= 0) *reinterpret_cast<uint4*>(p.out + at + 8 * (lane % LANES)) = *reinterpret_cast<const uint4*>(Qg + kt_at(q4 * 32 + of, lane % LANES));
            }
        }
        kp_tc_fence_before();
        if (__builtin_expect(!ok, 0)) { if (lane == 0) atomicExch(&g_kv4_tc_status, 1); }
    }
    kp_tc_fence_before();
    __syncthreads();
    if (warp == 12) kp_tmem_dealloc(tmem_base, 512);
    if (!SPLIT) return;

    kv4_cluster_sync();
    if (warp < 8) kt_join_shares<HD>(p, sm, rank, kvh, tile, row0, cta_col0, n_here);
    kv4_cluster_sync();                                 // (nobody leaves while its shares are read)
}

// The sum of 2^(score - lse) over the 128 columns of a tile, of those from lo to hi (MASKED), for this thread's key: S of tensor memory
// times kappa and the column's factor is the score.
template <bool MASKED>
__device__ __forceinline__ float kt_column_sum(uint32_t tmem_s, const float4* col, float kappa, int lo, int hi) {
    float part = 0.f;
    const float2 k2 = make_float2(kappa, kappa);
#pragma unroll 1
    for (int e = 0; e < 128; e += 32) {
        uint32_t s[32];
        kp_tmem_ld32(tmem_s + e, s);
        const uint32_t there = kt_bits(lo - e, hi - e);
        float2 a[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            const float4 f = col[(e + j) >> 1];            // (factor, lse) of two columns
            float2 x = kt_fma2(make_float2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), k2, make_float2(0.f, 0.f));
            x = make_float2(kv4_exp2(fmaf(x.x, f.x, -f.y)), kv4_exp2(fmaf(x.y, f.z, -f.w)));
            if (MASKED) {
                if (!(there & (1u << j))) x.x = 0.f;
                if (!(there & (2u << j))) x.y = 0.f;
            }
            a[(j >> 1) & 1] = kt_add2(a[(j >> 1) & 1], x);
        }
        const float2 t = kt_add2(a[0], a[1]);
        part += t.x + t.y;
    }
    return part;
}

// ---- mass.  A cluster of CTAs per (128 keys, kv head, segment): S^T = K Q^T with a thread a key, so that a key's weights add up in its
// thread.  The operands of Q and the columns' (factor, lse) are those that the kernel above left, brought by bulk copies into a ring; the two groups
// of 128 threads take the tiles of 128 columns in turn.  The CTAs of a cluster share the columns out (the first keys of a prompt are
// read by all of it), and their sums are added in order.  2,048 rows of 32 heads over 8 of 64: 38 us, of which the exponentials are 16.  (Two tiles of
// keys a CTA for each image, to halve their way from L2: slower by 4 to 5 us there, with one CTA's start for twice the keys.)
template <int HD>
__global__ void __launch_bounds__(Kt<HD>::MASS_THREADS, 2)
kv4_tc_mass_kernel(const Kv4TcArgs p) {
    using S = Kt<HD>;
    constexpr int QST = S::QST;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    unsigned char* Ks = sm;                            // OPER
    unsigned char* Qs = Ks + S::OPER;                  // [QST] IMAGE
    uint64_t* bars = reinterpret_cast<uint64_t*>(Qs + QST * S::IMAGE);
    uint64_t* k_full = bars;
    uint64_t* q_full = bars + 1; uint64_t* q_empty = bars + 4;                   // [QST]
    uint64_t* s_full = bars + 7; uint64_t* s_free = bars + 9;                    // [group]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* tops = abort_flag + 1;               // [4]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    kp_pdl_begin();
    const int n_ctas = p.cluster, rank = blockIdx.x % n_ctas, R = p.H / p.G;
    // the first keys first, of all heads and segments: most rows read them
    const int place = blockIdx.x / n_ctas, kvh = place % p.G, seg = place / p.G % p.n_seg, k0 = place / p.G / p.n_seg * KT_ROWS;
    const int n_rows = p.cu_rows[seg + 1] - p.cu_rows[seg], pos0 = p.seg_pos[seg], n_cols = n_rows * R;
    // keys that any row reads, and columns that read any of this CTA's, in tiles of 128 from column 0; this CTA has every n_ctas-th tile
    const int last = min(pos0 + n_rows - 1, p.max_blocks * p.ps - 1), first = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
    const int c_lo = max(0, k0 - pos0) * R;
    const int c_hi = (p.window > 0 ? min(n_rows - 1, k0 - pos0 + KT_ROWS - 2 + p.window) : n_rows - 1) * R + R - 1;
    if (n_rows < p.min_rows || k0 > last || k0 + KT_ROWS - 1 < first || c_hi < c_lo) return;       // (all of a cluster or none)
    const int j_lo = c_lo / 128 + rank, n_j = max(0, (c_hi / 128 - j_lo + n_ctas) / n_ctas);
    if (threadIdx.x == 0) {
        kp_mbar_init(k_full, 128);
        for (int i = 0; i < QST; i++) { kp_mbar_init(&q_full[i], 1); kp_mbar_init(&q_empty[i], 1 + 128); }
        for (int i = 0; i < 2; i++) { kp_mbar_init(&s_full[i], 1); kp_mbar_init(&s_free[i], 128); }
        *abort_flag = 0;
        kp_mbar_init_fence();
    }
    if (warp == 8) kp_tmem_alloc(tmem_slot, 256);
    kp_tc_fence_before();
    __syncthreads();
    kp_tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    float sum = 0.f;                                   // this key's weight here, and where its mass lies
    float* to = nullptr;

    if (warp == 8) {
        // ---- copies and products
        const int top_tile = kt_first_tile(p, seg, R, lane);
        auto load = [&](int i) {
            const int st = i % QST, j = j_lo + i * n_ctas;
            const size_t tile_id = ((size_t)kvh * p.n_tiles + top_tile - (j >> 1)) * 2 + (j & 1);
            kp_mbar_expect_tx_warp(&q_full[st], S::IMAGE);
            kp_bulk_g2s_warp(Qs + st * S::IMAGE, p.q_image + tile_id * S::OPER, S::OPER, &q_full[st]);
            kp_bulk_g2s_warp(Qs + st * S::IMAGE + S::OPER, p.col + tile_id * 128, 1024, &q_full[st]);
        };
        for (int i = 0; i < QST && i < n_j; i++) load(i);
        bool ok = n_j == 0 || kt_wait(k_full, 0);
        for (int i = 0; i < n_j && ok; i++) {
            const int st = i % QST, g = i & 1, use = i >> 1;                     // S of group g for the use-th time
            ok = kt_wait(&q_full[st], (i / QST) & 1) && kt_wait(&s_free[g], (use & 1) ^ 1);
            if (!ok) break;
            kp_tc_fence_after();
            kt_issue_s<HD>(tmem_base + g * 128, Ks, Qs + st * S::IMAGE);
            kp_umma_commit_warp(&s_full[g]);
            kp_umma_commit_warp(&q_empty[st]);
            // the stage of the tile before is asked for again once that tile's columns have been read
            if (i > 0 && i - 1 + QST < n_j) {
                ok = kt_wait(&q_empty[(i - 1) % QST], ((i - 1) / QST) & 1);
                if (ok) load(i - 1 + QST);
            }
        }
        if (!ok) {
            if (lane == 0) { *abort_flag = 1; atomicExch(&g_kv4_tc_status, 1); }
            kp_linger_after_failure();                 // copies may still be under way
        }
    } else {
        const int g = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane, key = k0 + r;
        const bool there = key >= first && key <= last;
        if (g == 0) {
            const int page = there ? p.block_table[(size_t)seg * p.max_blocks + (key >> p.ps_log2)] : 0;
            KtRow<HD> x;
            x.load(p.pages + ((size_t)page * p.G + kvh) * (size_t)kv4_page_bytes(p.ps, HD), key & (p.ps - 1), p.ps, there, false);
            if (there && rank == 0) to = p.mass + ((size_t)page * p.G + kvh) * p.ps + (key & (p.ps - 1));
            int ek = -100;
#pragma unroll
            for (int y = 0; y < S::NG; y++) ek = max(ek, kt_exponent(x.r[y]));
            ek = __reduce_max_sync(0xffffffffu, ek);
            if (lane == 0) tops[warp] = ek;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            kt_write_key<HD>(Ks, r, x, max(max(tops[0], tops[1]), max(tops[2], tops[3])));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            kp_mbar_arrive(k_full);
        }
        const uint32_t tmem_s = tmem_base + g * 128 + ((uint32_t)(q4 * 32) << 16);
        // columns that read this key
        const int mine_lo = max(0, key - pos0) * R;
        const int mine_hi = !there ? -1 : (p.window > 0 ? min(n_rows, key - pos0 + p.window) * R : n_cols) - 1;
        bool ok = n_j == 0 || kp_mbar_wait_bounded(k_full, 0);
        const float kappa = kt_pow2(max(max(tops[0], tops[1]), max(tops[2], tops[3])) - 7);
#pragma unroll 1
        for (int i = g; i < n_j; i += 2) {
            const int st = i % QST, use = i >> 1, c0 = (j_lo + i * n_ctas) * 128;
            if (ok && (*abort_flag || !kp_mbar_wait_bounded(&s_full[g], use & 1))) ok = false;
            // (the copies of the columns' factors arrived before the product that this waits for was issued; the wait makes them visible)
            if (ok && !kp_mbar_wait_bounded(&q_full[st], (i / QST) & 1)) ok = false;
            kp_tc_fence_after();
            const float4* col = reinterpret_cast<const float4*>(Qs + st * S::IMAGE + S::OPER);
            const bool masked = __any_sync(0xffffffffu, c0 < mine_lo || c0 + 127 > mine_hi);
            sum += masked ? kt_column_sum<true>(tmem_s, col, kappa, mine_lo - c0, mine_hi - c0) : kt_column_sum<false>(tmem_s, col, kappa, 0, 127);
            kp_tc_fence_before();
            kp_mbar_arrive(&s_free[g]);
            kp_mbar_arrive(&q_empty[st]);
        }
        if (__builtin_expect(!ok, 0)) { if (lane == 0) atomicExch(&g_kv4_tc_status, 1); sum = 0.f; }
    }
    kp_tc_fence_before();
    __syncthreads();
    if (warp == 8) kp_tmem_dealloc(tmem_base, 256);
    float* join = reinterpret_cast<float*>(Ks);        // [group][key]; the cluster's first CTA adds them up, in order
    if (warp < 8) join[threadIdx.x] = sum;
    if (n_ctas > 1) kv4_cluster_sync(); else __syncthreads();
    if (to) {
        float all = sum + join[128 + threadIdx.x];
        for (int r = 1; r < n_ctas; r++) all += kv4_peer(join + threadIdx.x, r) + kv4_peer(join + 128 + threadIdx.x, r);
        kv4_add_mass(to, all);
    }
    if (n_ctas > 1) kv4_cluster_sync();                 // (nobody leaves while its sums are read)
}

template <int HD>
static int kt_run(Kv4TcArgs a, int max_context, long long busy, cudaStream_t st) {
    using S = Kt<HD>;
    static std::atomic<unsigned long long> ready{0}, ready_split{0}, ready_mass{0};
    int e = kp_smem_limit(kv4_tc_kernel<HD, false>, S::SMEM, ready);
    if (!e) e = kp_smem_limit(kv4_tc_kernel<HD, true>, S::SMEM, ready_split);
    if (e) return e;
    // The mass in clusters of four where that many CTAs fit the GPU at once and each has four tiles of columns or more, else one CTA a tile of
    // keys: a CTA's start (its keys' codes, the first images) takes as long as several tiles of columns.  Measured, attention and mass, one
    // CTA against four: 2048 rows of 32 heads over 8 126 us against 93, 512 rows 41 against 30; 8 x 256 rows 45 against 48, 300 rows behind
    // 4096 keys 137 against 154, 4 x 1024 behind 1024 223 against 243.
    const int tiles = (max_context + KT_ROWS - 1) / KT_ROWS;
    const long long places = (long long)tiles * a.n_seg * a.G;
    // A tile's keys over as many CTAs, up to 16 (8 is what clusters may have without being let), as the GPU holds clusters of, where each has a tile of
    // keys and there are three or more:
    // the join costs less than the second tile.  Measured with 32 heads over 8, one CTA a tile against the rule's: 64 rows behind 16000 keys
    // 249 us against 41 (45 with at most eight; over 2 kv heads 247, 32 and 44), 300 behind 4096 79 against 37, 512 behind 1024 32 against 24, 64 behind
    // 512 18.5 against 15; 256 rows and no
    // more (two tiles of keys) 13.1 against 14.6, 1024 behind 4096, whose pairs would not all be there at once, 87 against 97.
    const int reach = a.window > 0 && a.window + 256 / (a.H / a.G) < max_context ? a.window + 256 / (a.H / a.G) : max_context;
    a.split = 1;
    for (int n = KT_MOST; n > 1 && a.split == 1; n--)
        if (busy * a.G <= kv4_fit<kv4_tc_kernel<HD, true>>(n, S::THREADS, S::SMEM) && (reach + KT_ROWS - 1) / KT_ROWS >= max(n, 3)) a.split = n;
    if ((long long)a.n_tiles * a.G > 2147483647LL || (a.mass && places > 2147483647LL)) return KP_ERR_UNSUPPORTED;
    const Kv4Launch l((unsigned)a.n_tiles * a.G, a.split, S::THREADS, S::SMEM, st);
    cudaError_t c = cudaLaunchKernelEx(&l.cfg, a.split > 1 ? kv4_tc_kernel<HD, true> : kv4_tc_kernel<HD, false>, a);
    if (c) return (int)c;
    if (a.mass) {
        e = kp_smem_limit(kv4_tc_mass_kernel<HD>, S::MASS_SMEM, ready_mass);
        if (e) return e;
        a.cluster = places <= 148 && a.n_tiles - a.n_seg >= 8 * a.n_seg ? 4 : 1;
        const Kv4Launch l((unsigned)places, a.cluster, S::MASS_THREADS, S::MASS_SMEM, st);
        c = cudaLaunchKernelEx(&l.cfg, kv4_tc_mass_kernel<HD>, a);
        if (c) return (int)c;
    }
    return kp_launch_status();
}

extern "C" {

// Bytes of the operand image and of the columns' factors that a call with mass needs beside each other (16-byte aligned).
long long kp_kv4_tc_scratch(int n_rows, int n_seg, int H, int G, int hd) {
    const long long tiles = ((long long)n_rows * (H / G) + 255) / 256 + n_seg;
    return tiles * G * 2 * ((hd / 64) * 16384 + KT_EXT + 1024);
}

// The segments of at least min_rows rows (bfloat16, head size 64 or 128); scratch (with mass): kp_kv4_tc_scratch bytes.
int kp_kv4_attention_tc(const void* q, long long ldq, const void* pages, const int* block_table, int max_blocks, const int* cu_rows,
                        const int* seg_pos, int n_seg, void* out, long long ldo, float scale, int window, int ps, int H, int G, int hd, int n_rows,
                        int min_rows, int max_rows, int max_context, float* mass, void* scratch, void* stream) {
    if (n_rows <= 0 || n_seg <= 0) return 0;
    if (G < 1 || H < 1 || H % G || max_rows < 1 || ps < 16 || (ps & (ps - 1)) || window < 0 || n_seg > 65535 || G > 65535 || min_rows < 1 || !(scale > 0.f) ||
        (((uintptr_t)pages | (uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) & 15) || (ldq & 7) || (ldo & 7) || (mass && !scratch))
        return KP_ERR_BAD_ARG;
    const int R = H / G;
    const long long tiles = ((long long)n_rows * R + 255) / 256 + n_seg;
    // about how many tiles there are: as where each segment has max_rows rows
    const long long busy = max(tiles - n_seg, (long long)(n_rows / max_rows) * (((long long)max_rows * R + 255) / 256));
    Kv4TcArgs a = {};
    a.q = (const bf16*)q; a.ldq = ldq; a.out = (bf16*)out; a.ldo = ldo; a.pages = (const unsigned char*)pages;
    a.block_table = block_table; a.max_blocks = max_blocks; a.cu_rows = cu_rows; a.seg_pos = seg_pos;
    a.scale = scale; a.window = window; a.ps = ps; a.H = H;
    while ((1 << a.ps_log2) < ps) a.ps_log2++;
    a.G = G; a.mass = mass; a.min_rows = min_rows; a.n_seg = n_seg; a.n_tiles = (int)tiles;
    if (mass) {
        a.q_image = (unsigned char*)scratch;
        a.col = (float2*)((unsigned char*)scratch + (size_t)tiles * G * 2 * ((hd / 64) * 16384 + KT_EXT));
    }
    if (hd == 64) return kt_run<64>(a, max_context, busy, (cudaStream_t)stream);
    if (hd == 128) return kt_run<128>(a, max_context, busy, (cudaStream_t)stream);
    return KP_ERR_UNSUPPORTED;
}

}  // extern "C"
