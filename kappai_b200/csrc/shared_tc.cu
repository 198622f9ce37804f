// The prefix's part of attention behind a shared prefix (shared.cuh) on the 5th-generation tensor cores: bfloat16, heads of 64 or 128 values, pages
// of which a tile of 128 keys is made.
//
// Columns.  T = 128 / R rows of a group (rounded down) with their R query heads of a kv head are the 128 rows of an MMA tile: the queries come by one
// TMA box a 64 values, (64 values, R heads, T rows).  A CTA has two such sets of columns, and
//   1 warp asks for K and V, a box a page, into a ring of tiles of 128 keys;
//   1 warp issues  S = Q K^T  and  O += P V  (tcgen05.mma; S and O in tensor memory);
//   2 x 4 warps have a thread a column: S from tensor memory, softmax, P (bfloat16, by up to 2^-8 of each weight) back to tensor memory, where it is the A
//   operand of the second product.  With heads of 128 tensor memory has no room for P beside S and O: it takes half of S, which has been read by then.
// More than 128 columns: the two sets are different columns and read the same tiles.  Up to 128: both sets are the same columns and take a chunk of keys
// each, so that the tensor core and the loads go on for one while the other is at its exponentials.
//
// A column's reference m follows its largest score in steps of at least 2^8 (O is rescaled in tensor memory only then): weights are at most 2^8.  The
// prefix's last page may hold anything behind the prefix: those scores are set to -inf, and the values' rows to zeros.
// Every mbarrier wait is bounded; one that gives up sets the status word, and the CTA frees its tensor memory and returns.
#include "shared.cuh"
#include "tcgen05.cuh"

KP_STATUS_WORD(g_shared_tc_status, shared_tc)          // 0 ok; 1: a bounded wait gave up

#define SC_KEYS 128                                    // keys a tile, and columns a set
#define SC_THREADS 320

template <int HD, bool SPLIT>
struct Sc {
    static constexpr int NB = HD / 64, TILE = NB * 16384;
    static constexpr bool ALIAS = HD == 128;           // P lies in S's columns 64..127, not in columns of its own
    static constexpr int Q_TILES = SPLIT ? 1 : 2;
    static constexpr int ST = HD == 64 ? (SPLIT ? 6 : 5) : (SPLIT ? 3 : 2);
    static constexpr int S_COL = 0, O_COL = 256, P_COL = ALIAS ? 64 : 256 + 2 * HD, P_STEP = ALIAS ? 128 : 64;      // columns of tensor memory (of set 0)
    static constexpr int N_BARS = 1 + 4 * ST + 8;
    static constexpr size_t SMEM = 1024 + (size_t)Q_TILES * TILE + (size_t)ST * 2 * TILE + N_BARS * 8 + 16;
    static_assert(SMEM <= KP_SMEM_MAX, "more shared memory than a CTA has");
};

__device__ __forceinline__ float sc_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two float32 operations at once
__device__ __forceinline__ float2 sc_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 sc_add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ uint32_t sc_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// D (+)= A B with A in tensor memory (a lane a row, a column two consecutive elements), by an elected lane of a warp in step
__device__ __forceinline__ void sc_umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
// a wait of a warp in step, which gives up as one
__device__ __forceinline__ bool sc_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, kp_mbar_wait_bounded(bar, parity)); }

// grid: (CTAs that share a prefix, kv heads, groups x tiles of columns); SPLIT: both sets are the same columns, with a chunk of keys each
template <int HD, bool SPLIT>
__global__ void __launch_bounds__(SC_THREADS, 1)
shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmC, const __grid_constant__ ShArgs p) {
    using C = Sc<HD, SPLIT>;
    constexpr int ST = C::ST;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    unsigned char* Qs = sm;                            // [Q_TILES] TILE
    unsigned char* Ks = Qs + C::Q_TILES * C::TILE;     // [ST] TILE
    unsigned char* Vs = Ks + ST * C::TILE;             // [ST] TILE
    uint64_t* q_full = reinterpret_cast<uint64_t*>(Vs + ST * C::TILE);
    uint64_t* k_full = q_full + 1;   uint64_t* k_empty = k_full + ST;      // [ST] each
    uint64_t* v_full = k_empty + ST; uint64_t* v_empty = v_full + ST;
    uint64_t* s_full = v_empty + ST; uint64_t* s_free = s_full + 2;        // [2] each: by set
    uint64_t* p_full = s_free + 2;   uint64_t* o_done = p_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    kp_pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.y, group = blockIdx.z / p.tiles, R = p.H / p.G, T = SC_KEYS / R;
    const int s0 = max(0, min(p.group_seqs[group], p.n_seq)), s1 = max(s0, min(p.group_seqs[group + 1], p.n_seq));
    if (s0 == s1) return;
    const int P = sh_prefix(p, group), first = sh_row(p, s0), rows = sh_row(p, s1) - first;
    const int tile_row = blockIdx.z % p.tiles * (SPLIT ? T : 2 * T);       // the tile's first row in the group
    const int chunk0 = SPLIT ? 2 * blockIdx.x : blockIdx.x;
    if (tile_row >= rows || chunk0 * p.chunk >= P) return;
    const int sets = SPLIT ? (P > (chunk0 + 1) * p.chunk ? 2 : 1) : (rows - tile_row > T ? 2 : 1);
    // keys of the sets: from key_lo(g) on, n_kt(g) tiles; below key_hi
    auto key_lo = [&](int g) { return (chunk0 + (SPLIT ? g : 0)) * p.chunk; };
    auto key_hi = [&](int g) { return min(P, key_lo(g) + p.chunk); };
    auto n_kt = [&](int g) { return g < sets ? (key_hi(g) - key_lo(g) + SC_KEYS - 1) / SC_KEYS : 0; };
    const int n0 = n_kt(0), n1 = n_kt(1);
    // tiles are counted over both sets where each has its own: the stage of a tile is its number modulo ST
    auto number = [&](int i, int g) { return SPLIT ? min(i, n0) + min(i, n1) + (g && i < n0 ? 1 : 0) : i; };

    if (threadIdx.x == 0) {
        kp_mbar_init(q_full, 1);
        for (int i = 0; i < ST; i++) { kp_mbar_init(&k_full[i], 1); kp_mbar_init(&k_empty[i], 1); kp_mbar_init(&v_full[i], 1); kp_mbar_init(&v_empty[i], 1); }
        for (int i = 0; i < 2; i++) { kp_mbar_init(&s_full[i], 1); kp_mbar_init(&s_free[i], 128); kp_mbar_init(&p_full[i], 128); kp_mbar_init(&o_done[i], 1); }
        *abort_flag = 0;
        kp_mbar_init_fence();
    }
    if (warp == 8) kp_tmem_alloc(tmem_slot, 512);
    kp_tc_fence_before();
    __syncthreads();
    kp_tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 9) {
        // ---- loads
        const int box = min(p.ps, SC_KEYS), n_box = SC_KEYS / box;
        const int* bt = p.table + (size_t)s0 * p.width;
        if (lane == 0) {
            const int q_tiles = SPLIT ? 1 : sets;
            kp_mbar_expect_tx(q_full, q_tiles * C::NB * T * R * 128);
            for (int g = 0; g < q_tiles; g++)
                for (int y = 0; y < C::NB; y++)
                    kp_tma_load_3d(Qs + g * C::TILE + y * 16384, &tmQ, y * 64, kvh * R, first + tile_row + g * T, q_full);
        }
        __syncwarp();
        bool ok = true;
        auto page_of = [&](int i, int g) {             // of this lane's box of a tile
            const int key = key_lo(g) + i * SC_KEYS + lane * box;
            return i < (g ? n1 : n0) && lane < n_box && key < key_hi(g) ? bt[key / p.ps] : -1;
        };
        auto load = [&](unsigned char* dst, int page, int i, int g, int kv, uint64_t* bar) {
            const int hi = key_hi(g), key0 = key_lo(g) + i * SC_KEYS, key = key0 + lane * box;
            const bool mine = lane < n_box && key < hi && (unsigned)page < (unsigned long long)p.n_pages;
            const int count = __popc(__ballot_sync(0xffffffffu, mine));
            if (lane == 0) kp_mbar_expect_tx(bar, count * box * C::NB * 128);
            __syncwarp();
            if (mine) {
                const int row = ((page * 2 + kv) * p.G + kvh) * p.ps + key % p.ps;
                for (int y = 0; y < C::NB; y++) kp_tma_load_2d(dst + y * 16384 + lane * box * 128, &tmC, y * 64, row, bar);
            }
            __syncwarp();
        };
        const int n_max = max(n0, n1);
        int page[2] = {page_of(0, 0), SPLIT ? page_of(0, 1) : -1};
        for (int i = 0; i < n_max && ok; i++)
#pragma unroll
            for (int g = 0; g < (SPLIT ? 2 : 1); g++) {
                if (i >= (g ? n1 : n0)) continue;
                const int u = number(i, g), st = u % ST, par = ((u / ST) & 1) ^ 1;
                if (*abort_flag || !sc_wait(&k_empty[st], par)) { ok = false; break; }
                load(Ks + st * C::TILE, page[g], i, g, 0, &k_full[st]);
                if (!sc_wait(&v_empty[st], par)) { ok = false; break; }
                load(Vs + st * C::TILE, page[g], i, g, 1, &v_full[st]);
                page[g] = page_of(i + 1, g);
            }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(&g_shared_tc_status, 1); }
    } else if (warp == 8) {
        // ---- the tensor core's work
        constexpr uint32_t idesc_s = kp_umma_idesc(128, 128), idesc_pv = kp_umma_idesc(128, HD, true);
        auto issue_s = [&](int i, int g) {
            const int u = number(i, g), st = u % ST;
            if (!sc_wait(&k_full[st], (u / ST) & 1) || (!C::ALIAS && i > 0 && !sc_wait(&s_free[g], (i - 1) & 1))) return false;
            kp_tc_fence_after();
#pragma unroll
            for (int y = 0; y < C::NB; y++)
                kp_umma_bf16_box(tmem_base + C::S_COL + 128 * g, kp_umma_desc(kp_smem_u32(Qs + (SPLIT ? 0 : g) * C::TILE + y * 16384)),
                                 kp_umma_desc(kp_smem_u32(Ks + st * C::TILE + y * 16384)), idesc_s, y > 0);
            kp_umma_commit_warp(&s_full[g]);
            if (SPLIT || g == sets - 1) kp_umma_commit_warp(&k_empty[st]);
            return true;
        };
        auto issue_pv = [&](int i, int g) {
            const int u = number(i, g), st = u % ST;
            if (!sc_wait(&v_full[st], (u / ST) & 1) || !sc_wait(&p_full[g], i & 1)) return false;
            kp_tc_fence_after();
            const int left = key_hi(g) - key_lo(g) - i * SC_KEYS;
            if (left < SC_KEYS && (SPLIT || g == 0)) {
                // what lies behind the prefix has weight 0, and must not be NaN or infinite
                for (int y = 0; y < C::NB; y++)
                    for (int e = left * 8 + lane; e < SC_KEYS * 8; e += 32) *reinterpret_cast<uint4*>(Vs + st * C::TILE + y * 16384 + e * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            const uint32_t va = kp_smem_u32(Vs + st * C::TILE);
#pragma unroll
            for (int kk = 0; kk < SC_KEYS / 16; kk++)
                sc_umma_ts(tmem_base + C::O_COL + HD * g, tmem_base + C::P_COL + C::P_STEP * g + 8 * kk,
                           HD == 64 ? kp_umma_desc(va + kk * 2048) : kp_umma_desc_mn(va + kk * 2048, 16384), idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
            kp_umma_commit_warp(&o_done[g]);
            if (SPLIT || g == sets - 1) kp_umma_commit_warp(&v_empty[st]);
            return true;
        };
        bool ok = sc_wait(q_full, 0);
        for (int g = 0; g < sets && ok; g++) ok = issue_s(0, g);
        const int n_max = max(n0, n1);
        // (a set's products run in the order in which they are issued: where P lies in S, the next S comes behind the product that reads it)
        for (int i = 0; i < n_max && ok; i++)
            for (int g = 0; g < sets && ok; g++) {
                if (i >= (g ? n1 : n0)) continue;
                const bool more = i + 1 < (g ? n1 : n0);
                ok = C::ALIAS ? issue_pv(i, g) && (!more || issue_s(i + 1, g)) : (!more || issue_s(i + 1, g)) && issue_pv(i, g);
            }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(&g_shared_tc_status, 1); }
    } else {
        // ---- the columns: warps 0-3 set 0, warps 4-7 set 1; thread r of a set has column r, row r / R and head r % R
        const int g = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane;
        const int row = tile_row + (SPLIT ? 0 : g * T) + r / R;
        const bool live = r < T * R && row < rows;
        const bool any = __any_sync(0xffffffffu, live);                    // (a warp without a column only keeps the others' count)
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t tmem_s = tmem_base + C::S_COL + 128 * g + lane_off, tmem_o = tmem_base + C::O_COL + HD * g + lane_off;
        const uint32_t tmem_p = tmem_base + C::P_COL + C::P_STEP * g + lane_off;
        const float sl2 = p.scale * 1.4426950408889634f;
        const int n = g ? n1 : n0, lo = key_lo(g), hi = key_hi(g);
        bool ok = true;
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            if (ok && (*abort_flag || !kp_mbar_wait_bounded(&s_full[g], i & 1))) ok = false;
            kp_tc_fence_after();
            const int left = hi - lo - i * SC_KEYS;                        // keys from this tile on
            if (any) {
                uint32_t s[4][32];
#pragma unroll
                for (int e = 0; e < 4; e++) kp_tmem_ld32_issue(tmem_s + 32 * e, s[e]);
                kp_tmem_ld_wait();
                if (!C::ALIAS) { kp_tc_fence_before(); kp_mbar_arrive(&s_free[g]); }       // the next tile's S may be computed
                if (left < SC_KEYS) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int j = 0; j < 32; j++) if (e * 32 + j >= left) s[e][j] = 0xff800000u;
                }
                float t[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    t[e] = fmaxf(__uint_as_float(s[e][0]), __uint_as_float(s[e][1]));
#pragma unroll
                    for (int j = 2; j < 32; j += 2) t[e] = sc_max3(t[e], __uint_as_float(s[e][j]), __uint_as_float(s[e][j + 1]));
                }
                const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * sl2;
                const float m_new = top > m + 8.0f ? top : m;              // (the first: m = -inf)
                const float corr = m_new == m ? 1.0f : sh_exp2(m - m_new);
                const float sub = m_new == -INFINITY ? 0.f : m_new;
                const float2 f2 = make_float2(sl2, sl2), sub2 = make_float2(-sub, -sub);
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t w[2][32];
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float2 x = sc_fma2(make_float2(__uint_as_float(s[e][j]), __uint_as_float(s[e][j + 1])), f2, sub2);
                        x.x = sh_exp2(x.x);
                        x.y = sh_exp2(x.y);
                        sums[e & 1] = sc_add2(sums[e & 1], x);
                        w[e >> 1][(e & 1) * 16 + (j >> 1)] = sc_pack(x.x, x.y);
                    }
                // the product of the tile before has read P and added to O
                if (i > 0 && ok && !kp_mbar_wait_bounded(&o_done[g], (i - 1) & 1)) ok = false;
                if (i > 0 && __any_sync(0xffffffffu, live && corr != 1.0f)) {
                    kp_tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < HD; d += 32) {
                        uint32_t v[32];
                        kp_tmem_ld32(tmem_o + d, v);
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
                        kp_tmem_st32(tmem_o + d, v);
                    }
                }
                kp_tmem_st32(tmem_p, w[0]);
                kp_tmem_st32(tmem_p + 32, w[1]);
                kp_tmem_st_wait();
                sums[0] = sc_add2(sums[0], sums[1]);
                l = l * corr + (sums[0].x + sums[0].y);
                m = m_new;
            } else {
                if (!C::ALIAS) kp_mbar_arrive(&s_free[g]);
                // (p_full's count is of one tile: nobody arrives for a tile before all have for the one before)
                if (i > 0 && ok && !kp_mbar_wait_bounded(&o_done[g], (i - 1) & 1)) ok = false;
            }
            kp_tc_fence_before();
            kp_mbar_arrive(&p_full[g]);
        }
        if (n > 0) {
            if (ok && !kp_mbar_wait_bounded(&o_done[g], (n - 1) & 1)) ok = false;
            kp_tc_fence_after();
            if (any) {
                const size_t at = ((size_t)(first + row) * p.H + kvh * R + r % R) * p.n_chunks + chunk0 + (SPLIT ? g : 0);
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t v[32];
                    kp_tmem_ld32(tmem_o + d, v);
                    if (live && ok) {
                        uint4* dst = reinterpret_cast<uint4*>(p.part_o + at * HD + d);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) dst[j >> 2] = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    }
                }
                if (live && ok) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
                kp_tc_fence_before();
            }
        }
        if (__builtin_expect(!ok, 0)) {
            *abort_flag = 1;
            atomicExch(&g_shared_tc_status, 1);
            kp_linger_after_failure();
        }
    }
    kp_tc_fence_before();
    __syncthreads();
    if (warp == 8) { kp_tc_fence_after(); kp_tmem_dealloc(tmem_base, 512); }
}

template <int HD, bool SPLIT>
static int sc_launch(const ShArgs& a, const CUtensorMap& tq, const CUtensorMap& tc, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(shared_prefix_tc_kernel<HD, SPLIT>, Sc<HD, SPLIT>::SMEM, ready);
    if (e) return e;
    const int ctas = SPLIT ? (a.n_chunks + 1) / 2 : a.n_chunks;
    cudaError_t c = kp_launch_pdl(shared_prefix_tc_kernel<HD, SPLIT>, dim3(ctas, a.G, a.n_groups * a.tiles), dim3(SC_THREADS), Sc<HD, SPLIT>::SMEM, st, tq, tc, a);
    return c ? (int)c : kp_launch_status();
}

// The first launch (kp_attention_shared makes the second one): split: a tile of columns is T = 128 / R rows and a CTA takes two chunks, else 2 T rows and one.
extern "C" int kp_attention_shared_prefix_tc(const void* q, long long ldq, const void* cache, long long n_pages, const int* table, int width, const int* cu_rows,
                                             const int* group_seqs, const int* prefix_len, int n, int n_seq, int n_groups, float* part_o, float* part_ml, int n_chunks,
                                             int chunk, float scale, int ps, int H, int G, int hd, int max_prefix, int tiles, int split, void* stream) {
    if (n <= 0 || n_seq <= 0 || n_groups <= 0 || max_prefix <= 0) return 0;
    if (G < 1 || G > 65535 || H < 1 || H % G || H / G > SC_KEYS || ps < 8 || ps % 8 || !(ps % SC_KEYS == 0 || SC_KEYS % ps == 0) || width < 1 ||
        (long long)width * ps > (1 << 30) || n_pages < 1 || n_pages * 2 * G * ps >= 2147483647LL || chunk < SC_KEYS || chunk % SC_KEYS || n_chunks < 1 ||
        n_chunks > SH_MAX_CHUNKS || (long long)n_chunks * chunk < max_prefix || tiles < 1 || (long long)n_groups * tiles > 65535 || (ldq & 7) || !(scale > 0.f) ||
        (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)part_o) & 15) || (hd != 64 && hd != 128))
        return KP_ERR_UNSUPPORTED;
    const int R = H / G, T = SC_KEYS / R;
    CUtensorMap tq, tc;
    KpEncodeTiledFn fn = kp_encode_tiled_fn();
    if (!fn) return KP_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)H, (cuuint64_t)n};
    cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ldq * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)R, (cuuint32_t)T};
    cuuint32_t estr[3] = {1, 1, 1};
    if (fn(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return KP_ERR_UNSUPPORTED;
    int e = kp_make_map_bf16_2d(&tc, cache, (unsigned long long)n_pages * 2 * G * ps, hd, hd, 64, ps < SC_KEYS ? ps : SC_KEYS);
    if (e) return e;
    ShArgs a = {};
    a.q = q; a.ldq = ldq; a.cache = cache; a.n_pages = n_pages; a.table = table; a.width = width; a.cu_rows = cu_rows; a.group_seqs = group_seqs;
    a.prefix_len = prefix_len; a.n = n; a.n_seq = n_seq; a.n_groups = n_groups; a.part_o = part_o; a.part_ml = part_ml; a.n_chunks = n_chunks; a.chunk = chunk;
    a.tiles = tiles; a.scale = scale; a.ps = ps; a.H = H; a.G = G; a.max_prefix = max_prefix;
    const cudaStream_t st = (cudaStream_t)stream;
    if (hd == 64) return split ? sc_launch<64, true>(a, tq, tc, st) : sc_launch<64, false>(a, tq, tc, st);
    return split ? sc_launch<128, true>(a, tq, tc, st) : sc_launch<128, false>(a, tq, tc, st);
}
