// The prefix's part of attention behind a shared prefix (shared.cuh) on the 5th-generation tensor cores: bfloat16, heads of 64 or 128 values, pages
// of which a tile of 128 keys is made.
//
// Columns.  T = 128 / R rows of a group (rounded down) with their R query heads of a kv head are the 128 rows of an MMA tile: the queries come by one
// TMA box a 64 values, (64 values, R heads, T rows).  A CTA has two such sets of rows, and
//   1 warp asks for K and V, a box a page, into a ring of tiles of 128 keys;
//   1 warp issues  S = Q K^T  and  O += P V  (tcgen05.mma; S and O in tensor memory);
//   2 x 4 warps have a thread a row: S from tensor memory, softmax, P (bfloat16, by up to 2^-8 of each weight) back to tensor memory, where it is the A
//   operand of the second product.  With heads of 128 tensor memory has no room for P beside S and O: it takes half of S, which has been read by then.
// More than 128 columns: the two sets are different columns and read the same tiles.  Up to 128: both are the same columns and take turns at the tiles, so
// that the tensor core and the loads go on for one while the other is at its exponentials.  Up to 64: each set has the columns twice, and the second copy
// takes the second half of every tile's keys (P is zero in the other half), so that all warps have exponentials to do, half as many each: 24 rows of
// two heads behind 120001 keys 62 us, 56 so.  What a column's copies have is joined through shared memory at the end.
//
// Bound by its loads with few columns (24 rows of two heads of 64 behind 120001 keys: 53 us in all, 6.2 TB/s while its tiles run), by the chain of a tile with many
// (256 columns with heads of 128: 3 to 3.5 us a tile of 128 keys, of which products are 1.5).
//
// A column's reference m follows its largest score in steps of at least 2^8 (O is rescaled in tensor memory only then): weights are at most 2^8.  The
// prefix's last page may hold anything behind the prefix: those scores are set to -inf, and the values' rows to zeros.  (All rows of a group read all of
// the prefix: a value that is not finite belongs in every one of them.  Up to 64 columns an infinite one comes out as NaN, 0 times infinity.)
// Every mbarrier wait is bounded; one that gives up sets the status word, and the CTA frees its tensor memory and returns.
#include "shared.cuh"
#include "tcgen05.cuh"

KP_STATUS_WORD(g_shared_tc_status, shared_tc)          // 0 ok; 1: a bounded wait gave up

#define SC_KEYS 128                                    // keys a tile, and columns a set
#define SC_THREADS 320

// MODE 0: 256 columns a CTA; 1: 128, the sets in turn; 2: 64, the copies of a set with half a tile each
template <int HD, int MODE>
struct Sc {
    static constexpr int NB = HD / 64, TILE = NB * 16384;
    static constexpr bool ALIAS = HD == 128;           // P lies in S's columns 64..127, not in columns of its own
    static constexpr int Q_TILES = MODE ? 1 : 2;
    static constexpr int ST = HD == 64 ? (MODE ? 6 : 5) : (MODE ? 3 : 2);
    static constexpr int S_COL = 0, O_COL = 256, P_COL = ALIAS ? 64 : 256 + 2 * HD, P_STEP = ALIAS ? 128 : 64;      // columns of tensor memory (of set 0)
    static constexpr int N_BARS = 1 + 4 * ST + 8;
    static constexpr int COLS = MODE == 2 ? 64 : 128, PARTS = MODE == 2 ? 4 : 2;       // columns of a set, and copies of each (MODE > 0)
    static constexpr int LDO = HD + 4;
    static constexpr size_t SMEM = 1024 + (size_t)Q_TILES * TILE + (size_t)ST * 2 * TILE + N_BARS * 8 + 16;
    static_assert(SMEM <= KP_SMEM_MAX, "more shared memory than a CTA has");
    static_assert(!MODE || (PARTS - 1) * COLS * LDO * 4 + PARTS * COLS * 8 <= ST * 2 * TILE, "the join takes the ring's place");
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

// 32 bytes, a whole sector, at a 32-byte boundary
__device__ __forceinline__ void sc_store32(float* dst, float4 a, float4 b) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(dst), "f"(a.x), "f"(a.y), "f"(a.z), "f"(a.w), "f"(b.x), "f"(b.y), "f"(b.z), "f"(b.w) : "memory");
}
__device__ __forceinline__ void sc_sync_rows() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// grid: chunks of a prefix, kv heads, groups x tiles of columns (sh_grid), or with a budget so many CTAs, which find theirs
template <int HD, int MODE>
__global__ void __launch_bounds__(SC_THREADS, 1)
shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmC, const __grid_constant__ ShArgs p) {
    using C = Sc<HD, MODE>;
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
    const int R = p.H / p.G, T = C::COLS / R;
    const ShPlace place(p);
    int chunk = blockIdx.x, kvh = place.g, group = place.i / p.tiles, tile = place.i % p.tiles;
    const int chunk_keys = sh_chunk(p, lane);
    if (p.budget) {
        // this CTA's place in the list of (group, chunk, tile, kv head)
        const int per = p.tiles * p.G, mine = lane < p.n_groups ? (sh_prefix(p, lane) + chunk_keys - 1) / chunk_keys * per : 0;
        int run = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const int o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
        const unsigned hit = __ballot_sync(0xffffffffu, (int)blockIdx.x < run);
        if (!hit) return;
        group = __ffs(hit) - 1;
        const int at = blockIdx.x - __shfl_sync(0xffffffffu, run - mine, group);
        chunk = at / per;
        tile = at % per / p.G;
        kvh = at % p.G;
    } else if (group >= p.n_groups) return;
    const int g0 = p.group_seqs[group], g1 = p.group_seqs[group + 1], P = sh_prefix(p, group);
    const int s0 = max(0, min(g0, p.n_seq)), s1 = max(s0, min(g1, p.n_seq));
    if (s0 == s1) return;
    const int first = sh_row(p, s0), rows = sh_row(p, s1) - first;
    const int tile_row = tile * (MODE ? T : 2 * T);                        // the tile's first row in the group
    const int k_lo = chunk * chunk_keys, k_hi = min(P, k_lo + chunk_keys);
    if (tile_row >= rows || k_lo >= k_hi) return;
    const int n_tiles = (k_hi - k_lo + SC_KEYS - 1) / SC_KEYS;
    const int sets = MODE ? (n_tiles > 1 ? 2 : 1) : (rows - tile_row > T ? 2 : 1);
    // tiles of the sets: the i-th of set g is tile number(i, g), whose keys begin at key_of
    const int n0 = MODE ? (n_tiles + 1) / 2 : n_tiles, n1 = sets < 2 ? 0 : (MODE ? n_tiles / 2 : n_tiles);
    auto number = [&](int i, int g) { return MODE ? 2 * i + g : i; };
    auto key_of = [&](int i, int g) { return k_lo + number(i, g) * SC_KEYS; };

    // the first loads are under way while tensor memory is allocated
    const int box = min(p.ps, SC_KEYS), n_box = SC_KEYS / box;
    const int* bt = p.table + (size_t)s0 * p.width;
    auto page_of = [&](int i, int g) {                 // of this lane's box of a tile
        const int key = key_of(i, g) + lane * box;
        return i < (g ? n1 : n0) && lane < n_box && key < k_hi ? bt[sh_block(p, key)] : -1;
    };
    auto load = [&](unsigned char* dst, int page, int i, int g, int kv, uint64_t* bar) {
        const int key = key_of(i, g) + lane * box;
        const bool mine = lane < n_box && key < k_hi && (unsigned)page < (unsigned long long)p.n_pages;
        const int count = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) kp_mbar_expect_tx(bar, count * box * C::NB * 128);
        __syncwarp();
        if (mine) {
            const int row = ((page * 2 + kv) * p.G + kvh) * p.ps + key - sh_block(p, key) * p.ps;
            for (int y = 0; y < C::NB; y++) kp_tma_load_2d(dst + y * 16384 + lane * box * 128, &tmC, y * 64, row, bar);
        }
        __syncwarp();
    };
    int page[2];
    if (warp == 9) {
        page[0] = page_of(0, 0);
        page[1] = MODE ? page_of(0, 1) : -1;
        if (lane == 0) {
            kp_mbar_init(q_full, 1);
            for (int i = 0; i < ST; i++) { kp_mbar_init(&k_full[i], 1); kp_mbar_init(&k_empty[i], 1); kp_mbar_init(&v_full[i], 1); kp_mbar_init(&v_empty[i], 1); }
            for (int i = 0; i < 2; i++) { kp_mbar_init(&s_full[i], 1); kp_mbar_init(&s_free[i], 128); kp_mbar_init(&p_full[i], 128); kp_mbar_init(&o_done[i], 1); }
            *abort_flag = 0;
            kp_mbar_init_fence();
            const int q_tiles = MODE ? MODE : sets;    // (MODE 2: the same rows twice, 64 rows of the tile apart)
            kp_mbar_expect_tx(q_full, q_tiles * C::NB * T * R * 128);
            for (int g = 0; g < q_tiles; g++)
                for (int y = 0; y < C::NB; y++)
                    kp_tma_load_3d(Qs + g * (MODE ? 8192 : C::TILE) + y * 16384, &tmQ, y * 64, kvh * R, first + tile_row + (MODE ? 0 : g * T), q_full);
        }
        __syncwarp();
        load(Ks, page[0], 0, 0, 0, &k_full[0]);
        load(Vs, page[0], 0, 0, 1, &v_full[0]);
    }
    if (warp == 8) kp_tmem_alloc(tmem_slot, 512);
    kp_tc_fence_before();
    __syncthreads();
    kp_tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 9) {
        // ---- loads
        bool ok = true;
        page[0] = page_of(1, 0);
        for (int i = 0; i < n0 && ok; i++)
#pragma unroll
            for (int g = 0; g < (MODE ? 2 : 1); g++) {
                if (i >= (g ? n1 : n0) || (i == 0 && g == 0)) continue;
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
                kp_umma_bf16_box(tmem_base + C::S_COL + 128 * g, kp_umma_desc(kp_smem_u32(Qs + (MODE ? 0 : g) * C::TILE + y * 16384)),
                                 kp_umma_desc(kp_smem_u32(Ks + st * C::TILE + y * 16384)), idesc_s, y > 0);
            kp_umma_commit_warp(&s_full[g]);
            if (MODE || g == sets - 1) kp_umma_commit_warp(&k_empty[st]);
            return true;
        };
        auto issue_pv = [&](int i, int g) {
            const int u = number(i, g), st = u % ST;
            if (!sc_wait(&v_full[st], (u / ST) & 1) || !sc_wait(&p_full[g], i & 1)) return false;
            kp_tc_fence_after();
            const int left = k_hi - key_of(i, g);
            if (left < SC_KEYS && (MODE || g == 0)) {
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
            if (MODE || g == sets - 1) kp_umma_commit_warp(&v_empty[st]);
            return true;
        };
        bool ok = sc_wait(q_full, 0);
        for (int g = 0; g < sets && ok; g++) ok = issue_s(0, g);
        // (a set's products run in the order in which they are issued: where P lies in S, the next S comes behind the product that reads it)
        for (int i = 0; i < n0 && ok; i++)
            for (int g = 0; g < sets && ok; g++) {
                if (i >= (g ? n1 : n0)) continue;
                const bool more = i + 1 < (g ? n1 : n0);
                ok = C::ALIAS ? issue_pv(i, g) && (!more || issue_s(i + 1, g)) : (!more || issue_s(i + 1, g)) && issue_pv(i, g);
            }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(&g_shared_tc_status, 1); }
    } else {
        // ---- the rows of the tile: warps 0-3 set 0, warps 4-7 set 1; thread r of a set has row r: column c, row c / R of the group's and head c % R
        const int g = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane, c = MODE == 2 ? r & 63 : r, half = MODE == 2 ? q4 >> 1 : 0;
        constexpr int NS = MODE == 2 ? 2 : 4;                              // keys of a tile that a thread takes, in thirty-twos
        const int row = tile_row + (MODE ? 0 : g * T) + c / R;
        const bool live = c < T * R && row < rows;
        const bool any = __any_sync(0xffffffffu, live);                    // (a warp without a column only keeps the others' count)
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t tmem_s = tmem_base + C::S_COL + 128 * g + lane_off, tmem_o = tmem_base + C::O_COL + HD * g + lane_off;
        const uint32_t tmem_p = tmem_base + C::P_COL + C::P_STEP * g + lane_off;
        const float sl2 = p.scale * 1.4426950408889634f;
        const int n = g ? n1 : n0;
        bool ok = true;
        float m = -INFINITY, l = 0.f;
        auto no_weights = [&] {                                            // in the half of the tile that the other copy takes
            uint32_t zero[32];
#pragma unroll
            for (int j = 0; j < 32; j++) zero[j] = 0u;
            kp_tmem_st32(tmem_p + 32 * (half ^ 1), zero);
        };
        if (MODE == 2 && !C::ALIAS && any) { no_weights(); kp_tmem_st_wait(); }
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            if (ok && (*abort_flag || !kp_mbar_wait_bounded(&s_full[g], i & 1))) ok = false;
            kp_tc_fence_after();
            const int left = k_hi - key_of(i, g) - 64 * half;              // keys from this thread's first one on
            if (any) {
                uint32_t s[NS][32];
#pragma unroll
                for (int e = 0; e < NS; e++) kp_tmem_ld32_issue(tmem_s + 64 * half + 32 * e, s[e]);
                kp_tmem_ld_wait();
                if (!C::ALIAS) { kp_tc_fence_before(); kp_mbar_arrive(&s_free[g]); }       // the next tile's S may be computed
                if (left < NS * 32) {
#pragma unroll
                    for (int e = 0; e < NS; e++)
#pragma unroll
                        for (int j = 0; j < 32; j++) if (e * 32 + j >= left) s[e][j] = 0xff800000u;
                }
                float top = -INFINITY;
#pragma unroll
                for (int e = 0; e < NS; e++) {
                    float t = fmaxf(__uint_as_float(s[e][0]), __uint_as_float(s[e][1]));
#pragma unroll
                    for (int j = 2; j < 32; j += 2) t = sc_max3(t, __uint_as_float(s[e][j]), __uint_as_float(s[e][j + 1]));
                    top = fmaxf(top, t);
                }
                top *= sl2;
                const float m_new = top > m + 8.0f ? top : m;              // (the first: m = -inf)
                const float corr = m_new == m ? 1.0f : sh_exp2(m - m_new);
                const float sub = m_new == -INFINITY ? 0.f : m_new;
                const float2 f2 = make_float2(sl2, sl2), sub2 = make_float2(-sub, -sub);
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t w[NS / 2][32];
#pragma unroll
                for (int e = 0; e < NS; e++)
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
#pragma unroll
                for (int e = 0; e < NS / 2; e++) kp_tmem_st32(tmem_p + 32 * (half + e), w[e]);
                if (MODE == 2 && C::ALIAS) no_weights();
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
        if (n > 0 && ok && !kp_mbar_wait_bounded(&o_done[g], (n - 1) & 1)) ok = false;
        kp_tc_fence_after();
        const size_t at = ((size_t)(first + row) * p.H + kvh * R + c % R) * p.n_chunks + chunk;
        if constexpr (MODE == 0) {
            if (any && n > 0) {
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t v[32];
                    kp_tmem_ld32(tmem_o + d, v);
                    if (live && ok) {
                        auto four = [&](int j) { return make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])); };
#pragma unroll
                        for (int j = 0; j < 32; j += 8) sc_store32(p.part_o + at * HD + d + j, four(j), four(j + 4));
                    }
                }
                if (live && ok) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
            }
        } else {
            // the copies of a column, joined where the ring was: all products are done
            const int part = MODE == 2 ? 2 * g + half : g;
            float* O = reinterpret_cast<float*>(Ks);                        // [PARTS - 1][COLS][LDO]
            float2* ml = reinterpret_cast<float2*>(O + (C::PARTS - 1) * C::COLS * C::LDO);
            sc_sync_rows();
            ml[part * C::COLS + c] = make_float2(m, l);
            sc_sync_rows();
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int e = 0; e < C::PARTS; e++) M = fmaxf(M, ml[e * C::COLS + c].x);
            const float u = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int e = 0; e < C::PARTS; e++) L += sh_exp2(ml[e * C::COLS + c].x - u) * ml[e * C::COLS + c].y;
            const float f = sh_exp2(m - u);
            if (part && any) {
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t v[32];
                    kp_tmem_ld32(tmem_o + d, v);
                    float4* dst = reinterpret_cast<float4*>(O + ((part - 1) * C::COLS + c) * C::LDO + d);
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        dst[j >> 2] = n ? make_float4(__uint_as_float(v[j]) * f, __uint_as_float(v[j + 1]) * f, __uint_as_float(v[j + 2]) * f, __uint_as_float(v[j + 3]) * f)
                                        : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            sc_sync_rows();
            if (!part && any) {
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t v[32];
                    kp_tmem_ld32(tmem_o + d, v);
                    if (live && ok) {
                        auto four = [&](int j) {
                            float4 x = make_float4(__uint_as_float(v[j]) * f, __uint_as_float(v[j + 1]) * f, __uint_as_float(v[j + 2]) * f, __uint_as_float(v[j + 3]) * f);
#pragma unroll
                            for (int e = 0; e < C::PARTS - 1; e++) {
                                const float4 y = *reinterpret_cast<const float4*>(O + (e * C::COLS + c) * C::LDO + d + j);
                                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                            }
                            return x;
                        };
#pragma unroll
                        for (int j = 0; j < 32; j += 8) sc_store32(p.part_o + at * HD + d + j, four(j), four(j + 4));
                    }
                }
                if (live && ok) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(M, L);
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

template <int HD, int MODE>
static int sc_launch(const ShArgs& a, const CUtensorMap& tq, const CUtensorMap& tc, cudaStream_t st) {
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(shared_prefix_tc_kernel<HD, MODE>, Sc<HD, MODE>::SMEM, ready);
    if (e) return e;
    const dim3 grid = a.budget ? dim3(a.budget) : sh_grid(a.n_chunks, a.G, a.n_groups * a.tiles);
    cudaError_t c = kp_launch_pdl(shared_prefix_tc_kernel<HD, MODE>, grid, dim3(SC_THREADS), Sc<HD, MODE>::SMEM, st, tq, tc, a);
    return c ? (int)c : kp_launch_status();
}

// The first launch (kp_attention_shared makes the second one).  mode 0: a tile of columns is 2 T rows, T = 128 / R; 1: T rows; 2: 64 / R rows.  budget > 0: `chunk`
// is the least that a chunk has, and the launch has so many CTAs.
extern "C" int kp_attention_shared_prefix_tc(const void* q, long long ldq, const void* cache, long long n_pages, const int* table, int width, const int* cu_rows,
                                             const int* group_seqs, const int* prefix_len, int n, int n_seq, int n_groups, float* part_o, float* part_ml, int n_chunks,
                                             int chunk, float scale, int ps, int H, int G, int hd, int max_prefix, int tiles, int mode, int budget, void* stream) {
    if (n <= 0 || n_seq <= 0 || n_groups <= 0 || max_prefix <= 0) return 0;
    if (G < 1 || H < 1 || H % G || mode < 0 || mode > 2 || H / G > (mode == 2 ? 64 : 128) || ps < 8 || ps % 8 || !(ps % SC_KEYS == 0 || SC_KEYS % ps == 0) ||
        width < 1 || (long long)width * ps > (1 << 30) || n_pages < 1 || n_pages * 2 * G * ps >= 2147483647LL || chunk < SC_KEYS || chunk % SC_KEYS || n_chunks < 1 ||
        n_chunks > SH_MAX_CHUNKS || (long long)n_chunks * chunk < max_prefix || tiles < 1 || !sh_grid_ok(n_groups, tiles, G) || (ldq & 7) || !(scale > 0.f) ||
        (((uintptr_t)q | (uintptr_t)cache) & 15) || ((uintptr_t)part_o & 31) || (hd != 64 && hd != 128) || budget < 0 ||
        (budget && (n_groups > 32 || (long long)n_groups * tiles * G > budget)))
        return KP_ERR_UNSUPPORTED;
    const int R = H / G, T = (mode == 2 ? 64 : 128) / R;
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
    a.budget = budget; a.group_tiles = tiles; a.tiles = tiles; a.scale = scale; a.ps = ps; a.ps_log2 = -1; a.H = H; a.G = G; a.max_prefix = max_prefix;
    for (int i = 0; i < 31; i++) if (ps == 1 << i) a.ps_log2 = i;
    const cudaStream_t st = (cudaStream_t)stream;
    switch (mode * 256 + hd) {
        case 64: return sc_launch<64, 0>(a, tq, tc, st);
        case 128: return sc_launch<128, 0>(a, tq, tc, st);
        case 256 + 64: return sc_launch<64, 1>(a, tq, tc, st);
        case 256 + 128: return sc_launch<128, 1>(a, tq, tc, st);
        case 512 + 64: return sc_launch<64, 2>(a, tq, tc, st);
        default: return sc_launch<128, 2>(a, tq, tc, st);
    }
}
