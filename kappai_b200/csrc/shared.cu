// Attention behind a shared prefix (shared.cuh): both launches for any head size and page size (bfloat16; shared_f32.cu builds the same for float32).
//
// A CTA takes a tile of columns through a range of keys in tiles of 64 (or 32) that wait in shared memory some tiles ahead, page by page.
//   bfloat16 (mma.sync): with 8 or 16 columns every one of four warps takes a quarter of the tile's keys, and the products have the keys, then the values as
//   their 16 rows and the columns as their 8: the 4 heads of a decoded token fill half of a product, not a quarter.  With up to 64 every warp takes 16 of the
//   columns.  Scores, weights and output stay in registers.  Weights are rounded to bfloat16 as they enter the product with V, by up to 2^-8 of each, as the
//   output itself is.
//   float32 (FMA, two at a time: sums over the heads' even and odd places, pairs of values): a thread has some columns times some keys of the scores, then the
//   same columns times some values of the output; weights pass through shared memory of their warp.  Nothing is rounded below 32 bits.
// Tiles come by TMA from a warp of its own where the sizes allow it (bfloat16, pages of which a tile is made): four warps
// that also copied, 16 bytes a thread with a page to find for each, took twice the time.  Elsewhere by cp.async.
// A key that a column does not read has no part in it, finite or not: in a tile with such keys the values that are not finite are taken out of the
// product and added to the columns that do read them.
// Every mbarrier wait is bounded; one that gives up sets the status word.
#include <cooperative_groups.h>

#include "mma.cuh"
#include "shared.cuh"

namespace cg = cooperative_groups;

#ifdef SH_F32
typedef float ShT;
#define SH_DTYPE KP_DTYPE_F32
#define SH_ENTRY kp_attention_shared_f32
#define SH_32(launch, ...) launch<HD, 32, TMA>(__VA_ARGS__)      // (tiles of 32 columns: float32 only)
KP_STATUS_WORD(g_shared_status, shared_f32)
#else
typedef bf16 ShT;
#define SH_DTYPE KP_DTYPE_BF16
#define SH_ENTRY kp_attention_shared
#define SH_32(launch, ...) KP_ERR_UNSUPPORTED
KP_STATUS_WORD(g_shared_status, shared)                // 0 ok; 1: a bounded wait gave up
#endif

// Keys of a box of own keys: of a sequence's last keys fewer come for nothing.  1424 tiles of columns with 19 to 34, heads of 256, boxes of 64 keys 77 us, of
// 16 67.
#define SH_OWN_BOX 16
#define SH_WORKERS 128                                 // threads of the four warps that compute

template <typename T, int HD, int BM, bool TMA>
struct Sh {
    static constexpr bool MMA = sizeof(T) == 2, KEYS = MMA && BM <= 16;     // KEYS: the warps share the keys, not the columns
    static constexpr int THREADS = TMA ? SH_WORKERS + 32 : SH_WORKERS;
    static constexpr int KT = MMA ? 64 : 32;                                // keys a tile
    static constexpr int E = 16 / sizeof(T);                                // values of 16 bytes
    static constexpr int LD = HD + E;                                       // a row in shared memory: 16 bytes more, so that rows lie in different banks
    static constexpr int BW = HD % 64 ? 32 : 64;                            // values of a row of a TMA box
    static constexpr int TILE = KT * (TMA ? HD : LD);                       // values of K's tile, or of V's (TMA: BW values a row, swizzled)
    static constexpr int CH = HD / E, NI = (KT * CH + SH_WORKERS - 1) / SH_WORKERS;
    static constexpr int PAIR = 2 * TILE * (int)sizeof(T);
    // (float32: few, so that there is room for three CTAs an SM: with one a warp has a scheduler to itself and issues in one cycle of three)
    static constexpr int ST = TMA ? (HD == 32 ? 4 : (HD <= 96 ? 3 : 2)) : !MMA ? (HD < 96 ? 3 : 2) : (4 * PAIR <= 100 * 1024 ? 4 : (3 * PAIR <= 110 * 1024 ? 3 : 2));
    static constexpr int MR = BM / 8;                                       // columns of a thread (FMA)
    static constexpr int Q_BYTES = BM * LD * sizeof(T);
    static constexpr int RING = ST * PAIR;
    static constexpr int P_BYTES = MMA ? 4 * 256 * 4 : BM * (KT + 4) * 4;   // weights (MMA: only where values are not finite)
    static constexpr int PARTS = KEYS ? 4 : 1;                              // outputs of the warps, then the joined one
    static constexpr int LDO = HD + 4;                                      // (columns in different banks)
    static constexpr int O_BYTES = (PARTS > 1 ? PARTS + 1 : 1) * BM * LDO * 4;
    // CTAs an SM that registers are to allow: as many as shared memory does
    static constexpr int CTAS = !TMA ? 1 : (BM <= 16 ? (HD <= 64 ? 4 : (HD <= 128 ? (BM == 8 ? 3 : 2) : (BM == 8 ? 2 : 1))) : (HD <= 128 ? 2 : 1));
    static constexpr int ML_BYTES = (PARTS + 1) * BM * 2 * 4;
    static constexpr int MAIN = RING > O_BYTES ? RING : O_BYTES;            // the output takes the ring's place
    static constexpr int PAD = TMA ? 1024 : 0;                              // the ring starts on a multiple of 1024 bytes
    static constexpr size_t SMEM = PAD + MAIN + Q_BYTES + P_BYTES + ML_BYTES + 2 * ST * 8;
    static constexpr size_t MOST = SMEM + BM * (SH_MAX_CLUSTER + SH_MAX_CHUNKS) * 4;      // with the weights of the join
    static_assert(MOST <= KP_SMEM_MAX, "more shared memory than a CTA has");
};

// a CTA's shared memory
template <typename T, int HD, int BM, bool TMA>
struct ShMem {
    typedef Sh<T, HD, BM, TMA> C;
    unsigned char* ring; T* Qs; unsigned char* P; float* ml; uint64_t* full; uint64_t* empty; float* wts;
    __device__ __forceinline__ ShMem(unsigned char* smem, int main) {
        ring = TMA ? reinterpret_cast<unsigned char*>(((uintptr_t)smem + 1023) & ~(uintptr_t)1023) : smem;
        Qs = reinterpret_cast<T*>(ring + main);
        P = reinterpret_cast<unsigned char*>(Qs) + C::Q_BYTES;
        ml = reinterpret_cast<float*>(P + C::P_BYTES);
        full = reinterpret_cast<uint64_t*>(ml + C::ML_BYTES / 4);
        empty = full + C::ST;
        wts = reinterpret_cast<float*>(empty + C::ST);                      // [BM][parts]
    }
};
__device__ __forceinline__ void sh_sync_workers() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// not a number, or infinite
__device__ __forceinline__ bool sh_odd(float v) { return !(fabsf(v) <= 3.402823466e38f); }
// two float32 operations at once
__device__ __forceinline__ float2 sh_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)), "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
// an 8 x 8 matrix of bfloat16, a row four lanes, turned over
__device__ __forceinline__ uint32_t sh_transposed(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t sh_finite2(uint32_t r) {                // a pair of bfloat16, zeros for what is not finite
    if ((r & 0x7f80u) == 0x7f80u) r &= 0xffff0000u;
    if ((r & 0x7f800000u) == 0x7f800000u) r &= 0x0000ffffu;
    return r;
}

// The loads of the keys k0 .. k1 - 1 of a block-table row, by a warp of their own: a box of p.box keys a lane, those that have any of them.  Tiles start at multiples of KT.
template <typename T, int HD, int BM>
__device__ __forceinline__ bool sh_load(const ShArgs& p, const CUtensorMap& tm, const ShMem<T, HD, BM, true>& sm, const int* bt, int g, int k0, int k1) {
    typedef Sh<T, HD, BM, true> C;
    constexpr int KT = C::KT;
    const int lane = threadIdx.x & 31, box = p.box, n_box = KT / box, t0 = k0 / KT, t1 = k1 > k0 ? (k1 + KT - 1) / KT : t0;
    auto page_of = [&](int t) {
        const int key = t * KT + lane * box;
        return t < t1 && lane < n_box && key < k1 && key + box > k0 ? __ldg(bt + sh_block(p, key)) : -1;
    };
    int page = page_of(t0), st = 0, round = 0;
    for (int t = t0; t < t1; t++) {
        const int key = t * KT + lane * box;
        if (!__all_sync(0xffffffffu, kp_mbar_wait_bounded(&sm.empty[st], (round & 1) ^ 1))) return false;
        const bool mine = (unsigned)page < (unsigned long long)p.n_pages;  // (-1: not this lane's)
        const int count = __popc(__ballot_sync(0xffffffffu, mine));
        if (lane == 0) kp_mbar_expect_tx(&sm.full[st], 2 * count * box * HD * 2);
        __syncwarp();
        if (mine) {
            const int row = (page * 2 * p.G + g) * p.ps + (key - sh_block(p, key) * p.ps);
            unsigned char* dst = sm.ring + st * C::PAIR + lane * box * C::BW * 2;
#pragma unroll
            for (int y = 0; y < HD / C::BW; y++) {
                kp_tma_load_2d(dst + y * KT * C::BW * 2, &tm, y * C::BW, row, &sm.full[st]);
                kp_tma_load_2d(dst + C::PAIR / 2 + y * KT * C::BW * 2, &tm, y * C::BW, row + p.G * p.ps, &sm.full[st]);
            }
        }
        __syncwarp();
        if (++st == p.stages) { st = 0; round++; }
        page = page_of(t + 1);
    }
    return true;
}

// One tile of BM columns, of which `live` are there, through the keys k0 .. k1 - 1 of the block-table row bt, by the four warps; column c reads those below
// lim(c) <= k1 (all of them those below k1 unless OWN).  Leaves
// O [BM][HD] at the ring's place and (m, l) [BM] in ml.  False if a wait gave up.
template <typename T, int HD, int BM, bool TMA, bool OWN, typename Lim>
__device__ __forceinline__ bool sh_tile(const ShArgs& p, const ShMem<T, HD, BM, TMA>& sm, const int* bt, int g, int live, int k0, int k1, int lim_min, Lim lim) {
    typedef Sh<T, HD, BM, TMA> C;
    constexpr int KT = C::KT, LD = C::LD, TILE = C::TILE, CH = C::CH, NI = C::NI, ST = C::ST, E = C::E;
    T* ring = reinterpret_cast<T*>(sm.ring);
    const T* Qs = sm.Qs;
    float* ml = sm.ml;
    unsigned char* Pbuf = sm.P;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* cache = (const T*)p.cache;
    const size_t plane = (size_t)p.G * p.ps * HD, page_stride = 2 * plane;
    const int base = k0 / KT * KT, n_tiles = k1 > k0 ? (k1 - base + KT - 1) / KT : 0;
    bool ok = true;

    int page[NI];                                                           // of the tile that is asked for next
    auto find = [&](int t) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int key = base + t * KT + (tid + i * SH_WORKERS) / CH;
            page[i] = key >= k0 && key < k1 ? __ldg(bt + sh_block(p, key)) : -1;
        }
    };
    auto ask = [&](int t) {
        T* Kt = ring + (t % ST) * 2 * TILE;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int at = tid + i * SH_WORKERS, j = at / CH, e = (at % CH) * E;
            if ((KT * CH) % SH_WORKERS && at >= KT * CH) break;
            const int key = base + t * KT + j;
            const bool there = (unsigned)page[i] < (unsigned long long)p.n_pages;
            const T* src = cache + (size_t)(there ? page[i] : 0) * page_stride + ((size_t)g * p.ps + (there ? key - sh_block(p, key) * p.ps : 0)) * HD + e;
            cp_async16(Kt + j * LD + e, src, there);
            cp_async16(Kt + TILE + j * LD + e, src + plane, there);
        }
    };
    if constexpr (!TMA) {
        find(0);
#pragma unroll
        for (int t = 0; t < ST - 1; t++) {
            if (t < n_tiles) { ask(t); find(t + 1); }
            cp_async_commit();
        }
    }
    int st = 0, round = 0;                                                  // the tile's stage, and how often it has been used
    auto begin = [&](int t) {                                               // tile t is there
        if constexpr (TMA) {
            if (ok && !kp_mbar_wait_bounded(&sm.full[st], round & 1)) ok = false;
        } else {
            cp_async_wait<ST - 2>();
            __syncthreads();
            if (t + ST - 1 < n_tiles) { ask(t + ST - 1); find(t + ST); }
            cp_async_commit();
        }
    };
    auto end = [&] {                                                        // and has been read
        if constexpr (TMA) {
            __syncwarp();
            if (lane == 0) kp_mbar_arrive(&sm.empty[st]);
        }
        if (++st == (TMA ? p.stages : ST)) { st = 0; round++; }
    };
    auto finish = [&] {                                                     // the ring has been read: the output takes its place
        if constexpr (!TMA) cp_async_wait<0>();
        sh_sync_workers();
    };
    // a value's place in a tile (TMA: rows of 64 or 32 values, 16-byte pieces in the order that the swizzle gives them)
    auto at_ = [&](const T* tile, int row, int col) {
        if constexpr (!TMA) return tile + row * LD + col;
        else return tile + col / C::BW * (KT * C::BW) + row * C::BW + ((col % C::BW / 8 ^ (C::BW == 64 ? row & 7 : (row >> 1) & 3)) << 3) + (col & 7);
    };
    const float sl2 = p.scale * 1.4426950408889634f;                        // scores in units of log2

    if constexpr (C::KEYS) {
        constexpr int NT = BM / 8;
        const int kw = warp * 16, r = lane >> 2, c2 = (lane & 3) * 2;       // this warp's keys; this lane's key (and + 8) and columns (and + 1) of a product
        int lm[NT][2];
        uint32_t qf[HD / 16][NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            lm[n][0] = lim(n * 8 + c2);
            lm[n][1] = lim(n * 8 + c2 + 1);
#pragma unroll
            for (int k = 0; k < HD / 32; k++) {
                uint32_t b[4];
                ldmatrix_x4(b, Qs + (n * 8 + (lane & 7)) * LD + k * 32 + (lane >> 3) * 8);
                qf[2 * k][n][0] = b[0]; qf[2 * k][n][1] = b[1];
                qf[2 * k + 1][n][0] = b[2]; qf[2 * k + 1][n][1] = b[3];
            }
        }
        float o[HD / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int d = 0; d < HD / 16; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[d][n][e] = 0.f;
        }
        for (int t = 0; t < n_tiles; t++) {
            begin(t);
            const T* Kt = ring + st * 2 * TILE;
            const T* Vt = Kt + TILE;
            const int key0 = base + t * KT + kw;
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                uint32_t a[4];
                ldmatrix_x4(a, at_(Kt, kw + (lane & 15), k * 16 + (lane >> 4) * 8));
#pragma unroll
                for (int n = 0; n < NT; n++) mma_bf16(s[n], a[0], a[1], a[2], a[3], qf[k][n][0], qf[k][n][1]);
            }
            const bool masked = key0 + 16 > lim_min || key0 < k0;
            uint32_t b[NT][2];                                              // the weights, columns by keys
            bool grown = false;
            float f[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (masked)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = key0 + r + (e >> 1) * 8;
                        if (key >= lm[n][e & 1] || key < k0) s[n][e] = -INFINITY;
                    }
                float u[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float top = fmaxf(s[n][e], s[n][2 + e]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float now = fmaxf(m[n][e], top * sl2);
                    u[e] = now == -INFINITY ? 0.f : now;
                    grown |= now > m[n][e];
                    f[n][e] = sh_exp2(m[n][e] - u[e]);                      // (m = -inf: 0)
                    m[n][e] = now;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] = sh_exp2(fmaf(s[n][e], sl2, -u[e & 1]));
                l[n][0] = l[n][0] * f[n][0] + (s[n][0] + s[n][2]);
                l[n][1] = l[n][1] * f[n][1] + (s[n][1] + s[n][3]);
                b[n][0] = sh_transposed(pack_bf16(s[n][0], s[n][1]));
                b[n][1] = sh_transposed(pack_bf16(s[n][2], s[n][3]));
            }
            if (__any_sync(0xffffffffu, grown))
#pragma unroll
                for (int d = 0; d < HD / 16; d++)
#pragma unroll
                    for (int n = 0; n < NT; n++) { o[d][n][0] *= f[n][0]; o[d][n][1] *= f[n][1]; o[d][n][2] *= f[n][0]; o[d][n][3] *= f[n][1]; }
            uint32_t keep[2] = {0xffffffffu, 0xffffffffu};                  // keys that are there: c2 and the next, and eight further
            if (masked)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int key = key0 + h * 8 + c2;
                    if (key < k0 || key >= k1) keep[h] &= 0xffff0000u;
                    if (key + 1 < k0 || key + 1 >= k1) keep[h] &= 0x0000ffffu;
                }
            bool odd = false;
#pragma unroll
            for (int d = 0; d < HD / 16; d++) {
                uint32_t a[4];
                ldmatrix_x4_trans(a, at_(Vt, kw + (lane & 7) + ((lane >> 4) << 3), d * 16 + ((lane >> 3) & 1) * 8));
                if (masked)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        a[e] &= keep[e >> 1];
                        if constexpr (OWN) {
                            const uint32_t g_ = sh_finite2(a[e]);
                            odd |= g_ != a[e];
                            a[e] = g_;
                        }
                    }
#pragma unroll
                for (int n = 0; n < NT; n++) mma_bf16(o[d][n], a[0], a[1], a[2], a[3], b[n][0], b[n][1]);
            }
            if (OWN && masked && __any_sync(0xffffffffu, odd)) {
                // values that are not finite, key by key, to the columns that read them
                float* P = reinterpret_cast<float*>(Pbuf) + warp * 256;     // [column][16 keys]
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) P[(n * 8 + c2 + (e & 1)) * 16 + r + (e >> 1) * 8] = s[n][e];
                __syncwarp();
#pragma unroll 1
                for (int i = max(0, k0 - key0); i < 16; i++)
#pragma unroll
                    for (int d = 0; d < HD / 16; d++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float x = to_f32(*at_(Vt, kw + i, d * 16 + h * 8 + r));
                            if (sh_odd(x))
#pragma unroll
                                for (int n = 0; n < NT; n++)
#pragma unroll
                                    for (int e = 0; e < 2; e++)
                                        if (key0 + i < lm[n][e]) o[d][n][2 * h + e] += P[(n * 8 + c2 + e) * 16 + i] * x;
                        }
                __syncwarp();
            }
            end();
        }
        finish();
        constexpr int LDO = C::LDO;
        float* O = reinterpret_cast<float*>(sm.ring);
        float* Ow = O + (1 + warp) * BM * LDO;                              // [0]: the joined one
        float* mw = ml + (1 + warp) * BM * 2;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c = n * 8 + c2 + e;
                l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
                l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
                l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
                if (c >= live) continue;
                if (!r) { mw[2 * c] = m[n][e]; mw[2 * c + 1] = l[n][e]; }
#pragma unroll
                for (int d = 0; d < HD / 16; d++) { Ow[c * LDO + d * 16 + r] = o[d][n][e]; Ow[c * LDO + d * 16 + 8 + r] = o[d][n][2 + e]; }
            }
        sh_sync_workers();
        for (int i = tid; i < live * (HD / 4); i += SH_WORKERS) {
            const int c = i / (HD / 4), d = i % (HD / 4) * 4;
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 1; w < 5; w++) M = fmaxf(M, ml[(w * BM + c) * 2]);
            const float u = M == -INFINITY ? 0.f : M;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 1; w < 5; w++) {
                const float g_ = sh_exp2(ml[(w * BM + c) * 2] - u);
                const float4 x = *reinterpret_cast<const float4*>(O + (w * BM + c) * LDO + d);
                L += g_ * ml[(w * BM + c) * 2 + 1];
                acc.x += g_ * x.x; acc.y += g_ * x.y; acc.z += g_ * x.z; acc.w += g_ * x.w;
            }
            *reinterpret_cast<float4*>(O + c * LDO + d) = acc;
            if (!d) { ml[2 * c] = M; ml[2 * c + 1] = L; }
        }
    } else if constexpr (C::MMA) {
        constexpr int NK = KT;
        constexpr bool QREG = HD <= 128;
        const int c0 = warp * 16;
        const int r0 = c0 + (lane >> 2), r1 = r0 + 8;
        const int lim0 = lim(r0), lim1 = lim(r1);
        uint32_t qf[QREG ? HD / 16 : 1][4];
        const T* qrow = Qs + (c0 + (lane & 15)) * LD + (lane >> 4) * 8;
        if constexpr (QREG) {
#pragma unroll
            for (int k = 0; k < HD / 16; k++) ldmatrix_x4(qf[k], qrow + k * 16);
        }
        float o[HD / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 8; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[d][e] = 0.f;
        for (int t = 0; t < n_tiles; t++) {
            begin(t);
            const T* Kt = ring + st * 2 * TILE;
            const T* Vt = Kt + TILE;
            const int key0 = base + t * KT;
            float s[NK / 8][4];
#pragma unroll
            for (int j = 0; j < NK / 8; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[j][e] = 0.f;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                uint32_t a[4];
                if constexpr (QREG) {
#pragma unroll
                    for (int e = 0; e < 4; e++) a[e] = qf[k][e];
                } else ldmatrix_x4(a, qrow + k * 16);
#pragma unroll
                for (int j = 0; j < NK / 16; j++) {
                    uint32_t b[4];
                    ldmatrix_x4(b, at_(Kt, j * 16 + (lane & 7) + ((lane >> 4) << 3), k * 16 + ((lane >> 3) & 1) * 8));
                    mma_bf16(s[2 * j], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma_bf16(s[2 * j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
            }
            const bool masked = key0 + NK > lim_min || key0 < k0;
            unsigned odd = 0;                                               // stretches of 16 keys that have values that are not finite
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < NK / 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if (masked) {
                        const int key = key0 + j * 8 + (lane & 3) * 2 + e;
                        if (key >= lim0 || key < k0) s[j][e] = -INFINITY;
                        if (key >= lim1 || key < k0) s[j][2 + e] = -INFINITY;
                    }
                    t0 = fmaxf(t0, s[j][e]);
                    t1 = fmaxf(t1, s[j][2 + e]);
                }
            t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1)); t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
            t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1)); t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
            const float n0 = fmaxf(m0, t0 * sl2), n1 = fmaxf(m1, t1 * sl2);
            const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;
            if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
                const float f0 = sh_exp2(m0 - u0), f1 = sh_exp2(m1 - u1);   // (m = -inf: 0)
                l0 *= f0; l1 *= f1;
#pragma unroll
                for (int d = 0; d < HD / 8; d++) { o[d][0] *= f0; o[d][1] *= f0; o[d][2] *= f1; o[d][3] *= f1; }
                m0 = n0; m1 = n1;
            }
#pragma unroll
            for (int j = 0; j < NK / 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    s[j][e] = sh_exp2(fmaf(s[j][e], sl2, -u0));
                    s[j][2 + e] = sh_exp2(fmaf(s[j][2 + e], sl2, -u1));
                    l0 += s[j][e];
                    l1 += s[j][2 + e];
                }
#pragma unroll
            for (int j = 0; j < NK / 16; j++) {
                uint32_t a[4] = {pack_bf16(s[2 * j][0], s[2 * j][1]), pack_bf16(s[2 * j][2], s[2 * j][3]), pack_bf16(s[2 * j + 1][0], s[2 * j + 1][1]),
                                 pack_bf16(s[2 * j + 1][2], s[2 * j + 1][3])};
                uint32_t keep[2] = {0xffffffffu, 0xffffffffu};              // keys that are there: 2 (lane % 4) and the next, and eight further
                if (masked)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int key = key0 + j * 16 + h * 8 + (lane & 3) * 2;
                        if (key < k0 || key >= k1) keep[h] &= 0xffff0000u;
                        if (key + 1 < k0 || key + 1 >= k1) keep[h] &= 0x0000ffffu;
                    }
#pragma unroll
                for (int d = 0; d < HD / 16; d++) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, at_(Vt, j * 16 + (lane & 15), d * 16 + (lane >> 4) * 8));
                    if (masked)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            b[e] &= keep[e & 1];
                            if constexpr (OWN) {
                                const uint32_t f = sh_finite2(b[e]);
                                odd |= (unsigned)(f != b[e]) << j;
                                b[e] = f;
                            }
                        }
                    mma_bf16(o[2 * d], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma_bf16(o[2 * d + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
            }
            if constexpr (OWN) {
                // values that are not finite, key by key, to the columns that read them
                odd = __reduce_or_sync(0xffffffffu, odd);
                float* P = reinterpret_cast<float*>(Pbuf) + warp * 256;
#pragma unroll 1
                for (int j = 0; odd >> j; j++) {
                    if (!((odd >> j) & 1)) continue;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float w = s[h][e];
#pragma unroll
                            for (int i = 1; i < NK / 16; i++) w = i == j ? s[2 * i + h][e] : w;
                            P[((lane >> 2) + (e >> 1) * 8) * 16 + h * 8 + (lane & 3) * 2 + (e & 1)] = w;
                        }
                    __syncwarp();
#pragma unroll 1
                    for (int i = 0; i < 16; i++) {
                        const int key = key0 + j * 16 + i;
                        const float p0 = P[(lane >> 2) * 16 + i], p1 = P[((lane >> 2) + 8) * 16 + i];
#pragma unroll
                        for (int d = 0; d < HD / 8; d++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                const float x = to_f32(*at_(Vt, j * 16 + i, d * 8 + (lane & 3) * 2 + e));
                                if (sh_odd(x) && key >= k0) {
                                    if (key < lim0) o[d][e] += p0 * x;
                                    if (key < lim1) o[d][2 + e] += p1 * x;
                                }
                            }
                    }
                    __syncwarp();
                }
            }
            end();
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        finish();
        float* O = reinterpret_cast<float*>(sm.ring);
        constexpr int LDO = C::LDO;
#pragma unroll
        for (int d = 0; d < HD / 8; d++) {
            *reinterpret_cast<float2*>(O + r0 * LDO + d * 8 + (lane & 3) * 2) = make_float2(o[d][0], o[d][1]);
            *reinterpret_cast<float2*>(O + r1 * LDO + d * 8 + (lane & 3) * 2) = make_float2(o[d][2], o[d][3]);
        }
        if (!(lane & 3)) { ml[2 * r0] = m0; ml[2 * r0 + 1] = l0; ml[2 * r1] = m1; ml[2 * r1 + 1] = l1; }
    } else {
        constexpr int MR = C::MR, KJ = KT / 16, DJ = HD / 32;
        const int tr = tid >> 4, tc = tid & 15;
        float* P = reinterpret_cast<float*>(Pbuf);
        float2 o[MR][DJ];
        float m[MR], l[MR];
        int lm[MR];
#pragma unroll
        for (int r = 0; r < MR; r++) {
            m[r] = -INFINITY; l[r] = 0.f; lm[r] = lim(tr * MR + r);
#pragma unroll
            for (int d = 0; d < DJ; d++) o[r][d] = make_float2(0.f, 0.f);
        }
        for (int t = 0; t < n_tiles; t++) {
            begin(t);
            const float* Kt = reinterpret_cast<const float*>(ring) + (t % ST) * 2 * TILE;
            const float* Vt = Kt + TILE;
            const float* Qf = reinterpret_cast<const float*>(Qs) + tr * MR * LD;
            const int key0 = base + t * KT;
            float2 s2[MR][KJ];                                              // even and odd places of the heads
#pragma unroll
            for (int r = 0; r < MR; r++)
#pragma unroll
                for (int j = 0; j < KJ; j++) s2[r][j] = make_float2(0.f, 0.f);
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                float4 k[KJ];
#pragma unroll
                for (int j = 0; j < KJ; j++) k[j] = *reinterpret_cast<const float4*>(Kt + (tc + 16 * j) * LD + d);
#pragma unroll
                for (int r = 0; r < MR; r++) {
                    const float4 q = *reinterpret_cast<const float4*>(Qf + r * LD + d);
#pragma unroll
                    for (int j = 0; j < KJ; j++)
                        s2[r][j] = sh_fma2(make_float2(q.x, q.y), make_float2(k[j].x, k[j].y), sh_fma2(make_float2(q.z, q.w), make_float2(k[j].z, k[j].w), s2[r][j]));
                }
            }
            const bool masked = key0 + KT > lim_min || key0 < k0;
#pragma unroll
            for (int r = 0; r < MR; r++) {
                float top = -INFINITY, s[KJ];
#pragma unroll
                for (int j = 0; j < KJ; j++) {
                    s[j] = s2[r][j].x + s2[r][j].y;
                    if (masked && (key0 + tc + 16 * j >= lm[r] || key0 + tc + 16 * j < k0)) s[j] = -INFINITY;
                    top = fmaxf(top, s[j]);
                }
#pragma unroll
                for (int x = 8; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                const float n = fmaxf(m[r], top * sl2), u = n == -INFINITY ? 0.f : n;
                const float f = exp2f(m[r] - u);
                m[r] = n;
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < DJ; d++) { o[r][d].x *= f; o[r][d].y *= f; }
#pragma unroll
                for (int j = 0; j < KJ; j++) {
                    const float e = exp2f(fmaf(s[j], sl2, -u));
                    l[r] += e;
                    P[(tr * MR + r) * (KT + 4) + tc + 16 * j] = e;
                }
            }
            __syncwarp();                                                   // (a column's weights are made and read by one half of a warp)
            if (!masked) {
#pragma unroll 2
                for (int j = 0; j < KT; j += 4) {
                    float2 v[4][DJ];
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int d = 0; d < DJ; d++) v[i][d] = *reinterpret_cast<const float2*>(Vt + (j + i) * LD + d * 32 + tc * 2);
#pragma unroll
                    for (int r = 0; r < MR; r++) {
                        const float4 w = *reinterpret_cast<const float4*>(P + (tr * MR + r) * (KT + 4) + j);
                        const float2 wx = make_float2(w.x, w.x), wy = make_float2(w.y, w.y), wz = make_float2(w.z, w.z), ww = make_float2(w.w, w.w);
#pragma unroll
                        for (int d = 0; d < DJ; d++) o[r][d] = sh_fma2(wx, v[0][d], sh_fma2(wy, v[1][d], sh_fma2(wz, v[2][d], sh_fma2(ww, v[3][d], o[r][d]))));
                    }
                }
            } else {
#pragma unroll 1
                for (int j = max(0, k0 - key0); j < KT; j++)
#pragma unroll
                    for (int r = 0; r < MR; r++)
                        if (key0 + j < lm[r]) {
                            const float w = P[(tr * MR + r) * (KT + 4) + j];
#pragma unroll
                            for (int d = 0; d < DJ; d++) o[r][d] = sh_fma2(make_float2(w, w), *reinterpret_cast<const float2*>(Vt + j * LD + d * 32 + tc * 2), o[r][d]);
                        }
            }
            __syncwarp();
        }
        finish();
        float* O = reinterpret_cast<float*>(sm.ring);
#pragma unroll
        for (int r = 0; r < MR; r++) {
            const int c = tr * MR + r;
#pragma unroll
            for (int d = 0; d < DJ; d++) *reinterpret_cast<float2*>(O + c * C::LDO + d * 32 + tc * 2) = o[r][d];
#pragma unroll
            for (int x = 8; x; x >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
            if (!tc) { ml[2 * c] = m[r]; ml[2 * c + 1] = l[r]; }
        }
    }
    return ok;
}

// the queries of BM columns from column c0 of the rows row0 .., by the four warps: zeros behind the last
template <typename T, int HD, int BM, bool TMA>
__device__ __forceinline__ void sh_queries(const ShArgs& p, T* Qs, int row0, int n_cols, int c0, int g, int R) {
    typedef Sh<T, HD, BM, TMA> C;
    const T* q = (const T*)p.q + (size_t)row0 * p.ldq + (size_t)g * R * HD;
    for (int i = threadIdx.x; i < BM * C::CH; i += SH_WORKERS) {
        const int c = i / C::CH, e = i % C::CH * C::E, col = c0 + c;
        const T* src = q + (size_t)(col / R) * p.ldq + (col % R) * HD + e;
        T* dst = Qs + c * C::LD + e;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (col < n_cols) {
            if (p.q_vec) x = *reinterpret_cast<const uint4*>(src);
            else {
                T* y = reinterpret_cast<T*>(&x);
#pragma unroll
                for (int j = 0; j < C::E; j++) y[j] = src[j];
            }
        }
        *reinterpret_cast<uint4*>(dst) = x;
    }
    sh_sync_workers();
}
template <typename T, int HD, int BM, bool TMA>
__device__ __forceinline__ void sh_init(const ShMem<T, HD, BM, TMA>& sm) {
    if (TMA && threadIdx.x == 0) {
        for (int i = 0; i < Sh<T, HD, BM, TMA>::ST; i++) { kp_mbar_init(&sm.full[i], 1); kp_mbar_init(&sm.empty[i], 4); }
        kp_mbar_init_fence();
    }
}
// queries, loads and the tile by the warps whose work they are; then everyone has the output
template <typename T, int HD, int BM, bool TMA, bool OWN, typename Lim>
__device__ __forceinline__ void sh_work(const ShArgs& p, const CUtensorMap& tm, const ShMem<T, HD, BM, TMA>& sm, const int* bt, int g, int R, int row0, int n_cols, int c0,
                                        int k0, int k1, int lim_min, Lim lim) {
    bool ok = true;
    if (TMA && threadIdx.x >= SH_WORKERS) {
        if constexpr (TMA) ok = sh_load(p, tm, sm, bt, g, k0, k1);
    } else {
        sh_queries<T, HD, BM, TMA>(p, sm.Qs, row0, n_cols, c0, g, R);
        ok = sh_tile<T, HD, BM, TMA, OWN>(p, sm, bt, g, min(BM, n_cols - c0), k0, k1, lim_min, lim);
    }
    if (__builtin_expect(!ok, 0)) {
        atomicExch(&g_shared_status, 1);
        kp_linger_after_failure();
    }
    __syncthreads();
}

// ---- first launch: a chunk of a group's prefix for a tile of its columns.  A tile of 64 keys takes a CTA of 64 columns 0.75, 1.5 and 1.8 us with heads of 64,
// 128 and 256, one of 8 columns 0.3, 0.4 and 0.5: a chain of loads from shared memory, products and exponentials.  What only rows that stand among the
// keys need (values that are not finite) is left out: with it the wide ones fetched instructions for most of their time (4.9 us with heads of 256).
template <typename T, int HD, int BM, bool TMA>
__global__ void __launch_bounds__(Sh<T, HD, BM, TMA>::THREADS, Sh<T, HD, BM, TMA>::CTAS)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ ShArgs p) {
    kp_pdl_begin();
    extern __shared__ __align__(16) unsigned char smem[];
    const ShMem<T, HD, BM, TMA> sm(smem, p.main);
    const ShPlace at(p);
    const int chunk = blockIdx.x, g = at.g, group = at.i / p.tiles, c0 = at.i % p.tiles * BM, R = p.H / p.G;
    if (group >= p.n_groups) return;
    const int s0 = max(0, min(p.group_seqs[group], p.n_seq)), s1 = max(s0, min(p.group_seqs[group + 1], p.n_seq));
    const int P = sh_prefix(p, group), k0 = chunk * p.chunk, k1 = min(P, k0 + p.chunk);
    if (s0 == s1 || k0 >= k1) return;
    const int row0 = sh_row(p, s0), n_cols = max(0, sh_row(p, s1) - row0) * R;
    if (c0 >= n_cols) return;
    sh_init(sm);
    __syncthreads();
    sh_work<T, HD, BM, TMA, false>(p, tm, sm, p.table + (size_t)s0 * p.width, g, R, row0, n_cols, c0, k0, k1, k1, [&](int) { return k1; });
    const float* O = reinterpret_cast<const float*>(sm.ring);
    for (int i = threadIdx.x; i < BM * HD / 4; i += Sh<T, HD, BM, TMA>::THREADS) {
        const int c = i / (HD / 4), d = i % (HD / 4) * 4, col = c0 + c;
        if (col >= n_cols) break;
        const size_t to = ((size_t)(row0 + col / R) * p.H + g * R + col % R) * p.n_chunks + chunk;
        *reinterpret_cast<float4*>(p.part_o + to * HD + d) = *reinterpret_cast<const float4*>(O + c * Sh<T, HD, BM, TMA>::LDO + d);
        if (!d) *reinterpret_cast<float2*>(p.part_ml + to * 2) = make_float2(sm.ml[2 * c], sm.ml[2 * c + 1]);
    }
}

// ---- second launch: a sequence's own keys, shared out over a cluster, and the join.  Bound by its loads where there are many keys (256 sequences with 100 to
// 700 of them, 8 kv heads of 128: 74 us, 5.6 TB/s), by the latencies of one CTA where there are few (64 with up to 500, heads of 64: 10 us behind the prefix).
template <typename T, int HD, int BM, bool TMA>
__global__ void __launch_bounds__(Sh<T, HD, BM, TMA>::THREADS, Sh<T, HD, BM, TMA>::CTAS)
shared_own_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ ShArgs p) {
    // With a first launch its inputs are ready: all CTAs of that one have waited for the kernels before it by the time that this one may start.
    KP_TRACE_MARK(0);
    if (p.alone) pdl_wait();
    typedef Sh<T, HD, BM, TMA> C;
    constexpr int KT = C::KT, THREADS = C::THREADS;
    extern __shared__ __align__(16) unsigned char smem[];
    const ShMem<T, HD, BM, TMA> sm(smem, p.main);
    float* ml = sm.ml;
    float* wts = sm.wts;
    __shared__ int s_group, s_prefix, s_chunk;
    cg::cluster_group cluster = cg::this_cluster();
    const int n_cl = gridDim.x, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const ShPlace at(p);
    const int g = at.g, seq = at.i / p.tiles, c0 = at.i % p.tiles * BM, R = p.H / p.G;
    if (seq >= p.n_seq) return;
    // (all of these loads under way together)
    const bool look = tid < p.n_groups;
    int from = look ? p.group_seqs[tid] : 0, to = look ? p.group_seqs[tid + 1] : 0, len = look ? sh_prefix(p, tid) : 0;
    const int row0 = sh_row(p, seq), n_cols = max(0, sh_row(p, seq + 1) - row0) * R, pos0 = max(-p.n, min(p.seg_pos[seq], p.width * p.ps));
    // Clusters without rows make room for those that have some.  The first place's stay: they wait for the first launch as all with rows do, so that this one
    // ends behind it, which what comes next relies on.
    const bool work = c0 < n_cols;                           // (the same for all CTAs of a cluster)
    if (!work && at.i) return;
    sh_init(sm);
    if (tid == 0) s_group = -1;
    __syncthreads();
    for (int i = tid;;) {
        if (from <= seq && seq < to) { s_group = i; s_prefix = len; }
        if ((i += THREADS) >= p.n_groups) break;
        from = p.group_seqs[i]; to = p.group_seqs[i + 1]; len = sh_prefix(p, i);
    }
    __syncthreads();
    const int group = s_group, P = group >= 0 ? s_prefix : 0;
    if (work) {
        const int last = pos0 + (min(n_cols, c0 + BM) - 1) / R;                     // position of the tile's last row
        const int end = max(P, (int)min((long long)last + 1, (long long)p.width * p.ps));
        const int t0 = P / KT, per = ((end + KT - 1) / KT - t0 + n_cl - 1) / n_cl;  // whole tiles of keys, and a CTA's
        const int k0 = min(end, max(P, (t0 + part * per) * KT)), k1 = min(end, (t0 + (part + 1) * per) * KT);
        sh_work<T, HD, BM, TMA, true>(p, tm, sm, p.table + (size_t)seq * p.width, g, R, row0, n_cols, c0, k0, k1, min(k1, pos0 + c0 / R + 1),
                [&](int c) { return min(k1, pos0 + (c0 + c) / R + 1); });
    }
    if (p.budget) {
        if (warp == 0) { const int c = sh_chunk(p, lane); if (lane == 0) s_chunk = c; }
        __syncthreads();
    }
    KP_TRACE_MARK(1);
    if (!p.alone) pdl_wait();                                // the prefix's parts are there
    pdl_launch_dependents();
    if (!work) return;
    if (n_cl > 1) cluster.sync();
    const int chunk = p.budget ? s_chunk : p.chunk, n_pre = group >= 0 ? (P + chunk - 1) / chunk : 0, n_parts = n_cl + n_pre, ld_w = n_cl + p.n_chunks;
    const float* O = reinterpret_cast<const float*>(sm.ring);
    // the parts' weights: 2^(m - M) / sum 2^(m - M) l.  The cluster's CTAs share the columns.
    for (int c = part + warp * n_cl; c < BM && c0 + c < n_cols; c += n_cl * (THREADS / 32)) {
        const int col = c0 + c;
        const float* pre = p.part_ml + ((size_t)(row0 + col / R) * p.H + g * R + col % R) * p.n_chunks * 2;
        float m[3], l[3], M = -INFINITY;
#pragma unroll
        for (int i = 0; i < 3; i++) {
            const int x = lane + 32 * i;
            m[i] = -INFINITY; l[i] = 0.f;
            if (x < n_parts) {
                const float2 v = x < n_cl ? *reinterpret_cast<const float2*>((n_cl > 1 ? cluster.map_shared_rank(ml, x) : ml) + 2 * c)
                                          : __ldcg(reinterpret_cast<const float2*>(pre + 2 * (x - n_cl)));
                m[i] = v.x; l[i] = v.y;
            }
            M = fmaxf(M, m[i]);
        }
        M = warp_max(M);
        const float u = M == -INFINITY ? 0.f : M;
        float L = 0.f;
#pragma unroll
        for (int i = 0; i < 3; i++) { m[i] = exp2f(m[i] - u); L += m[i] * l[i]; }
        L = warp_sum(L);
        const float inv = L == 0.f ? 0.f : 1.f / L;          // (no key: zeros)
#pragma unroll
        for (int i = 0; i < 3; i++) if (lane + 32 * i < n_parts) wts[c * ld_w + lane + 32 * i] = m[i] * inv;
    }
    __syncthreads();
    constexpr int D4 = HD / 4;
    const int mine = (min(BM, n_cols - c0) - part + n_cl - 1) / n_cl;               // columns part, part + n_cl, ...
    for (int i = tid; i < mine * D4; i += THREADS) {
        const int c = part + i / D4 * n_cl, d = i % D4 * 4, col = c0 + c;
        const size_t row = row0 + col / R;
        const float* w = wts + c * ld_w;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4 x) { a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w; };
        for (int x = 0; x < n_cl; x++) add(w[x], *reinterpret_cast<const float4*>((n_cl > 1 ? cluster.map_shared_rank(O, x) : O) + c * C::LDO + d));
        const float* pre = p.part_o + (row * p.H + g * R + col % R) * p.n_chunks * HD + d;
#pragma unroll 4
        for (int x = 0; x < n_pre; x++) add(w[n_cl + x], __ldcg(reinterpret_cast<const float4*>(pre + (size_t)x * HD)));
        T* dst = (T*)p.out + row * p.ldo + (size_t)(g * R + col % R) * HD + d;
        if constexpr (sizeof(T) == 2) {
            const uint2 y = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
            if (p.out_vec) *reinterpret_cast<uint2*>(dst) = y;
            else {
                const T* v = reinterpret_cast<const T*>(&y);
#pragma unroll
                for (int e = 0; e < 4; e++) dst[e] = v[e];
            }
        } else {
            if (p.out_vec) *reinterpret_cast<float4*>(dst) = a;
            else { dst[0] = a.x; dst[1] = a.y; dst[2] = a.z; dst[3] = a.w; }
        }
    }
    if (n_cl > 1) cluster.sync();                            // (its shared memory is read until then)
}

template <int HD, int BM, bool TMA>
static int sh_prefix_launch(const CUtensorMap& tm, ShArgs a, cudaStream_t st) {
    typedef Sh<ShT, HD, BM, TMA> C;
    a.stages = C::ST;
    a.main = C::MAIN;
    a.box = min(a.ps, C::KT);
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(shared_prefix_kernel<ShT, HD, BM, TMA>, C::SMEM, ready, true);
    if (e) return e;
    cudaError_t c = kp_launch_pdl(shared_prefix_kernel<ShT, HD, BM, TMA>, sh_grid(a.n_chunks, a.G, a.n_groups * a.tiles), dim3(C::THREADS), C::SMEM, st, tm, a);
    return c ? (int)c : kp_launch_status();
}
template <int HD, int BM, bool TMA>
static int sh_own_launch(const CUtensorMap& tm, ShArgs a, int ctas, int own_keys, cudaStream_t st) {
    typedef Sh<ShT, HD, BM, TMA> C;
    // No more stages than a CTA has tiles, so that more CTAs fit an SM: 1424 tiles of columns with 19 to 34 own keys, heads of 256, 102 us with two
    // stages, 77 with one.
    a.stages = TMA ? max(1, min(C::ST, (own_keys / ctas + C::KT - 1) / C::KT)) : C::ST;
    a.main = max(a.stages * C::PAIR, C::O_BYTES);
    a.box = min(a.ps, SH_OWN_BOX);
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(shared_own_kernel<ShT, HD, BM, TMA>, C::MOST, ready, true);
    if (e) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = sh_grid(ctas, a.G, a.n_seq * a.tiles);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = C::SMEM - C::MAIN + a.main + (size_t)BM * (ctas + a.n_chunks) * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t c = cudaLaunchKernelEx(&cfg, shared_own_kernel<ShT, HD, BM, TMA>, tm, a);
    return c ? (int)c : kp_launch_status();
}
template <int HD, bool TMA>
static int sh_run_tma(const CUtensorMap& tm, const CUtensorMap& own, ShArgs& a, int tile, int group_tiles, int own_tile, int own_tiles, int own_ctas, int own_keys, int with_prefix, cudaStream_t st) {
    if (with_prefix) {
        a.tiles = group_tiles;
        int e;
        switch (tile) {
            case 8: e = sh_prefix_launch<HD, 8, TMA>(tm, a, st); break;
            case 16: e = sh_prefix_launch<HD, 16, TMA>(tm, a, st); break;
            case 32: e = SH_32(sh_prefix_launch, tm, a, st); break;
            default: e = sh_prefix_launch<HD, 64, TMA>(tm, a, st);
        }
        if (e) return e;
    }
    a.tiles = own_tiles;
    switch (own_tile) {
        case 8: return sh_own_launch<HD, 8, TMA>(own, a, own_ctas, own_keys, st);
        case 16: return sh_own_launch<HD, 16, TMA>(own, a, own_ctas, own_keys, st);
        case 32: return SH_32(sh_own_launch, own, a, own_ctas, own_keys, st);
        default: return sh_own_launch<HD, 64, TMA>(own, a, own_ctas, own_keys, st);
    }
}
// the cache as rows of a key's (or value's) hd numbers of a head, in boxes of bw of them (32 or 64: swizzled over 64 or 128 bytes) by the keys of a page, `most` at
// most
static int sh_make_map(CUtensorMap* map, const ShArgs& a, int hd, int bw, int most) {
    KpEncodeTiledFn fn = kp_encode_tiled_fn();
    if (!fn) return KP_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)a.n_pages * 2 * a.G * a.ps}, strides[1] = {(cuuint64_t)hd * 2};
    cuuint32_t box[2] = {(cuuint32_t)bw, (cuuint32_t)(a.ps < most ? a.ps : most)}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.cache), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              bw == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0 : KP_ERR_UNSUPPORTED;
}
template <int HD>
static int sh_run(ShArgs& a, int tile, int group_tiles, int own_tile, int own_tiles, int own_ctas, int own_keys, int with_prefix, cudaStream_t st) {
    alignas(64) CUtensorMap tm = {};
    if constexpr (sizeof(ShT) == 2) {
        typedef Sh<ShT, HD, 16, true> C;
        if (a.ps % 8 == 0 && (a.ps % C::KT == 0 || C::KT % a.ps == 0) && a.n_pages * 2 * a.G * a.ps < 2147483647LL) {
            alignas(64) CUtensorMap own;
            int e = with_prefix ? sh_make_map(&tm, a, HD, C::BW, C::KT) : 0;
            if (!e) e = sh_make_map(&own, a, HD, C::BW, SH_OWN_BOX);
            if (e) return e;
            return sh_run_tma<HD, true>(tm, own, a, tile, group_tiles, own_tile, own_tiles, own_ctas, own_keys, with_prefix, st);
        }
    }
    return sh_run_tma<HD, false>(tm, tm, a, tile, group_tiles, own_tile, own_tiles, own_ctas, own_keys, with_prefix, st);
}

// The first launch in its tcgen05 form (kp_attention_shared_prefix_tc)
typedef int (*ShPrefixTc)(const void*, long long, const void*, long long, const int*, int, const int*, const int*, const int*, int, int, int, float*, float*, int, int,
                          float, int, int, int, int, int, int, int, int, void*);

// tile, own_tile: columns of a tile, 8, 16, 32 (float32) or 64, of the first and of the second launch; n_chunks = 0: there is no prefix; own_keys: a
// sequence's own keys, about.  prefix_tc: the first
// launch's tcgen05 form, or null; mode, budget: its arguments.
extern "C" int SH_ENTRY(const void* q, long long ldq, const void* cache, long long n_pages, const int* table, int width, const int* cu_rows, const int* seg_pos,
                        const int* group_seqs, const int* prefix_len, int n, int n_seq, int n_groups, void* out, long long ldo, float* part_o,
                        float* part_ml, int n_chunks, int chunk, float scale, int ps, int H, int G, int hd, int max_prefix, int tile, int group_tiles,
                        int own_tile, int own_tiles, int own_ctas, int own_keys, void* prefix_tc, int mode, int budget, void* stream) {
    if (n <= 0 || n_seq <= 0) return 0;
    const int elt = sizeof(ShT), with_prefix = n_chunks > 0 && !prefix_tc, prefix_done = n_chunks > 0 && prefix_tc;
    if (G < 1 || H < 1 || H % G || ps < 1 || width < 1 || (long long)width * ps > (1 << 30) || n_pages < 1 || n_groups < 0 || chunk < 1 ||
        n_chunks < 0 || n_chunks > SH_MAX_CHUNKS || ((with_prefix || prefix_done) && (n_chunks < 1 || (long long)n_chunks * chunk < max_prefix)) ||
        (tile != 8 && tile != 16 && tile != 32 && tile != 64) || (own_tile != 8 && own_tile != 16 && own_tile != 32 && own_tile != 64) || group_tiles < 1 || own_tiles < 1 || own_ctas < 1 || own_ctas > SH_MAX_CLUSTER || own_keys < 0 ||
        !sh_grid_ok(n_groups, group_tiles, G) || !sh_grid_ok(n_seq, own_tiles, G) || ((uintptr_t)cache & 15) || ((uintptr_t)q & (elt - 1)) ||
        ((uintptr_t)out & (elt - 1)) || !(scale > 0.f) || (with_prefix && chunk % 64) || budget < 0 || (budget && (n_groups > 32 || (long long)n_groups * group_tiles * G > budget || chunk % 128)))
        return KP_ERR_BAD_ARG;
    int ps_log2 = -1;
    for (int i = 0; i < 31; i++) if (ps == 1 << i) ps_log2 = i;
    ShArgs a = {q, ldq, ((uintptr_t)q & 15) == 0 && ldq * elt % 16 == 0, cache, n_pages, table, width, cu_rows, seg_pos, group_seqs, prefix_len, n, n_seq, n_groups,
                out, ldo, ((uintptr_t)out & 15) == 0 && ldo * elt % 16 == 0, part_o, part_ml, n_chunks, chunk, prefix_done ? budget : 0, group_tiles, 1, !(with_prefix || prefix_done), scale, ps, ps_log2,
                H, G, with_prefix || prefix_done ? max_prefix : 0, 0, 0, 0};
    const cudaStream_t st = (cudaStream_t)stream;
    if (prefix_done) {
        const int e = ((ShPrefixTc)prefix_tc)(q, ldq, cache, n_pages, table, width, cu_rows, group_seqs, prefix_len, n, n_seq, n_groups, part_o, part_ml, n_chunks, chunk,
                                              scale, ps, H, G, hd, max_prefix, group_tiles, mode, budget, stream);
        if (e) return e;
    }
#define SH_HD(D) case D: return sh_run<D>(a, tile, group_tiles, own_tile, own_tiles, own_ctas, own_keys, with_prefix, st)
    switch (hd) {
        SH_HD(32);
        SH_HD(64);
        SH_HD(96);
        SH_HD(128);
        SH_HD(192);
        SH_HD(256);
        default: return KP_ERR_UNSUPPORTED;
    }
}
