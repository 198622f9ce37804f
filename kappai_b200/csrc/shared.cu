// Attention behind a shared prefix (shared.cuh): both launches for any type, head size and page size.
//
// A CTA of four warps takes a tile of columns through a range of keys in tiles that cp.async brings to shared memory some tiles ahead, page by page.
//   bfloat16 (mma.sync): with up to 16 columns every warp takes a quarter of the tile's keys, with up to 64 every warp 16 of the columns; scores, weights and
//   output stay in registers.  Weights are rounded to bfloat16 as they enter the product with V, by up to 2^-8 of each, as the output itself is.
//   float32 (FMA): a thread has some columns times some keys of the scores, then the same columns times some values of the output; weights pass through shared
//   memory of their warp.  Nothing is rounded below 32 bits.
// A key that a column does not read has no part in it, finite or not: a tile with such a key takes the values that are not finite out of the
// product and adds them to the columns that do read them.
#include <cooperative_groups.h>

#include "mma.cuh"
#include "shared.cuh"

namespace cg = cooperative_groups;

#define SH_THREADS 128

template <typename T, int HD, int BM>
struct Sh {
    static constexpr bool MMA = sizeof(T) == 2;
    static constexpr int KT = MMA || HD <= 128 ? 64 : 32;                   // keys a tile
    static constexpr int E = 16 / sizeof(T);                                // values of 16 bytes
    static constexpr int LD = HD + E;                                       // a row in shared memory: 16 bytes more, so that rows lie in different banks
    static constexpr int TILE = KT * LD;                                    // values of K's tile, or of V's
    static constexpr int CH = HD / E, NI = (KT * CH + SH_THREADS - 1) / SH_THREADS;
    static constexpr int ST = 4 * TILE * (int)sizeof(T) * 2 <= 100 * 1024 ? 4 : (3 * TILE * (int)sizeof(T) * 2 <= 110 * 1024 ? 3 : 2);
    static constexpr int MR = BM / 8;                                       // columns of a thread (FMA)
    static constexpr int Q_BYTES = BM * LD * sizeof(T);
    static constexpr int RING = ST * 2 * TILE * (int)sizeof(T);
    static constexpr int P_BYTES = MMA ? 4 * 256 * 4 : BM * (KT + 4) * 4;   // weights (MMA: only where values are not finite)
    static constexpr int PARTS = MMA && BM == 16 ? 4 : 1;                   // outputs of the warps, then the joined one
    static constexpr int O_BYTES = (PARTS > 1 ? PARTS + 1 : 1) * BM * HD * 4;
    static constexpr int ML_BYTES = (PARTS + 1) * BM * 2 * 4;
    static constexpr int W_BYTES = BM * (SH_MAX_CLUSTER + SH_MAX_CHUNKS) * 4;
    static constexpr int MAIN = RING > O_BYTES ? RING : O_BYTES;            // the output takes the ring's place
    static constexpr size_t SMEM = Q_BYTES + MAIN + P_BYTES + ML_BYTES + W_BYTES;
    static_assert(SMEM <= KP_SMEM_MAX, "more shared memory than a CTA has");
};

// not a number, or infinite
__device__ __forceinline__ bool sh_odd(float v) { return !(fabsf(v) <= 3.402823466e38f); }
__device__ __forceinline__ uint32_t sh_finite2(uint32_t r) {                // a pair of bfloat16, zeros for what is not finite
    if ((r & 0x7f80u) == 0x7f80u) r &= 0xffff0000u;
    if ((r & 0x7f800000u) == 0x7f800000u) r &= 0x0000ffffu;
    return r;
}

// One tile of BM columns through the keys k0 .. k1 - 1 of the block-table row bt; column c reads those below lim(c).  Leaves O [BM][HD] and
// (m, l) [BM] in shared memory.
template <typename T, int HD, int BM, typename Lim>
__device__ __forceinline__ void sh_tile(const ShArgs& p, const T* Qs, unsigned char* main_, unsigned char* Pbuf, float* ml, const int* bt, int g, int k0, int k1,
                                        int lim_min, Lim lim) {
    typedef Sh<T, HD, BM> C;
    constexpr int KT = C::KT, LD = C::LD, TILE = C::TILE, CH = C::CH, NI = C::NI, ST = C::ST, E = C::E;
    T* ring = reinterpret_cast<T*>(main_);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* cache = (const T*)p.cache;
    const size_t plane = (size_t)p.G * p.ps * HD, page_stride = 2 * plane;
    const int n_tiles = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;

    int page[NI];                                                           // of the tile that is asked for next
    auto find = [&](int t) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int key = k0 + t * KT + (tid + i * SH_THREADS) / CH;
            page[i] = key < k1 ? __ldg(bt + sh_block(p, key)) : 0;
        }
    };
    auto ask = [&](int t) {
        T* Kt = ring + (t % ST) * 2 * TILE;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int at = tid + i * SH_THREADS, j = at / CH, e = (at % CH) * E;
            if ((KT * CH) % SH_THREADS && at >= KT * CH) break;
            const int key = k0 + t * KT + j;
            const bool there = key < k1 && (unsigned)page[i] < (unsigned long long)p.n_pages;
            const T* src = cache + (size_t)(there ? page[i] : 0) * page_stride + ((size_t)g * p.ps + (there ? key - sh_block(p, key) * p.ps : 0)) * HD + e;
            cp_async16(Kt + j * LD + e, src, there);
            cp_async16(Kt + TILE + j * LD + e, src + plane, there);
        }
    };
    find(0);
#pragma unroll
    for (int t = 0; t < ST - 1; t++) {
        if (t < n_tiles) { ask(t); find(t + 1); }
        cp_async_commit();
    }
    const float sl2 = p.scale * 1.4426950408889634f;                        // scores in units of log2

    if constexpr (C::MMA) {
        constexpr bool KEYS = BM == 16;                                     // the warps share the keys, not the columns
        constexpr int NK = KEYS ? KT / 4 : KT;                              // keys of a tile that a warp takes
        constexpr bool QREG = HD <= 128;
        const int c0 = KEYS ? 0 : warp * 16, kw = KEYS ? warp * NK : 0;
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
            cp_async_wait<ST - 2>();
            __syncthreads();
            if (t + ST - 1 < n_tiles) { ask(t + ST - 1); find(t + ST); }
            cp_async_commit();
            const T* Kt = ring + (t % ST) * 2 * TILE + kw * LD;
            const T* Vt = Kt + TILE;
            const int key0 = k0 + t * KT + kw;
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
                    ldmatrix_x4(b, Kt + (j * 16 + (lane & 7) + ((lane >> 4) << 3)) * LD + k * 16 + ((lane >> 3) & 1) * 8);
                    mma_bf16(s[2 * j], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma_bf16(s[2 * j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
            }
            const bool masked = key0 + NK > lim_min;
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < NK / 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if (masked) {
                        const int key = key0 + j * 8 + (lane & 3) * 2 + e;
                        if (key >= lim0) s[j][e] = -INFINITY;
                        if (key >= lim1) s[j][2 + e] = -INFINITY;
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
                const T* v = Vt + (j * 16 + (lane & 15)) * LD + (lane >> 4) * 8;
                bool odd = false;
#pragma unroll
                for (int d = 0; d < HD / 16; d++) {
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, v + d * 16);
                    if (masked)
#pragma unroll
                        for (int e = 0; e < 4; e++) { const uint32_t f = sh_finite2(b[e]); odd |= f != b[e]; b[e] = f; }
                    mma_bf16(o[2 * d], a[0], a[1], a[2], a[3], b[0], b[1]);
                    mma_bf16(o[2 * d + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
                }
                if (masked && __any_sync(0xffffffffu, odd)) {
                    // values that are not finite, key by key, to the columns that read them
                    float* P = reinterpret_cast<float*>(Pbuf) + warp * 256;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            P[(lane >> 2) * 16 + h * 8 + (lane & 3) * 2 + e] = s[2 * j + h][e];
                            P[((lane >> 2) + 8) * 16 + h * 8 + (lane & 3) * 2 + e] = s[2 * j + h][2 + e];
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
                                const float x = to_f32(Vt[(j * 16 + i) * LD + d * 8 + (lane & 3) * 2 + e]);
                                if (sh_odd(x)) {
                                    if (key < lim0) o[d][e] += p0 * x;
                                    if (key < lim1) o[d][2 + e] += p1 * x;
                                }
                            }
                    }
                    __syncwarp();
                }
            }
        }
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        cp_async_wait<0>();
        __syncthreads();                                                    // the ring has been read: the output takes its place
        float* O = reinterpret_cast<float*>(main_);
        if constexpr (!KEYS) {
#pragma unroll
            for (int d = 0; d < HD / 8; d++) {
                *reinterpret_cast<float2*>(O + r0 * HD + d * 8 + (lane & 3) * 2) = make_float2(o[d][0], o[d][1]);
                *reinterpret_cast<float2*>(O + r1 * HD + d * 8 + (lane & 3) * 2) = make_float2(o[d][2], o[d][3]);
            }
            if (!(lane & 3)) { ml[2 * r0] = m0; ml[2 * r0 + 1] = l0; ml[2 * r1] = m1; ml[2 * r1 + 1] = l1; }
        } else {
            float* Ow = O + (1 + warp) * 16 * HD;                           // [0]: the joined one
            float* mw = ml + 32 + warp * 32;
#pragma unroll
            for (int d = 0; d < HD / 8; d++) {
                *reinterpret_cast<float2*>(Ow + r0 * HD + d * 8 + (lane & 3) * 2) = make_float2(o[d][0], o[d][1]);
                *reinterpret_cast<float2*>(Ow + r1 * HD + d * 8 + (lane & 3) * 2) = make_float2(o[d][2], o[d][3]);
            }
            if (!(lane & 3)) { mw[2 * r0] = m0; mw[2 * r0 + 1] = l0; mw[2 * r1] = m1; mw[2 * r1 + 1] = l1; }
            __syncthreads();
            for (int i = tid; i < 16 * HD / 4; i += SH_THREADS) {
                const int c = i / (HD / 4), d = i % (HD / 4) * 4;
                float M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < 4; w++) M = fmaxf(M, ml[32 + w * 32 + 2 * c]);
                const float u = M == -INFINITY ? 0.f : M;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const float f = sh_exp2(ml[32 + w * 32 + 2 * c] - u);
                    const float4 x = *reinterpret_cast<const float4*>(O + (1 + w) * 16 * HD + c * HD + d);
                    L += f * ml[32 + w * 32 + 2 * c + 1];
                    acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
                }
                *reinterpret_cast<float4*>(O + c * HD + d) = acc;
                if (!d) { ml[2 * c] = M; ml[2 * c + 1] = L; }
            }
        }
    } else {
        constexpr int MR = C::MR, KJ = KT / 16, DJ = HD / 32;
        const int tr = tid >> 4, tc = tid & 15;
        float* P = reinterpret_cast<float*>(Pbuf);
        float o[MR][2 * DJ], m[MR], l[MR];
        int lm[MR];
#pragma unroll
        for (int r = 0; r < MR; r++) {
            m[r] = -INFINITY; l[r] = 0.f; lm[r] = lim(tr * MR + r);
#pragma unroll
            for (int d = 0; d < 2 * DJ; d++) o[r][d] = 0.f;
        }
        for (int t = 0; t < n_tiles; t++) {
            cp_async_wait<ST - 2>();
            __syncthreads();
            if (t + ST - 1 < n_tiles) { ask(t + ST - 1); find(t + ST); }
            cp_async_commit();
            const float* Kt = reinterpret_cast<const float*>(ring) + (t % ST) * 2 * TILE;
            const float* Vt = Kt + TILE;
            const float* Qf = reinterpret_cast<const float*>(Qs) + tr * MR * LD;
            const int key0 = k0 + t * KT;
            float s[MR][KJ];
#pragma unroll
            for (int r = 0; r < MR; r++)
#pragma unroll
                for (int j = 0; j < KJ; j++) s[r][j] = 0.f;
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                float4 k[KJ];
#pragma unroll
                for (int j = 0; j < KJ; j++) k[j] = *reinterpret_cast<const float4*>(Kt + (tc + 16 * j) * LD + d);
#pragma unroll
                for (int r = 0; r < MR; r++) {
                    const float4 q = *reinterpret_cast<const float4*>(Qf + r * LD + d);
#pragma unroll
                    for (int j = 0; j < KJ; j++) s[r][j] = fmaf(q.x, k[j].x, fmaf(q.y, k[j].y, fmaf(q.z, k[j].z, fmaf(q.w, k[j].w, s[r][j]))));
                }
            }
            const bool masked = key0 + KT > lim_min;
#pragma unroll
            for (int r = 0; r < MR; r++) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < KJ; j++) {
                    if (masked && key0 + tc + 16 * j >= lm[r]) s[r][j] = -INFINITY;
                    top = fmaxf(top, s[r][j]);
                }
#pragma unroll
                for (int x = 8; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                const float n = fmaxf(m[r], top * sl2), u = n == -INFINITY ? 0.f : n;
                const float f = exp2f(m[r] - u);
                m[r] = n;
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < 2 * DJ; d++) o[r][d] *= f;
#pragma unroll
                for (int j = 0; j < KJ; j++) {
                    const float e = exp2f(fmaf(s[r][j], sl2, -u));
                    l[r] += e;
                    P[(tr * MR + r) * (KT + 4) + tc + 16 * j] = e;
                }
            }
            __syncwarp();                                                   // (a column's weights are made and read by one half of a warp)
            if (!masked) {
#pragma unroll 1
                for (int j = 0; j < KT; j += 4) {
                    float2 v[4][DJ];
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int d = 0; d < DJ; d++) v[i][d] = *reinterpret_cast<const float2*>(Vt + (j + i) * LD + d * 32 + tc * 2);
#pragma unroll
                    for (int r = 0; r < MR; r++) {
                        const float4 w = *reinterpret_cast<const float4*>(P + (tr * MR + r) * (KT + 4) + j);
#pragma unroll
                        for (int d = 0; d < DJ; d++) {
                            o[r][2 * d] = fmaf(w.x, v[0][d].x, fmaf(w.y, v[1][d].x, fmaf(w.z, v[2][d].x, fmaf(w.w, v[3][d].x, o[r][2 * d]))));
                            o[r][2 * d + 1] = fmaf(w.x, v[0][d].y, fmaf(w.y, v[1][d].y, fmaf(w.z, v[2][d].y, fmaf(w.w, v[3][d].y, o[r][2 * d + 1]))));
                        }
                    }
                }
            } else {
#pragma unroll 1
                for (int j = 0; j < KT; j++)
#pragma unroll
                    for (int r = 0; r < MR; r++)
                        if (key0 + j < lm[r]) {
                            const float w = P[(tr * MR + r) * (KT + 4) + j];
#pragma unroll
                            for (int d = 0; d < DJ; d++) {
                                const float2 v = *reinterpret_cast<const float2*>(Vt + j * LD + d * 32 + tc * 2);
                                o[r][2 * d] = fmaf(w, v.x, o[r][2 * d]);
                                o[r][2 * d + 1] = fmaf(w, v.y, o[r][2 * d + 1]);
                            }
                        }
            }
            __syncwarp();
        }
        cp_async_wait<0>();
        __syncthreads();
        float* O = reinterpret_cast<float*>(main_);
#pragma unroll
        for (int r = 0; r < MR; r++) {
            const int c = tr * MR + r;
#pragma unroll
            for (int d = 0; d < DJ; d++) *reinterpret_cast<float2*>(O + c * HD + d * 32 + tc * 2) = make_float2(o[r][2 * d], o[r][2 * d + 1]);
#pragma unroll
            for (int x = 8; x; x >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
            if (!tc) { ml[2 * c] = m[r]; ml[2 * c + 1] = l[r]; }
        }
    }
    __syncthreads();
}

// the queries of BM columns from column c0 of the rows row0 ..: zeros behind the last
template <typename T, int HD, int BM>
__device__ __forceinline__ void sh_queries(const ShArgs& p, T* Qs, int row0, int n_cols, int c0, int g, int R) {
    typedef Sh<T, HD, BM> C;
    const T* q = (const T*)p.q + (size_t)row0 * p.ldq + (size_t)g * R * HD;
    for (int i = threadIdx.x; i < BM * C::CH; i += SH_THREADS) {
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
}

// ---- first launch: a chunk of a group's prefix for a tile of its columns
template <typename T, int HD, int BM>
__global__ void __launch_bounds__(SH_THREADS)
shared_prefix_kernel(const ShArgs p) {
    kp_pdl_begin();
    typedef Sh<T, HD, BM> C;
    extern __shared__ __align__(16) unsigned char smem[];
    T* Qs = reinterpret_cast<T*>(smem);
    unsigned char* main_ = smem + C::Q_BYTES;
    unsigned char* Pbuf = main_ + C::MAIN;
    float* ml = reinterpret_cast<float*>(Pbuf + C::P_BYTES);
    const int chunk = blockIdx.x, g = blockIdx.y, group = blockIdx.z / p.tiles, c0 = blockIdx.z % p.tiles * BM, R = p.H / p.G;
    const int s0 = max(0, min(p.group_seqs[group], p.n_seq)), s1 = max(s0, min(p.group_seqs[group + 1], p.n_seq));
    const int P = sh_prefix(p, group), k0 = chunk * p.chunk, k1 = min(P, k0 + p.chunk);
    if (s0 == s1 || k0 >= k1) return;
    const int row0 = sh_row(p, s0), n_cols = max(0, sh_row(p, s1) - row0) * R;
    if (c0 >= n_cols) return;
    sh_queries<T, HD, BM>(p, Qs, row0, n_cols, c0, g, R);
    __syncthreads();
    sh_tile<T, HD, BM>(p, Qs, main_, Pbuf, ml, p.table + (size_t)s0 * p.width, g, k0, k1, k1, [&](int) { return k1; });
    const float* O = reinterpret_cast<const float*>(main_);
    for (int i = threadIdx.x; i < BM * HD / 4; i += SH_THREADS) {
        const int c = i / (HD / 4), d = i % (HD / 4) * 4, col = c0 + c;
        if (col >= n_cols) break;
        const size_t at = ((size_t)(row0 + col / R) * p.H + g * R + col % R) * p.n_chunks + chunk;
        *reinterpret_cast<float4*>(p.part_o + at * HD + d) = *reinterpret_cast<const float4*>(O + c * HD + d);
        if (!d) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(ml[2 * c], ml[2 * c + 1]);
    }
}

// ---- second launch: a sequence's own keys, shared out over a cluster, and the join
template <typename T, int HD, int BM>
__global__ void __launch_bounds__(SH_THREADS)
shared_own_kernel(const ShArgs p) {
    // With a first launch its inputs are ready: all CTAs of that one have waited for the kernels before it by the time that this one may start.
    KP_TRACE_MARK(0);
    if (p.alone) pdl_wait();
    typedef Sh<T, HD, BM> C;
    extern __shared__ __align__(16) unsigned char smem[];
    T* Qs = reinterpret_cast<T*>(smem);
    unsigned char* main_ = smem + C::Q_BYTES;
    unsigned char* Pbuf = main_ + C::MAIN;
    float* ml = reinterpret_cast<float*>(Pbuf + C::P_BYTES);
    float* wts = ml + C::ML_BYTES / 4;                       // [BM][parts]
    __shared__ int s_group;
    cg::cluster_group cluster = cg::this_cluster();
    const int n_cl = gridDim.x, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.y, seq = blockIdx.z / p.tiles, c0 = blockIdx.z % p.tiles * BM, R = p.H / p.G;
    if (tid == 0) s_group = -1;
    __syncthreads();
    for (int i = tid; i < p.n_groups; i += SH_THREADS)
        if (p.group_seqs[i] <= seq && seq < p.group_seqs[i + 1]) s_group = i;
    const int row0 = sh_row(p, seq), n_cols = max(0, sh_row(p, seq + 1) - row0) * R, pos0 = max(-p.n, min(p.seg_pos[seq], p.width * p.ps));
    __syncthreads();
    const int group = s_group, P = group >= 0 ? sh_prefix(p, group) : 0;
    const bool work = c0 < n_cols;                           // (the same for all CTAs of a cluster)
    if (work) {
        const int last = pos0 + (min(n_cols, c0 + BM) - 1) / R;                     // position of the tile's last row
        const int end = (int)min((long long)last + 1, (long long)p.width * p.ps);
        const int per = (max(0, end - P) + n_cl * C::KT - 1) / (n_cl * C::KT) * C::KT;      // keys a CTA, in whole tiles
        const int k0 = P + part * per, k1 = min(end, k0 + per);
        sh_queries<T, HD, BM>(p, Qs, row0, n_cols, c0, g, R);
        __syncthreads();
        sh_tile<T, HD, BM>(p, Qs, main_, Pbuf, ml, p.table + (size_t)seq * p.width, g, k0, k1, min(k1, pos0 + c0 / R + 1),
                           [&](int c) { return min(k1, pos0 + (c0 + c) / R + 1); });
    }
    KP_TRACE_MARK(1);
    if (!p.alone) pdl_wait();                                // the prefix's parts are there
    pdl_launch_dependents();
    if (!work) return;
    if (n_cl > 1) cluster.sync();
    const int n_pre = group >= 0 ? (P + p.chunk - 1) / p.chunk : 0, n_parts = n_cl + n_pre;
    const float* O = reinterpret_cast<const float*>(main_);
    // the parts' weights: 2^(m - M) / sum 2^(m - M) l.  The cluster's CTAs share the columns.
    for (int c = part + warp * n_cl; c < BM && c0 + c < n_cols; c += n_cl * 4) {
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
        for (int i = 0; i < 3; i++) if (lane + 32 * i < n_parts) wts[c * (SH_MAX_CLUSTER + SH_MAX_CHUNKS) + lane + 32 * i] = m[i] * inv;
    }
    __syncthreads();
    constexpr int D4 = HD / 4;
    const int mine = (min(BM, n_cols - c0) - part + n_cl - 1) / n_cl;               // columns part, part + n_cl, ...
    for (int i = tid; i < mine * D4; i += SH_THREADS) {
        const int c = part + i / D4 * n_cl, d = i % D4 * 4, col = c0 + c;
        const size_t row = row0 + col / R;
        const float* w = wts + c * (SH_MAX_CLUSTER + SH_MAX_CHUNKS);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float f, const float4 x) { a.x += f * x.x; a.y += f * x.y; a.z += f * x.z; a.w += f * x.w; };
        for (int x = 0; x < n_cl; x++) add(w[x], *reinterpret_cast<const float4*>((n_cl > 1 ? cluster.map_shared_rank(O, x) : O) + c * HD + d));
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

template <typename T, int HD, int BM>
static int sh_prefix_launch(const ShArgs& a, cudaStream_t st) {
    typedef Sh<T, HD, BM> C;
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(shared_prefix_kernel<T, HD, BM>, C::SMEM, ready);
    if (e) return e;
    cudaError_t c = kp_launch_pdl(shared_prefix_kernel<T, HD, BM>, dim3(a.n_chunks, a.G, a.n_groups * a.tiles), dim3(SH_THREADS), C::SMEM, st, a);
    return c ? (int)c : kp_launch_status();
}
template <typename T, int HD, int BM>
static int sh_own_launch(const ShArgs& a, int ctas, cudaStream_t st) {
    typedef Sh<T, HD, BM> C;
    static std::atomic<unsigned long long> ready{0};
    int e = kp_smem_limit(shared_own_kernel<T, HD, BM>, C::SMEM, ready);
    if (e) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, a.G, a.n_seq * a.tiles);
    cfg.blockDim = dim3(SH_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t c = cudaLaunchKernelEx(&cfg, shared_own_kernel<T, HD, BM>, a);
    return c ? (int)c : kp_launch_status();
}

template <typename T, int HD>
static int sh_run(ShArgs& a, int tile, int group_tiles, int own_tile, int own_tiles, int own_ctas, int with_prefix, cudaStream_t st) {
    int e = 0;
    if (with_prefix) {
        a.tiles = group_tiles;
        e = tile == 16 ? sh_prefix_launch<T, HD, 16>(a, st) : sh_prefix_launch<T, HD, 64>(a, st);
        if (e) return e;
    }
    a.tiles = own_tiles;
    return own_tile == 16 ? sh_own_launch<T, HD, 16>(a, own_ctas, st) : sh_own_launch<T, HD, 64>(a, own_ctas, st);
}

// tile, own_tile: columns of a tile, 16 or 64, of the first and of the second launch; with_prefix: 0 where the prefix's parts come from another
// launch (prefix_done: it has been queued) or there is none.
extern "C" int kp_attention_shared(const void* q, long long ldq, const void* cache, long long n_pages, const int* table, int width, const int* cu_rows, const int* seg_pos,
                                   const int* group_seqs, const int* prefix_len, int n, int n_seq, int n_groups, void* out, long long ldo, float* part_o,
                                   float* part_ml, int n_chunks, int chunk, float scale, int ps, int H, int G, int hd, int max_prefix, int tile, int group_tiles,
                                   int own_tile, int own_tiles, int own_ctas, int with_prefix, int prefix_done, int dtype, void* stream) {
    if (n <= 0 || n_seq <= 0) return 0;
    const int elt = dtype == KP_DTYPE_F32 ? 4 : 2;
    if (G < 1 || G > 65535 || H < 1 || H % G || ps < 1 || width < 1 || (long long)width * ps > (1 << 30) || n_pages < 1 || n_groups < 0 || chunk < 1 ||
        n_chunks < 0 || n_chunks > SH_MAX_CHUNKS || ((with_prefix || prefix_done) && (n_chunks < 1 || (long long)n_chunks * chunk < max_prefix)) ||
        (tile != 16 && tile != 64) || (own_tile != 16 && own_tile != 64) || group_tiles < 1 || own_tiles < 1 || own_ctas < 1 || own_ctas > SH_MAX_CLUSTER ||
        (long long)n_groups * group_tiles > 65535 || (long long)n_seq * own_tiles > 65535 || ((uintptr_t)cache & 15) || ((uintptr_t)q & (elt - 1)) ||
        ((uintptr_t)out & (elt - 1)))
        return KP_ERR_BAD_ARG;
    int ps_log2 = -1;
    for (int i = 0; i < 31; i++) if (ps == 1 << i) ps_log2 = i;
    ShArgs a = {q, ldq, ((uintptr_t)q & 15) == 0 && ldq * elt % 16 == 0, cache, n_pages, table, width, cu_rows, seg_pos, group_seqs, prefix_len, n, n_seq, n_groups,
                out, ldo, ((uintptr_t)out & 15) == 0 && ldo * elt % 16 == 0, part_o, part_ml, n_chunks, chunk, 1, !(with_prefix || prefix_done), scale, ps, ps_log2,
                H, G, with_prefix || prefix_done ? max_prefix : 0};
    const cudaStream_t st = (cudaStream_t)stream;
#define SH_HD(D) case D: KP_DISPATCH_DTYPE(dtype, T, return sh_run<T, D>(a, tile, group_tiles, own_tile, own_tiles, own_ctas, with_prefix, st))
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
