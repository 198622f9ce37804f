// A cache of keys and values held in 4 bits: its bytes, and the warp-level attention over it that the kernels share.
//
// A page holds, for every kv head, one record of bytes about its `ps` keys (ps a multiple of 16):
//     key codes [ps][HD/2] | value codes [ps][HD/2] | key ranges [ps][NG] | value ranges [ps][NG]
// A row of HD values is cut into NG groups of GS = 64 values (32 where 64 does not divide HD).  A group has a scale s and
// a minimum z, both bfloat16 (a range in the low and the high half of 4 bytes), and 4-bit codes c (value 2i of the row in
// the low half of byte i): the value is s c + z.  Codes are integers, so what is read is exact up to that formula; bfloat16
// has the range of float32, so no key or value is too large for the cache, and the codes are taken against the rounded s
// and z, so their rounding is not added to the codes'.
//
// The arithmetic.  With q the query and k = s c + z,   q.k = sum over groups  s (q.c) + z (sum of q),
// so the codes themselves enter the matrix instructions and a scale is one multiplication a (key, group), not one a value.
// A code is an fp16 operand without any arithmetic: the bits 0000 0000 0000 cccc are the subnormal c 2^-24, and
// 0000 0000 cccc 0000 are c 2^-20, so eight codes of a word need four ANDs and one shift.  Queries enter as fp16 too, each
// scaled by a power of two of its own that brings its largest value to [2^14, 2^15): a bfloat16 query loses nothing that
// is above 2^-38 of its largest value.  float32 queries enter as two fp16 parts (22 bits).  The softmax weights p are
// multiplied with the values' scales and enter as fp16 (as two parts in the float32 form), with the running maximum in
// units that hold p s at or below 2^15: fp16's whole range, 39 binary orders, lies below the largest weight of a row.
// Scores, maxima, sums and accumulators are float32.
//
// Keys are the rows of the score product (m16n8k16: 16 keys x 8 queries), so that no row of the instruction is wasted where
// few queries share a kv head, and the values' dimensions are the rows of the second product; its P operand is the score
// accumulator turned by movmatrix.
#pragma once
#include <cuda_fp16.h>

#include "mma.cuh"

#define KV4_LOG2E 1.4426950408889634f

template <int HD>
struct Kv4 {
    static constexpr int GS = HD % 64 == 0 ? 64 : 32;      // values a group
    static constexpr int NG = HD / GS;                      // groups a row
    static constexpr int ROW = HD / 2;                      // bytes of a row's codes
    static constexpr int PP = ROW / 16;                     // 16-byte pieces of it
    static constexpr int KS = GS / 16;                      // steps of 16 values in a group
    static constexpr int MT = GS / 16;                      // tiles of 16 dimensions in a group
    // a block of 16 keys in shared memory: the four parts of the record, one behind the other
    static constexpr int V_OFF = 16 * ROW, KR_OFF = 32 * ROW, VR_OFF = KR_OFF + 64 * NG, BLOCK = VR_OFF + 64 * NG;
    // where a 16-byte piece of a key's row lies: rows whose length is a power of two have their pieces turned, so that the
    // rows read together do not meet in the same banks
    static __device__ __forceinline__ int piece(int key, int p) {
        if (PP == 4) return key * 4 + (p ^ (((key >> 1) & 1) << 1));
        if (PP == 8) return key * 8 + (p ^ ((key & 3) << 1));
        return key * PP + p;
    }
};
__host__ __device__ constexpr long long kv4_page_bytes(int page_size, int hd) {
    return (long long)page_size * (hd + 8 * (hd / (hd % 64 == 0 ? 64 : 32)));
}

__device__ __forceinline__ float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Packs (a, b) to fp16 and leaves in them what that did not take.
__device__ __forceinline__ uint32_t pack_f16_part(float& a, float& b) {
    const __half2 v = __floats2half2_rn(a, b);
    a -= __low2float(v);
    b -= __high2float(v);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// a range's two halves
__device__ __forceinline__ float kv4_scale(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float kv4_least(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }

// The key of a block's half that stands in row (or slot) g of the products' operands: with this order neither the key words
// (rows 0..3 and 4..7 together) nor the value words (slots 0, 2, 4, 6, then 1, 3, 5, 7) meet in a bank.
__device__ __forceinline__ int kv4_key_of(int g) { return (g & 1) ? 4 + (((g >> 1) + 2) & 3) : g >> 1; }

// ---- a block of 16 keys from its page's record to shared memory, by one warp (`rec`: record of (page, kv head), `off`: the
// block's first key in the page)
template <int HD>
__device__ __forceinline__ void kv4_load_block(unsigned char* dst, const unsigned char* __restrict__ rec, int off, int ps, int lane) {
    using F = Kv4<HD>;
    const unsigned char* kc = rec + (size_t)off * F::ROW;
    const unsigned char* vc = kc + (size_t)ps * F::ROW;
    const unsigned char* kr = rec + (size_t)ps * HD + (size_t)off * 4 * F::NG;
    const unsigned char* vr = kr + (size_t)ps * 4 * F::NG;
    constexpr int N = F::ROW;                              // 16-byte pieces of 16 rows of codes
#pragma unroll
    for (int i = 0; i < (N + 31) / 32; i++) {
        const int j = i * 32 + lane;
        if (N % 32 == 0 || j < N) {
            const int at = F::piece(j / F::PP, j % F::PP) * 16;
            cp_async16(dst + at, kc + j * 16, true);
            cp_async16(dst + F::V_OFF + at, vc + j * 16, true);
        }
    }
    static_assert(8 * F::NG <= 32, "the ranges of a block are at most a piece a lane");
    if (lane < 4 * F::NG) cp_async16(dst + F::KR_OFF + lane * 16, kr + lane * 16, true);
    else if (lane < 8 * F::NG) cp_async16(dst + F::VR_OFF + (lane - 4 * F::NG) * 16, vr + (lane - 4 * F::NG) * 16, true);
}

// ---- queries of a warp: 8 NT columns as B operands of the score product
template <int HD, int PARTS, int NT>
struct Kv4Q {
    uint32_t b[NT][PARTS][HD / 16][2];
    // for this thread's queries 2t and 2t + 1: the factors of s (q.(c - 8)) and of z + 8 s, and what the product starts from
    // (- 8 times the sum of q in the codes' unit; 0 where the operand is c - 8 itself)
    float fs[NT][2], fz[NT][Kv4<HD>::NG][2], init[NT][Kv4<HD>::NG][2];
};

// Loads column n-tile `nt`: `src` is the query of column lane / 4 (null: none).
template <int HD, int PARTS, int NT, bool CENTRE, typename T>
__device__ __forceinline__ void kv4_load_q(Kv4Q<HD, PARTS, NT>& Q, int nt, const T* src, float scale, int lane) {
    using F = Kv4<HD>;
    const int t = lane & 3;
    constexpr int W = F::GS / 4;                           // values of a group that a lane holds: 16 or 8 consecutive ones
    float v[F::NG][W];
    float top = 0.f;
#pragma unroll
    for (int y = 0; y < F::NG; y++)
#pragma unroll
        for (int i = 0; i < W; i++) {
            v[y][i] = src ? to_f32(src[y * F::GS + t * W + i]) : 0.f;
            top = fmaxf(top, fabsf(v[y][i]));
        }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^e brings the largest value to [2^14, 2^15); a query of zeros, or one that is not finite, stays as it is
    int e = 0;
    if (top > 0.f && top < INFINITY) e = min(14 - ilogbf(top), 100);
    const float up = ldexpf(1.0f, e);
    float sum[F::NG];
#pragma unroll
    for (int y = 0; y < F::NG; y++) {
        sum[y] = 0.f;
#pragma unroll
        for (int k = 0; k < F::KS; k++) {                  // step k: values (0, 4), (1, 5) of a word, then (2, 6), (3, 7), then the next word
            const int d = (k >> 1) * 8 + (k & 1) * 2;
            float x[4] = {v[y][d] * up, v[y][d + 4] * up, v[y][d + 1] * up * 0.0625f, v[y][d + 5] * up * 0.0625f};
#pragma unroll
            for (int p = 0; p < PARTS; p++) {
                const float w0 = x[0], w1 = x[1], w2 = x[2], w3 = x[3];
                Q.b[nt][p][y * F::KS + k][0] = pack_f16_part(x[0], x[1]);
                Q.b[nt][p][y * F::KS + k][1] = pack_f16_part(x[2], x[3]);
                // (an infinite value leaves NaN behind: the sum must not see more than what the operand holds)
                sum[y] += ((w0 - x[0]) + (w1 - x[1])) + 16.0f * ((w2 - x[2]) + (w3 - x[3]));
            }
        }
        sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], 1);
        sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], 2);
    }
    const float f = ldexpf(scale * KV4_LOG2E, -e);
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int from = (2 * t + i) * 4;                  // a lane whose column this is
        const float fi = __shfl_sync(0xffffffffu, f, from);
        Q.fs[nt][i] = CENTRE ? fi : fi * 16777216.0f;
#pragma unroll
        for (int y = 0; y < F::NG; y++) {
            const float qs = __shfl_sync(0xffffffffu, sum[y], from);
            Q.fz[nt][y][i] = fi * qs;
            Q.init[nt][y][i] = CENTRE ? 0.f : qs * (-8.0f / 16777216.0f);
        }
    }
}

// Two codes as an fp16 operand: as they are (CENTRE: about their middle, c - 8, exactly; what the sums of s c and of z have in
// common then cancels before it is rounded and not behind it.  The float32 form and what adds up weights take this one, for one
// subtraction more a pair of codes: without it such a weight is off by 1e-6, with it by 2e-7).
template <bool CENTRE, bool HIGH>
__device__ __forceinline__ uint32_t kv4_code(uint32_t w) {
    const uint32_t x = w & (HIGH ? 0x00f000f0u : 0x000f000fu);
    if (!CENTRE) return x;
    const uint32_t y = x | 0x64006400u;                    // 1024 + c, or 1024 + 16 c
    const uint32_t c = HIGH ? 0x64806480u : 0x64086408u;   // 1024 + 128, or 1024 + 8
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&y), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// the A operand of the score product: codes of group y of the keys in rows g and g + 8
template <int HD, bool CENTRE>
__device__ __forceinline__ void kv4_key_operand(uint32_t (&a)[Kv4<HD>::KS][4], const unsigned char* blk, int y, int lane) {
    using F = Kv4<HD>;
    const int key = kv4_key_of(lane >> 2), t = lane & 3;
    uint32_t w[2][F::GS / 32];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (F::GS == 64) {
            const uint2 x = *reinterpret_cast<const uint2*>(blk + F::piece(key + 8 * h, 2 * y + (t >> 1)) * 16 + (t & 1) * 8);
            w[h][0] = x.x; w[h][F::GS / 32 - 1] = x.y;
        } else {
            w[h][0] = *reinterpret_cast<const uint32_t*>(blk + F::piece(key + 8 * h, y) * 16 + t * 4);
        }
    }
#pragma unroll
    for (int i = 0; i < F::GS / 32; i++) {
        const uint32_t x = w[0][i], z = w[1][i], x8 = x >> 8, z8 = z >> 8;
        a[2 * i][0] = kv4_code<CENTRE, false>(x); a[2 * i][1] = kv4_code<CENTRE, false>(z);
        a[2 * i][2] = kv4_code<CENTRE, true>(x); a[2 * i][3] = kv4_code<CENTRE, true>(z);
        a[2 * i + 1][0] = kv4_code<CENTRE, false>(x8); a[2 * i + 1][1] = kv4_code<CENTRE, false>(z8);
        a[2 * i + 1][2] = kv4_code<CENTRE, true>(x8); a[2 * i + 1][3] = kv4_code<CENTRE, true>(z8);
    }
}

// Scores of a block's 16 keys, times scale and log2 e: s[nt][0, 1] of the key in row g and queries 2t, 2t + 1, s[nt][2, 3] of row g + 8.
template <int HD, int PARTS, int NT, bool CENTRE>
__device__ __forceinline__ void kv4_scores(float (&s)[NT][4], const unsigned char* blk, const Kv4Q<HD, PARTS, NT>& Q, int lane) {
    using F = Kv4<HD>;
    const int key = kv4_key_of(lane >> 2);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[nt][i] = 0.f;
#pragma unroll
    for (int y = 0; y < F::NG; y++) {
        uint32_t a[F::KS][4];
        kv4_key_operand<HD, CENTRE>(a, blk, y, lane);
        const uint32_t r0 = *reinterpret_cast<const uint32_t*>(blk + F::KR_OFF + (key * F::NG + y) * 4);
        const uint32_t r1 = *reinterpret_cast<const uint32_t*>(blk + F::KR_OFF + ((key + 8) * F::NG + y) * 4);
        const float s0 = kv4_scale(r0), z0 = fmaf(8.0f, s0, kv4_least(r0)), s1 = kv4_scale(r1), z1 = fmaf(8.0f, s1, kv4_least(r1));
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float acc[4] = {Q.init[nt][y][0], Q.init[nt][y][1], Q.init[nt][y][0], Q.init[nt][y][1]};
#pragma unroll
            for (int p = PARTS - 1; p >= 0; p--)           // (the small part first)
#pragma unroll
                for (int k = 0; k < F::KS; k++)
                    mma_f16(acc, a[k][0], a[k][1], a[k][2], a[k][3], Q.b[nt][p][y * F::KS + k][0], Q.b[nt][p][y * F::KS + k][1]);
            s[nt][0] += fmaf(acc[0] * s0, Q.fs[nt][0], z0 * Q.fz[nt][y][0]);
            s[nt][1] += fmaf(acc[1] * s0, Q.fs[nt][1], z0 * Q.fz[nt][y][1]);
            s[nt][2] += fmaf(acc[2] * s1, Q.fs[nt][0], z1 * Q.fz[nt][y][0]);
            s[nt][3] += fmaf(acc[3] * s1, Q.fs[nt][1], z1 * Q.fz[nt][y][1]);
        }
    }
}

// ---- the running softmax and output of a warp's queries
template <int HD, int PARTS, int NT>
struct Kv4Acc {
    float o[NT][HD / 16][4];                               // [dimension tile]: queries 2t, 2t + 1 of its dimension row g, then of row g + 8
    float z[NT][Kv4<HD>::NG][2];                           // this thread's share of sum p z
    float l[NT][2];                                        // and of sum p
    float m[NT][2];                                        // largest score so far (base 2)
    float shift[NT][2];                                    // what p is taken against: p = 2^(score - shift)
    float top_s;                                           // the values' largest scale so far
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < 2; i++) { l[nt][i] = 0.f; m[nt][i] = -INFINITY; shift[nt][i] = -INFINITY; }
#pragma unroll
            for (int y = 0; y < Kv4<HD>::NG; y++) z[nt][y][0] = z[nt][y][1] = 0.f;
#pragma unroll
            for (int j = 0; j < HD / 16; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[nt][j][i] = 0.f;
        }
        // Scales below 2^-60 are taken for that: with p s at most 2^15 the sum of p then stays below 2^75 times the number
        // of keys.  (Values of 2^-56 and less lose their last bits.)
        top_s = 8.673617379884035e-19f;
    }
    // After the scores' maxima: moves the shift, and with it what has been added up.
    __device__ __forceinline__ void rescale(const float (&mx)[NT][2], float ts) {
        top_s = fmaxf(top_s, ts);
        const float lg = (float)((int)(__float_as_uint(top_s) >> 23) - 126 - 15);      // 2^(lg + 15) >= top_s: p s <= 2^15
        bool moved = false;
        float corr[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[nt][i] = fmaxf(m[nt][i], mx[nt][i]);
                const float ns = m[nt][i] == -INFINITY ? -INFINITY : m[nt][i] + lg;
                corr[nt][i] = ns == shift[nt][i] ? 1.0f : kv4_exp2(shift[nt][i] - ns);
                moved = moved || ns != shift[nt][i];
                shift[nt][i] = ns;
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    l[nt][i] *= corr[nt][i];
#pragma unroll
                    for (int y = 0; y < Kv4<HD>::NG; y++) z[nt][y][i] *= corr[nt][i];
#pragma unroll
                    for (int j = 0; j < HD / 16; j++) { o[nt][j][i] *= corr[nt][i]; o[nt][j][2 + i] *= corr[nt][i]; }
                }
            }
        }
    }
    // Behind the last key: the threads' shares of the sums are added up (all get them).
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], d);
#pragma unroll
                    for (int y = 0; y < Kv4<HD>::NG; y++) z[nt][y][i] += __shfl_xor_sync(0xffffffffu, z[nt][y][i], d);
                }
            }
    }
    // value of dimension pair (d, d + 1), d = GS y + (GS / 8) g + 2 j, for query 2t + i
    static __device__ __forceinline__ int dim(int y, int j, int lane) { return y * Kv4<HD>::GS + (lane >> 2) * (Kv4<HD>::GS / 8) + 2 * j; }
    __device__ __forceinline__ float2 value(int nt, int y, int j, int i) const {
        const int e = y * Kv4<HD>::MT + j;
        constexpr float f0 = PARTS == 1 ? 16777216.0f : 1.0f, f1 = f0 / 16.0f;
        return make_float2(fmaf(o[nt][e][i], f0, z[nt][y][i]), fmaf(o[nt][e][2 + i], f1, z[nt][y][i]));
    }
};

// the values' ranges of the keys in rows g and g + 8, of group y (a key that is not there counts as zeros: whatever lies in
// its place must not reach a sum)
template <int HD>
__device__ __forceinline__ void kv4_value_ranges(uint32_t (&r)[2], const unsigned char* blk, int y, bool there0, bool there1, int lane) {
    using F = Kv4<HD>;
    const int key = kv4_key_of(lane >> 2);
    r[0] = there0 ? *reinterpret_cast<const uint32_t*>(blk + F::VR_OFF + (key * F::NG + y) * 4) : 0u;
    r[1] = there1 ? *reinterpret_cast<const uint32_t*>(blk + F::VR_OFF + ((key + 8) * F::NG + y) * 4) : 0u;
}

// Adds a block of 16 keys: p [nt][4] are its weights, laid out as the scores.
template <int HD, int PARTS, int NT>
__device__ __forceinline__ void kv4_add_block(Kv4Acc<HD, PARTS, NT>& A, const float (&p)[NT][4], const unsigned char* blk, bool there0, bool there1,
                                              int lane) {
    using F = Kv4<HD>;
    const int g = lane >> 2, t = lane & 3;
    const int ka = t, kb = 4 + ((t + 2) & 3);              // the keys in slots 2t and 2t + 1
#pragma unroll
    for (int y = 0; y < F::NG; y++) {
        uint32_t r[2];
        kv4_value_ranges<HD>(r, blk, y, there0, there1, lane);
        const float s0 = kv4_scale(r[0]), s1 = kv4_scale(r[1]);
        float z0 = kv4_least(r[0]), z1 = kv4_least(r[1]);
        if (PARTS > 1) { z0 = fmaf(8.0f, s0, z0); z1 = fmaf(8.0f, s1, z1); }
        uint32_t b[NT][PARTS][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            A.z[nt][y][0] = fmaf(p[nt][0], z0, fmaf(p[nt][2], z1, A.z[nt][y][0]));
            A.z[nt][y][1] = fmaf(p[nt][1], z0, fmaf(p[nt][3], z1, A.z[nt][y][1]));
            float w0 = p[nt][0] * s0, w1 = p[nt][1] * s0, w2 = p[nt][2] * s1, w3 = p[nt][3] * s1;
#pragma unroll
            for (int q = 0; q < PARTS; q++) {
                b[nt][q][0] = movmatrix_trans(PARTS == 1 ? pack_f16(w0, w1) : pack_f16_part(w0, w1));
                b[nt][q][1] = movmatrix_trans(PARTS == 1 ? pack_f16(w2, w3) : pack_f16_part(w2, w3));
            }
        }
        uint32_t u[2][F::GS / 32];                         // [keys 0..7, 8..15]: the codes of slots 2t and 2t + 1 side by side
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (F::GS == 64) {
                const int at = (g & 3) * 4;
                const uint32_t wa = *reinterpret_cast<const uint32_t*>(blk + F::V_OFF + F::piece(ka + 8 * h, 2 * y + (g >> 2)) * 16 + at);
                const uint32_t wb = *reinterpret_cast<const uint32_t*>(blk + F::V_OFF + F::piece(kb + 8 * h, 2 * y + (g >> 2)) * 16 + at);
                u[h][0] = __byte_perm(wa, wb, 0x5410);
                u[h][F::GS / 32 - 1] = __byte_perm(wa, wb, 0x7632);
            } else {
                const uint32_t wa = *reinterpret_cast<const uint16_t*>(blk + F::V_OFF + F::piece(ka + 8 * h, y) * 16 + g * 2);
                const uint32_t wb = *reinterpret_cast<const uint16_t*>(blk + F::V_OFF + F::piece(kb + 8 * h, y) * 16 + g * 2);
                u[h][0] = wa | (wb << 16);
            }
        }
#pragma unroll
        for (int j = 0; j < F::MT; j++) {                  // tile j: codes 2j (rows 0..7) and 2j + 1 (rows 8..15) of the lane's word
            const uint32_t x = u[0][j >> 1] >> ((j & 1) * 8), w = u[1][j >> 1] >> ((j & 1) * 8);
            const uint32_t a0 = kv4_code<(PARTS > 1), false>(x), a1 = kv4_code<(PARTS > 1), true>(x);
            const uint32_t a2 = kv4_code<(PARTS > 1), false>(w), a3 = kv4_code<(PARTS > 1), true>(w);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if (PARTS == 1) {
                    mma_f16(A.o[nt][y * F::MT + j], a0, a1, a2, a3, b[nt][0][0], b[nt][0][1]);
                } else {
                    // (the accumulator of the tensor core cuts off what it cannot hold; a block's sum is small, and joins
                    // the others by an addition that rounds)
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16(acc, a0, a1, a2, a3, b[nt][PARTS - 1][0], b[nt][PARTS - 1][1]);
                    mma_f16(acc, a0, a1, a2, a3, b[nt][0][0], b[nt][0][1]);
#pragma unroll
                    for (int i = 0; i < 4; i++) A.o[nt][y * F::MT + j][i] += acc[i];
                }
            }
        }
    }
}

// A tile of TB blocks (the first key's index is `key0`) against all of a warp's queries.  hi / lo: the last and the first key
// of this thread's queries; k_lo .. k_hi: the keys that any query of the call reads.  MASKED: some key may lie outside.
// KEEP: the scores of a column go to scores[nt][i] as well (null: it is none).
template <int HD, int PARTS, int NT, int TB, bool CENTRE, bool MASKED, bool KEEP>
__device__ __forceinline__ void kv4_tile(Kv4Acc<HD, PARTS, NT>& A, const Kv4Q<HD, PARTS, NT>& Q, const unsigned char* tile, int key0,
                                         const int (&hi)[NT][2], const int (&lo)[NT][2], int k_lo, int k_hi, int lane, float* const (&scores)[NT][2]) {
    using F = Kv4<HD>;
    const int key = kv4_key_of(lane >> 2);
    float s[TB][NT][4];
    float mx[NT][2], ts = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
    for (int b = 0; b < TB; b++) {
        const unsigned char* blk = tile + b * F::BLOCK;
        kv4_scores<HD, PARTS, NT, CENTRE>(s[b], blk, Q, lane);
        const int ka = key0 + b * 16 + key, kb = ka + 8;
        const bool t0 = !MASKED || (ka >= k_lo && ka <= k_hi), t1 = !MASKED || (kb >= k_lo && kb <= k_hi);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (MASKED) {
                    if (!(ka >= lo[nt][i] && ka <= hi[nt][i])) s[b][nt][i] = -INFINITY;
                    if (!(kb >= lo[nt][i] && kb <= hi[nt][i])) s[b][nt][2 + i] = -INFINITY;
                }
                if (KEEP && scores[nt][i]) { scores[nt][i][ka] = s[b][nt][i]; scores[nt][i][kb] = s[b][nt][2 + i]; }
                mx[nt][i] = fmaxf(mx[nt][i], fmaxf(s[b][nt][i], s[b][nt][2 + i]));
            }
#pragma unroll
        for (int y = 0; y < F::NG; y++) {
            uint32_t r[2];
            kv4_value_ranges<HD>(r, blk, y, t0, t1, lane);
            const float a = kv4_scale(r[0]), c = kv4_scale(r[1]);
            ts = fmaxf(ts, fmaxf(a < INFINITY ? a : 0.f, c < INFINITY ? c : 0.f));      // (a group that is not finite sets no scale)
        }
    }
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) {
        ts = fmaxf(ts, __shfl_xor_sync(0xffffffffu, ts, d));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) mx[nt][i] = fmaxf(mx[nt][i], __shfl_xor_sync(0xffffffffu, mx[nt][i], d));
    }
    A.rescale(mx, ts);
    float sh[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++) sh[nt][i] = A.shift[nt][i] == -INFINITY ? 0.f : A.shift[nt][i];
#pragma unroll
    for (int b = 0; b < TB; b++) {
        const unsigned char* blk = tile + b * F::BLOCK;
        const int ka = key0 + b * 16 + key, kb = ka + 8;
        const bool t0 = !MASKED || (ka >= k_lo && ka <= k_hi), t1 = !MASKED || (kb >= k_lo && kb <= k_hi);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                s[b][nt][i] = kv4_exp2(s[b][nt][i] - sh[nt][i]);
                s[b][nt][2 + i] = kv4_exp2(s[b][nt][2 + i] - sh[nt][i]);
                A.l[nt][i] += s[b][nt][i] + s[b][nt][2 + i];
            }
        kv4_add_block<HD, PARTS, NT>(A, s[b], blk, t0, t1, lane);
    }
}
