// A cache of keys and values held in 4 bits: its bytes, and the warp-level attention over it that the kernels share.
//
// A page holds, for every kv head, one record of bytes about its `ps` keys (ps a power of two, at least 16):
//     key codes [ps][HD/2] | value codes [ps][HD/2] | key ranges [ps][NG] | value ranges [ps][NG]
// A row of HD values is cut into NG groups of GS = 64 values (32 where 64 does not divide HD).  A group has a scale s and
// a minimum z, both bfloat16 (a range in the low and the high half of 4 bytes), and 4-bit codes c (value 2i of the row in
// the low half of byte i): the value is s c + z.  Codes are integers, so what is read is exact up to that formula.  bfloat16
// has the exponents of float32: values up to its largest, 3.39e38, have their place (larger ones count as infinite).  The codes are taken against
// the rounded s and z, which makes up for their rounding but at the group's edge: z, the nearest bfloat16 number, can lie up to 2^-8 |min| above the
// minimum, and values below z read as z.  That is more than half a step where |min| is more than 8.5 times the group's range.
//
// The arithmetic.  With q the query and k = s c + z,   q.k = sum over groups  s (q.c) + z (sum of q),
// so the codes themselves enter the matrix instructions and a scale is one multiplication a (key, group), not one a value.
// A code is an fp16 operand without any arithmetic: the bits 0000 0000 0000 cccc are the subnormal c 2^-24, and
// 0000 0000 cccc 0000 are c 2^-20, so eight codes of a word need four ANDs and one shift.  Queries enter as fp16 too,
// each scaled by a power of two that brings its largest value to [2^14, 2^15): what fp16 does not hold of a bfloat16 query
// is below 2^-35 of that value.  float32 queries enter as two fp16 parts (22 bits).  The softmax weights p are
// multiplied with the values' scales and enter as fp16 (as two parts in the float32 form), with the running maximum in
// units that hold p s at or below 2^15 (it follows the maxima in steps of 2^8 and more): at least 31 binary orders of fp16 lie
// below the largest weight of a row.  (s is the largest scale of the values so far: values 2^30 and more smaller than another of the same
// kv head lose bits to it.)
// Scores, maxima, sums and accumulators are float32.
//
// Keys are the rows of the score product (m16n8k16: 16 keys x 8 queries), so that no row of the instruction is wasted where
// few queries share a kv head, and the values' dimensions are the rows of the second product; its P operand is the score
// accumulator turned by movmatrix.
#pragma once
#include <cuda_fp16.h>

#include "mma.cuh"

#define KV4_LOG2E 1.4426950408889634f
#define KV4_LEAST_SCALE 8.271806125530277e-25f             // 2^-80

template <int HD>
struct Kv4 {
    static constexpr int GS = HD % 64 == 0 ? 64 : 32;      // values a group
    static constexpr int NG = HD / GS;                      // groups a row
    static constexpr int ROW = HD / 2;                      // bytes of a row's codes
    static constexpr int PP = ROW / 16;                     // 16-byte pieces of it
    static constexpr int KS = GS / 16;                      // steps of 16 values in a group
    static constexpr int MT = GS / 16;                      // tiles of 16 dimensions in a group
    // A tile of KEYS keys in shared memory: rows of key codes, rows of value codes, key ranges, value ranges.  Rows of 64 and 128 bytes
    // lie as the TMA's 64- and 128-byte swizzles put them (the tile on such a boundary), others as they are.
    static constexpr int bytes(int keys) { return keys * (HD + 8 * NG); }
    static __device__ __forceinline__ int turn(int key) { return PP == 4 ? (key >> 1) & 3 : (PP == 8 ? key & 7 : 0); }
    // Which of a block's 8 keys stands in row (or slot) g of the products' operands: in these orders neither the key words (rows
    // 0..3, rows 4..7) nor the value words (slots 0, 2, 4, 6, slots 1, 3, 5, 7) meet in a bank.
    static __device__ __forceinline__ int key_of(int g) { return (PP == 4 ? 0x32547160 : (PP == 8 ? 0x57136420 : 0x53427160)) >> (4 * g) & 7; }
};
__host__ __device__ constexpr long long kv4_page_bytes(int page_size, int hd) {
    return (long long)page_size * (hd + 8 * (hd / (hd % 64 == 0 ? 64 : 32)));
}

__device__ __forceinline__ float kv4_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
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
__device__ __forceinline__ bool kv4_finite(uint32_t r) { return (r & 0x7f80u) != 0x7f80u && (r & 0x7f800000u) != 0x7f800000u; }

// ---- a block of 16 keys from its page's record to shared memory by a warp's cp.async: row `at` of a tile of KEYS keys (`rec`:
// record of (page, kv head), `off`: the block's first key in the page)
template <int HD, int KEYS>
__device__ __forceinline__ void kv4_load_block(unsigned char* tile, int at, const unsigned char* __restrict__ rec, int off, int ps, int lane) {
    using F = Kv4<HD>;
    const unsigned char* kc = rec + (size_t)off * F::ROW;
    const unsigned char* vc = kc + (size_t)ps * F::ROW;
    const unsigned char* kr = rec + (size_t)ps * HD + (size_t)off * 4 * F::NG;
    const unsigned char* vr = kr + (size_t)ps * 4 * F::NG;
    constexpr int N = F::ROW;                              // 16-byte pieces of 16 rows of codes
    unsigned char* dst = tile + at * F::ROW;
#pragma unroll
    for (int i = 0; i < (N + 31) / 32; i++) {
        const int j = i * 32 + lane;
        if (N % 32 == 0 || j < N) {
            const int to = j / F::PP * F::ROW + ((j % F::PP) ^ F::turn(j / F::PP)) * 16;
            cp_async16(dst + to, kc + j * 16, true);
            cp_async16(dst + KEYS * F::ROW + to, vc + j * 16, true);
        }
    }
    static_assert(8 * F::NG <= 32, "the ranges of a block are at most a piece a lane");
    unsigned char* r = tile + KEYS * HD + at * 4 * F::NG;
    if (lane < 4 * F::NG) cp_async16(r + lane * 16, kr + lane * 16, true);
    else if (lane < 8 * F::NG) cp_async16(r + KEYS * 4 * F::NG + (lane - 4 * F::NG) * 16, vr + (lane - 4 * F::NG) * 16, true);
}
// Where a lane finds its part of a block of 16 keys of a tile of KEYS keys (the tile on a 128-byte boundary): offsets from the tile, for
// its first block.
template <int HD, int KEYS>
struct Kv4Block {
    int k, va, vb, r;                                      // its key words, its value words of slots 2t and 2t + 1, its key's ranges
    __device__ __forceinline__ explicit Kv4Block(int lane) {
        using F = Kv4<HD>;
        const int g = lane >> 2, t = lane & 3, key = F::key_of(g), ka = F::key_of(2 * t), kb = F::key_of(2 * t + 1);
        const int v = KEYS * F::ROW;
        if (F::GS == 64) {
            k = key * F::ROW + ((t >> 1) ^ F::turn(key)) * 16 + (t & 1) * 8;
            va = v + ka * F::ROW + ((g >> 2) ^ F::turn(ka)) * 16 + (g & 3) * 4;
            vb = v + kb * F::ROW + ((g >> 2) ^ F::turn(kb)) * 16 + (g & 3) * 4;
        } else {
            k = key * F::ROW + t * 4;
            va = v + ka * F::ROW + g * 2;
            vb = v + kb * F::ROW + g * 2;
        }
        r = KEYS * HD + key * 4 * F::NG;
    }
    // an offset of group 0, moved to group y (in rows whose pieces are turned the group's bits of the piece's number are exchanged)
    static __device__ __forceinline__ int group(int off, int y) {
        using F = Kv4<HD>;
        return F::PP == 4 || F::PP == 8 ? off ^ (y * 32) : off + y * (F::GS / 2);
    }
};

template <typename W>
__device__ __forceinline__ W kv4_at(const unsigned char* p) { return *reinterpret_cast<const W*>(p); }

// ---- queries of a warp: 8 NT columns as B operands of the score product
template <int HD, int PARTS, int NT>
struct Kv4Q {
    uint32_t b[NT][PARTS][HD / 16][2];
    float fs[NT][2];                                       // factor of s (q.c) for this thread's queries 2t and 2t + 1
    float fz[NT][Kv4<HD>::NG][2];                          // factor of z for them
};

// Loads the warp's columns: src[nt] is the query of column 8 nt + lane / 4 (null: none).
// N consecutive values, 16 bytes at a time where they lie so
template <int N>
__device__ __forceinline__ void kv4_values(float (&v)[N], const bf16* p) {
    if (((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            const uint4 x = reinterpret_cast<const uint4*>(p)[i];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; j++) { v[8 * i + 2 * j] = kv4_scale(w[j]); v[8 * i + 2 * j + 1] = kv4_least(w[j]); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = to_f32(p[i]);
    }
}
template <int N>
__device__ __forceinline__ void kv4_values(float (&v)[N], const float* p) {
    if (((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const float4 x = reinterpret_cast<const float4*>(p)[i];
            v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = p[i];
    }
}
template <int HD, int PARTS, int NT, bool CENTRE, typename T>
__device__ __forceinline__ void kv4_load_q(Kv4Q<HD, PARTS, NT>& Q, const T* const (&src)[NT], float scale, int lane) {
    using F = Kv4<HD>;
    const int t = lane & 3;
    constexpr int W = F::GS / 4;                           // values of a group that a lane holds: 16 or 8 consecutive ones
    // A power of two of each column's own brings its largest value to [2^14, 2^15): its neighbours' size has no part in what fp16 holds of it.
    // (A value that is not finite stays so.)
    float up[NT], f[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float top = 0.f;
        if (src[nt]) {
#pragma unroll
            for (int y = 0; y < F::NG; y++) {
                float v[W];
                kv4_values<W>(v, src[nt] + y * F::GS + t * W);
#pragma unroll
                for (int i = 0; i < W; i++) top = fmaxf(top, fabsf(v[i]));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = top > 0.f && top < INFINITY ? min(14 - ilogbf(top), 100) : 0;
        up[nt] = ldexpf(1.0f, e);
        f[nt] = ldexpf(scale * KV4_LOG2E, -e);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float theirs = __shfl_sync(0xffffffffu, f[nt], (2 * t + i) * 4);                      // (from a lane whose column this is)
            Q.fs[nt][i] = CENTRE ? theirs : theirs * 16777216.0f;
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int y = 0; y < F::NG; y++) {
            float v[W], sum = 0.f;
#pragma unroll
            for (int i = 0; i < W; i++) v[i] = 0.f;
            if (src[nt]) kv4_values<W>(v, src[nt] + y * F::GS + t * W);
#pragma unroll
            for (int i = 0; i < W; i++) v[i] *= up[nt];
#pragma unroll
            for (int k = 0; k < F::KS; k++) {              // step k: values (0, 4), (1, 5) of a word, then (2, 6), (3, 7), then the next word
                const int d = (k >> 1) * 8 + (k & 1) * 2;
                float x[4] = {v[d], v[d + 4], v[d + 1] * 0.0625f, v[d + 5] * 0.0625f};
#pragma unroll
                for (int p = 0; p < PARTS; p++) {
                    const float w0 = x[0], w1 = x[1], w2 = x[2], w3 = x[3];
                    Q.b[nt][p][y * F::KS + k][0] = pack_f16_part(x[0], x[1]);
                    Q.b[nt][p][y * F::KS + k][1] = pack_f16_part(x[2], x[3]);
                    sum += ((w0 - x[0]) + (w1 - x[1])) + 16.0f * ((w2 - x[2]) + (w3 - x[3]));      // of what the operand holds
                }
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                Q.fz[nt][y][i] = __shfl_sync(0xffffffffu, f[nt] * sum, (2 * t + i) * 4);
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
template <int HD, int KEYS, bool CENTRE>
__device__ __forceinline__ void kv4_key_operand(uint32_t (&a)[Kv4<HD>::KS][4], const unsigned char* tile, int at, const Kv4Block<HD, KEYS>& B, int y) {
    using F = Kv4<HD>;
    const unsigned char* p = tile + B.group(B.k, y) + at * F::ROW;
    uint32_t w[2][F::GS / 32];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (F::GS == 64) {
            const uint2 x = kv4_at<uint2>(p + 8 * h * F::ROW);
            w[h][0] = x.x; w[h][F::GS / 32 - 1] = x.y;
        } else {
            w[h][0] = kv4_at<uint32_t>(p + 8 * h * F::ROW);
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
template <int HD, int KEYS, int PARTS, int NT, bool CENTRE>
__device__ __forceinline__ void kv4_scores(float (&s)[NT][4], const unsigned char* tile, int at, const Kv4Block<HD, KEYS>& B,
                                           const Kv4Q<HD, PARTS, NT>& Q) {
    using F = Kv4<HD>;
#pragma unroll
    for (int y = 0; y < F::NG; y++) {
        uint32_t a[F::KS][4];
        kv4_key_operand<HD, KEYS, CENTRE>(a, tile, at, B, y);
        const unsigned char* r = tile + B.r + at * 4 * F::NG + y * 4;
        const uint32_t r0 = kv4_at<uint32_t>(r), r1 = kv4_at<uint32_t>(r + 32 * F::NG);
        float z0 = kv4_least(r0), s0 = kv4_scale(r0), z1 = kv4_least(r1), s1 = kv4_scale(r1);
        if (CENTRE) { z0 = fmaf(8.0f, s0, z0); z1 = fmaf(8.0f, s1, z1); }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = PARTS - 1; p >= 0; p--)           // (the small part first)
#pragma unroll
                for (int k = 0; k < F::KS; k++)
                    mma_f16(acc, a[k][0], a[k][1], a[k][2], a[k][3], Q.b[nt][p][y * F::KS + k][0], Q.b[nt][p][y * F::KS + k][1]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float fs = Q.fs[nt][i], fz = Q.fz[nt][y][i];
                s[nt][i] = fmaf(acc[i], s0 * fs, y == 0 ? z0 * fz : fmaf(z0, fz, s[nt][i]));
                s[nt][2 + i] = fmaf(acc[2 + i], s1 * fs, y == 0 ? z1 * fz : fmaf(z1, fz, s[nt][2 + i]));
            }
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
    float top_s;                                           // the values' largest scale so far, or 2^-80 of the largest minimum
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
        // Scales below 2^-90 are taken for that: with p s at most 2^15 the sum of p then stays below 2^105 times the number
        // of keys.  (Values of 2^-86 and less lose their last bits.)  Where a minimum is so much larger than the scales that p z would leave
        // float32 (a group of equal values has the scale 0), 2^-80 of it counts as a scale: p z stays below 2^95, its sum below 2^125.
        top_s = 8.077935669463161e-28f;
    }
    // Before a tile's weights: `mx` are the thread's largest scores of it, `ts` its largest scale of a value (see top_s).  The shift follows
    // the maxima in steps: only a score above the last one's by 8, or a larger scale, moves it (and what has been added up).
    __device__ __forceinline__ void follow(float (&mx)[NT][2], float ts) {
        bool above = ts > top_s;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) above = above || mx[nt][0] > m[nt][0] + 8.0f || mx[nt][1] > m[nt][1] + 8.0f;
        if (!__any_sync(0xffffffffu, above)) return;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 2; i++) mx[nt][i] = fmaxf(mx[nt][i], __shfl_xor_sync(0xffffffffu, mx[nt][i], d));
        // (the bound of the scales is a power of two, up to four times the largest: the next tiles' need not move it again)
        ts = warp_max(ts);
        if (ts > top_s) top_s = __uint_as_float(min((__float_as_uint(ts) >> 23) + 2u, 254u) << 23);
        const float lg = (float)((int)(__float_as_uint(top_s) >> 23) - 127 - 7);       // 2^(lg + 7) = top_s: p s <= 2^7, and 2^15 with the step
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                m[nt][i] = fmaxf(m[nt][i], mx[nt][i]);
                const float ns = m[nt][i] == -INFINITY ? -INFINITY : m[nt][i] + lg;
                const float corr = ns == shift[nt][i] ? 1.0f : kv4_exp2(shift[nt][i] - ns);
                shift[nt][i] = ns;
                l[nt][i] *= corr;
#pragma unroll
                for (int y = 0; y < Kv4<HD>::NG; y++) z[nt][y][i] *= corr;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) { o[nt][j][i] *= corr; o[nt][j][2 + i] *= corr; }
            }
    }
    // Behind the last key: the threads' shares of the sums are added up (all get them).  A column without a key has the shift -inf then; one
    // whose scores are all NaN has not.
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
                if (l[nt][i] != l[nt][i] && shift[nt][i] == -INFINITY) shift[nt][i] = 0.f;
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

// Adds a block of 16 keys: p [nt][4] are its weights, laid out as the scores; the values' ranges of group y in ranges[y].
template <int HD, int KEYS, int PARTS, int NT>
__device__ __forceinline__ void kv4_add_block(Kv4Acc<HD, PARTS, NT>& A, const float (&p)[NT][4], const unsigned char* tile, int at,
                                              const Kv4Block<HD, KEYS>& B, const uint32_t (&ranges)[Kv4<HD>::NG][2]) {
    using F = Kv4<HD>;
#pragma unroll
    for (int y = 0; y < F::NG; y++) {
        const float s0 = kv4_scale(ranges[y][0]), s1 = kv4_scale(ranges[y][1]);
        float z0 = kv4_least(ranges[y][0]), z1 = kv4_least(ranges[y][1]);
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
        const unsigned char *pa = tile + B.group(B.va, y) + at * F::ROW, *pb = tile + B.group(B.vb, y) + at * F::ROW;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if (F::GS == 64) {
                const uint32_t wa = kv4_at<uint32_t>(pa + 8 * h * F::ROW), wb = kv4_at<uint32_t>(pb + 8 * h * F::ROW);
                u[h][0] = __byte_perm(wa, wb, 0x5410);
                u[h][F::GS / 32 - 1] = __byte_perm(wa, wb, 0x7632);
            } else {
                const uint32_t wa = kv4_at<uint16_t>(pa + 8 * h * F::ROW), wb = kv4_at<uint16_t>(pb + 8 * h * F::ROW);
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

// TB blocks of a tile (from row `at` on, the first key's index is `key0`) against all of a warp's queries.  hi / lo: the last and the first key
// of this thread's queries; k_lo .. k_hi: the keys that any query of the call reads.  MASKED: some key may lie outside.
// KEEP: the scores of a column go to scores[nt][i] as well (null: it is none).
template <int HD, int KEYS, int PARTS, int NT, int TB, bool CENTRE, bool MASKED, bool KEEP>
__device__ __forceinline__ void kv4_tile(Kv4Acc<HD, PARTS, NT>& A, const Kv4Q<HD, PARTS, NT>& Q, const Kv4Block<HD, KEYS>& B, const unsigned char* tile, int at, int key0,
                                         const int (&hi)[NT][2], const int (&lo)[NT][2], int k_lo, int k_hi, int lane, float* const (&scores)[NT][2]) {
    using F = Kv4<HD>;
    const int key = F::key_of(lane >> 2);
    float s[TB][NT][4];
    uint32_t ranges[TB][F::NG][2];
    float mx[NT][2], ts = 0.f, tz = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) mx[nt][0] = mx[nt][1] = -INFINITY;
#pragma unroll
    for (int b = 0; b < TB; b++) {
        const int ka = key0 + b * 16 + key, kb = ka + 8;
#pragma unroll
        for (int y = 0; y < F::NG; y++) {
            const unsigned char* r = tile + B.r + (KEYS + at + b * 16) * 4 * F::NG + y * 4;
            ranges[b][y][0] = kv4_at<uint32_t>(r);
            ranges[b][y][1] = kv4_at<uint32_t>(r + 32 * F::NG);
            if (MASKED) {                                  // (a key that is not there counts as zeros: whatever lies in its place must not reach a sum)
                if (!(ka >= k_lo && ka <= k_hi)) ranges[b][y][0] = 0u;
                if (!(kb >= k_lo && kb <= k_hi)) ranges[b][y][1] = 0u;
            }
            ts = kv4_max3(ts, kv4_scale(ranges[b][y][0]), kv4_scale(ranges[b][y][1]));
            tz = kv4_max3(tz, fabsf(kv4_least(ranges[b][y][0])), fabsf(kv4_least(ranges[b][y][1])));
        }
        kv4_scores<HD, KEYS, PARTS, NT, CENTRE>(s[b], tile, at + b * 16, B, Q);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (MASKED) {
                    if (!(ka >= lo[nt][i] && ka <= hi[nt][i])) s[b][nt][i] = -INFINITY;
                    if (!(kb >= lo[nt][i] && kb <= hi[nt][i])) s[b][nt][2 + i] = -INFINITY;
                }
                if (KEEP && scores[nt][i]) { scores[nt][i][ka] = s[b][nt][i]; scores[nt][i][kb] = s[b][nt][2 + i]; }
                mx[nt][i] = kv4_max3(mx[nt][i], s[b][nt][i], s[b][nt][2 + i]);
            }
    }
    ts = fmaxf(ts, tz * KV4_LEAST_SCALE);
    if (ts == INFINITY) {                                  // (a group that is not finite sets no scale)
        ts = 0.f;
#pragma unroll
        for (int b = 0; b < TB; b++)
#pragma unroll
            for (int y = 0; y < F::NG; y++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float s = kv4_scale(ranges[b][y][i]), z = fabsf(kv4_least(ranges[b][y][i])), t = fmaxf(s, z * KV4_LEAST_SCALE);
                    if (s < INFINITY && z < INFINITY) ts = fmaxf(ts, t);
                }
    }
    A.follow(mx, ts);
    float sh[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int i = 0; i < 2; i++) sh[nt][i] = A.shift[nt][i] == -INFINITY ? 0.f : A.shift[nt][i];
#pragma unroll
    for (int b = 0; b < TB; b++) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                s[b][nt][i] = kv4_exp2(s[b][nt][i] - sh[nt][i]);
                s[b][nt][2 + i] = kv4_exp2(s[b][nt][2 + i] - sh[nt][i]);
                A.l[nt][i] += s[b][nt][i] + s[b][nt][2 + i];
            }
        if (MASKED) {                                      // a value that is not finite has no part in a column that does not read its key
            const int k[2] = {key0 + b * 16 + key, key0 + b * 16 + key + 8};
#pragma unroll
            for (int y = 0; y < F::NG; y++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (kv4_finite(ranges[b][y][h])) continue;
                    const float bad = kv4_scale(ranges[b][y][h]) * 0.f + kv4_least(ranges[b][y][h]);
                    ranges[b][y][h] = 0u;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            if (k[h] >= lo[nt][i] && k[h] <= hi[nt][i]) A.z[nt][y][i] += bad;
                }
        }
        kv4_add_block<HD, KEYS, PARTS, NT>(A, s[b], tile, at + b * 16, B, ranges[b]);
    }
}

// Adds a sequence's weights to a key's mass.  Each (sequence, kv head) adds once to a key in a launch, so the order of additions is fixed and the result's bits
// are; where several sequences' tables name the same page each one's weights arrive, in an order that is not.
__device__ __forceinline__ void kv4_add_mass(float* to, float w) {
    asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(to), "f"(w) : "memory");
}

// ---- CTAs of a cluster that share the keys of some columns
__device__ __forceinline__ void kv4_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t kv4_peer_at(const float* p, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(kp_smem_u32(p)), "r"(rank));
    return at;
}
// what lies at this place of the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ float kv4_peer(const float* p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(kv4_peer_at(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 kv4_peer4(const float* p, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(kv4_peer_at(p, rank)) : "memory");
    return v;
}
// A CTA's share of a tile of `cols` rows in shared memory: [column][HD] float32, each row divided by its own sum, shift [column], sum of p [column], and
// room for the weights of the join [column][most].  Four dimensions lie together, eight such places turned by the column.
__host__ __device__ constexpr int kv4_share_floats(int cols, int hd, int most) { return cols * (hd + 2 + most); }
__device__ __forceinline__ int kv4_share_at(int col, int d, int hd) { return col * hd + ((d >> 2 ^ (col & 7)) << 2) + (d & 3); }
__device__ __forceinline__ void kv4_share_sums(float* part, int cols, int hd, int col, float shift, float sum) {
    part[cols * hd + col] = shift;
    part[cols * (hd + 1) + col] = sum;
}
// Rows of this CTA's columns from the shares of the cluster's n CTAs (at most MOST), four dimensions a thread; BATCH loads from each are under way at once
template <typename T, int HD, int THREADS, bool ALIGNED, int STRIDE, int MOST, int BATCH, typename RowOf>
__device__ __forceinline__ void kv4_join_rows(const float* part, const float* weight, int rank, int n, int n_cols, RowOf row_of) {
    constexpr int LANES = HD / 4;
    for (int i0 = threadIdx.x; i0 < n_cols * LANES; i0 += THREADS * BATCH) {
        float4 v[BATCH][MOST];
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int i = i0 + b * THREADS, col = rank + i / LANES * n;
#pragma unroll
            for (int j = 0; j < MOST; j++)
                if (i < n_cols * LANES && j < n) v[b][j] = kv4_peer4(part + kv4_share_at(col, i % LANES * 4, HD), j);
        }
#pragma unroll
        for (int b = 0; b < BATCH; b++) {
            const int i = i0 + b * THREADS, col = rank + i / LANES * n;
            if (i >= n_cols * LANES) break;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int j = 0; j < MOST; j++)
                if (j < n) {
                    const float y = weight[col * STRIDE + j];
                    x = make_float4(fmaf(y, v[b][j].x, x.x), fmaf(y, v[b][j].y, x.y), fmaf(y, v[b][j].z, x.z), fmaf(y, v[b][j].w, x.w));
                }
            T* dst = row_of(col) + i % LANES * 4;
            if (ALIGNED) {
                *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
            } else {
                dst[0] = from_f32<T>(x.x); dst[1] = from_f32<T>(x.y); dst[2] = from_f32<T>(x.z); dst[3] = from_f32<T>(x.w);
            }
        }
    }
}
// The rows of n_here columns from the shares of the cluster's n CTAs, each weighted by its part of the sum, added in order, by THREADS threads, between
// two meetings of the cluster.  The CTAs share the columns out: this one has every n-th.  sums_of gets a column's shift and sum.  ALIGNED: bfloat16 rows
// on 8-byte boundaries.
template <typename T, int HD, int COLS, int THREADS, bool ALIGNED, int MOST, typename RowOf, typename SumsOf>
__device__ __forceinline__ void kv4_join_shares(float* part, int n, int rank, int n_here, RowOf row_of, SumsOf sums_of) {
    const float* stat = part + COLS * HD;
    float* weight = part + COLS * (HD + 2);
    const int col = rank + threadIdx.x * n;
    if (col < COLS) {
        float m[MOST], l[MOST], top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int j = 0; j < MOST; j++)
            if (j < n) { m[j] = kv4_peer(stat + col, j); l[j] = kv4_peer(stat + COLS + col, j); }
#pragma unroll
        for (int j = 0; j < MOST; j++) if (j < n) top = fmaxf(top, m[j]);
#pragma unroll
        for (int j = 0; j < MOST; j++)
            if (j < n) { l[j] *= kv4_exp2(m[j] - (top == -INFINITY ? 0.f : top)); sum += l[j]; }
#pragma unroll
        for (int j = 0; j < MOST; j++) if (j < n) weight[col * MOST + j] = sum == 0.f ? 0.f : l[j] / sum;
        sums_of(col, top, sum);
    }
    asm volatile("bar.sync 4, %0;" ::"n"(THREADS) : "memory");
    const int n_cta = (n_here + n - 1 - rank) / n;         // this CTA's columns
    if (n == 2) kv4_join_rows<T, HD, THREADS, ALIGNED, MOST, 2, 4>(part, weight, rank, n, n_cta, row_of);
    else if (n <= 4) kv4_join_rows<T, HD, THREADS, ALIGNED, MOST, 4, 2>(part, weight, rank, n, n_cta, row_of);
    else if (MOST == 8 || n <= 8) kv4_join_rows<T, HD, THREADS, ALIGNED, MOST, 8, 1>(part, weight, rank, n, n_cta, row_of);
    else kv4_join_rows<T, HD, THREADS, ALIGNED, MOST, MOST, 1>(part, weight, rank, n, n_cta, row_of);
}

// ---- launches of `places` clusters of `cluster` CTAs
struct Kv4Launch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    Kv4Launch(unsigned places, int cluster, int threads, size_t smem, cudaStream_t st) {
        cfg.gridDim = dim3(places * cluster);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = cluster > 1 ? 2 : 1;
    }
};
// clusters of n (at most 16; above 8 the kernel has to be let) CTAs of a kernel that the GPU holds at once (its limit of shared memory has been raised)
template <auto KERNEL>
static int kv4_fit(int n, int threads, size_t smem) {
    static std::atomic<int> known[64][17];                 // one more than the answer, by device
    int dev = 0, fit = 0;
    if (cudaGetDevice(&dev) || dev >= 64) return 0;
    if (const int k = known[dev][n]) return k - 1;
    const Kv4Launch l(1, n, threads, smem, nullptr);
    if ((n > 8 && cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) ||
        cudaOccupancyMaxActiveClusters(&fit, KERNEL, &l.cfg)) {
        cudaGetLastError();
        fit = 0;
    }
    known[dev][n] = fit + 1;
    return fit;
}
