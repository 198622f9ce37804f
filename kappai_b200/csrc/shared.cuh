// Attention of a batch whose sequences share a long prefix: what its kernels have in common.
//
// Sequences come in groups.  The block tables of a group's sequences begin alike: the first `prefix_len` keys are the same for all of them (a page in
// which the prefix ends is each sequence's own copy).  A row at position pos reads the keys 0 .. pos of its sequence,
//   o = sum_j exp(s_j) v_j / sum_j exp(s_j),   s_j = scale q k_j,
// and the sum falls in two: the keys below prefix_len, which all rows of the group read, and the sequence's own keys from there on.
//   The prefix: the rows of a group and the R = H / G query heads that share a kv head are one list of columns, c = row R + head, and a tile of columns
//   reads a chunk of the prefix's keys once for all of them.  It leaves (m, l, O) of each column: the largest score (in units of log2), sum
//   2^(s - m) and sum 2^(s - m) v.
//   The own keys: a tile of columns of one sequence, its keys shared out over the CTAs of a cluster.  The cluster then joins its parts with the
//   prefix's, M = max m, o = sum 2^(m - M) O / sum 2^(m - M) l, and writes the rows.
// Two launches: the second runs while the first is still at work and waits for it only before it joins.
//
// Scratch: part_o [n_rows][H][n_chunks][hd] and part_ml [n_rows][H][n_chunks][2], float32; chunks that a group's prefix does not reach are neither
// written nor read.
#pragma once
#include "common.cuh"

#define SH_MAX_CHUNKS 64
#define SH_MAX_CLUSTER 8

// The grid of a launch: x, kv heads, and places (a group's or a sequence's tiles of columns).  The third axis ends at 65535: places beyond that stand beside
// the others on the second one, the last of them perhaps too many.
#define SH_AXIS 65535
static inline dim3 sh_grid(int x, int G, int places) { return places <= SH_AXIS ? dim3(x, G, places) : dim3(x, G * ((places + SH_AXIS - 1) / SH_AXIS), SH_AXIS); }
static inline bool sh_grid_ok(int n, int tiles, int G) {
    const long long places = (long long)n * tiles;
    return places < 2147483647LL - SH_AXIS && (places + SH_AXIS - 1) / SH_AXIS * G <= SH_AXIS;
}

struct ShArgs {
    const void* q; long long ldq; int q_vec;                 // q_vec: rows start on 16-byte boundaries
    const void* cache; long long n_pages;
    const int* table; int width;
    const int* cu_rows; const int* seg_pos; const int* group_seqs; const int* prefix_len;
    int n, n_seq, n_groups;
    void* out; long long ldo; int out_vec;
    float* part_o; float* part_ml;
    int n_chunks, chunk;                                     // of a prefix, at most; keys a chunk
    int budget, group_tiles;                                 // budget > 0: chunks are as long as they must be for the first launch to have that many CTAs at
                                                             // most, and `chunk` at least (sh_chunk); tiles of columns of a group
    int tiles;                                               // of columns, of a group (first launch) or of a sequence (second)
    int alone;                                               // second launch: there was no first one
    float scale; int ps, ps_log2; int H, G, max_prefix;
    int box;                                                 // shared.cu: keys that a TMA load brings
    int stages, main;                                        // and stages of the ring that there is room for, and the bytes that it (and later the output) has
};

struct ShPlace {                                             // a CTA's kv head and place
    int g, i;
    __device__ __forceinline__ ShPlace(const ShArgs& p) {
        g = blockIdx.y;
        i = blockIdx.z;
        if (gridDim.y != p.G) { i += g / p.G * SH_AXIS; g %= p.G; }
    }
};
__device__ __forceinline__ int sh_prefix(const ShArgs& p, int group) {
    return max(0, min(min(p.prefix_len[group], p.max_prefix), p.width * p.ps));
}
__device__ __forceinline__ int sh_row(const ShArgs& p, int seq) { return max(0, min(p.cu_rows[seq], p.n)); }
__device__ __forceinline__ float sh_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Keys a chunk, found by a warp.  Prefixes differ, and only the device knows how long they are: of chunks cut for the longest alone the others' would leave
// SMs idle, or take a second turn for a few (five prefixes of 701 to 12000 keys, 4 kv heads: 46 us in 152 CTAs of 7 tiles).
__device__ __forceinline__ int sh_chunk(const ShArgs& p, int lane) {
    if (!p.budget) return p.chunk;
    const int n = lane < p.n_groups ? (sh_prefix(p, lane) + 127) / 128 : 0, per = p.group_tiles * p.G;
    // The least length with which the chunks are within the budget (a chunk a prefix always is), in doubled steps and then by bisection.  Mostly it is one of
    // the first (bisection alone takes 1.2 us longer then); with one prefix much longer than the others it is the hundredth: one of 200000 keys and 15 of
    // 300, 4 kv heads, counted up in ones 76 us, 71.5 so.
    auto fits = [&](int c) { return (long long)__reduce_add_sync(0xffffffffu, (n + c - 1) / c) * per <= p.budget; };
    int lo = (int)max((long long)p.chunk / 128, ((long long)__reduce_add_sync(0xffffffffu, n) * per + p.budget - 1) / p.budget);
    if (!fits(lo)) {
        int hi = lo + 1;
#pragma unroll 1
        for (int step = 2; !fits(hi); step *= 2) { lo = hi; hi += step; }       // (fits at the longest prefix at last)
#pragma unroll 1
        while (hi - lo > 1) {                                // (lo: does not fit; hi: does)
            const int mid = (lo + hi) >> 1;
            if (fits(mid)) hi = mid; else lo = mid;
        }
        lo = hi;
    }
    return lo * 128;
}
// the page of a key and its place there
__device__ __forceinline__ int sh_block(const ShArgs& p, int key) { return p.ps_log2 >= 0 ? key >> p.ps_log2 : key / p.ps; }
