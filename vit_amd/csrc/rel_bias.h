// Learned relative position bias by buckets, as the attention kernels use it (attention_rel.hip, attention_rel_bwd.hip).
//
// Tokens are `prefix` tokens without a place, then the cells of a grid_h x grid_w grid in row order (a sequence is a grid of
// one row). bias(i, j, h) = table[bucket(i, j), h]; for two grid tokens the bucket depends on their offset only:
//   offset index = code(i) - code(j) + center,   code = y (2 gw - 1) + x,   center = (gh - 1)(2 gw - 1) + gw - 1
// counts the (2 gh - 1)(2 gw - 1) offsets without gaps, so one subtraction of two per-token numbers addresses the head's
// bias by offset, expanded into LDS once per workgroup (codes of a block's tokens are monotone: only the slice of offsets that
// its queries / keys can reach is expanded). Three more entries follow the offsets: prefix query on a grid key, grid query on a
// prefix key, prefix on prefix.
#pragma once
#include "vit_common.h"
#include <math.h>

struct RelGeo {
    const float* table;    // [num_buckets, heads]
    const int* bucket_of;  // [offsets + 3] or null: the index itself
    int prefix, gw, grid, center, offsets, num_buckets, heads;
    float inv_scale, inv_gw;
};

constexpr float kRelMasked = -1e30f;  // a table entry below this masks its offset (a mask written as a type's lowest value)

__device__ __forceinline__ int rel_code(const RelGeo& g, int token) {
    int p = token - g.prefix;
    p = p < 0 ? 0 : p;
    p = p > g.grid - 1 ? g.grid - 1 : p;
    // row of the cell: (p + 1/2) / gw is at least 1 / (2 gw) from a whole number, 16 times what rounding adds for p < 2^14 and more
    return p + (int)(((float)p + 0.5f) * g.inv_gw) * (g.gw - 1);
}
// bias of an offset index in units of the raw product (divided by the softmax scale): the start value of the product's
// accumulator, so that adding it costs nothing
template <int U>
__device__ __forceinline__ void rel_entries(const RelGeo& g, const int (&index)[U], int head, float (&v)[U]) {  // the loads of all U together
    int b[U];
#pragma unroll
    for (int j = 0; j < U; ++j) b[j] = index[j];
    if (g.bucket_of) {
#pragma unroll
        for (int j = 0; j < U; ++j) b[j] = g.bucket_of[index[j]];
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int c = b[j] < 0 ? 0 : b[j] < g.num_buckets ? b[j] : g.num_buckets - 1;
        v[j] = g.table[(size_t)c * g.heads + head];
    }
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = b[j] < 0 || b[j] >= g.num_buckets ? 0.f : v[j] < kRelMasked ? -INFINITY : v[j] * g.inv_scale;
}
__device__ __forceinline__ float rel_entry(const RelGeo& g, int index, int head) {
    const int at[1] = {index};
    float v[1];
    rel_entries<1>(g, at, head, v);
    return v[0];
}
// The slice of offsets that the queries first .. last of a block reach over all keys (query), or the keys first .. last over all
// queries: entries lo .. lo + n - 1. Behind it in LDS, with a prefix: span + 1 copies of the entry of a prefix token on the other side,
// which that token's made-up code addresses like an offset (so it needs no test), the entry of a prefix token on the block's side, and
// that of a pair of them.
struct RelSlice {
    int lo, n, span, c0, c1;
    __device__ RelSlice(const RelGeo& g, int first, int last, bool query) {  // uniform arguments: kept in scalar registers
        c0 = __builtin_amdgcn_readfirstlane(rel_code(g, first));
        c1 = __builtin_amdgcn_readfirstlane(rel_code(g, last));
        const int cmax = __builtin_amdgcn_readfirstlane(rel_code(g, g.prefix + g.grid - 1));
        lo = (query ? c0 - cmax : -c1) + g.center;
        span = c1 - c0;
        n = span + cmax + 1;
    }
};
// All threads of the workgroup.
__device__ __forceinline__ void rel_expand(const RelGeo& g, float* T, const RelSlice& s, bool query, int head) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (opaque: nothing of this is worth a register in the loops around it)
    for (int i = tid; i < s.n; i += 4 * blockDim.x) {  // four entries' loads under way at once
        int at[4];
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            at[j] = i + j * (int)blockDim.x;
            at[j] = s.lo + (at[j] < s.n ? at[j] : s.n - 1);
        }
        rel_entries<4>(g, at, head, v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * (int)blockDim.x < s.n) T[i + j * (int)blockDim.x] = v[j];
    }
    if (g.prefix) {
        const float other = rel_entry(g, g.offsets + (query ? 1 : 0), head);
        for (int i = tid; i <= s.span; i += blockDim.x) T[s.n + i] = other;
        if (tid < 2) T[s.n + s.span + 1 + tid] = rel_entry(g, g.offsets + (tid ? 2 : query ? 0 : 1), head);
    }
}
// 4 * code of a row's token, rows being the side that is not the block's
__device__ __forceinline__ int rel_row_code(const RelGeo& g, const RelSlice& s, bool query, int token) {
    if (token < g.prefix) return 4 * (query ? s.c0 + g.center - s.lo - s.n : s.n + s.c1 - g.center + s.lo);
    return 4 * rel_code(g, token);
}

// Start values of a 32 x 32 product tile whose register e is row row0 + (e & 3) + 8 (e >> 2) + 4 hi and whose lane is the column.
// Everything is in bytes, so that an entry costs one subtraction and one read: `codes` are the 32 rows' codes in LDS; QLANE (the lane
// is the query, rows are keys): an entry is at `at` - code, otherwise at `at` + code.
typedef __attribute__((address_space(3))) const float* lds_float;
__device__ __forceinline__ int rel_lds(const float* T) { return (int)(uintptr_t)LDS_PTR((void*)T); }
template <bool QLANE>
struct RelLane {
    int at, mask, both;  // mask: 0 on a lane with a prefix token (`at` is then its entry, whatever the row); both: address of the pair's entry
    bool any;            // wave-uniform: the wave has such lanes
    __device__ RelLane() {}
    __device__ RelLane(const RelGeo& g, const RelSlice& s, const float* T, int token, int last) {
        const bool lp = token < g.prefix;
        const int c = rel_code(g, token < last ? token : last);
        at = rel_lds(T) + 4 * (lp ? s.n + s.span + 1 : g.center - s.lo + (QLANE ? c : -c));
        mask = lp ? 0 : -1;
        both = __builtin_amdgcn_readfirstlane(rel_lds(T) + 4 * (s.n + s.span + 2));
        any = __any(lp);
    }
};
template <bool QLANE>
__device__ __forceinline__ void rel_tile(f32x16& s, const int* codes, const RelLane<QLANE>& l, int hi, int prefix, int row0) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    int c[16];
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
        const i32x4 v = *(const i32x4*)(codes + 8 * g4 + 4 * hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) c[g4 * 4 + j] = v[j];
    }
    if (l.any) {
        int lim = prefix - row0 - 4 * hi;
        asm volatile("" : "+v"(lim));  // (opaque: 16 lane masks would be hoisted into 32 SGPRs)
        if (l.mask) lim = -64;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int m = c[e] & l.mask, at = QLANE ? l.at - m : l.at + m;
            s[e] = *(lds_float)(uintptr_t)((e & 3) + 8 * (e >> 2) < lim ? l.both : at);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = *(lds_float)(uintptr_t)(QLANE ? l.at - c[e] : l.at + c[e]);
    }
}

// ---- A row's level: what its probabilities are taken against, p = 2^(s c - level), s a raw score (product + bias / scale), c = scale log2 e.
// It is held in two parts, level = M c + m. A row has M = 0 and m = its running maximum, rounded: fma(s, c, -m) takes it off the unrounded
// s c, and what m was rounded by is a factor of the whole row that the sum of the row has too. But that factor is 2^(half an ulp of m): from
// |m| = 2^31 on it leaves fp32's range (every key of the row at a finite mask of -1e10, say: NaN or zeros). So a row further than kRelFar
// from zero has M = its raw maximum and m = 0: s - M is exact where p is not small. One subtraction a score, made only where a row of the wave
// needs it (`far`, wave-uniform).
constexpr float kRelFloor = -1e35f;    // a level never falls below this: masked scores (-inf) then have probability 0
constexpr float kRelFar = 16777216.f;  // 2^24: the factor is at most 2^0.5 up to here
struct RelLevel {
    float M = 0.f, m = kRelFloor;
    bool far = false;
    // how far (base 2) the row's scores, `mx` their largest, rise above the level
    __device__ __forceinline__ float excess(float mx, float c) const { return fmaf(mx - M, c, -m); }
    // the level of a row whose largest score so far is `mx`
    __device__ __forceinline__ void set(float mx, float c) {
        const float p = mx * c;
        const bool over = p > kRelFloor, f = over && fabsf(p) > kRelFar;
        M = f ? mx : 0.f;
        m = f ? 0.f : over ? p : kRelFloor;
        far = __any(f);
    }
    // raised to `mx` where that is above it (all lanes together); returns the factor of what was summed against the old one
    __device__ __forceinline__ float raise(float mx, float c) {
        const bool up = excess(mx, c) > 0.f;
        const float p = mx * c;
        const bool f = fabsf(p) > kRelFar;
        if (!far && !__any(up && f)) {
            const float m1 = fmaxf(m, p), factor = __builtin_amdgcn_exp2f(m - m1);
            m = m1;
            return factor;
        }
        const float M1 = up ? f ? mx : 0.f : M, m1 = up ? f ? 0.f : p : m;
        const float factor = __builtin_amdgcn_exp2f(fmaf(M - M1, c, m - m1));
        M = M1;
        m = m1;
        far = __any(M != 0.f);
        return factor;
    }
    // scores to exponents' arguments, in place
    __device__ __forceinline__ void arguments(f32x16& s, float c) const {
        if (far) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] -= M;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], c, -m);
    }
    // base-2 log-sum-exp from the row's sum
    __device__ __forceinline__ float log_sum(float sum, float c) const { return fmaf(M, c, m + log2f(sum)); }
};

// ---- The gradient's probabilities. P = 2^(s c - lse) from the forward's base-2 log-sum-exp is off by the factor 2^(lse's rounding, up to half
// an ulp) for the whole row: nothing up to |lse| = 2^8 (2^-17), 4 % at a finite mask of -1e6, any factor at -1e9. Rows beyond kRelFarSum
// therefore have their statistic in two parts, P = 2^((s - M) c - L) with M the row's raw maximum and L = log2 of its sum against M, made anew
// from the scores where dQ is made and handed to the other launches; every other row has M = 0, L = lse, and its one fma as before.
constexpr float kRelFarSum = 256.f;
__device__ __forceinline__ bool rel_far(float lse) { return fabsf(lse) > kRelFarSum && lse < INFINITY; }
// (M, L) of 32 queries on the lane (fragments qf) over all keys of their sample, read from memory tile by tile: the same instructions in the
// same order as in the products of the gradient, so the scores are theirs bit for bit (at 1e9 one ulp of a score is a factor of 2^92).
// One wave, no barrier; `bias` (rl's expansion) is complete.
template <int DH>
__device__ __forceinline__ void rel_far_rows(const RelGeo& g, const RelSlice& sl, const RelLane<true>& rl, const bf16x8 (&qf)[DH / 16],
                                             const unsigned char* keys, int pitch, int nb, int lane, float c, float& M, float& L) {
    const int r = lane & 31, hi = lane >> 5;
    float top = -INFINITY, sum = 0.f;
    for (int key0 = 0; key0 < nb; key0 += 32) {
        f32x16 s;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int token = key0 + (e & 3) + 8 * (e >> 2) + 4 * hi;
            const int at = rl.at - (rel_row_code(g, sl, true, token) & rl.mask);
            s[e] = *(lds_float)(uintptr_t)(token < g.prefix && !rl.mask ? rl.both : at);
        }
        const unsigned char* kp = keys + (size_t)(key0 + r < nb ? key0 + r : nb - 1) * pitch + hi * 16;
#pragma unroll
        for (int ks = 0; ks < DH / 16; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(kp + ks * 32), qf[ks], s, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (key0 + (e & 3) + 8 * (e >> 2) + 4 * hi >= nb) s[e] = -INFINITY;
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
        mx = fmaxf(top, max_across_halves(mx));
        const float base = mx > -INFINITY ? mx : 0.f;  // (no key so far: every probability 0)
        float add = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) add += __builtin_amdgcn_exp2f((s[e] - base) * c);
        sum = fmaf(sum, __builtin_amdgcn_exp2f((top - base) * c), add);
        top = mx;
    }
    sum += __shfl_xor(sum, 32, 64);
    M = top > -INFINITY ? top : 0.f;
    L = top > -INFINITY ? log2f(sum) : INFINITY;
}

// ---- host side
// Largest slice of offsets that a block of `block` consecutive tokens needs: all codes of the other side plus its own span
// (floats, with what stands behind the slice)
static inline int rel_slice_max(int gh, int gw, int block) {
    const int grid = gh * gw;
    const int max_code = (gh - 1) * (2 * gw - 1) + gw - 1;
    const int last = block - 1 < grid - 1 ? block - 1 : grid - 1;
    // a block that starts in column x > 0 spans one row border more than one that starts at 0
    const int borders = (last + gw - 1) / gw;
    int span = last + (borders < gh - 1 ? borders : gh - 1) * (gw - 1);
    if (span > max_code) span = max_code;
    return max_code + 2 * span + 4;
}
constexpr int kRelSliceCap = 16384;  // floats: 64 KiB of LDS
int rel_make_geo(const char* who, const vit_rel_pos* pos, const float* table, int heads, float scale, RelGeo* out, int* seq);
