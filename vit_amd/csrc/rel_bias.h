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

struct RelGeo {
    const float* table;    // [num_buckets, heads]
    const int* bucket_of;  // [offsets + 3] or null: the index itself
    int prefix, gw, grid, center, offsets, num_buckets, heads;
    float inv_scale;
};

constexpr float kRelMasked = -1e30f;  // a table entry below this masks its offset (a mask written as a type's lowest value)

__device__ __forceinline__ int rel_code(const RelGeo& g, int token) {
    int p = token - g.prefix;
    p = p < 0 ? 0 : p;
    p = p > g.grid - 1 ? g.grid - 1 : p;
    return p + (p / g.gw) * (g.gw - 1);
}
// bias of an offset index in units of the raw product (divided by the softmax scale): the start value of the product's
// accumulator, so that adding it costs nothing
__device__ __forceinline__ float rel_entry(const RelGeo& g, int index, int head) {
    const int b = g.bucket_of ? g.bucket_of[index] : index;
    if (b < 0 || b >= g.num_buckets) return 0.f;
    const float v = g.table[(size_t)b * g.heads + head];
    return v < kRelMasked ? -INFINITY : v * g.inv_scale;
}
// The block of LDS that one head's product tiles start from: entries lo .. lo + n - 1 of the offsets, then the three prefix
// entries. All threads of the workgroup.
__device__ __forceinline__ void rel_expand(const RelGeo& g, float* T, int lo, int n, int head) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) T[i] = rel_entry(g, lo + i, head);
    if (g.prefix && threadIdx.x < 3) T[n + threadIdx.x] = rel_entry(g, g.offsets + threadIdx.x, head);
}
// The slice that the queries first .. last of a block reach over all keys (QUERY), or the keys first .. last over all queries.
// lane_add / row_add make an index into it: query code + .. - key code, both sides' constant on the lane (QLANE) or the row.
struct RelSlice {
    int lo, n;
    __device__ RelSlice(const RelGeo& g, int first, int last, bool query) {
        const int c0 = rel_code(g, first), c1 = rel_code(g, last), cmax = rel_code(g, g.prefix + g.grid - 1);
        lo = (query ? c0 - cmax : -c1) + g.center;
        n = c1 - c0 + cmax + 1;
    }
};

// Start values of a 32 x 32 product tile whose register e is row row0 + (e & 3) + 8 (e >> 2) + 4 hi and whose lane is the column.
// QLANE: the lane is the query (rows are keys): index = lane_code - code; otherwise index = code - lane_code, where either the
// lane's or the rows' codes already hold center - lo. `codes`: the 32 rows' codes in LDS; n: the slice's length.
template <bool QLANE>
__device__ __forceinline__ void rel_tile(f32x16& s, const float* T, const int* codes, int lane_code, int hi, int prefix, int n, int lane_tok,
                                         int row0) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    if (row0 < prefix || __any(lane_tok < prefix)) {  // wave-uniform: only tiles that hold a prefix token
        int lim = prefix - row0 - 4 * hi;
        asm volatile("" : "+v"(lim));  // (opaque: 16 lane masks would be hoisted into 32 SGPRs)
        const bool lp = lane_tok < prefix;
        const int one = n + (lp ? (QLANE ? 0 : 1) : (QLANE ? 1 : 0));  // entry of a pair with a prefix row / without, by the lane's side
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const i32x4 c = *(const i32x4*)(codes + 8 * g4 + 4 * hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool rp = 8 * g4 + j < lim;
                int at = QLANE ? lane_code - c[j] : c[j] - lane_code;
                at = lp || rp ? one : at;
                at = lp && rp ? n + 2 : at;
                s[g4 * 4 + j] = T[at];
            }
        }
    } else {
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const i32x4 c = *(const i32x4*)(codes + 8 * g4 + 4 * hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[g4 * 4 + j] = T[QLANE ? lane_code - c[j] : c[j] - lane_code];
        }
    }
}

// ---- host side
// Largest slice of offsets that a block of `block` consecutive tokens needs: all codes of the other side plus its own span
// (floats, with the three prefix entries)
static inline int rel_slice_max(int gh, int gw, int block) {
    const int grid = gh * gw;
    const int max_code = (gh - 1) * (2 * gw - 1) + gw - 1;
    const int last = block - 1 < grid - 1 ? block - 1 : grid - 1;
    // a block that starts in column x > 0 spans one row border more than one that starts at 0
    int span = last + ((last + gw - 1) / gw) * (gw - 1);
    if (span > max_code) span = max_code;
    return max_code + span + 1 + 3;
}
constexpr int kRelSliceCap = 16384;  // floats: 64 KiB of LDS
int rel_make_geo(const char* who, const vit_rel_pos* pos, const float* table, int heads, float scale, RelGeo* out, int* seq);
