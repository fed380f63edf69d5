// Backward of attention with a learned relative position bias (attention_rel.hip; bias as in rel_bias.h):
//
//   s = scale q.k + bias,  P = exp2(s log2 e - lse),  dP = dO V^T,  delta = rowsum(dO * O),  dS = P * (dP - delta)
//   dQ = scale dS K,  dK = scale sum_heads dS^T Q,  dV = sum_heads P^T dO,  d_table[b, h] = sum of dS over (sample, i, j) in bucket b
//
// Launches, none with atomics (bitwise reproducible):
//   1 dQ: 32 queries a wave on the lane, keys streamed through LDS. delta from the wave's own rows of dO and O carries the
//     rounding of O and of the P that made it (about 2^-9), which is nothing beside dQ's own rounding but would stay in the
//     fp32 sums of dS that make d_table. Rows of the true dS sum to zero (the P of a row sum to 1), so the row sums of the dS
//     computed with the rounded delta, kept in fp32 beside the products, are its error: delta + sum is written for 2 and 3. Rows whose lse is
//     far from zero get their statistic again, in two parts (rel_bias.h), before the products: for this launch and for 2 and 3.
//   2 dK, dV: 32 keys a wave on the lane, the queries of every head of the group streamed through LDS.
//   3 bias: one block of (query, key) of one head and a range of samples per workgroup. The bias depends on the pair and not on the
//     sample, and so does the place of dS in its gradient: dS is summed over the samples in registers, and only the sum is folded by
//     offset (below) -- no scatter in the loop over samples. P and dP are computed again for it (2 products more).
//   4 offsets: adds the blocks' folded sums per offset in a fixed order; 5 (only with a map) adds the offsets of a bucket.
//
// Roundings: P and dS are rounded to bf16 for the products that make dQ, dK, dV (by at most 2^-8 of each, as P is in the forward: the matrix
// instructions take bf16 operands), and those when they are stored. d_table is made of the unrounded fp32 dS.
//
// Folding: pair (i, j) of a block has linear offset o = i - j, and the grid offset is dx = o mod gw (class 0: x_i >= dx, no row border
// between) or that - gw (class 1): 2 sums for each diagonal of the block, whatever the grid's width, then three for the prefix classes.
#include "lds_image.h"
#include "rel_bias.h"
#include <math.h>

// launches 1 and 2 in one pass where a head fits the LDS (attention_rel_bwd_dh64.hip)
bool attention_rel_bwd_dh64_eligible(int N, int heads, int kv_heads, int head_dim);
int launch_attention_rel_bwd_dh64(const RelGeo& geo, const void* qkv, const void* out, const void* dout, const float* lse, float* ndelta, float* rows,
                                  int* met, void* dqkv, const int* lengths, int batch, int N, int heads, float scale, hipStream_t stream);

namespace {

constexpr float LOG2E = 1.4426950408889634f;
enum { MODE_DQ = 0, MODE_DKV = 1 };

struct RelBwdArgs {
    const bf16_t* qkv;
    const bf16_t* out;
    const bf16_t* dout;
    const float* lse;
    float* ndelta;  // [B, H, N]: -delta
    float* rows;    // [2][B, H, N]: M and L of the rows (rel_bias.h). One pass: only where lse is far from zero
    bf16_t* dqkv;
    int* met;      // one pass: [workgroups][8]
    float* part;   // [splits][H][tq][tk][fp]: folded sums of the blocks
    float* doff;   // [H][offsets + 3] (with a map)
    float* dtable;
    const int* by_bucket;
    const int* bucket_start;
    const int* lengths;
    RelGeo geo;
    int B, N, H, HK;
    int splits, tq, tk, bq, bk, fp;  // bias gradient: sample ranges, query / key blocks, their sizes, pitch of their sums
    float scale, scale_log2e;
    __device__ float* row_M(int b, int h) const { return rows + ((size_t)b * H + h) * N; }
    __device__ float* row_L(int b, int h) const { return rows + ((size_t)(B + b) * H + h) * N; }
};

__device__ __forceinline__ bf16x8 pack8b(const f32x16& p, int s) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16_t)p[8 * s + e];
    return o;
}
__device__ __forceinline__ int sample_length(const int* lengths, int b, int N) {
    if (!lengths) return N;
    const int n = lengths[b];
    return n < 0 ? 0 : n > N ? N : n;
}

// Buffers of a chunk of 32 inner rows: two images, (L, -delta, M) of queries, codes; a multiple of 256 (LdsImage::step)
constexpr int CR = 32;
template <int DH, int MODE>
constexpr int chunk_bytes() { return 2 * CR * LdsImage<DH>::ROW + (MODE == MODE_DKV ? 512 : 256); }

// One chunk's products, for 32 outer rows on the lane: `buf` its buffer (at LDS address img; ro: of the lane's first row piece). DQ: oL the
// second part of the row's statistic; far: the wave has rows with a first part, which stands in LDS at Mr (not worth a register)
template <int DH, int MODE>
__device__ __forceinline__ void chunk_products(const RelBwdArgs& a, const unsigned char* buf, int img, int ro, const TrRead<DH>& tr,
                                               const RelLane<MODE == MODE_DQ>& rl, const bf16x8 (&f1)[DH / 16], const bf16x8 (&f2)[DH / 16], bool far,
                                               const float* Mr, float oL, float oD, f32x16 (&acc1)[(DH + 31) / 32],
                                               f32x16 (&acc2)[(DH + 31) / 32], float& dsum, int row0, int nb, int hi) {
    using I = LdsImage<DH>;
    constexpr int KS = DH / 16, DB = (DH + 31) / 32, IMG = CR * I::ROW, BUF = chunk_bytes<DH, MODE>();
    f32x16 s, dp;
    rel_tile(s, (const int*)(buf + BUF - CR * 4), rl, hi, a.geo.prefix, row0);
    if constexpr (MODE == MODE_DQ) {
        // (from zero here and for the bias, delta taken off behind the products: what the matrix instructions cut off their sums is then
        // the same in both, and delta's correction holds it. Started from -delta they left
        // d_table 1.7e-6 off with 12 x 1001 tokens in 8 buckets, 7e-7 now.)
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = 0.f;
    } else {  // (from -delta: a cut-off of 2^-24 is nothing beside the rounding of these sums to bf16)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const f32x4 Dl = *(const f32x4*)(buf + 2 * IMG + CR * 4 + (8 * g4 + 4 * hi) * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) dp[g4 * 4 + j] = Dl[j];
        }
    }
    int ka = ro;
    asm volatile("" : "+v"(ka));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_chunk(I::step(ka, ks)), f1[ks], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_chunk(I::step(ka, ks) + IMG), f2[ks], dp, 0, 0, 0);
    }
    if (row0 + CR > nb) {
        int lim = nb - row0 - 4 * hi;
        asm volatile("" : "+v"(lim));
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if ((e & 3) + 8 * (e >> 2) >= lim) s[e] = -INFINITY;
    }
    if constexpr (MODE == MODE_DQ) {
        if (far) {
            int tid = threadIdx.x;
            asm volatile("" : "+v"(tid));
            const float M = Mr[tid & 31];
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] -= M;
        }
    } else {
        const float* const Ms = (const float*)(buf + 2 * IMG + 2 * CR * 4);
        if (__any(Ms[threadIdx.x & 31] != 0.f)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] -= Ms[(e & 3) + 8 * (e >> 2) + 4 * hi];
        }
    }
    const unsigned t1 = (unsigned)img, t2 = t1 + IMG;
    bf16x8 xt[DB];
    if constexpr (MODE == MODE_DQ) {
        tr.template read_step<0>(xt, t1);
        float sum = 0.f;  // (a chunk's terms first: fewer roundings at the size of the row's sum)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -oL));  // P^T
            dp[e] -= oD;
            sum = fmaf(s[e], dp[e], sum);
        }
        dsum += sum;
        if (nb <= CR) {
            // All of the row is here: delta's error leaves dS before it is rounded. (With few keys it is a large part of dS, up to twice
            // dQ's rounding for 3 keys; with more than a chunk of them it is below a twentieth.)
            const float err = dsum + __shfl_xor(dsum, 32, 64);
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] -= err;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= dp[e];  // dS^T
        const bf16x8 x0 = pack8b(s, 0), x1 = pack8b(s, 1);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc1[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[d], x0, acc1[d], 0, 0, 0);
        tr.template read_step<1>(xt, t1);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc1[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[d], x1, acc1[d], 0, 0, 0);
    } else {
        tr.template read_step<0>(xt, t2);
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const f32x4 L = *(const f32x4*)(buf + 2 * IMG + (8 * g4 + 4 * hi) * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = g4 * 4 + j;
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -L[j]));  // P
                dp[e] *= s[e];                                                    // dS
            }
        }
        const bf16x8 p0 = pack8b(s, 0), p1 = pack8b(s, 1), d0 = pack8b(dp, 0), d1 = pack8b(dp, 1);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc2[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[d], p0, acc2[d], 0, 0, 0);
        tr.template read_step<1>(xt, t2);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc2[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[d], p1, acc2[d], 0, 0, 0);
        tr.template read_step<0>(xt, t1);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc1[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[d], d0, acc1[d], 0, 0, 0);
        tr.template read_step<1>(xt, t1);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc1[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[d], d1, acc1[d], 0, 0, 0);
    }
}

// what the registers allow without a spill (a spilled register's reload waits for all loads under way)
constexpr int bwd_waves_per_simd(int dh, int mode) { return mode == MODE_DQ ? (dh <= 96 ? 3 : 2) : dh <= 64 ? 3 : dh <= 96 ? 2 : 1; }
// A workgroup of up to 4 waves takes 32 outer rows a wave of one (sample, head); the inner rows come in chunks of 32 by LDS-DMA into two
// buffers, the next chunk under the products of this one, in images that serve row reads and transposed reads alike. 4 x 1025 tokens, 16
// heads of 80: dQ 71 us, dK and dV 75 us, bound by the steps' chains (4400 cycles at three waves a SIMD, 5500 at two, of which the next
// chunk's loads take 800 to 1300: spread over the products they cost more). Whole sequences staged at once took 1.5 and 1.7 times as long.
template <int DH, int MODE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(bwd_waves_per_simd(DH, MODE)))) void attn_rel_bwd_kernel(const RelBwdArgs a) {
    using I = LdsImage<DH>;
    constexpr int KS = DH / 16, DB = (DH + 31) / 32, IMG = CR * I::ROW, BUF = chunk_bytes<DH, MODE>();
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    float* const T = (float*)(smem + 2 * BUF);
    const int lds0 = (int)(uintptr_t)LDS_PTR(smem);
    const int N = a.N, H = a.H, HK = a.HK;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
    const int r = lane & 31, hi = lane >> 5;
    const int OH = MODE == MODE_DQ ? H : HK;  // outer heads
    const int b = blockIdx.x / OH, oh = blockIdx.x - b * OH, group = H / HK;
    const int pitch = (H + 2 * HK) * DH * 2, opitch = H * DH * 2;
    const int nb = __builtin_amdgcn_readfirstlane(sample_length(a.lengths, b, N));
    // with lengths the last blocks first (only long samples have them), else last (the sequence may end inside one)
    const int blk0 = (a.lengths ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * nw * 32;
    const int blk1 = min(blk0 + nw * 32, N) - 1;
    const int o0 = blk0 + wave * 32, row = o0 + r;
    const unsigned char* base = (const unsigned char*)a.qkv + (size_t)b * N * pitch;
    const unsigned char* gbase = (const unsigned char*)a.dout + (size_t)b * N * opitch;
    const int hk = MODE == MODE_DQ ? oh / group : oh;
    const int nheads = MODE == MODE_DQ ? 1 : group;
    const int nc = blk0 < nb ? (nb + CR - 1) / CR : 0, steps = nc * nheads;
    const RelSlice sl(a.geo, blk0, blk1, MODE == MODE_DQ);  // over all keys / all queries

    const LdsFill<DH> fill(lane);
    auto stage = [&](int step, int h, int c) {
        const int row0 = c * CR;
        unsigned char* const dst = smem + (step & 1) * BUF;
        // rows behind the sample re-read its last one: what is masked is still finite
        const __amdgpu_buffer_rsrc_t r1 = head_resource<DH>(base + (size_t)(MODE == MODE_DQ ? H + hk : h) * DH * 2, N, pitch);
        const __amdgpu_buffer_rsrc_t r2 = MODE == MODE_DQ ? head_resource<DH>(base + (size_t)(H + HK + hk) * DH * 2, N, pitch)
                                                          : head_resource<DH>(gbase + (size_t)h * DH * 2, N, opitch);
        int ln = lane;
        asm volatile("" : "+v"(ln));  // (opaque: what follows is made here, not kept in registers over the products)
        fill.chunk(r1, dst, CR, wave, nw, row0, nb - 1, pitch);
        fill.chunk(r2, dst + IMG, CR, wave, nw, row0, nb - 1, MODE == MODE_DQ ? pitch : opitch);
        if constexpr (MODE == MODE_DKV) {
            if (wave == 0) {  // the queries' L, -delta and M
                int q = row0 + ln;
                q = q < nb ? q : nb - 1;
                auto row_values = [&](const float* p, int place) {
                    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (unsigned)N * 4, 0x00020000);
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(dst + 2 * IMG + place * CR * 4), 4, q * 4, 0, 0, 0);
                };
                if (ln < CR) {
                    row_values(a.row_L(b, h), 0);
                    row_values(a.ndelta + ((size_t)b * H + h) * N, 1);
                    row_values(a.row_M(b, h), 2);
                }
            }
        }
        if (ln < CR && wave == nw - 1) *(int*)(dst + BUF - CR * 4 + ln * 4) = rel_row_code(a.geo, sl, MODE == MODE_DQ, row0 + ln);
    };
    if (steps > 0) stage(0, MODE == MODE_DQ ? oh : oh * group, 0);

    // ---- outer fragments
    const int orow = row < nb ? row : (nb > 0 ? nb - 1 : 0);
    bf16x8 f1[KS], f2[KS];
    float oL = INFINITY, oD = 0.f;
    if constexpr (MODE == MODE_DQ) {
        const size_t at = ((size_t)b * N + orow) * opitch + (size_t)oh * DH * 2 + hi * 16;
        float d = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            f1[ks] = *(const bf16x8*)(base + (size_t)orow * pitch + (size_t)oh * DH * 2 + ks * 32 + hi * 16);
            f2[ks] = *(const bf16x8*)((const unsigned char*)a.dout + at + ks * 32);
            const bf16x8 ov = *(const bf16x8*)((const unsigned char*)a.out + at + ks * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) d = fmaf((float)f2[ks][e], (float)ov[e], d);
        }
        oD = d + __shfl_xor(d, 32, 64);
        if (row < nb) oL = a.lse[((size_t)b * H + oh) * N + row]; else oD = 0.f;
    } else {
        const unsigned char* kp = base + (size_t)orow * pitch + (size_t)(H + hk) * DH * 2 + hi * 16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            f1[ks] = *(const bf16x8*)(kp + ks * 32);
            f2[ks] = *(const bf16x8*)(kp + (size_t)HK * DH * 2 + ks * 32);
        }
    }
    rel_expand(a.geo, T, sl, MODE == MODE_DQ, MODE == MODE_DQ ? oh : oh * group);
    const RelLane<MODE == MODE_DQ> rl(a.geo, sl, T, row, N - 1);
    const TrRead<DH> tr(lane);
    float* const Mr = T + sl.n + sl.span + 3 + wave * 32;
    bool far = false;  // DQ: the wave has rows of the two-part statistic
    if constexpr (MODE == MODE_DQ) {
        const bool f = rel_far(oL);
        far = __any(f);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");  // T is whole
        if (far) {
            float M, L;
            rel_far_rows<DH>(a.geo, sl, rl, f1, base + (size_t)(H + hk) * DH * 2, pitch, nb, lane, a.scale_log2e, M, L);
            if (f) oL = L;
            Mr[r] = f ? M : 0.f;  // (both halves of the wave write it)
        }
    }
    const int ro = lds0 + I::at(r, hi);
    f32x16 acc1[DB], acc2[DB];  // DQ: acc1 = dQ^T.  DKV: acc1 = dK^T, acc2 = dV^T
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) { acc1[d][e] = 0.f; acc2[d][e] = 0.f; }
    float dsum = 0.f;  // DQ: row sum of dS
    int c = 0, head = MODE == MODE_DQ ? oh : oh * group;
    for (int step = 0; step < steps; ++step) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");  // the chunk is whole; nobody reads the other buffer (and at c = 0 T) any more
        if (MODE == MODE_DKV && c == 0 && step > 0) {  // the next head of the group
            rel_expand(a.geo, T, sl, false, head);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            asm volatile("s_barrier" ::: "memory");
        }
        if (step + 1 < steps) stage(step + 1, c + 1 == nc ? head + 1 : head, c + 1 == nc ? 0 : c + 1);
        const int img = (step & 1) * BUF, row0 = c * CR;
        const unsigned char* const buf = smem + img;
        chunk_products<DH, MODE>(a, buf, lds0 + img, ro + img, tr, rl, f1, f2, far, Mr, oL, oD, acc1, acc2, dsum, row0, nb, hi);
        if (++c == nc) { c = 0; ++head; }
    }
    if constexpr (MODE == MODE_DQ) {
        dsum += __shfl_xor(dsum, 32, 64);
        if (row < N && hi == 0) {
            a.ndelta[((size_t)b * H + oh) * N + row] = oL < INFINITY ? -(oD + dsum) : 0.f;
            a.row_M(b, oh)[row] = far ? Mr[r] : 0.f;
            a.row_L(b, oh)[row] = oL;
        }
    }
    // ---- store (rows behind the sample's length: zeros)
    if (row < N) {
        const bool live = row < nb;
        bf16_t* dst = a.dqkv + (((size_t)b * N + row) * (H + 2 * HK) + (MODE == MODE_DQ ? oh : H + oh)) * DH;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int d0 = d * 32 + 8 * g4 + 4 * hi;
                if (d0 < DH) {
                    bf16x4 v, w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = (bf16_t)(live ? acc1[d][g4 * 4 + e] * a.scale : 0.f);
                        w[e] = (bf16_t)(live ? acc2[d][g4 * 4 + e] : 0.f);
                    }
                    *(bf16x4*)(dst + d0) = v;
                    if constexpr (MODE == MODE_DKV) *(bf16x4*)(dst + (size_t)HK * DH + d0) = w;
                }
            }
    }
}

// ---- sums of dS over samples, folded by offset. Grid: (query blocks * key blocks, H, splits). A wave has 32 queries and KT tiles of
// 32 keys; K and V of the block's keys come by LDS-DMA one sample ahead (two buffers), the wave's own Q and dO rows one sample ahead
// in registers, so a sample costs one barrier and its loads have a sample's products to land. 256 x 197 tokens, 12 heads of 64: 115 us,
// 4 x 1025, 16 heads of 80: 98 us (of a workgroup's 80 000 cycles there 17 000 go by before the first product, 10 000 in the fold). Folded a
// strip of 32 keys at a time by the whole workgroup it took 1.1 and 1.25 times as long.
template <int DH, int KT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void attn_rel_bias_grad_kernel(const RelBwdArgs a) {
    using I = LdsImage<DH>;
    constexpr int KS = DH / 16, ROWS = KT * 32, IMG = ROWS * I::ROW;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    // [2][K image, V image], the keys' codes, the expansion; after the samples what the fold needs
    int* const codes = (int*)(smem + 4 * IMG);
    float* const T = (float*)(codes + ROWS);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
    const int r = lane & 31, hi = lane >> 5;
    const int N = a.N, H = a.H, HK = a.HK, B = a.B;
    const int tq = blockIdx.x / a.tk, tk = blockIdx.x - tq * a.tk;
    const int h = blockIdx.y, hk = h / (H / HK);
    const int blk0 = tq * nw * 32, q0 = blk0 + wave * 32, q = q0 + r, k0 = tk * ROWS;
    const int pitch = (H + 2 * HK) * DH * 2, opitch = H * DH * 2;
    const int b0 = (int)((int64_t)B * blockIdx.z / a.splits), b1 = (int)((int64_t)B * (blockIdx.z + 1) / a.splits);
    const int blk1 = blk0 + nw * 32 < N ? blk0 + nw * 32 - 1 : N - 1;

    auto next_sample = [&](int b) {  // the first from b on that has a pair in this block
        while (b < b1) {
            const int nb = sample_length(a.lengths, b, N);
            if (nb > blk0 && nb > k0) break;
            ++b;
        }
        return b;
    };
    // a part of a sample's loads: this wave's pieces i0, i0 + 1 .. of the K and V images, part of its query rows
    const int pieces = (ROWS + nw * I::RPI - 1) / (nw * I::RPI);  // a wave has per image
    auto stage = [&](int b, int nb, int buf, int i0, int i1) {
        const char* base = (const char*)a.qkv + (size_t)b * N * pitch + (size_t)(H + hk) * DH * 2;
        const __amdgpu_buffer_rsrc_t kr = head_resource<DH>(base, N, pitch), vr = head_resource<DH>(base + (size_t)HK * DH * 2, N, pitch);
        unsigned char* const dst = smem + buf * 2 * IMG;
        // whole tiles up to the sample's last key (rows behind it re-read that key: what is masked is still finite)
        const int need = nb - k0 < ROWS ? (nb - k0 + 31) & ~31 : ROWS;
        int ln = lane;
        asm volatile("" : "+v"(ln));  // (opaque: the lane offsets are made here, not kept in registers over the products)
        for (int i = i0; i < i1; ++i) {
            const int row = (i * nw + wave) * I::RPI;
            if (row < need) {
                I::dma(kr, dst, row, ROWS, k0, nb - 1, pitch, ln);
                I::dma(vr, dst + IMG, row, ROWS, k0, nb - 1, pitch, ln);
            }
        }
    };
    bf16x8 fq[KS], fo[KS], nq[KS], no[KS];
    float L = INFINITY, D = 0.f, nL = INFINITY, nD = 0.f;
    auto load_rows = [&](int b, int nb, int ks0, int ks1) {
        int ql = q;
        asm volatile("" : "+v"(ql));
        const int qr = ql < nb ? ql : nb - 1;
        const char* qp = (const char*)a.qkv + (size_t)b * N * pitch + (size_t)h * DH * 2;  // (uniform bases, 32-bit lane offsets)
        const char* op = (const char*)a.dout + (size_t)b * N * opitch + (size_t)h * DH * 2;
        const unsigned qo = (unsigned)(qr * pitch + hi * 16), oo = (unsigned)(qr * opitch + hi * 16);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            if (ks < ks0 || ks >= ks1) continue;
            nq[ks] = *(const bf16x8*)(qp + qo + ks * 32);
            no[ks] = *(const bf16x8*)(op + oo + ks * 32);
        }
        if (ks1 == KS) {
            const size_t at = ((size_t)b * H + h) * N;
            nL = (a.lse + at)[qr];
            nD = (a.ndelta + at)[qr];
        }
    };
    f32x16 acc[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;

    int b = next_sample(b0), buf = 0;
    int nb = b < b1 ? sample_length(a.lengths, b, N) : 0;
    if (b < b1) {
        load_rows(b, nb, 0, KS);
        stage(b, nb, 0, 0, pieces);
    }
    const RelSlice sl(a.geo, blk0, blk1, true);  // (under the first sample's loads)
    rel_expand(a.geo, T, sl, true, h);
    for (int i = tid; i < ROWS; i += blockDim.x) codes[i] = rel_row_code(a.geo, sl, true, k0 + i);
    const RelLane<true> rl(a.geo, sl, T, q, N - 1);
    bool far = false;  // the wave has met rows of the two-part statistic
    while (b < b1) {
        const int bn = next_sample(b + 1), nnb = bn < b1 ? sample_length(a.lengths, bn, N) : 0;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // this sample's images are whole; nobody reads the other buffer any more
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { fq[ks] = nq[ks]; fo[ks] = no[ks]; }
        const bool f = rel_far(nL);
        far |= __any(f);
        L = f ? INFINITY : nL;  // P = exp2(.. - inf) = 0 for rows that come behind the loop
        D = nD;
        const unsigned char* Kb = smem + buf * 2 * IMG;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int key0 = k0 + t * 32;
            if (bn < b1) {  // the next sample's loads, some a tile: all at once they would block the wave at the CU's memory queue
                load_rows(bn, nnb, t * KS / KT, (t + 1) * KS / KT);
                stage(bn, nnb, buf ^ 1, t * pieces / KT, (t + 1) * pieces / KT);
            }
            if (q0 < nb && key0 < nb) {
                f32x16 s, dp;
                rel_tile(s, codes + t * 32, rl, hi, a.geo.prefix, key0);
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const int off = I::at(t * 32 + r, ks * 2 + hi);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(Kb + off), fq[ks], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(Kb + IMG + off), fo[ks], dp, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -L));
                    dp[e] += D;
                }
                if (key0 + 32 > nb || (nb < N && q0 + 32 > nb)) {
                    // pairs behind the sample, chosen and not made zero by P alone: what is made of its last rows may be NaN (queries behind
                    // the longest sample there can be: once, in the fold)
                    int lim = q < nb ? nb - key0 - 4 * hi : -64;
                    asm volatile("" : "+v"(lim));
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool on = (e & 3) + 8 * (e >> 2) < lim;
                        s[e] = on ? s[e] : 0.f;
                        dp[e] = on ? dp[e] : 0.f;
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][e] = fmaf(s[e], dp[e], acc[t][e]);
            }
        }
        b = bn;
        nb = nnb;
        buf ^= 1;
    }

    // ---- rows whose lse is far from zero, against their two-part statistic; slow, from memory (no barrier)
    if (far) {
        for (b = next_sample(b0); b < b1; b = next_sample(b + 1)) {
            nb = sample_length(a.lengths, b, N);
            L = q < nb ? a.lse[((size_t)b * H + h) * N + q] : INFINITY;
            const bool f = rel_far(L);
            if (!__any(f)) continue;
            load_rows(b, nb, 0, KS);
            float M = 0.f;
            L = INFINITY;
            if (f) {
                M = a.row_M(b, h)[q];
                L = a.row_L(b, h)[q];
            }
            const unsigned char* kv = (const unsigned char*)a.qkv + (size_t)b * N * pitch + (size_t)(H + hk) * DH * 2 + hi * 16;
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const int key0 = k0 + t * 32;
                if (key0 >= nb) break;
                const unsigned char* kp = kv + (size_t)(key0 + r < nb ? key0 + r : nb - 1) * pitch;
                f32x16 s, dp;
                rel_tile(s, codes + t * 32, rl, hi, a.geo.prefix, key0);
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(kp + ks * 32), nq[ks], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(kp + (size_t)HK * DH * 2 + ks * 32), no[ks], dp, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool on = f && key0 + (e & 3) + 8 * (e >> 2) + 4 * hi < nb;
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[e] - M, a.scale_log2e, -L)), d = dp[e] + nD;
                    acc[t][e] = fmaf(on ? p : 0.f, on ? d : 0.f, acc[t][e]);
                }
            }
        }
    }

    // ---- fold. Each wave its own 32 x 32 tiles through LDS: lane (r, hi) adds the pairs (i, j = (i + r) mod 32), i = 16 hi .. 16 hi + 15,
    // which lie on two diagonals, i - j = -r and, past the tile's edge, 32 - r; the first of tile t is the second of tile t + 1.
    float* const S = (float*)smem + wave * (32 * 33);  // [32][33]
    float* const V = (float*)smem + nw * (32 * 33);    // [nw][KT + 1][class][32]: offset q0 - k0 + 32 - 32 slot - r
    float* const P3 = V + nw * (KT + 1) * 64;          // [nw][3]
    const int prefix = a.geo.prefix, gw = a.geo.gw;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, c0 = 0.f, c1 = 0.f;
    auto modw = [&](int v) {
        v %= gw;
        return v < 0 ? v + gw : v;
    };
    auto emit = [&](int slot, float v0, float v1) {
        v0 += __shfl_xor(v0, 32, 64);
        v1 += __shfl_xor(v1, 32, 64);
        V[((wave * (KT + 1) + slot) * 2 + hi) * 32 + r] = hi ? v1 : v0;
    };
    __syncthreads();
    const int x0 = modw(q0 + 16 * hi - prefix);  // column of the lane's first query (a prefix token's is not used)
    int dx = modw(q0 - k0 - r), dx2 = modw(q0 - k0 + 32 - r);
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        __builtin_amdgcn_wave_barrier();  // (the last tile's reads come first)
#pragma unroll
        for (int e = 0; e < 16; ++e) S[r * 33 + (e & 3) + 8 * (e >> 2) + 4 * hi] = q < N ? acc[t][e] : 0.f;
        __builtin_amdgcn_wave_barrier();
        float a10 = 0.f, a11 = 0.f, a20 = 0.f, a21 = 0.f;
        if (q0 < prefix || k0 + t * 32 < prefix) {  // a tile with prefix tokens: those pairs in three sums of their own
            const int lq = prefix - q0, lk = prefix - (k0 + t * 32);
            int x = x0;
            for (int n = 0; n < 16; ++n) {
                const int i = 16 * hi + n, j = (i + r) & 31;
                const float v = S[i * 33 + j];
                const bool grid = i >= lq && j >= lk, wrap = i + r >= 32, low = x >= (wrap ? dx2 : dx);
                a10 += grid && !wrap && low ? v : 0.f;
                a11 += grid && !wrap && !low ? v : 0.f;
                a20 += grid && wrap && low ? v : 0.f;
                a21 += grid && wrap && !low ? v : 0.f;
                s0 += i < lq && j >= lk ? v : 0.f;
                s1 += i >= lq && j < lk ? v : 0.f;
                s2 += i < lq && j < lk ? v : 0.f;
                x = x + 1 == gw ? 0 : x + 1;
            }
        } else {
            int x = x0;
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                const int i = 16 * hi + n;
                const float v = S[i * 33 + ((i + r) & 31)];
                const bool wrap = i + r >= 32, low = x >= (wrap ? dx2 : dx);
                const float v0 = low ? v : 0.f, v1 = low ? 0.f : v;
                a10 += wrap ? 0.f : v0;
                a11 += wrap ? 0.f : v1;
                a20 += wrap ? v0 : 0.f;
                a21 += wrap ? v1 : 0.f;
                x = x + 1 == gw ? 0 : x + 1;
            }
        }
        emit(t, c0 + a20, c1 + a21);
        c0 = a10, c1 = a11;
        dx2 = dx;
        dx = modw(dx - 32);
    }
    emit(KT, c0, c1);
    if (prefix > 0) {
        s0 = wave_sum(s0);
        s1 = wave_sum(s1);
        s2 = wave_sum(s2);
    }
    if (lane == 0) { P3[wave * 3] = s0; P3[wave * 3 + 1] = s1; P3[wave * 3 + 2] = s2; }
    __syncthreads();
    const int fold = 2 * (nw * 32 + ROWS - 1);  // place v: offset blk0 - k0 + v - (ROWS - 1)
    float* dst = a.part + ((((size_t)blockIdx.z * H + h) * a.tq + tq) * a.tk + tk) * a.fp;
    for (int i = tid; i < fold; i += blockDim.x) {
        const int o = (i >> 1) - (ROWS - 1), m = (o + 32 * KT + 31) / 32 - KT;  // o = 32 m - r
        float v = 0.f;
        for (int w = 0; w < nw; ++w) {
            const int slot = w + 1 - m;
            if (slot >= 0 && slot <= KT) v += V[((w * (KT + 1) + slot) * 2 + (i & 1)) * 32 + 32 * m - o];
        }
        dst[i] = v;
    }
    if (tid < 3) {
        float v = 0.f;
        for (int w = 0; w < nw; ++w) v += P3[w * 3 + tid];
        dst[fold + tid] = v;
    }
}

// ---- per offset: the blocks' folded sums in a fixed order. A lane has an offset index (neighbours read neighbours) of one head, a
// workgroup's waves share its (split, query block) pairs
constexpr int kOffsetWaves = 16;
__global__ __launch_bounds__(64 * kOffsetWaves) void attn_rel_offset_kernel(const RelBwdArgs a, float* dst, int stride_h, int stride_o) {
    __shared__ float sums[kOffsetWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int idx = blockIdx.x * 64 + lane, h = blockIdx.y;
    const int offsets = a.geo.offsets, all = offsets + (a.geo.prefix ? 3 : 0);
    const int gw = a.geo.gw, rows = 2 * gw - 1;
    const int dyi = idx / rows, dx = idx - dyi * rows - (gw - 1), dy = dyi - (a.geo.center / rows);
    const int o = dy * gw + dx, cls = dx < 0 ? 1 : 0;
    const int bq = a.bq, bk = a.bk, fold = bq + bk - 1;  // queries, keys of a block, diagonals
    float s = 0.f;
    if (idx < offsets) {
        for (int i = wave; i < a.splits * a.tq; i += kOffsetWaves) {
            const int sp = i / a.tq, tq = i - sp * a.tq;
            const float* p = a.part + (((size_t)sp * a.H + h) * a.tq + tq) * a.tk * a.fp;
            // key blocks that hold a key i - o of the block's queries
            const int j0 = tq * bq - o, j1 = j0 + bq - 1;  // keys of its first and last query
            const int t0 = j0 > 0 ? j0 / bk : 0, t1 = j1 < 0 ? -1 : j1 / bk;
            for (int tk = t0; tk <= t1 && tk < a.tk; ++tk) s += p[(size_t)tk * a.fp + 2 * (o - (tq * bq - tk * bk) + bk - 1) + cls];
        }
    } else if (idx < all) {  // the prefix classes: only the first blocks have any
        for (int i = wave; i < a.splits * a.tq; i += kOffsetWaves) {
            const int sp = i / a.tq, tq = i - sp * a.tq;
            const float* p = a.part + (((size_t)sp * a.H + h) * a.tq + tq) * a.tk * a.fp;
            for (int tk = 0; tk < (tq == 0 ? a.tk : 1); ++tk) s += p[(size_t)tk * a.fp + 2 * fold + idx - offsets];
        }
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave > 0 || idx >= all) return;
    s = 0.f;
#pragma unroll
    for (int w = 0; w < kOffsetWaves; ++w) s += sums[w][lane];
    dst[(size_t)h * stride_h + (size_t)idx * stride_o] = s;
}
// ---- per bucket: its offsets' sums in the map's order
__global__ __launch_bounds__(256) void attn_rel_bucket_kernel(const RelBwdArgs a) {
    const int lane = threadIdx.x & 63;
    const int bucket = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y;
    if (bucket >= a.geo.num_buckets) return;
    const int total = a.geo.offsets + (a.geo.prefix ? 3 : 0);
    float s = 0.f;
    if (a.geo.bucket_of) {
        int i0 = a.bucket_start[bucket], i1 = a.bucket_start[bucket + 1];
        i0 = i0 < 0 ? 0 : i0;
        i1 = i1 > total ? total : i1;
        for (int i = i0 + lane; i < i1; i += 64) {
            const int at = a.by_bucket[i];
            if (at >= 0 && at < total) s += a.doff[(size_t)h * total + at];
        }
    } else if (lane == 0 && bucket < total) {
        s = a.doff[(size_t)h * total + bucket];
    }
    s = wave_sum(s);
    if (lane == 0) a.dtable[(size_t)bucket * a.H + h] = s;
}

// ---- the same for few outer rows: a workgroup has 32 of them, its waves share the inner chunks (wave w takes w, w + waves, .., each through
// its own buffer, no barrier between), and their sums are added through LDS.
constexpr int split_waves_most(int dh, int mode) { return mode == MODE_DKV && dh > 96 ? 4 : 8; }  // (two waves a SIMD have 256 registers each)
template <int DH, int MODE>
__global__ __launch_bounds__(64 * split_waves_most(DH, MODE)) void attn_rel_bwd_split_kernel(const RelBwdArgs a, int tile0) {
    using I = LdsImage<DH>;
    constexpr int KS = DH / 16, DB = (DH + 31) / 32, IMG = CR * I::ROW, BUF = chunk_bytes<DH, MODE>(), OUT = MODE == MODE_DQ ? 3 : 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
    const int r = lane & 31, hi = lane >> 5;
    unsigned char* const rows = smem + (size_t)nw * BUF;  // images of the outer rows: DQ Q, dO, O;  DKV K, V
    float* const sums = (float*)(rows + OUT * IMG);       // [nw][32]: DQ the waves' row sums of dS
    float* const T = sums + nw * 32;
    unsigned char* const buf = smem + (size_t)wave * BUF;
    const int img = (int)(uintptr_t)LDS_PTR(buf);
    const int N = a.N, H = a.H, HK = a.HK;
    const int OH = MODE == MODE_DQ ? H : HK;  // outer heads
    const int b = blockIdx.x / OH, oh = blockIdx.x - b * OH, group = H / HK;
    const int pitch = (H + 2 * HK) * DH * 2, opitch = H * DH * 2;
    const int nb = __builtin_amdgcn_readfirstlane(sample_length(a.lengths, b, N));
    const int o0 = (tile0 + blockIdx.y) * 32, row = o0 + r;
    const unsigned char* base = (const unsigned char*)a.qkv + (size_t)b * N * pitch;
    const unsigned char* gbase = (const unsigned char*)a.dout + (size_t)b * N * opitch;
    const int hk = MODE == MODE_DQ ? oh / group : oh, head0 = MODE == MODE_DQ ? oh : oh * group;
    const int nheads = MODE == MODE_DQ ? 1 : group;
    const int nc = o0 < nb ? (nb + CR - 1) / CR : 0;
    const RelSlice sl(a.geo, o0, min(o0 + 31, N - 1), MODE == MODE_DQ);
    const LdsFill<DH> fill(lane);
    auto stage = [&](int h, int c) {  // the wave's next chunk
        const int row0 = c * CR;
        // rows behind the sample re-read its last one: what is masked is still finite
        const __amdgpu_buffer_rsrc_t r1 = head_resource<DH>(base + (size_t)(MODE == MODE_DQ ? H + hk : h) * DH * 2, N, pitch);
        const __amdgpu_buffer_rsrc_t r2 = MODE == MODE_DQ ? head_resource<DH>(base + (size_t)(H + HK + hk) * DH * 2, N, pitch)
                                                          : head_resource<DH>(gbase + (size_t)h * DH * 2, N, opitch);
        fill.chunk(r1, buf, CR, 0, 1, row0, nb - 1, pitch);
        fill.chunk(r2, buf + IMG, CR, 0, 1, row0, nb - 1, MODE == MODE_DQ ? pitch : opitch);
        if constexpr (MODE == MODE_DKV) {
            int q = row0 + lane;
            q = q < nb ? q : nb - 1;
            auto row_values = [&](const float* p, int place) {
                const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (unsigned)N * 4, 0x00020000);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LDS_PTR(buf + 2 * IMG + place * CR * 4), 4, q * 4, 0, 0, 0);
            };
            if (lane < CR) {
                row_values(a.row_L(b, h), 0);
                row_values(a.ndelta + ((size_t)b * H + h) * N, 1);
                row_values(a.row_M(b, h), 2);
            }
        }
        if (lane < CR) *(int*)(buf + BUF - CR * 4 + lane * 4) = rel_row_code(a.geo, sl, MODE == MODE_DQ, row0 + lane);
    };
    if (nc > 0) {
        if constexpr (MODE == MODE_DQ) {
            fill.chunk(head_resource<DH>(base + (size_t)oh * DH * 2, N, pitch), rows, CR, wave, nw, o0, nb - 1, pitch);
            fill.chunk(head_resource<DH>(gbase + (size_t)oh * DH * 2, N, opitch), rows + IMG, CR, wave, nw, o0, nb - 1, opitch);
            const unsigned char* ob = (const unsigned char*)a.out + (size_t)b * N * opitch + (size_t)oh * DH * 2;
            fill.chunk(head_resource<DH>(ob, N, opitch), rows + 2 * IMG, CR, wave, nw, o0, nb - 1, opitch);
        } else {
            fill.chunk(head_resource<DH>(base + (size_t)(H + hk) * DH * 2, N, pitch), rows, CR, wave, nw, o0, nb - 1, pitch);
            fill.chunk(head_resource<DH>(base + (size_t)(H + HK + hk) * DH * 2, N, pitch), rows + IMG, CR, wave, nw, o0, nb - 1, pitch);
        }
        if (wave < nc) stage(head0, wave);
    }
    float oL = INFINITY, oD = 0.f;
    if (MODE == MODE_DQ && row < nb) oL = a.lse[((size_t)b * H + oh) * N + row];
    rel_expand(a.geo, T, sl, MODE == MODE_DQ, head0);
    const RelLane<MODE == MODE_DQ> rl(a.geo, sl, T, row, N - 1);
    const TrRead<DH> tr(lane);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the outer rows, T
    bf16x8 f1[KS], f2[KS];
    if (nc > 0) {
        float d = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            f1[ks] = *(const bf16x8*)(rows + I::at(r, 2 * ks + hi));
            f2[ks] = *(const bf16x8*)(rows + IMG + I::at(r, 2 * ks + hi));
            if constexpr (MODE == MODE_DQ) {
                const bf16x8 ov = *(const bf16x8*)(rows + 2 * IMG + I::at(r, 2 * ks + hi));
#pragma unroll
                for (int e = 0; e < 8; ++e) d = fmaf((float)f2[ks][e], (float)ov[e], d);
            }
        }
        if (MODE == MODE_DQ && row < nb) oD = d;
        if constexpr (MODE == MODE_DQ) oD += __shfl_xor(oD, 32, 64);
    }
    float* const Mr = sums + wave * 32;
    bool far = false;  // DQ: the wave has rows of the two-part statistic
    if constexpr (MODE == MODE_DQ) {
        const bool f = rel_far(oL);
        far = __any(f);
        if (far) {  // (every wave for itself: they share the queries)
            float M, L;
            rel_far_rows<DH>(a.geo, sl, rl, f1, base + (size_t)(H + hk) * DH * 2, pitch, nb, lane, a.scale_log2e, M, L);
            if (f) oL = L;
            Mr[r] = f ? M : 0.f;  // (both halves of the wave write it)
        }
    }
    f32x16 acc1[DB], acc2[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) { acc1[d][e] = 0.f; acc2[d][e] = 0.f; }
    float dsum = 0.f;
    for (int g = 0; g < nheads; ++g) {
        if (g > 0) {  // the next head of the group
            __syncthreads();
            rel_expand(a.geo, T, sl, false, head0 + g);
            __syncthreads();
        }
        for (int c = wave; c < nc; c += nw) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            chunk_products<DH, MODE>(a, buf, img, img + I::at(r, hi), tr, rl, f1, f2, far, Mr, oL, oD, acc1, acc2, dsum, c * CR, nb, hi);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the chunk's reads are over)
            if (c + nw < nc) stage(head0 + g, c + nw);
            else if (g + 1 < nheads) stage(head0 + g + 1, wave);
        }
    }
    // ---- the waves' sums
    if constexpr (MODE == MODE_DQ) {
        dsum += __shfl_xor(dsum, 32, 64);
        if (wave == 0 && hi == 0 && row < N) {
            a.row_M(b, oh)[row] = far ? Mr[r] : 0.f;
            a.row_L(b, oh)[row] = oL;
        }
        if (hi == 0) sums[wave * 32 + r] = dsum;
    }
    float* const part = (float*)smem;  // [nw] of BUF bytes: [DH][32]
    auto add = [&](f32x16 (&acc)[DB], bf16_t* dst, int rowel, float scale) {
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int dd = d * 32 + (e & 3) + 8 * (e >> 2) + 4 * hi;
                if (dd < DH) part[(size_t)wave * (BUF / 4) + dd * 32 + r] = acc[d][e];
            }
        __syncthreads();
        for (int i = tid; i < 32 * (DH / 8); i += blockDim.x) {
            const int q = i & 31, d0 = (i >> 5) * 8;
            if (o0 + q >= N) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
            for (int w = 0; w < nw; ++w)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += part[(size_t)w * (BUF / 4) + (d0 + e) * 32 + q];
            bf16x8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (bf16_t)(o0 + q < nb ? v[e] * scale : 0.f);  // (rows behind the sample's length: zeros)
            *(bf16x8*)(dst + (size_t)(o0 + q) * rowel + d0) = o;
        }
    };
    const int rowel = (H + 2 * HK) * DH;
    bf16_t* dst = a.dqkv + (size_t)b * N * rowel + (size_t)(MODE == MODE_DQ ? oh : H + oh) * DH;
    add(acc1, dst, rowel, a.scale);
    if constexpr (MODE == MODE_DKV) add(acc2, dst + (size_t)HK * DH, rowel, 1.f);
    if constexpr (MODE == MODE_DQ) {
        if (wave == 0 && hi == 0 && row < N) {
            float t = 0.f;
            for (int w = 0; w < nw; ++w) t += sums[w * 32 + r];
            a.ndelta[((size_t)b * H + oh) * N + row] = oL < INFINITY ? -(oD + t) : 0.f;
        }
    }
}

// rows of a launch's blocks: equal blocks of up to `most` waves
int block_rows(int n32, int most) { return ceil_div(n32, ceil_div(n32, most)) * 32; }
// few enough tiles of 32 rows that the waves of a workgroup share one
// Whole calls (replayed) in us, this / the kernels that share inner chunks, 12 heads of 64 (tiles a CU in brackets): 577 tokens, 1 sample [0.9]
// 44 / 82, 2 [1.8] 68 / 89, 4 [3.6] 110 / 98; against one pass (attention_rel_bwd_dh64.hip) 197 tokens, 1 sample [0.3] 30 / 39, 4 [1.3] 45 / 42;
// 8 heads over 4 of 128, 512 tokens, 1 sample [0.5, 0.25 for dK, dV] 51 / 131
bool attn_rel_few_rows(int64_t tiles, int ncu, bool one_pass) { return 2 * tiles <= (one_pass ? 2 : 5) * (int64_t)ncu; }

template <int DH, int MODE>
int launch_split(const RelBwdArgs& a, const vit_rel_pos* pos, int tile0, int tiles, hipStream_t stream) {
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, 32);
    const int n32 = ceil_div(a.N, 32);
    int waves = n32 < split_waves_most(DH, MODE) ? n32 : split_waves_most(DH, MODE);
    auto need = [&](int w) {
        return (size_t)w * (chunk_bytes<DH, MODE>() + 128) + (MODE == MODE_DQ ? 3 : 2) * CR * LdsImage<DH>::ROW + (size_t)slice * 4;
    };
    while (waves > 1 && need(waves) > 160 * 1024) --waves;
    auto kern = attn_rel_bwd_split_kernel<DH, MODE>;
    static PerDeviceInt attr_set;
    std::atomic<int>* as = attr_set.slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(kern, dim3(a.B * (MODE == MODE_DQ ? a.H : a.HK), tiles), dim3(waves * 64), need(waves), stream, a, tile0);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

template <int DH, int MODE>
int launch_part(const RelBwdArgs& a, const vit_rel_pos* pos, int ncu, hipStream_t stream) {
    const int n32 = ceil_div(a.N, 32), items = a.B * (MODE == MODE_DQ ? a.H : a.HK);
    int blocks = ceil_div(n32, 4), waves = block_rows(n32, 4) / 32, tail = 0;
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, waves * 32);
    if (attn_rel_few_rows((int64_t)items * n32, ncu, false)) return launch_split<DH, MODE>(a, pos, 0, n32, stream);
    constexpr int kFarRows = MODE == MODE_DQ ? 128 : 0;  // floats behind the expansion
    size_t lds = (size_t)2 * chunk_bytes<DH, MODE>() + (size_t)(slice + kFarRows) * 4;
    if (!a.lengths && n32 > 4 && n32 % 4 && (int64_t)items * (n32 % 4) <= ncu) {
        // Tiles behind the last whole block of 4 that would start a round of workgroups of their own: by the waves of workgroups instead
        // (4 x 1025 tokens, 16 heads of 80, dK and dV: 127 us with the 33rd tile as a ninth block, 75 + 19 so)
        const int big = rel_slice_max(pos->grid_h, pos->grid_w, 128);
        const size_t big_lds = (size_t)2 * chunk_bytes<DH, MODE>() + (size_t)(big + kFarRows) * 4;
        const int by_lds = (int)(160 * 1024 / big_lds), by_regs = bwd_waves_per_simd(DH, MODE);
        const int64_t slots = (int64_t)ncu * (by_lds < by_regs ? by_lds : by_regs), full = (int64_t)items * (n32 / 4);
        if (big <= kRelSliceCap && (full + items + slots - 1) / slots > (full + slots - 1) / slots) {
            waves = 4;
            blocks = n32 / 4;
            tail = n32 % 4;
            lds = big_lds;
        }
    }
    auto kern = attn_rel_bwd_kernel<DH, MODE>;
    static PerDeviceInt attr_set;
    std::atomic<int>* as = attr_set.slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(kern, dim3(items, blocks), dim3(waves * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return tail ? launch_split<DH, MODE>(a, pos, blocks * 4, tail, stream) : VIT_OK;
}

struct Workspace {
    size_t delta, rows, met, part, doff, bytes;
    int splits, tq, tk, bq, bk, fp;
};
// LDS of the bias gradient's workgroups: two buffers of K and V images, codes, expansion (up to the limit of entries blocks of 2 key tiles
// fit at every head dim)
size_t bias_lds(int head_dim, int kt, int slice) {
    const int ch = head_dim / 8, row = (ch == 8 || ch == 16 ? ch : ch + 1) * 16;
    return (size_t)4 * kt * 32 * row + (size_t)(kt * 32 + slice) * 4;
}
int plan_workspace(const vit_rel_pos* pos, int batch, int heads, int head_dim, Workspace* w) {
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    const int N = pos->prefix + pos->grid_h * pos->grid_w, n32 = ceil_div(N, 32);
    // query blocks of up to 8 waves, all alike; key blocks of 7 tiles where that is the whole sequence (one block: Q, dO, K, V are read
    // once a sample) and the head dim leaves the registers room for it (a spilled register's reload waits for all loads under
    // way), else 4 tiles, 2 for head_dim 128 and where the expansion of a long sequence leaves the images less
    w->tq = ceil_div(n32, 8);
    w->bq = block_rows(n32, 8);
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, w->bq);
    w->bk = (head_dim <= 64 && n32 > 4 && n32 <= 7 ? 7 : head_dim <= 112 && bias_lds(head_dim, 4, slice) <= 160 * 1024 ? 4 : 2) * 32;
    // Few samples: blocks of 1, 2 or 4 key tiles, the smallest that gives each CU at most one block and three (block, sample) pairs. us at
    // 7 / 4 / 2 / 1 tiles, 12 heads of 64 x 197 tokens: 1 sample 26 / 19 / 13 / 11, 8: 27 / 20 / 16 / 16, 64: 50 / 48 / 52 / 68; 577 tokens
    // (more blocks than CUs at 2 tiles): 1 sample - / 20 / 25 / 26, 64: - / 274 / 363 / 464
    for (int kt = 1; kt * 32 < w->bk; kt *= 2) {
        const int64_t blocks = (int64_t)heads * w->tq * ceil_div(n32, kt);
        if (blocks <= ncu && blocks * batch <= 3 * (int64_t)ncu) {
            w->bk = kt * 32;
            break;
        }
    }
    w->tk = ceil_div(N, w->bk);
    w->fp = 2 * (w->bq + w->bk - 1) + 4;
    // enough sample ranges to give every CU a workgroup, whole samples each
    int64_t s = ncu / ((int64_t)heads * w->tq * w->tk);
    w->splits = s < 1 ? 1 : s > batch ? batch : (int)s;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    w->delta = 0;
    w->rows = up((size_t)batch * heads * N * 4);
    w->met = w->rows + up((size_t)batch * heads * N * 8);
    w->part = w->met + up((size_t)ncu * 8 * 4);
    w->doff = w->part + up((size_t)w->splits * heads * w->tq * w->tk * w->fp * 4);
    w->bytes = w->doff + up((size_t)heads * ((size_t)(2 * pos->grid_h - 1) * (2 * pos->grid_w - 1) + 3) * 4);
    return VIT_OK;
}

template <int DH, int KT>
int launch_bias_grad(const RelBwdArgs& a, const vit_rel_pos* pos, hipStream_t stream) {
    const int nw = a.bq / 32;
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, a.bq);
    size_t lds = bias_lds(DH, KT, slice);
    const size_t fold = (size_t)nw * (32 * 33 + (KT + 1) * 64 + 3) * 4;
    if (lds < fold) lds = fold;
    auto kern = attn_rel_bias_grad_kernel<DH, KT>;
    static PerDeviceInt attr_set;
    std::atomic<int>* as = attr_set.slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(kern, dim3(a.tq * a.tk, a.H, a.splits), dim3(nw * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

template <int DH>
int launch_all(RelBwdArgs a, const vit_rel_pos* pos, hipStream_t stream) {
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    if (attention_rel_bwd_dh64_eligible(a.N, a.H, a.HK, DH) && !attn_rel_few_rows((int64_t)a.B * a.H * ceil_div(a.N, 32), ncu, true)) {
        VIT_TRY_RC(launch_attention_rel_bwd_dh64(a.geo, a.qkv, a.out, a.dout, a.lse, a.ndelta, a.rows, a.met, a.dqkv, a.lengths, a.B, a.N, a.H, a.scale, stream));
    } else {
        VIT_TRY_RC((launch_part<DH, MODE_DQ>(a, pos, ncu, stream)));
        VIT_TRY_RC((launch_part<DH, MODE_DKV>(a, pos, ncu, stream)));
    }
    if (!a.dtable) return VIT_OK;
    if (a.bk == 32) VIT_TRY_RC((launch_bias_grad<DH, 1>(a, pos, stream)));
    else if (a.bk == 7 * 32) VIT_TRY_RC((launch_bias_grad<DH, (DH <= 64 ? 7 : DH <= 112 ? 4 : 2)>(a, pos, stream)));
    else if (a.bk == 4 * 32) VIT_TRY_RC((launch_bias_grad<DH, (DH <= 112 ? 4 : 2)>(a, pos, stream)));
    else VIT_TRY_RC((launch_bias_grad<DH, 2>(a, pos, stream)));
    const int total = a.geo.offsets + (a.geo.prefix ? 3 : 0);
    // without a map, and with nothing in the table behind the offsets, the offset sums are the table's gradient
    const bool direct = !a.geo.bucket_of && a.geo.num_buckets == total;
    hipLaunchKernelGGL(attn_rel_offset_kernel, dim3(ceil_div(total, 64), a.H), dim3(64 * kOffsetWaves), 0, stream, a, direct ? a.dtable : a.doff,
                       direct ? 1 : total, direct ? a.H : 1);
    VIT_CHECK_HIP(hipGetLastError());
    if (!direct) {
        hipLaunchKernelGGL(attn_rel_bucket_kernel, dim3(ceil_div(a.geo.num_buckets, 4), a.H), dim3(256), 0, stream, a);
        VIT_CHECK_HIP(hipGetLastError());
    }
    return VIT_OK;
}

}  // namespace

extern "C" size_t vit_attention_rel_bwd_workspace_bytes(const vit_rel_pos* pos, int batch, int heads, int head_dim) {
    Workspace w{};
    if (!pos || batch <= 0 || heads <= 0 || pos->prefix < 0 || pos->grid_h <= 0 || pos->grid_w <= 0 ||
        (int64_t)pos->grid_h * pos->grid_w > 16384 || plan_workspace(pos, batch, heads, head_dim, &w) != VIT_OK)
        return 0;
    return w.bytes;
}

extern "C" int vit_attention_rel_bwd(const vit_rel_pos* pos, const void* qkv, const float* table, const int32_t* lengths, const void* out,
                                     const void* d_out, const float* lse, void* dqkv, float* d_table, void* workspace,
                                     size_t workspace_bytes, int batch, int heads, int kv_heads, int head_dim, float scale, void* stream) {
    VIT_REQUIRE(qkv && out && d_out && lse && dqkv && workspace, "vit_attention_rel_bwd: null argument");
    VIT_REQUIRE(batch > 0 && heads > 0 && kv_heads > 0 && heads <= 65535 && (int64_t)batch * heads < (1 << 22),
                "vit_attention_rel_bwd: empty or too large a problem");
    VIT_REQUIRE(heads % kv_heads == 0, "vit_attention_rel_bwd: heads %d is not a multiple of kv_heads %d", heads, kv_heads);
    VIT_REQUIRE(head_dim % 16 == 0 && head_dim >= 16 && head_dim <= 128,
                "vit_attention_rel_bwd: head_dim must be a multiple of 16 in [16,128], got %d", head_dim);
    VIT_REQUIRE((((uintptr_t)qkv | (uintptr_t)out | (uintptr_t)d_out | (uintptr_t)dqkv | (uintptr_t)workspace) & 15) == 0,
                "vit_attention_rel_bwd: tensors must be 16-byte aligned");
    RelBwdArgs a{};
    VIT_TRY_RC(rel_make_geo("vit_attention_rel_bwd", pos, table, heads, scale, &a.geo, &a.N));
    VIT_REQUIRE((int64_t)a.N * (heads + 2 * kv_heads) * head_dim * 2 < (1LL << 31), "vit_attention_rel_bwd: one sample's qkv rows exceed 2 GiB");
    VIT_REQUIRE(!d_table || !pos->bucket_of || (pos->by_bucket && pos->bucket_start),
                "vit_attention_rel_bwd: the gradient of a mapped table needs the map's inverse");
    // (every limit before the first launch: a refused call writes nothing)
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, block_rows(ceil_div(a.N, 32), d_table ? 8 : 4));
    VIT_REQUIRE(slice <= kRelSliceCap, "vit_attention_rel_bwd: a %d x %d grid needs %d bias entries at once, %d fit", pos->grid_h, pos->grid_w, slice, kRelSliceCap);
    Workspace w{};
    VIT_TRY_RC(plan_workspace(pos, batch, heads, head_dim, &w));
    if (workspace_bytes < w.bytes)
        return vit_set_error(VIT_E_NOMEM, "vit_attention_rel_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, w.bytes);
    a.qkv = (const bf16_t*)qkv;
    a.out = (const bf16_t*)out;
    a.dout = (const bf16_t*)d_out;
    a.lse = lse;
    a.dqkv = (bf16_t*)dqkv;
    a.ndelta = (float*)((char*)workspace + w.delta);
    a.rows = (float*)((char*)workspace + w.rows);
    a.met = (int*)((char*)workspace + w.met);
    a.part = (float*)((char*)workspace + w.part);
    a.doff = (float*)((char*)workspace + w.doff);
    a.dtable = d_table;
    a.by_bucket = pos->by_bucket;
    a.bucket_start = pos->bucket_start;
    a.lengths = lengths;
    a.B = batch;
    a.H = heads;
    a.HK = kv_heads;
    a.splits = w.splits;
    a.tq = w.tq;
    a.tk = w.tk;
    a.bq = w.bq;
    a.bk = w.bk;
    a.fp = w.fp;
    a.scale = scale;
    a.scale_log2e = scale * LOG2E;
#define RELB_CASE(DHV) \
    case DHV: return launch_all<DHV>(a, pos, (hipStream_t)stream);
    switch (head_dim) {
        RELB_CASE(16) RELB_CASE(32) RELB_CASE(48) RELB_CASE(64) RELB_CASE(80) RELB_CASE(96) RELB_CASE(112) RELB_CASE(128)
    }
#undef RELB_CASE
    return vit_set_error(VIT_E_INVALID, "vit_attention_rel_bwd: unsupported head_dim %d", head_dim);
}
