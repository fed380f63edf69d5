// Backward of attention with a learned relative position bias (attention_rel_bwd.hip: same mathematics), launches 1 and 2 in one pass:
// head_dim 64, 97..224 tokens, as many key as query heads. A sample's Q, K, V and dO of one head fit the LDS whole (4 x 28 KiB), each
// once: an image serves row reads and transposed reads alike (lds_image.h), so nothing is written to LDS but by LDS-DMA. One persistent
// workgroup per CU, one wave per 32 tokens, walks (head, sample) items:
//   A  the wave's 32 queries on the lane, all keys: dQ, and delta with its correction (for the bias sums too);
//   B  the wave's 32 keys on the lane, all queries: dK, dV.
// Two barriers an item, all loads a phase ahead: the next item's K, V images and every wave's own Q, dO, O rows (registers) come under B,
// whose images are Q and dO; those come under A, whose images are K and V (an L2 hit: the rows went to registers one phase before).
//
// 256 x 197 tokens, 12 heads: 245 us for 620 MB and 7 products of 32 x 32 x 64 a pair of tiles. Bound by each wave's chain of matrix and
// vector instructions (two waves a SIMD with 252 registers each; those two kinds overlap by about 30 %). As two chunked launches: 152 +
// 207 us. Fragments fetched a tile ahead or two tiles a step spilled and took longer; waves started at an offset gained 2 %.
#include "lds_image.h"
#include "rel_bias.h"
#include <math.h>

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int DH = 64;
using I = LdsImage<DH>;
constexpr int kRows = 224;               // rows of an image: fixed, so that images and row arrays lie at constant distances
constexpr int IMG = kRows * I::ROW;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct RelBwd64Args {
    const unsigned char* qkv;
    const unsigned char* out;
    const unsigned char* dout;
    const float* lse;
    float* ndelta;
    float* rows;  // [2][B, H, N]: M and L of rows whose lse is far from zero (rel_bias.h), for the bias sums
    int* met;     // [grid][8]: whether a workgroup's waves have met such rows
    unsigned char* dqkv;
    const int* lengths;
    RelGeo geo;
    int B, N, H, nitems;
    float scale, scale_log2e;
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ bf16x8 pack8(const f32x16& p, int s) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (bf16_t)p[8 * s + e];
    return o;
}
// 32 rows x 64 values read transposed: A fragments [k-step][32-value block]. addr[d][half]: lane addresses of rows 0..7 / 8..15.
// The wait is in the same statement: the compiler holds its outputs as written when it ends. (Through the builtin every such read
// would also wait for all LDS-DMA under way.)
template <int OFF>
__device__ __forceinline__ void tr_read(bf16x8 (&f)[2][2], const unsigned (&addr)[2][2], unsigned base) {
    short4v v[8];
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:%13\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %10 offset:%13\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(addr[0][0] + base), "v"(addr[0][1] + base), "v"(addr[1][0] + base), "v"(addr[1][1] + base), "n"(OFF), "n"(OFF + 16 * I::ROW)
                 : "memory");
#pragma unroll
    for (int k = 0; k < 4; ++k)
        f[k >> 1][k & 1] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v[2 * k], v[2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ int sample_length(const int* lengths, int b, int N) {
    if (!lengths) return N;
    const int n = lengths[b];
    return n < 0 ? 0 : n > N ? N : n;
}
// A wave's 32 rows between memory and its registers go through a 4-KiB LDS block of its own: a memory instruction then touches 8
// whole rows, not 32 quarters of rows (which cost the CU's address unit four times as much: 57 cycles an instruction, measured).
// Loads: 8 lanes a row, piece i rows 8 i ..; the block is wave-private and a wave's LDS operations execute in order: no barrier.
__device__ __forceinline__ void turn_rows(bf16x8 (&f)[4], const bf16x8 (&v)[4], unsigned char* blk, const int (&ro)[4], int lane) {
    asm volatile("" : "+v"(lane));  // (opaque here and below: these addresses are not worth registers over the products)
#pragma unroll
    for (int i = 0; i < 4; ++i) *(bf16x8*)(blk + I::at(8 * i + (lane >> 3), lane & 7)) = v[i];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) f[ks] = *(const bf16x8*)(blk + ro[ks]);
}
// accumulator (lane = token row, registers = head dims) * mul -> bf16 rows, zeros from row nb on; row0 + 31 may lie behind the resource
__device__ __forceinline__ void store_rows(f32x16 (&acc)[2], float mul, __amdgpu_buffer_rsrc_t dst, unsigned char* blk, int row0, int nb, int pitch, int lane) {
    asm volatile("" : "+v"(lane));
    if (row0 + 32 > nb && row0 + (lane & 31) >= nb) {  // (not by a factor of 0: they are sums of the last row's values, which may be NaN)
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (bf16_t)(acc[d][g4 * 4 + e] * mul);
            *(bf16x4*)(blk + I::at(lane & 31, d * 4 + g4) + (lane >> 5) * 8) = v;
        }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + (lane >> 3);
        const u32x4 v = *(const u32x4*)(blk + I::at(row, lane & 7));
        __builtin_amdgcn_raw_buffer_store_b128(v, dst, (row0 + row) * pitch + (lane & 7) * 16, 0, 0);
    }
}

// FAR: the launch behind the other, for the items that have rows far from zero: once more, with the two-part statistic and nothing loaded
// ahead, over what that launch left for them. (A kernel of its own: a branch for such rows anywhere in the other costs it 11 us at 256 x 197
// tokens, this one's early end 4.6. A gradient of which every row is such takes 1077 instead of 361 us.)
template <bool FAR>
__global__ __launch_bounds__(448) __attribute__((amdgpu_waves_per_eu(2, 2))) void attn_rel_bwd_dh64_kernel(const RelBwd64Args a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int N = a.N, H = a.H, B = a.B;
    unsigned char* const Ki = smem;
    unsigned char* const Vi = Ki + IMG;
    unsigned char* const Qi = Vi + IMG;
    unsigned char* const Gi = Qi + IMG;  // dO
    float* const rowL = (float*)(Gi + IMG);
    float* const rowD = rowL + kRows;
    int* const codes = (int*)(rowD + kRows);
    int* const codesq = codes + kRows;  // the keys' codes for A, the queries' for B
    unsigned char* const blk = (unsigned char*)(codesq + kRows) + (threadIdx.x >> 6) * 32 * I::ROW;  // this wave's
    float* const T = (float*)((unsigned char*)(codesq + kRows) + kRows * I::ROW);
    const unsigned lds0 = (unsigned)(uintptr_t)LDS_PTR(smem);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hi = lane >> 5;
    const int o0 = wave * 32, row = o0 + r;
    const int pitch = 3 * H * DH * 2, opitch = H * DH * 2;

    const int per = a.nitems / (int)gridDim.x, extra = a.nitems - per * (int)gridDim.x, wg = blockIdx.x;
    const int first = wg * per + (wg < extra ? wg : extra), last = first + per + (wg < extra ? 1 : 0);
    if (first >= last) return;  // uniform
    if (FAR && !__any((lane & 7) * 64 < (int)blockDim.x && a.met[wg * 8 + (lane & 7)])) return;  // uniform

    // ---- lane geometry
    int ro[4];  // row reads: chunk ks * 2 + hi of row r of a tile
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) ro[ks] = I::at(r, ks * 2 + hi);
    unsigned tr[2][2];
    {
        const int g = lane >> 4, i16 = lane & 15;
        const int key = 4 * (g >> 1) + (i16 >> 2), c = (g & 1) * 2 + ((i16 & 3) >> 1), sub = (i16 & 1) * 8;
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int half = 0; half < 2; ++half) tr[d][half] = lds0 + (unsigned)(I::at(key + 8 * half, d * 4 + c) + sub);
    }
    // one expansion for A (queries of the block on the lane) and one for B (keys): whole sequences, so the offsets are the same, what
    // stands behind them is not
    const RelSlice sa(a.geo, 0, N - 1, true), sb(a.geo, 0, N - 1, false);
    float* const Tb = T + sa.n + sa.span + 3;
    float* const rowM = Tb + sb.n + sb.span + 3;  // FAR
    int* const flags = (int*)(rowM + kRows);       // FAR: of the waves
    const RelLane<true> la(a.geo, sa, T, row, N - 1);
    const RelLane<false> lb(a.geo, sb, Tb, row, N - 1);
    for (int i = tid; i < kRows; i += blockDim.x) {
        codes[i] = rel_row_code(a.geo, sa, true, i);
        codesq[i] = rel_row_code(a.geo, sb, false, i);
    }

    // ---- staging: this wave's 32 rows of an image, four instructions
    auto rsrc_of = [&](const unsigned char* base, int b, int p, int col) { return head_resource<DH>(base + (size_t)b * N * p + (size_t)col * (DH * 2), N, p); };
    auto stage = [&](__amdgpu_buffer_rsrc_t rs, unsigned char* img, int p, int nb, int i) {
        int ln = lane;
        asm volatile("" : "+v"(ln));  // (opaque: the pieces' lane offsets are made here, not kept in registers over the products)
        const int lastr = nb > 0 ? nb - 1 : 0;  // rows behind the sample re-read its last row: what is masked is still finite
        I::dma(rs, img, o0 + i * 8, kRows, 0, lastr, p, ln);
    };
    auto stage_kv = [&](int item, int nb, int i) {
        const int h = item / B, b = item - h * B;
        stage(rsrc_of(a.qkv, b, pitch, H + h), Ki, pitch, nb, i);
        stage(rsrc_of(a.qkv, b, pitch, 2 * H + h), Vi, pitch, nb, i);
    };
    auto stage_qg = [&](int item, int nb, int i) {
        const int h = item / B, b = item - h * B;
        stage(rsrc_of(a.qkv, b, pitch, h), Qi, pitch, nb, i);
        stage(rsrc_of(a.dout, b, opitch, h), Gi, opitch, nb, i);
    };
    bf16x8 nq[4], ng[4], no[4];
    float nL = INFINITY;
    auto load_rows = [&](int item, int nb) {  // the wave's own queries: Q, dO, O rows, 8 lanes a row
        const int h = item / B, b = item - h * B, lastr = nb > 0 ? nb - 1 : 0;
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const unsigned char* qp = a.qkv + (size_t)b * N * pitch + (size_t)h * (DH * 2);
        const unsigned char* gp = a.dout + (size_t)b * N * opitch + (size_t)h * (DH * 2);
        const unsigned char* op = a.out + (size_t)b * N * opitch + (size_t)h * (DH * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int rr = o0 + 8 * i + (ln >> 3);
            rr = rr < lastr ? rr : lastr;
            const unsigned c = (unsigned)(ln & 7) * 16, qo = (unsigned)(rr * pitch) + c, oo = (unsigned)(rr * opitch) + c;
            nq[i] = *(const bf16x8*)(qp + qo);
            ng[i] = *(const bf16x8*)(gp + oo);
            no[i] = *(const bf16x8*)(op + oo);
        }
        const int orow = row < lastr ? row : lastr;
        nL = (a.lse + ((size_t)b * H + h) * N)[orow];
    };
    int item = first, thead = -1;
    auto length_of = [&](int item) { return __builtin_amdgcn_readfirstlane(sample_length(a.lengths, item % B, N)); };
    int nb = length_of(item);
    if constexpr (!FAR) {
        for (int i = 0; i < 4; ++i) stage_kv(item, nb, i);
        load_rows(item, nb);
    }
    asm volatile("" ::: "memory");
    wait_vm<0>();
    // (seen as complete here, so that the loop's wait for them counts the stores behind them on every path)
#pragma unroll
    for (int ks = 0; ks < 4 && !FAR; ++ks) asm volatile("" : "+v"(nq[ks]), "+v"(ng[ks]), "+v"(no[ks]));
    if constexpr (!FAR) asm volatile("" : "+v"(nL));
    f32x16 acc1[2], acc2[2];
    bool met = false;
    while (item < last) {
        const int h = item / B, b = item - h * B;
        const int ntb = (nb + 31) >> 5;
        const int nnb = item + 1 < last ? length_of(item + 1) : 0;
        if constexpr (FAR) {
            int rw = row;
            asm volatile("" : "+v"(rw));
            const bool f = __any(rw < nb && rel_far((a.lse + ((size_t)b * H + h) * N)[rw < nb ? rw : 0]));
            __syncthreads();  // nobody reads the last item's images any more
            if (lane == 0) flags[wave] = f;
            __syncthreads();
            if (!__any((lane & 7) * 64 < (int)blockDim.x && flags[lane & 7])) {  // uniform
                ++item;
                nb = nnb;
                continue;
            }
            for (int i = 0; i < 4; ++i) stage_kv(item, nb, i);
            load_rows(item, nb);
            asm volatile("" ::: "memory");
            wait_vm<0>();
        } else {
            // this wave's pieces and rows have landed: everything but the previous item's dK / dV stores (8, issued behind them)
            wait_vm<8>();
        }
        asm volatile("s_barrier" ::: "memory");  // 1: K, V images are whole; Q, dO images and T are free
        if (h != thead) {  // uniform
            rel_expand(a.geo, T, sa, true, h);
            rel_expand(a.geo, Tb, sb, false, h);
            thead = h;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            asm volatile("s_barrier" ::: "memory");
        }

        // ================= A: dQ
        bf16x8 f1[4], f2[4];
        float oL = row < nb ? nL : INFINITY, oD = 0.f;
        if constexpr (!FAR) met |= __any(rel_far(oL));
        // delta: dO . O in the rows' own lanes, 8 a row
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float d = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) d = fmaf((float)ng[i][e], (float)no[i][e], d);
            d = dpp_add<0xB1>(d);   // quad_perm 1,0,3,2
            d = dpp_add<0x4E>(d);   // quad_perm 2,3,0,1
            d = dpp_add<0x141>(d);  // row_half_mirror
            if ((lane & 7) == 0) rowD[o0 + 8 * i + (lane >> 3)] = d;
        }
        turn_rows(f1, nq, blk, ro, lane);
        turn_rows(f2, ng, blk, ro, lane);
        if (row < nb) oD = rowD[row];
        if constexpr (FAR) {
            float M, L;
            rel_far_rows<DH>(a.geo, sa, la, f1, a.qkv + (size_t)b * N * pitch + (size_t)(H + h) * (DH * 2), pitch, nb, lane, a.scale_log2e, M, L);
            const bool f = rel_far(oL);
            int rw = row;
            asm volatile("" : "+v"(rw));  // (opaque here and below, as above)
            rowM[rw] = f ? M : 0.f;       // (both halves of the wave write it)
            if (f) {
                oL = L;
                a.rows[((size_t)b * H + h) * N + rw] = M;
                a.rows[((size_t)(B + b) * H + h) * N + rw] = L;
            }
        }
        if (ntb == 1 && o0 < nb) {
            // One tile of keys: delta's error (the row's sum of dS) leaves delta before dS is made and rounded. (With few keys it is a large
            // part of dS, up to twice dQ's rounding for 3 keys; with more than a tile of them it is below a twentieth.)
            f32x16 s, dp;
            rel_tile(s, codes, la, hi, a.geo.prefix, 0);
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(Ki + ro[ks]), f1[ks], s, 0, 0, 0);
                dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(Vi + ro[ks]), f2[ks], dp, 0, 0, 0);
            }
            int rw = row, lim = nb - 4 * hi;
            asm volatile("" : "+v"(rw), "+v"(lim));
            const float M = FAR ? rowM[rw] : 0.f;
            float err = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float x = (e & 3) + 8 * (e >> 2) < lim ? fmaf(s[e] - M, a.scale_log2e, -oL) : -INFINITY;
                err = fmaf(__builtin_amdgcn_exp2f(x), dp[e] - oD, err);
            }
            oD += err + __shfl_xor(err, 32, 64);
        }
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc1[d][e] = 0.f;
        float dsum = 0.f;
        if (o0 < nb) {
            for (int t = 0; t < ntb; ++t) {
                const int key0 = t * 32, tb = t * 32 * I::ROW;
                f32x16 s, dp;
                bf16x8 kf[4], vf[4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    kf[ks] = *(const bf16x8*)(Ki + tb + ro[ks]);
                    vf[ks] = *(const bf16x8*)(Vi + tb + ro[ks]);
                }
                rel_tile(s, codes + key0, la, hi, a.geo.prefix, key0);
                if (t < 4) stage_qg(item, nb, t);  // (a piece a tile: all at once the CU's memory queue would block the wave)
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] = 0.f;  // (delta comes off behind the products, as in the bias launch: the same roundings in both)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], f1[ks], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[ks], f2[ks], dp, 0, 0, 0);
                }
                if constexpr (FAR) {
                    int rw = row;
                    asm volatile("" : "+v"(rw));
                    const float M = rowM[rw];
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] -= M;
                }
                bf16x8 kt[2][2];
                tr_read<0>(kt, tr, (unsigned)tb);
                if (key0 + 32 > nb) {
                    int lim = nb - key0 - 4 * hi;
                    asm volatile("" : "+v"(lim));
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if ((e & 3) + 8 * (e >> 2) >= lim) s[e] = -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -oL)) * (dp[e] - oD);  // dS^T
                    dsum += s[e];
                }
#pragma unroll
                for (int sk = 0; sk < 2; ++sk) {
                    const bf16x8 x = pack8(s, sk);
                    acc1[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[sk][0], x, acc1[0], 0, 0, 0);
                    acc1[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[sk][1], x, acc1[1], 0, 0, 0);
                }
            }
        }
        for (int i = o0 < nb ? ntb : 0; i < 4; ++i) stage_qg(item, nb, i);
        dsum += __shfl_xor(dsum, 32, 64);
        oD = oL < INFINITY ? oD + dsum : 0.f;
        if (hi == 0) {
            rowL[row] = oL;
            rowD[row] = -oD;
            int rw = row;
            if constexpr (FAR) asm volatile("" : "+v"(rw));
            if (rw < N) a.ndelta[((size_t)b * H + h) * N + rw] = -oD;
        }
        // the wave's own keys for B
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            f1[ks] = *(const bf16x8*)(Ki + o0 * I::ROW + ro[ks]);
            f2[ks] = *(const bf16x8*)(Vi + o0 * I::ROW + ro[ks]);
        }
        wait_vm<0>();  // Q, dO images (issued a phase ago)
        auto dst = [&](int col) { return head_resource<DH>(a.dqkv + (size_t)b * N * pitch + (size_t)col * (DH * 2), N, pitch); };
        store_rows(acc1, a.scale, dst(h), blk, o0, nb, pitch, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(f1[0]), "+v"(f1[1]), "+v"(f1[2]), "+v"(f1[3]), "+v"(f2[0]), "+v"(f2[1]), "+v"(f2[2]), "+v"(f2[3])::"memory");
        asm volatile("s_barrier" ::: "memory");  // 2: Q, dO images, the rows' L and delta are whole; K, V images are free
        const bool more = !FAR && item + 1 < last;

        // ================= B: dK, dV
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) { acc1[d][e] = 0.f; acc2[d][e] = 0.f; }
        if (o0 < nb) {
            for (int t = 0; t < ntb; ++t) {
                const int tb = t * 32 * I::ROW;
                if (more && t < 4) stage_kv(item + 1, nnb, t);
                f32x16 s, dp;
                bf16x8 rf[4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) rf[ks] = *(const bf16x8*)(Qi + tb + ro[ks]);
                rel_tile(s, codesq + t * 32, lb, hi, a.geo.prefix, t * 32);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rf[ks], f1[ks], s, 0, 0, 0);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) rf[ks] = *(const bf16x8*)(Gi + tb + ro[ks]);
                if constexpr (FAR) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] -= rowM[t * 32 + (e & 3) + 8 * (e >> 2) + 4 * hi];
                }
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const f32x4 Dl = *(const f32x4*)(rowD + t * 32 + 8 * g4 + 4 * hi);
#pragma unroll
                    for (int j = 0; j < 4; ++j) dp[g4 * 4 + j] = Dl[j];
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rf[ks], f2[ks], dp, 0, 0, 0);
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const f32x4 L = *(const f32x4*)(rowL + t * 32 + 8 * g4 + 4 * hi);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = g4 * 4 + j;
                        s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -L[j]));  // P
                        dp[e] *= s[e];                                                    // dS
                    }
                }
                bf16x8 xt[2][2];
                tr_read<IMG>(xt, tr, (unsigned)(2 * IMG + tb));
#pragma unroll
                for (int sk = 0; sk < 2; ++sk) {
                    const bf16x8 x = pack8(s, sk);
                    acc2[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[sk][0], x, acc2[0], 0, 0, 0);
                    acc2[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[sk][1], x, acc2[1], 0, 0, 0);
                }
                tr_read<0>(xt, tr, (unsigned)(2 * IMG + tb));
#pragma unroll
                for (int sk = 0; sk < 2; ++sk) {
                    const bf16x8 x = pack8(dp, sk);
                    acc1[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[sk][0], x, acc1[0], 0, 0, 0);
                    acc1[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xt[sk][1], x, acc1[1], 0, 0, 0);
                }
            }
        }
        if (more) {
            for (int i = o0 < nb ? ntb : 0; i < 4; ++i) stage_kv(item + 1, nnb, i);
            load_rows(item + 1, nnb);
        }
        asm volatile("" ::: "memory");  // (the eight stores stay behind the loads: the counted wait above)
        store_rows(acc1, a.scale, dst(H + h), blk, o0, nb, pitch, lane);
        store_rows(acc2, 1.f, dst(2 * H + h), blk, o0, nb, pitch, lane);
        ++item;
        nb = nnb;
    }
    if (!FAR && lane == 0) a.met[wg * 8 + wave] = met;
}

}  // namespace

// whole heads of 97..224 tokens, as many key as query heads
bool attention_rel_bwd_dh64_eligible(int N, int heads, int kv_heads, int head_dim) { return head_dim == 64 && heads == kv_heads && N > 96 && N <= 224; }

int launch_attention_rel_bwd_dh64(const RelGeo& geo, const void* qkv, const void* out, const void* dout, const float* lse, float* ndelta, float* rows,
                                  int* met, void* dqkv, const int* lengths, int batch, int N, int heads, float scale, hipStream_t stream) {
    RelBwd64Args a{};
    a.qkv = (const unsigned char*)qkv;
    a.out = (const unsigned char*)out;
    a.dout = (const unsigned char*)dout;
    a.lse = lse;
    a.ndelta = ndelta;
    a.rows = rows;
    a.met = met;
    a.dqkv = (unsigned char*)dqkv;
    a.lengths = lengths;
    a.geo = geo;
    a.B = batch;
    a.N = N;
    a.H = heads;
    a.nitems = batch * heads;
    a.scale = scale;
    a.scale_log2e = scale * LOG2E;
    const int nt = ceil_div(N, 32);
    const size_t lds = (size_t)kRows * (5 * I::ROW + 16) + (size_t)(geo.offsets * 3 + 8) * 4;  // (span <= offsets / 2)
    const size_t lds_far = lds + (size_t)(kRows + 8) * 4;
    VIT_REQUIRE(lds_far <= 160 * 1024, "attention_rel_bwd: %d offsets do not fit the LDS", geo.offsets);
    static PerDeviceInt attr_set;
    std::atomic<int>* as = attr_set.slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute((const void*)attn_rel_bwd_dh64_kernel<false>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        VIT_CHECK_HIP(hipFuncSetAttribute((const void*)attn_rel_bwd_dh64_kernel<true>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    const int grid = a.nitems < ncu ? a.nitems : ncu;
    hipLaunchKernelGGL(attn_rel_bwd_dh64_kernel<false>, dim3(grid), dim3(nt * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(attn_rel_bwd_dh64_kernel<true>, dim3(grid), dim3(nt * 64), lds_far, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}
