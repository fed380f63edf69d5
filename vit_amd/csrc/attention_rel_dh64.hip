// Attention with a learned relative position bias (attention_rel.hip: same mathematics), head_dim 64, bf16, whole sequences:
// the persistent LDS-DMA ring of attention_dh64.hip with the bias in front of its products.
//
// What the bias adds. The offsets' bias of one head (rel_bias.h) sits in LDS beside the ring, and a tile's 32 x 32 product starts
// from it: per score one subtraction for the address and one ds_read_b32. Lanes are consecutive queries, so the 64 lanes of a
// read touch about 36 consecutive words (no bank conflicts) wherever the grid's rows do not break. Workgroups take contiguous
// ranges of items ordered (head, query block, sample): the expansion is made again only when head or query block change, which a
// workgroup meets once or twice, behind a barrier pair of its own.
//
// Bound by the waves' own chains (about 140 vector instructions of 4 cycles and 16 exponentials beside 8 matrix instructions a tile, of
// which a quarter overlap). 256 x 197 tokens, 12 heads: 90 us (310 MB: 3.4 TB/s; attention without a bias 77 us); 32 x 577, 16 heads: 100 us
// (0.44 PFLOP/s; without 77 us). Whole-sequence images staged at once took 142 and 173 us; the idle eighth wave's place passed round the SIMDs gained
// nothing.
#include "rel_bias.h"
#include <math.h>
#include <type_traits>

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int DH = 64;
constexpr int SLOT = 8192;   // one tile: K 32 x 128 B, then V 32 x 128 B
constexpr int NW = 8;        // waves per workgroup
constexpr int NQ = 4;        // Q DMA pieces per wave and item
constexpr int QSLOT = 4096;  // one wave's 32 query rows x 128 B
constexpr float kDeferLog2 = 6.0f;  // the running max is left alone until a score outgrows it by more than this (base 2)

struct RelRingArgs {
    const unsigned char* qkv;
    bf16_t* out;
    float* lse;
    RelGeo geo;
    int B, N, H, HK, qblocks, nitems;
    float scale_log2e;
};

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
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// R: ring depth, tiles. LDS: R slots, NW query slots, the keys' codes, the expansion.
template <int R, bool LSE>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(4, 4))) void attention_rel_dh64_kernel(const RelRingArgs a) {
    constexpr int ST = 4 + (LSE ? 1 : 0);  // vector-memory stores an active wave issues per item
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const unsigned smem_lds = (unsigned)(uintptr_t)LDS_PTR(smem);
    const int N = a.N, H = a.H;
    const int nt = (N + 31) >> 5;  // key tiles per item
    int* const codes = (int*)(smem + R * SLOT + NW * QSLOT);
    float* const T = (float*)(codes + nt * 32);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, hi = lane >> 5;
    const int rs2 = (H + 2 * a.HK) * DH * 2;  // token stride, bytes
    const int group = H / a.HK;
    const int per = a.nitems / (int)gridDim.x, extra = a.nitems - per * (int)gridDim.x;
    const int wg = blockIdx.x;
    const int first = wg * per + (wg < extra ? wg : extra);
    const int nmy = per + (wg < extra ? 1 : 0);
    if (nmy <= 0) return;  // uniform

    struct Item { int b, h, qb; };
    auto item_at = [&](int j) {
        const int i = first + j, hq = i / a.B;
        Item t;
        t.b = i - hq * a.B;
        t.h = hq / a.qblocks;
        t.qb = hq - t.h * a.qblocks;
        return t;
    };
    // buffer resource over the rows of one packed head of one sample: N rows of 128 bytes, rs2 apart
    auto head_rsrc = [&](int b, int head) {
        const unsigned char* base = a.qkv + (size_t)b * N * rs2 + (size_t)head * (DH * 2);
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (unsigned)(N - 1) * (unsigned)rs2 + (unsigned)(DH * 2), 0x00020000);
    };
    auto kv_rsrc = [&](const Item& t) { return head_rsrc(t.b, H + t.h / group + (wave < 4 ? 0 : a.HK)); };

    // ---- DMA piece of this wave: rows 8 (wave & 3).. of K (wave < 4) or V (wave >= 4)
    const int prow = 8 * (wave & 3) + (lane >> 3);
    const int ppos = lane & 7;
    const int pchunk = (wave < 4) ? (ppos ^ ((prow >> 1) & 7)) : (ppos ^ (((prow >> 1) & 1) << 2));
    const unsigned pconst = (unsigned)(pchunk * 16);
    unsigned char* const pdst = smem + (wave < 4 ? 0 : 4096) + (wave & 3) * 1024;
    auto dma_tile = [&](__amdgpu_buffer_rsrc_t rsrc, int t, int slot) {
        const int lim = N - 1 - t * 32;  // rows past the sequence re-read its last row (their scores are masked)
        const int row = prow < lim ? prow : lim;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, LDS_PTR(pdst + slot * SLOT), 16, (int)((unsigned)row * (unsigned)rs2 + pconst), t * 32 * rs2, 0, 0);
    };

    // ---- read-side lane geometry
    const int ksw = (r >> 1) & 7;
    unsigned kro[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) kro[ks] = (unsigned)(r * 128 + (((ks * 2 + hi) ^ ksw) << 4));
    const int g = lane >> 4, i16 = lane & 15;
    const int tr_key = 4 * (g >> 1) + (i16 >> 2);
    const int tr_col = ((g & 1) * 16 + 4 * (i16 & 3)) * 2;
    const int vsw = (tr_key >> 1) & 1;
    unsigned vro[2];
#pragma unroll
    for (int d = 0; d < 2; ++d) vro[d] = (unsigned)(4096 + tr_key * 128 + ((d ^ vsw) << 6) + tr_col);

    unsigned char* const qslot = smem + R * SLOT + wave * QSLOT;
    auto dma_q = [&](const Item& t) {
        const __amdgpu_buffer_rsrc_t rsrc = head_rsrc(t.b, t.h);
        const int q0 = (t.qb * NW + wave) * 32;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int row = 8 * i + (lane >> 3);
            const int c = ppos ^ ((row >> 1) & 7);
            int qr = q0 + row;
            if (qr > N - 1) qr = N - 1;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, LDS_PTR(qslot + i * 1024), 16, qr * rs2 + c * 16, 0, 0, 0);
        }
    };
    bf16x8 qf[4];

    // ---- prologue: the expansion of the first item's head, then Q of item 0 and the first R - 1 tiles
    Item cur = item_at(0);
    RelLane<true> rl;
    auto expand = [&](const Item& t) {  // all threads, between barriers
        const int blk0 = t.qb * NW * 32;
        const int blk1 = blk0 + NW * 32 < N ? blk0 + NW * 32 - 1 : N - 1;
        const RelSlice sl(a.geo, blk0, blk1, true);
        rel_expand(a.geo, T, sl, true, t.h);
        for (int i = tid; i < nt * 32; i += NW * 64) codes[i] = rel_row_code(a.geo, sl, true, i);
        rl = RelLane<true>(a.geo, sl, T, blk0 + wave * 32 + r, N - 1);
    };
    expand(cur);
    wait_vm<0>();  // (the expansion's own loads: the counted waits below start from none outstanding)
    __syncthreads();

    int q0 = (cur.qb * NW + wave) * 32;
    __amdgpu_buffer_rsrc_t prs = kv_rsrc(cur);  // resource of the item the DMA cursor is in
    dma_q(cur);
    int pj = 0, pt = 0;  // DMA cursor: item index in this workgroup's range, tile
    auto dma_next = [&](int slot) {
        dma_tile(prs, pt, slot);
        // past the end the cursor stays on the last tile (a dummy re-fetch keeps the counts uniform)
        if (pt + 1 < nt) {
            ++pt;
        } else if (pj + 1 < nmy) {
            ++pj;
            pt = 0;
            prs = kv_rsrc(item_at(pj));
        }
    };
#pragma unroll
    for (int s = 0; s < R - 1; ++s) dma_next(s);

    f32x16 o[2];  // written by the first tile of every item
    RelLevel level;
    float l_run = 0.f;
    int slot = 0, pslot = R - 1;
    bool prev_active = false;  // did this wave store outputs for the previous item
    bool fresh = true;         // the expansion is this item's
    auto tile_step = [&](auto FIRSTC, int j, int p, bool active) {
        constexpr bool FIRST = decltype(FIRSTC)::value;
        {
            // counted wait: this wave's piece of the current tile has landed. Younger operations that may stay in flight: R - 2
            // DMAs; while p <= R - 2 also the previous item's ST stores and, from p = 1, the NQ loads of the Q prefetch
            const bool inwin = p <= R - 2;
            const bool stin = inwin && prev_active;
            const bool qin = inwin && p >= 1;
            if (stin) {
                if (qin) wait_vm<R - 2 + NQ + ST>(); else wait_vm<R - 2 + ST>();
            } else {
                if (qin) wait_vm<R - 2 + NQ>(); else wait_vm<R - 2>();
            }
        }
        asm volatile("s_barrier" ::: "memory");  // every wave's piece landed; the previous tile's slot is free
        if constexpr (FIRST) {
            if (!fresh) {  // uniform over the workgroup: another head or query block (nobody reads T any more: the barrier above)
                expand(cur);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                asm volatile("s_barrier" ::: "memory");
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) qf[ks] = *(const bf16x8*)(qslot + kro[ks]);
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(qf[0]), "+v"(qf[1]), "+v"(qf[2]), "+v"(qf[3])::"memory");
            dma_q(item_at(j + 1 < nmy ? j + 1 : j));  // (clamped: every item issues the same number of DMAs)
        }
        dma_next(pslot);
        pslot = pslot + 1 == R ? 0 : pslot + 1;

        if (active) {
            const unsigned char* Kb = smem + slot * SLOT;
            const unsigned kb_lds = smem_lds + (unsigned)(slot * SLOT);
            const int key0 = p * 32;
            f32x16 s;
            rel_tile(s, codes + key0, rl, hi, a.geo.prefix, key0);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const bf16x8 kf = *(const bf16x8*)(Kb + kro[ks]);
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[ks], s, 0, 0, 0);
            }
            // V^T fragments, issued now and waited for just before the PV products (inline asm: through the builtin the compiler
            // orders every such read behind vmcnt(0), which would drain the ring it reads from)
            short4v vl[8];
            {
                const unsigned va0 = kb_lds + vro[0], va1 = kb_lds + vro[1];
                asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:1024\n\t"
                             "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:1024\n\t"
                             "ds_read_b64_tr_b16 %4, %8 offset:2048\n\tds_read_b64_tr_b16 %5, %8 offset:3072\n\t"
                             "ds_read_b64_tr_b16 %6, %9 offset:2048\n\tds_read_b64_tr_b16 %7, %9 offset:3072"
                             : "=&v"(vl[0]), "=&v"(vl[1]), "=&v"(vl[2]), "=&v"(vl[3]), "=&v"(vl[4]), "=&v"(vl[5]), "=&v"(vl[6]), "=&v"(vl[7])
                             : "v"(va0), "v"(va1)
                             : "memory");
            }
            if (key0 + 32 > N) {  // wave-uniform: only the last tile of the sequence
                int lim = N - key0 - 4 * hi;
                asm volatile("" : "+v"(lim));  // (opaque: the 16 lane masks would be hoisted into 32 SGPRs)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if ((e & 3) + 8 * (e >> 2) >= lim) s[e] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            mx = max_across_halves(mx);
            if constexpr (FIRST) {
                level.set(mx, a.scale_log2e);
            } else {
                // rescale only when a score outgrows the running max by more than kDeferLog2: P stays <= 2^kDeferLog2 until then
                if (__any(level.excess(mx, a.scale_log2e) > kDeferLog2)) {
                    const float alpha = level.raise(mx, a.scale_log2e);
                    l_run *= alpha;
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
                }
            }
            float psum = 0.f;
            level.arguments(s, a.scale_log2e);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e]);
                psum += s[e];
            }
            if constexpr (FIRST) l_run = psum; else l_run += psum;
            asm volatile("s_waitcnt lgkmcnt(0)"
                         : "+v"(vl[0]), "+v"(vl[1]), "+v"(vl[2]), "+v"(vl[3]), "+v"(vl[4]), "+v"(vl[5]), "+v"(vl[6]), "+v"(vl[7])::"memory");
#pragma unroll
            for (int sk = 0; sk < 2; ++sk) {
                const bf16x8 pb = pack8(s, sk);
                const short8v b0 = __builtin_shufflevector(vl[4 * sk + 0], vl[4 * sk + 1], 0, 1, 2, 3, 4, 5, 6, 7);
                const short8v b1 = __builtin_shufflevector(vl[4 * sk + 2], vl[4 * sk + 3], 0, 1, 2, 3, 4, 5, 6, 7);
                if (FIRST && sk == 0) {
                    const f32x16 z = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    o[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b0), pb, z, 0, 0, 0);
                    o[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b1), pb, z, 0, 0, 0);
                } else {
                    o[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b0), pb, o[0], 0, 0, 0);
                    o[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, b1), pb, o[1], 0, 0, 0);
                }
            }
        }
        slot = slot + 1 == R ? 0 : slot + 1;
    };

    for (int j = 0; j < nmy; ++j) {
        const bool active = q0 < N;  // wave-uniform
        tile_step(std::true_type{}, j, 0, active);
        for (int p = 1; p < nt; ++p) tile_step(std::false_type{}, j, p, active);

        // ---- item finished: ST stores per active wave, never waited for explicitly
        if (active) {
            const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
            const bool live = l_tot > 0.f || l_tot != l_tot;  // (a NaN row stays one)
            const float inv = live ? __builtin_amdgcn_rcpf(l_tot) : 0.f;
            if constexpr (LSE) {
                if (hi == 0 && q0 + r < N) a.lse[((size_t)cur.b * H + cur.h) * N + q0 + r] = live ? level.log_sum(l_tot, a.scale_log2e) : INFINITY;
            }
            // the lane halves trade 8-byte pieces (v_permlane32_swap): every lane stores 8 consecutive head dims, 16 bytes; rows
            // >= N are out of the resource's range
            const int D = H * DH;
            const __amdgpu_buffer_rsrc_t orsrc = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(a.out + (size_t)cur.b * N * D + (size_t)cur.h * DH), 0, (unsigned)(N - 1) * (unsigned)(D * 2) + (unsigned)(DH * 2), 0x00020000);
            const unsigned ooff = (q0 + r < N) ? (unsigned)(q0 + r) * (unsigned)(D * 2) + (unsigned)(16 * hi) : 0x80000000u;
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                unsigned w[4][2];
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    bf16x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (bf16_t)(o[d][g4 * 4 + e] * inv);
                    const u32x2 u = __builtin_bit_cast(u32x2, v);
                    w[g4][0] = u[0];
                    w[g4][1] = u[1];
                }
#pragma unroll
                for (int pr = 0; pr < 2; ++pr) {
                    u32x4 pk;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const auto sw = __builtin_amdgcn_permlane32_swap(w[2 * pr][k], w[2 * pr + 1][k], false, false);
                        pk[k] = (unsigned)sw[0];
                        pk[2 + k] = (unsigned)sw[1];
                    }
                    __builtin_amdgcn_raw_buffer_store_b128(pk, orsrc, (int)(ooff + (unsigned)(d * 64 + 32 * pr)), 0, 0);
                }
            }
        }
        prev_active = active;
        if (j + 1 < nmy) {
            const Item nx = item_at(j + 1);
            fresh = nx.h == cur.h && nx.qb == cur.qb;
            cur = nx;
            q0 = (cur.qb * NW + wave) * 32;
        }
    }
    wait_vm<0>();  // the dummy DMAs of the tail must land before the LDS is released
}

size_t ring_lds(int R, int N, int slice) { return (size_t)R * SLOT + NW * QSLOT + (size_t)((N + 31) / 32 * 32 + slice) * 4; }

template <int R>
int launch_ring(const RelRingArgs& a, size_t lds, hipStream_t stream) {
    static PerDeviceInt resident_of[2];  // workgroups per CU by LSE: 2 when two fit, per device (attribute set along)
    const bool lse = a.lse != nullptr;
    const void* kern = lse ? (const void*)attention_rel_dh64_kernel<R, true> : (const void*)attention_rel_dh64_kernel<R, false>;
    std::atomic<int>* rs = resident_of[lse].slot();
    if (!rs || !rs->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (rs) rs->store(1, std::memory_order_relaxed);
    }
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    const int resident = ncu * (lds <= 80 * 1024 ? 2 : 1);
    const int grid = a.nitems < resident ? a.nitems : resident;
    if (lse) hipLaunchKernelGGL((attention_rel_dh64_kernel<R, true>), dim3(grid), dim3(NW * 64), lds, stream, a);
    else hipLaunchKernelGGL((attention_rel_dh64_kernel<R, false>), dim3(grid), dim3(NW * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

}  // namespace

// Takes it: whole sequences of at least 4 key tiles (the counted waits assume an item's stores and Q loads are out of the window
// before the next item's), one sample's rows within 32-bit offsets, the LDS. us, this / the chunked kernel of attention_rel.hip: 256 x 197
// tokens x 12 heads 86 / 108, 16 x 1024 x 16 102 / 117, 32 x 577 x 16 97 / 95.
bool attention_rel_dh64_eligible(const vit_rel_pos* pos, int batch, int heads, int kv_heads) {
    const int N = pos->prefix + pos->grid_h * pos->grid_w;
    if (N <= 96 || (long)N * (heads + 2 * kv_heads) * DH * 2 >= (1L << 31)) return false;
    return ring_lds(3, N, rel_slice_max(pos->grid_h, pos->grid_w, NW * 32)) <= 160 * 1024;
}

int launch_attention_rel_dh64(const vit_rel_pos* pos, const RelGeo& geo, const void* qkv, void* out, float* lse, int batch, int heads, int kv_heads,
                              float scale, hipStream_t stream) {
    RelRingArgs a{};
    a.qkv = (const unsigned char*)qkv;
    a.out = (bf16_t*)out;
    a.lse = lse;
    a.geo = geo;
    a.B = batch;
    a.N = pos->prefix + pos->grid_h * pos->grid_w;
    a.H = heads;
    a.HK = kv_heads;
    a.qblocks = ceil_div(ceil_div(a.N, 32), NW);
    const int64_t nitems = (int64_t)batch * heads * a.qblocks;
    VIT_REQUIRE(nitems < (1LL << 31), "attention_rel: too many (sample, head, query block) items");
    a.nitems = (int)nitems;
    a.scale_log2e = scale * LOG2E;
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, NW * 32);
    // the deepest ring that leaves two workgroups a CU, else the deepest that fits one
    for (size_t room : {(size_t)80 * 1024, (size_t)160 * 1024}) {
        if (ring_lds(5, a.N, slice) <= room) return launch_ring<5>(a, ring_lds(5, a.N, slice), stream);
        if (ring_lds(4, a.N, slice) <= room) return launch_ring<4>(a, ring_lds(4, a.N, slice), stream);
        if (ring_lds(3, a.N, slice) <= room) return launch_ring<3>(a, ring_lds(3, a.N, slice), stream);
    }
    return vit_set_error(VIT_E_INVALID, "attention_rel: no ring fits %d tokens", a.N);
}
