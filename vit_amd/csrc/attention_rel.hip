// Attention with a learned relative position bias by buckets, forward: out = softmax(scale Q K^T + bias) V, the bias of
// rel_bias.h. Same dataflow as attention.hip (query on the lane: S^T = K Q^T, online softmax, O^T += V^T P^T, no score
// matrix in memory); the product's accumulator starts from the bias, read from the head's LDS expansion.
//
// Beyond attention.hip: per-sample lengths (keys behind them are never read, queries behind them give zeros), key / value
// heads shared by groups of query heads, entries that mask (a query whose every key is masked gives zeros and lse = +inf).
//
// Roundings: scores, maxima, sums and the output are fp32. The bf16 kernels round the probabilities to bf16 for the second product (by at most
// 2^-8 of each: the matrix instructions take bf16 operands; their sum is of the unrounded ones) and the output when it is stored. Against the
// definition in 64 bits that is 2.3e-3 of the output where rounding the stored output alone leaves 1.7e-3 (fp32 mode: 4e-7).
#include "lds_image.h"
#include "rel_bias.h"
#include <math.h>

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct RelFwdArgs {
    const void* qkv;
    void* out;
    float* lse;
    const int* lengths;
    RelGeo geo;
    int N, H, HK;
    float scale_log2e;
};

constexpr float kDeferLog2 = 6.0f;  // the running max is left alone until a score outgrows it by more than this (base 2)
constexpr int KCH = 32;             // keys of a staged chunk
constexpr int NWAVE = 4;            // waves of a workgroup

__device__ __forceinline__ bf16x8 pack8(const f32x16& p, int s) {
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

// bf16, any head dim and length. A workgroup of up to 4 waves takes 32 queries a wave of one (sample, head); keys and values come in chunks
// of 32 by LDS-DMA into two buffers, the next chunk under the products of this one: one barrier a chunk, and three or four workgroups a CU
// to fill what a wave waits for. Bound by the vector instructions (softmax, bias addresses) that the matrix instructions only partly cover:
// 4 x 1025 tokens, 16 heads of 80: 60 us, 0.36 PFLOP/s; 6 samples of up to 1777 tokens, 16 heads of 128 over 4 of keys: 111 to 187 us by their
// lengths. With whole sequences staged, one workgroup a CU, these took 1.1 and 1.3 times as long.
template <int DH>
__global__ __launch_bounds__(64 * NWAVE) __attribute__((amdgpu_waves_per_eu(DH <= 64 ? 4 : 3))) void attention_rel_bf16_kernel(const RelFwdArgs a) {
    using I = LdsImage<DH>;
    constexpr int KS = DH / 16, DB = (DH + 31) / 32, IMG = KCH * I::ROW;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int N = a.N, H = a.H;
    int* const codes = (int*)(smem + 4 * IMG);  // [2][KCH]; images: [2][K, V]
    float* const T = (float*)(codes + 2 * KCH);
    const unsigned lds0 = (unsigned)(uintptr_t)LDS_PTR(smem);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
    const int r = lane & 31, hi = lane >> 5;
    const int b = blockIdx.x / H, h = blockIdx.x - b * H, hk = h / (H / a.HK);
    const int pitch = (H + 2 * a.HK) * DH * 2;
    const unsigned char* base = (const unsigned char*)a.qkv + (size_t)b * N * pitch;
    const int nb = __builtin_amdgcn_readfirstlane(sample_length(a.lengths, b, N));
    // with lengths the last blocks first (only long samples have them), else last (the sequence may end inside one)
    const int blk0 = (a.lengths ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * nw * 32, blk1 = blk0 + nw * 32 - 1;
    const int q0 = blk0 + wave * 32, q = q0 + r;
    const int nc = blk0 < nb ? (nb + KCH - 1) / KCH : 0;  // (a block of rows behind the sample only stores zeros)

    const __amdgpu_buffer_rsrc_t kr = head_resource<DH>(base + (size_t)(H + hk) * DH * 2, N, pitch);
    const __amdgpu_buffer_rsrc_t vr = head_resource<DH>(base + (size_t)(H + a.HK + hk) * DH * 2, N, pitch);
    const RelSlice sl(a.geo, blk0, blk1 < N ? blk1 : N - 1, true);
    const LdsFill<DH> fill(lane);
    auto stage = [&](int c) {
        unsigned char* const dst = smem + (c & 1) * 2 * IMG;
        // (rows behind the sample re-read its last key: what is masked is still finite)
        fill.chunk(kr, dst, KCH, wave, nw, c * KCH, nb - 1, pitch);
        fill.chunk(vr, dst + IMG, KCH, wave, nw, c * KCH, nb - 1, pitch);
        for (int i = tid; i < KCH; i += blockDim.x) codes[(c & 1) * KCH + i] = rel_row_code(a.geo, sl, true, c * KCH + i);
    };
    if (nc > 0) stage(0);
    bf16x8 qf[KS];
    {
        const int qrow = q < nb ? q : (nb > 0 ? nb - 1 : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const bf16x8*)(base + (size_t)qrow * pitch + (size_t)h * DH * 2 + ks * 32 + hi * 16);
    }
    rel_expand(a.geo, T, sl, true, h);
    const RelLane<true> rl(a.geo, sl, T, q, N - 1);
    const TrRead<DH> tr(lane);
    const int ro = (int)lds0 + I::at(r, hi);

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    RelLevel level;
    float l_run = 0.f;
    for (int c = 0; c < nc; ++c) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");  // the chunk is whole; nobody reads the other buffer any more
        if (c + 1 < nc) stage(c + 1);
        const int img = (c & 1) * 2 * IMG;
        {
            const int key0 = c * KCH;
            f32x16 s;
            rel_tile(s, codes + (c & 1) * KCH, rl, hi, a.geo.prefix, key0);
            int ka = ro + img;
            asm volatile("" : "+v"(ka));
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_chunk(I::step(ka, ks)), qf[ks], s, 0, 0, 0);
            const unsigned vimg = lds0 + (unsigned)(img + IMG);
            bf16x8 vt[2][DB];
            if constexpr (DB == 4) tr.template read_step<0>(vt[0], vimg);  // (32 registers at once would cost a wave a SIMD)
            else tr.read(vt, vimg);
            if (key0 + 32 > nb) {
                int lim = nb - key0 - 4 * hi;
                asm volatile("" : "+v"(lim));  // (opaque: the 16 lane masks would be hoisted into 32 SGPRs)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if ((e & 3) + 8 * (e >> 2) >= lim) s[e] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            mx = max_across_halves(mx);
            // rescale only when a score outgrows the running max by more than kDeferLog2: P stays <= 2^kDeferLog2 until then
            if (__any(level.excess(mx, a.scale_log2e) > kDeferLog2)) {
                const float alpha = level.raise(mx, a.scale_log2e);
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
            }
            float psum = 0.f;
            level.arguments(s, a.scale_log2e);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e]);
                psum += s[e];
            }
            l_run += psum;
#pragma unroll
            for (int sk = 0; sk < 2; ++sk) {
                if constexpr (DB == 4)
                    if (sk == 1) tr.template read_step<1>(vt[1], vimg);
                const bf16x8 pb = pack8(s, sk);
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt[sk][d], pb, o[d], 0, 0, 0);
            }
        }
    }

    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const bool live = q < nb && (l_tot > 0.f || l_tot != l_tot);  // (a NaN row stays one)
    const float inv = 1.0f / l_tot;
    if (q < N) {
        if (a.lse != nullptr && hi == 0) a.lse[((size_t)b * H + h) * N + q] = live ? level.log_sum(l_tot, a.scale_log2e) : INFINITY;
        const size_t at = ((size_t)b * N + q) * H * DH + (size_t)h * DH;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int d0 = d * 32 + 8 * g4 + 4 * hi;
                if (d0 < DH) {
                    bf16x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (bf16_t)(live ? o[d][g4 * 4 + e] * inv : 0.f);
                    *(bf16x4*)((bf16_t*)a.out + at + d0) = v;
                }
            }
    }
}

template <int DH>
int launch_rel_bf16(RelFwdArgs a, const vit_rel_pos* pos, int batch, hipStream_t stream) {
    const int n32 = ceil_div(a.N, 32), qblocks = ceil_div(n32, NWAVE), waves = ceil_div(n32, qblocks);  // equal blocks
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, waves * 32);
    const size_t lds = (size_t)4 * KCH * LdsImage<DH>::ROW + (size_t)(2 * KCH + slice) * 4;
    static PerDeviceInt attr_set;
    std::atomic<int>* as = attr_set.slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute((const void*)attention_rel_bf16_kernel<DH>, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(attention_rel_bf16_kernel<DH>, dim3(batch * a.H, qblocks), dim3(waves * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

}  // namespace

// persistent LDS-DMA ring for head_dim 64 and whole sequences (attention_rel_dh64.hip)
bool attention_rel_dh64_eligible(const vit_rel_pos* pos, int batch, int heads, int kv_heads);
int launch_attention_rel_dh64(const vit_rel_pos* pos, const RelGeo& geo, const void* qkv, void* out, float* lse, int batch, int heads, int kv_heads,
                              float scale, hipStream_t stream);

// fp32, and bf16 with few query rows: the waves of a workgroup share the keys (attention_rel_split.hip)
bool attention_rel_split_eligible(const vit_rel_pos* pos, int batch, int heads, int dtype, int ncu);
int launch_attention_rel_split(const vit_rel_pos* pos, const RelGeo& geo, const void* qkv, const int* lengths, void* out, float* lse, int batch, int heads,
                               int kv_heads, int head_dim, float scale, int dtype, int ncu, hipStream_t stream);

int rel_make_geo(const char* who, const vit_rel_pos* pos, const float* table, int heads, float scale, RelGeo* out, int* seq) {
    VIT_REQUIRE(pos && table, "%s: null argument", who);
    VIT_REQUIRE(pos->prefix >= 0 && pos->prefix <= 32, "%s: prefix must be in [0, 32], got %d", who, pos->prefix);
    VIT_REQUIRE(pos->grid_h > 0 && pos->grid_w > 0 && (int64_t)pos->grid_h * pos->grid_w <= 16384,
                "%s: bad grid %d x %d", who, pos->grid_h, pos->grid_w);
    VIT_REQUIRE(scale >= 1e-6f && scale <= 1e6f, "%s: scale must be in [1e-6, 1e6]", who);
    const int offsets = (2 * pos->grid_h - 1) * (2 * pos->grid_w - 1);
    VIT_REQUIRE(pos->num_buckets > 0 && (pos->bucket_of || pos->num_buckets >= offsets + (pos->prefix ? 3 : 0)),
                "%s: %d buckets without a map for %d offsets", who, pos->num_buckets, offsets);
    *out = RelGeo{table, pos->bucket_of, pos->prefix, pos->grid_w, pos->grid_h * pos->grid_w, (pos->grid_h - 1) * (2 * pos->grid_w - 1) + pos->grid_w - 1,
                  offsets, pos->num_buckets, heads, 1.0f / scale, 1.0f / (float)pos->grid_w};
    *seq = pos->prefix + pos->grid_h * pos->grid_w;
    return VIT_OK;
}

extern "C" int vit_attention_rel_fwd(const vit_rel_pos* pos, const void* qkv, const float* table, const int32_t* lengths, void* out,
                                     float* lse, int batch, int heads, int kv_heads, int head_dim, float scale, int dtype,
                                     void* stream) {
    VIT_REQUIRE(qkv && out, "vit_attention_rel_fwd: null argument");
    VIT_REQUIRE(batch > 0 && heads > 0 && kv_heads > 0 && (int64_t)batch * heads < (1 << 22), "vit_attention_rel_fwd: empty or too large a problem");
    VIT_REQUIRE(heads % kv_heads == 0, "vit_attention_rel_fwd: heads %d is not a multiple of kv_heads %d", heads, kv_heads);
    VIT_REQUIRE(head_dim % 16 == 0 && head_dim >= 16 && head_dim <= 128,
                "vit_attention_rel_fwd: head_dim must be a multiple of 16 in [16,128], got %d", head_dim);
    VIT_REQUIRE(dtype == VIT_BF16 || dtype == VIT_F32, "vit_attention_rel_fwd: bad dtype %d", dtype);
    VIT_REQUIRE(!lse || dtype == VIT_BF16, "vit_attention_rel_fwd: the log-sum-exp output is bf16-mode only");
    VIT_REQUIRE((((uintptr_t)qkv | (uintptr_t)out) & 15) == 0, "vit_attention_rel_fwd: tensors must be 16-byte aligned");
    RelFwdArgs a{};
    VIT_TRY_RC(rel_make_geo("vit_attention_rel_fwd", pos, table, heads, scale, &a.geo, &a.N));
    a.qkv = qkv;
    a.out = out;
    a.lse = lse;
    a.lengths = lengths;
    a.H = heads;
    a.HK = kv_heads;
    a.scale_log2e = scale * LOG2E;
    VIT_REQUIRE((int64_t)a.N * (heads + 2 * kv_heads) * head_dim * (dtype == VIT_BF16 ? 2 : 4) < (1LL << 31), "vit_attention_rel_fwd: one sample's qkv rows exceed 2 GiB");
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, 128);
    VIT_REQUIRE(slice <= kRelSliceCap, "vit_attention_rel_fwd: a %d x %d grid needs %d bias entries at once, %d fit", pos->grid_h, pos->grid_w, slice, kRelSliceCap);
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    if (attention_rel_split_eligible(pos, batch, heads, dtype, ncu))
        return launch_attention_rel_split(pos, a.geo, qkv, lengths, out, lse, batch, heads, kv_heads, head_dim, scale, dtype, ncu, (hipStream_t)stream);
    if (head_dim == 64 && !lengths && attention_rel_dh64_eligible(pos, batch, heads, kv_heads))
        return launch_attention_rel_dh64(pos, a.geo, qkv, out, lse, batch, heads, kv_heads, scale, (hipStream_t)stream);
#define REL_CASE(DHV) \
    case DHV: return launch_rel_bf16<DHV>(a, pos, batch, (hipStream_t)stream);
    switch (head_dim) {
        REL_CASE(16) REL_CASE(32) REL_CASE(48) REL_CASE(64) REL_CASE(80) REL_CASE(96) REL_CASE(112) REL_CASE(128)
    }
#undef REL_CASE
    return vit_set_error(VIT_E_INVALID, "vit_attention_rel_fwd: unsupported head_dim %d", head_dim);
}
