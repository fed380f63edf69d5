// Attention with a learned relative position bias by buckets, forward: out = softmax(scale Q K^T + bias) V, the bias of
// rel_bias.h. Same dataflow as attention.hip (query on the lane: S^T = K Q^T, online softmax, O^T += V^T P^T, no score
// matrix in memory); the product's accumulator starts from the bias, read from the head's LDS expansion.
//
// Beyond attention.hip: per-sample lengths (keys behind them are never read, queries behind them give zeros), key / value
// heads shared by groups of query heads, entries that mask (a query whose every key is masked gives zeros and lse = +inf).
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
    int N, H, HK, KC, slice;  // slice: floats of LDS for the expansion
    float scale_log2e;
};

template <int DH>
struct RGeo {
    static constexpr int KSTEPS = DH / 16;
    static constexpr int DB = (DH + 31) / 32;
    static constexpr int KS = DH * 2 + 16;     // K row stride, bytes
    static constexpr int VS = (DB | 1) * 64;   // V row stride, bytes (odd multiple of 64)
    static constexpr int CHUNKS = DH / 8;
};

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

template <int DH>
__global__ __launch_bounds__(512) void attention_rel_bf16_kernel(const RelFwdArgs a) {
    using G = RGeo<DH>;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int KC = a.KC, N = a.N, H = a.H;
    unsigned char* Kl = smem;
    unsigned char* Vl = smem + (size_t)KC * G::KS;
    int* codes = (int*)(Vl + (size_t)KC * G::VS);
    float* T = (float*)(codes + KC);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nwaves = blockDim.x >> 6;
    const int r = lane & 31, hi = lane >> 5;
    const int b = blockIdx.x / H, h = blockIdx.x - b * H, hk = h / (H / a.HK);
    const size_t rs = (size_t)(H + 2 * a.HK) * DH;
    const bf16_t* base = (const bf16_t*)a.qkv + (size_t)b * N * rs;
    const bf16_t* kbase = base + (size_t)(H + hk) * DH;
    const bf16_t* vbase = kbase + (size_t)a.HK * DH;
    const int nb = sample_length(a.lengths, b, N);

    const int blk0 = blockIdx.y * nwaves * 32;
    const int q0 = blk0 + wave * 32, q = q0 + r;
    const int qrow = q < nb ? q : (nb > 0 ? nb - 1 : 0);
    bf16x8 qf[G::KSTEPS];
#pragma unroll
    for (int ks = 0; ks < G::KSTEPS; ++ks) qf[ks] = *(const bf16x8*)(base + (size_t)qrow * rs + (size_t)h * DH + ks * 16 + hi * 8);

    const int blk1 = blk0 + nwaves * 32 - 1;
    const RelSlice sl(a.geo, blk0, blk1 < N ? blk1 : N - 1, true);
    rel_expand(a.geo, T, sl, true, h);
    const RelLane<true> rl(a.geo, sl, T, q, N - 1);

    f32x16 o[G::DB];
#pragma unroll
    for (int d = 0; d < G::DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    const int g = lane >> 4, i16 = lane & 15;
    const int tr_key = 4 * (g >> 1) + (i16 >> 2);
    const int tr_col = ((g & 1) * 16 + 4 * (i16 & 3)) * 2;

    for (int kc0 = 0; kc0 < nb; kc0 += KC) {
        int nkeys = nb - kc0;
        nkeys = nkeys > KC ? KC : (nkeys + 31) & ~31;
        __syncthreads();
        const int total = nkeys * G::CHUNKS;
        for (int idx = tid; idx < total; idx += blockDim.x) {
            const int key = idx / G::CHUNKS, c = idx - key * G::CHUNKS;
            int gk = kc0 + key;
            if (gk > nb - 1) gk = nb - 1;  // pad keys re-read the last row (their scores are masked)
            *(bf16x8*)(Kl + (size_t)key * G::KS + c * 16) = *(const bf16x8*)(kbase + (size_t)gk * rs + c * 8);
            *(bf16x8*)(Vl + (size_t)key * G::VS + c * 16) = *(const bf16x8*)(vbase + (size_t)gk * rs + c * 8);
        }
        for (int i = tid; i < nkeys; i += blockDim.x) codes[i] = rel_row_code(a.geo, sl, true, kc0 + i);
        __syncthreads();

        for (int t = 0; t < nkeys >> 5; ++t) {
            const int key0 = kc0 + t * 32;
            f32x16 s;
            rel_tile(s, codes + t * 32, rl, hi, a.geo.prefix, key0);
            const unsigned char* kp = Kl + (size_t)(t * 32 + r) * G::KS + hi * 16;
#pragma unroll
            for (int ks = 0; ks < G::KSTEPS; ++ks)
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(kp + ks * 32), qf[ks], s, 0, 0, 0);
            if (key0 + 32 > nb) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (key0 + (e & 3) + 8 * (e >> 2) + 4 * hi >= nb) s[e] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            mx = max_across_halves(mx);
            const float m_new = fmaxf(m_run, mx * a.scale_log2e);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;  // nothing but masked keys so far
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
            m_run = m_new;
            float psum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e] * a.scale_log2e - m_use);
                psum += s[e];
            }
            l_run = l_run * alpha + psum;
            if (__any(alpha != 1.f)) {
#pragma unroll
                for (int d = 0; d < G::DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
            }
#pragma unroll
            for (int sk = 0; sk < 2; ++sk) {
                const bf16x8 pb = pack8(s, sk);
                const unsigned char* vp = Vl + (size_t)(t * 32 + 16 * sk + tr_key) * G::VS + tr_col;
#pragma unroll
                for (int d = 0; d < G::DB; ++d) {
                    const short4v lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(vp + d * 64));
                    const short4v hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(vp + 8 * G::VS + d * 64));
                    const short8v both = __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, both), pb, o[d], 0, 0, 0);
                }
            }
        }
    }

    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const bool any = l_tot > 0.f || l_tot != l_tot;  // (a NaN row stays one)
    const bool live = q < nb && any;
    const float inv = 1.0f / l_tot;
    if (q < N) {
        if (a.lse != nullptr && hi == 0) a.lse[((size_t)b * H + h) * N + q] = live ? m_run + log2f(l_tot) : INFINITY;
        const size_t at = ((size_t)b * N + q) * H * DH + (size_t)h * DH;
#pragma unroll
        for (int d = 0; d < G::DB; ++d)
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

// ---- fp32: the same structure on v_mfma_f32_32x32x2_f32 (exact fp32 products)
template <int DH>
__global__ __launch_bounds__(512) void attention_rel_f32_kernel(const RelFwdArgs a) {
    constexpr int DB = (DH + 31) / 32;
    constexpr int KSF = DH + 1;   // K row stride, floats (odd: conflict-free column reads)
    constexpr int VSF = DB * 32;  // V row stride, floats
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int KC = a.KC, N = a.N, H = a.H;
    int* codes = (int*)smem;
    float* Kl = (float*)(codes + KC);
    float* Vl = Kl + (size_t)KC * KSF;
    float* T = Vl + (size_t)KC * VSF;

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nwaves = blockDim.x >> 6;
    const int r = lane & 31, hi = lane >> 5;
    const int b = blockIdx.x / H, h = blockIdx.x - b * H, hk = h / (H / a.HK);
    const size_t rs = (size_t)(H + 2 * a.HK) * DH;
    const float* base = (const float*)a.qkv + (size_t)b * N * rs;
    const float* kbase = base + (size_t)(H + hk) * DH;
    const float* vbase = kbase + (size_t)a.HK * DH;
    const int nb = sample_length(a.lengths, b, N);

    const int blk0 = blockIdx.y * nwaves * 32;
    const int q0 = blk0 + wave * 32, q = q0 + r;
    const int qrow = q < nb ? q : (nb > 0 ? nb - 1 : 0);
    float qf[DH / 2];
#pragma unroll
    for (int t = 0; t < DH / 2; ++t) qf[t] = base[(size_t)qrow * rs + (size_t)h * DH + 2 * t + hi];

    const int blk1 = blk0 + nwaves * 32 - 1;
    const RelSlice sl(a.geo, blk0, blk1 < N ? blk1 : N - 1, true);
    rel_expand(a.geo, T, sl, true, h);
    const RelLane<true> rl(a.geo, sl, T, q, N - 1);

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    for (int kc0 = 0; kc0 < nb; kc0 += KC) {
        int nkeys = nb - kc0;
        nkeys = nkeys > KC ? KC : (nkeys + 31) & ~31;
        __syncthreads();
        for (int idx = tid; idx < nkeys * VSF; idx += blockDim.x) {
            const int key = idx / VSF, c = idx - key * VSF;
            const int gk = kc0 + key;
            float kv = 0.f, vv = 0.f;
            if (gk < nb && c < DH) {
                kv = kbase[(size_t)gk * rs + c];
                vv = vbase[(size_t)gk * rs + c];
            }
            if (c < DH) Kl[(size_t)key * KSF + c] = kv;
            Vl[(size_t)key * VSF + c] = vv;
        }
        for (int i = tid; i < nkeys; i += blockDim.x) codes[i] = rel_row_code(a.geo, sl, true, kc0 + i);
        __syncthreads();

        for (int t = 0; t < nkeys >> 5; ++t) {
            const int key0 = kc0 + t * 32;
            f32x16 s;
            rel_tile(s, codes + t * 32, rl, hi, a.geo.prefix, key0);
            const float* kp = Kl + (size_t)(t * 32 + r) * KSF + hi;
#pragma unroll
            for (int kk = 0; kk < DH / 2; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x2f32(kp[2 * kk], qf[kk], s, 0, 0, 0);
            if (key0 + 32 > nb) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (key0 + (e & 3) + 8 * (e >> 2) + 4 * hi >= nb) s[e] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float m_new = fmaxf(m_run, mx * a.scale_log2e);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = exp2f(m_run - m_use);
            m_run = m_new;
            float psum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = exp2f(fmaf(s[e], a.scale_log2e, -m_use));
                psum += s[e];
            }
            l_run = l_run * alpha + psum;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
            // k-step e pairs key (e & 3) + 8 (e >> 2) [lanes 0-31] with the same + 4 [lanes 32-63]: what register e holds
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float* vp = Vl + (size_t)(t * 32 + (e & 3) + 8 * (e >> 2) + 4 * hi) * VSF + r;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vp[d * 32], s[e], o[d], 0, 0, 0);
            }
        }
    }

    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const bool live = q < nb && (l_tot > 0.f || l_tot != l_tot);
    const float inv = 1.0f / l_tot;
    if (q < N) {
        float* op = (float*)a.out + ((size_t)b * N + q) * H * DH + (size_t)h * DH;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int d0 = d * 32 + 8 * g4 + 4 * hi;
                if (d0 < DH) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = live ? o[d][g4 * 4 + e] * inv : 0.f;
                    *(f32x4*)(op + d0) = v;
                }
            }
    }
}

// waves per block: cover ceil(N / 32) query tiles with the least padding, prefer more waves
int pick_waves(int N, int* qblocks) {
    const int n32 = ceil_div(N, 32);
    int best_w = 1, best_cost = 1 << 30;
    for (int w = 8; w >= 1; --w) {
        if (w < 4 && n32 >= 4) break;
        const int cost = ceil_div(n32, w) * w;
        if (cost < best_cost) { best_cost = cost; best_w = w; }
    }
    *qblocks = ceil_div(n32, best_w);
    return best_w;
}

template <int DH>
int launch_rel(RelFwdArgs a, const vit_rel_pos* pos, int batch, int dtype, hipStream_t stream) {
    int qblocks;
    const int waves = pick_waves(a.N, &qblocks);
    const int per_key = dtype == VIT_BF16 ? RGeo<DH>::KS + RGeo<DH>::VS + 4 : (DH + 1 + (DH + 31) / 32 * 32 + 1) * 4;
    a.slice = rel_slice_max(pos->grid_h, pos->grid_w, waves * 32);
    VIT_REQUIRE(a.slice <= kRelSliceCap, "attention_rel: a %d x %d grid needs %d bias entries at once, %d fit", pos->grid_h, pos->grid_w, a.slice, kRelSliceCap);
    int KC = 80 * 1024 / per_key / 32 * 32;
    const int npad = (a.N + 31) / 32 * 32;
    if (KC > npad) KC = npad;
    a.KC = KC;
    const size_t lds = (size_t)KC * per_key + (size_t)a.slice * 4;
    const void* kern = dtype == VIT_BF16 ? (const void*)attention_rel_bf16_kernel<DH> : (const void*)attention_rel_f32_kernel<DH>;
    static PerDeviceInt attr_set[2];
    std::atomic<int>* as = attr_set[dtype].slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    if (dtype == VIT_BF16) hipLaunchKernelGGL(attention_rel_bf16_kernel<DH>, dim3(batch * a.H, qblocks), dim3(waves * 64), lds, stream, a);
    else hipLaunchKernelGGL(attention_rel_f32_kernel<DH>, dim3(batch * a.H, qblocks), dim3(waves * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

}  // namespace

// persistent LDS-DMA ring for head_dim 64 and whole sequences (attention_rel_dh64.hip)
bool attention_rel_dh64_eligible(const vit_rel_pos* pos, int batch, int heads, int kv_heads);
int launch_attention_rel_dh64(const vit_rel_pos* pos, const RelGeo& geo, const void* qkv, void* out, float* lse, int batch, int heads, int kv_heads,
                              float scale, hipStream_t stream);

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
                  offsets, pos->num_buckets, heads, 1.0f / scale};
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
    if (dtype == VIT_BF16 && head_dim == 64 && !lengths && attention_rel_dh64_eligible(pos, batch, heads, kv_heads))
        return launch_attention_rel_dh64(pos, a.geo, qkv, out, lse, batch, heads, kv_heads, scale, (hipStream_t)stream);
#define REL_CASE(DHV) \
    case DHV: return launch_rel<DHV>(a, pos, batch, dtype, (hipStream_t)stream);
    switch (head_dim) {
        REL_CASE(16) REL_CASE(32) REL_CASE(48) REL_CASE(64) REL_CASE(80) REL_CASE(96) REL_CASE(112) REL_CASE(128)
    }
#undef REL_CASE
    return vit_set_error(VIT_E_INVALID, "vit_attention_rel_fwd: unsupported head_dim %d", head_dim);
}
