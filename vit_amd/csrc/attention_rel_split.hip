// Attention with a learned relative position bias (the mathematics of attention_rel.hip) with a workgroup for 32 queries of one (sample,
// head) whose waves share the keys: wave w takes the tiles w, w + waves, .., and the waves' running maxima, sums and outputs are joined
// through LDS. Every fp32 call comes here, and bf16 calls with few queries: one image of 197 tokens and 12 heads is 84 workgroups, where
// the kernels that share staged keys between 128 or 256 queries have 24 or 12 that walk all tiles one after the other.
//
// bf16 is bound by latency here: the workgroup's queries and each wave's first key and value tile are on their way (LDS-DMA, whole rows)
// before the bias is expanded, and a wave's next tiles come under its softmax; there is no barrier between the first and the join.
// fp32 is bound by the matrix instructions (64 cycles for 4096 operations).
//
// Which calls, measured in us, this kernel / the shared ones (bf16; workgroups here per CU in brackets):
//   197 tokens x 12 heads x 64   samples 1 [0.3]: 6.5 / 11.7   4 [1.3]: 7.6 / 11.8   8 [2.6]: 9.1 / 12.1   16 [5.3]: 15.5 / 12.4
//   1025 x 16 x 80               samples 1 [2.1]: 32 / 45      2 [4.1]: 49 / 48      4 [8.3]: 85 / 60
//   256 x 8 x 128                samples 8 [2]: 10.7 / 16.6    16 [4]: 18.8 / 18.0
// so up to 4 a CU. Waves of a workgroup: 8 while there is a CU for each, else 4, more of which fit a CU at once (us at 8 / 4 waves):
//   bf16 197 x 12 x 64, samples 1: 6.5 / 6.7, 8: 11.8 / 9.1;  577 x 12 x 64, samples 1: 8.4 / 9.8, 8: 35 / 32
//   fp32 197 x 12 x 64, samples 1: 10.2 / 10.5, 4: 18.0 / 15.3, 32: 97 / 68;  577, samples 16: 258 / 186 (its matrix instructions: 115)
// fp32 with 128 to 256 queries on shared keys took 3 times as long for 4 x 197 tokens, 1.3 for 32 x 197, 1.8 for 32 x 577.
#include "lds_image.h"
#include "rel_bias.h"
#include <math.h>

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct RelSplitArgs {
    const void* qkv;
    void* out;
    float* lse;
    const int* lengths;
    RelGeo geo;
    int N, H, HK;
    float scale_log2e;
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

// ---- one tile's softmax step: s in, probabilities out; o rescaled where a row's maximum rose
template <int DB>
__device__ __forceinline__ void soft_step(f32x16& s, f32x16 (&o)[DB], RelLevel& level, float& l_run, int key0, int nb, int hi, float scale_log2e) {
    if (key0 + 32 > nb) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (key0 + (e & 3) + 8 * (e >> 2) + 4 * hi >= nb) s[e] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = max_across_halves(mx);
    if (__any(level.excess(mx, scale_log2e) > 0.f)) {
        const float alpha = level.raise(mx, scale_log2e);
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
    }
    float psum = 0.f;
    level.arguments(s, scale_log2e);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(s[e]);
        psum += s[e];
    }
    l_run += psum;
}

// ---- the join. Regions of `region` floats a wave: O^T [DH][32]; ml: [waves][32] of (m, M, sum, -), the rows' levels and sums
template <typename T, int DH, bool MIXED>  // MIXED: row i of block d is value DB i + d, not 32 d + i
__device__ __forceinline__ void join(const f32x16 (&o)[(DH + 31) / 32], const RelLevel& level, float l_run, float c, float* regions, int region, float* ml, T* out,
                                     float* lse, int q0, int nb, int N, int row_elems, int wave, int nw, int lane) {
    const int r = lane & 31, hi = lane >> 5;
    float* mine = regions + (size_t)wave * region;
#pragma unroll
    for (int d = 0; d < (DH + 31) / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int i = (e & 3) + 8 * (e >> 2) + 4 * hi, dd = MIXED ? i * ((DH + 31) / 32) + d : d * 32 + i;
            if (dd < DH) mine[dd * 32 + r] = o[d][e];
        }
    l_run += __shfl_xor(l_run, 32, 64);
    if (hi == 0) {
        *(f32x4*)(ml + (wave * 32 + r) * 4) = f32x4{level.m, level.M, l_run, 0.f};
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * (DH / 8); i += blockDim.x) {
        const int q = i & 31, d0 = (i >> 5) * 8;
        if (q0 + q >= N) continue;
        auto row = [&](int w) { return *(const f32x4*)(ml + (w * 32 + q) * 4); };
        RelLevel top;  // the highest of the waves' levels
        top.m = row(0)[0], top.M = row(0)[1];
        auto above = [&](const f32x4& v) { return fmaf(v[1] - top.M, c, v[0] - top.m); };
        for (int w = 1; w < nw; ++w) {
            const f32x4 v = row(w);
            const bool higher = above(v) > 0.f;
            top.m = higher ? v[0] : top.m;
            top.M = higher ? v[1] : top.M;
        }
        float l = 0.f, v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        for (int w = 0; w < nw; ++w) {
            const f32x4 x = row(w);
            const float f = __builtin_amdgcn_exp2f(above(x));
            l = fmaf(f, x[2], l);
            const float* p = regions + (size_t)w * region + d0 * 32 + q;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(f, p[e * 32], v[e]);
        }
        const bool live = q0 + q < nb && (l > 0.f || l != l);  // (a NaN row stays one)
        const float inv = 1.0f / l;
        T* dst = out + (size_t)(q0 + q) * row_elems + d0;
        if constexpr (sizeof(T) == 2) {
            bf16x8 w;
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = (bf16_t)(live ? v[e] * inv : 0.f);
            *(bf16x8*)dst = w;
        } else {
            f32x4 a, c;
#pragma unroll
            for (int e = 0; e < 4; ++e) { a[e] = live ? v[e] * inv : 0.f; c[e] = live ? v[4 + e] * inv : 0.f; }
            *(f32x4*)dst = a;
            *(f32x4*)(dst + 4) = c;
        }
        if (lse != nullptr && d0 == 0) lse[q0 + q] = live ? top.log_sum(l, c) : INFINITY;
    }
}

// One wave's region: its key tile and, bf16, its value tile; then its part of the join. Rows of DH values of `size` bytes.
constexpr int split_image(int dh, int size) {
    const int ch = dh * size / 16;
    return 32 * 16 * (ch == 8 || ch == 16 || ch == 32 ? ch : ch + 1);
}
constexpr int split_region(int dh, int size) {  // bytes
    const int images = (size == 2 ? 2 : 1) * split_image(dh, size), joined = 32 * dh * 4;
    return images > joined ? images : joined;
}

template <typename T, int DH>
struct Split {  // what both kernels start with
    static constexpr int IMG = split_image(DH, sizeof(T)), REGION = split_region(DH, sizeof(T));
    using I = LdsImage<DH * (int)sizeof(T) / 2>;
    int lane, wave, nw, r, hi, b, h, nb, q0, q, nt, pitch;
    unsigned char *qimg, *region;
    float *regions, *ml, *bias;
    int* codes;
    __amdgpu_buffer_rsrc_t kr, vr;
    RelLane<true> rl;
    __device__ __forceinline__ void tile(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int t) const {
        for (int i = 0; i < 32; i += I::RPI) I::dma(rsrc, dst, i, 32, t * 32, nb - 1, pitch, lane);
    }
    __device__ __forceinline__ Split(const RelSplitArgs& a, unsigned char* smem) {
        const int tid = threadIdx.x, H = a.H, N = a.N;
        lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
        r = lane & 31, hi = lane >> 5;
        qimg = smem;
        regions = (float*)(smem + IMG);
        region = smem + IMG + (size_t)wave * REGION;
        ml = (float*)(smem + IMG + (size_t)nw * REGION);
        codes = (int*)(ml + nw * 128);
        bias = (float*)(codes + ((N + 31) >> 5) * 32);
        b = blockIdx.x / H, h = blockIdx.x - b * H;
        const int hk = h / (H / a.HK);
        pitch = (H + 2 * a.HK) * DH * (int)sizeof(T);
        const unsigned char* base = (const unsigned char*)a.qkv + (size_t)b * N * pitch;
        nb = __builtin_amdgcn_readfirstlane(sample_length(a.lengths, b, N));
        q0 = blockIdx.y * 32, q = q0 + r;
        nt = q0 < nb ? (nb + 31) >> 5 : 0;
        const __amdgpu_buffer_rsrc_t qr = head_resource<DH * (int)sizeof(T) / 2>(base + (size_t)h * DH * sizeof(T), N, pitch);
        kr = head_resource<DH * (int)sizeof(T) / 2>(base + (size_t)(H + hk) * DH * sizeof(T), N, pitch);
        vr = head_resource<DH * (int)sizeof(T) / 2>(base + (size_t)(H + a.HK + hk) * DH * sizeof(T), N, pitch);
        if (nt > 0) {
            for (int i = wave * I::RPI; i < 32; i += nw * I::RPI) I::dma(qr, qimg, i, 32, q0, nb - 1, pitch, lane);
            if (wave < nt) {
                tile(kr, region, wave);
                if (sizeof(T) == 2) tile(vr, region + IMG, wave);
            }
        }
        const RelSlice sl(a.geo, q0, q0 + 31 < N ? q0 + 31 : N - 1, true);
        rel_expand(a.geo, bias, sl, true, h);
        for (int i = tid; i < nt * 32; i += blockDim.x) codes[i] = rel_row_code(a.geo, sl, true, i);
        rl = RelLane<true>(a.geo, sl, bias, q, N - 1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // bias, codes, queries
    }
};

template <int DH>
__global__ __launch_bounds__(512) void attention_rel_split_bf16_kernel(const RelSplitArgs a) {
    using S = Split<bf16_t, DH>;
    using I = typename S::I;
    constexpr int KS = DH / 16, DB = (DH + 31) / 32;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const S w(a, smem);
    const TrRead<DH> tr(w.lane);
    const unsigned vimg = (unsigned)(uintptr_t)LDS_PTR(w.region) + S::IMG;
    bf16x8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const bf16x8*)(w.qimg + I::at(w.r, 2 * ks + w.hi));
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    RelLevel level;
    float l_run = 0.f;
    for (int t = w.wave; t < w.nt; t += w.nw) {
        f32x16 s;
        rel_tile(s, w.codes + t * 32, w.rl, w.hi, a.geo.prefix, t * 32);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this tile's rows
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(w.region + I::at(w.r, 2 * ks + w.hi)), qf[ks], s, 0, 0, 0);
        bf16x8 vt[2][DB];
        tr.read(vt, vimg);
        if (t + w.nw < w.nt) {  // (the keys' and the values' reads are over) the next tile's rows under this one's softmax
            asm volatile("" : "+v"(s));
            w.tile(w.kr, w.region, t + w.nw);
            w.tile(w.vr, w.region + S::IMG, t + w.nw);
        }
        soft_step<DB>(s, o, level, l_run, t * 32, w.nb, w.hi, a.scale_log2e);
#pragma unroll
        for (int sk = 0; sk < 2; ++sk) {
            const bf16x8 pb = pack8(s, sk);
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt[sk][d], pb, o[d], 0, 0, 0);
        }
    }
    join<bf16_t, DH, false>(o, level, l_run, a.scale_log2e, w.regions, S::REGION / 4, w.ml, (bf16_t*)a.out + ((size_t)w.b * a.N * a.H + w.h) * DH,
                            a.lse ? a.lse + ((size_t)w.b * a.H + w.h) * a.N : nullptr, w.q0, w.nb, a.N, a.H * DH, w.wave, w.nw, w.lane);
}

// ---- fp32 on v_mfma_f32_32x32x2_f32 (exact fp32 products). The k-steps of Q K^T pair value kk of a row's first half with kk of its
// second, so a lane's part of a row is contiguous; values come straight from memory to the lanes that hold them in the product: row i of
// value block d is value DB i + d, so a lane's DB values stand together.
template <int DH>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(DH <= 64 ? 3 : 2))) void attention_rel_split_f32_kernel(const RelSplitArgs a) {
    using S = Split<float, DH>;
    using I = typename S::I;
    constexpr int DB = (DH + 31) / 32, CH = DH / 8;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const S w(a, smem);
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    RelLevel level;
    float l_run = 0.f;
    for (int t = w.wave; t < w.nt; t += w.nw) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this tile's keys
        // values: key (e & 3) + 8 (e >> 2) + 4 hi of the tile, what register e of s holds
        float vf[16][DB];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            int key = t * 32 + (e & 3) + 8 * (e >> 2) + 4 * w.hi;
            key = key < w.nb ? key : w.nb - 1;
            // (lanes behind the head's width hold values of the next head or, behind the last row, zeros: rows of O that nothing reads)
            const int at = key * w.pitch + w.r * DB * 4;
            if constexpr (DB == 1) vf[e][0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(w.vr, at, 0, 0));
            else if constexpr (DH % DB != 0) {  // (a lane's values straddle the head's end)
#pragma unroll
                for (int d = 0; d < DB; ++d) vf[e][d] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(w.vr, at + 4 * d, 0, 0));
            } else {
                typedef float fvec __attribute__((ext_vector_type(DB)));
                fvec v;
                if constexpr (DB == 2) v = __builtin_bit_cast(fvec, __builtin_amdgcn_raw_buffer_load_b64(w.vr, at, 0, 0));
                else if constexpr (DB == 3) v = __builtin_bit_cast(fvec, __builtin_amdgcn_raw_buffer_load_b96(w.vr, at, 0, 0));
                else v = __builtin_bit_cast(fvec, __builtin_amdgcn_raw_buffer_load_b128(w.vr, at, 0, 0));
#pragma unroll
                for (int d = 0; d < DB; ++d) vf[e][d] = v[d];
            }
        }
        f32x16 s;
        rel_tile(s, w.codes + t * 32, w.rl, w.hi, a.geo.prefix, t * 32);
        int opaque = 0;
        asm volatile("" : "+s"(opaque));  // (the queries stay in LDS: their registers would cost a wave a SIMD)
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const f32x4 kf = *(const f32x4*)(w.region + I::at(w.r, w.hi * CH + i));
            const f32x4 qf = *(const f32x4*)(w.qimg + opaque + I::at(w.r, w.hi * CH + i));
#pragma unroll
            for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[j], s, 0, 0, 0);
        }
        asm volatile("" : "+v"(s));
        if (t + w.nw < w.nt) w.tile(w.kr, w.region, t + w.nw);  // (this tile's reads are over)
        soft_step<DB>(s, o, level, l_run, t * 32, w.nb, w.hi, a.scale_log2e);
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[e][d], s[e], o[d], 0, 0, 0);
    }
    join<float, DH, true>(o, level, l_run, a.scale_log2e, w.regions, S::REGION / 4, w.ml, (float*)a.out + ((size_t)w.b * a.N * a.H + w.h) * DH, nullptr, w.q0,
                          w.nb, a.N, a.H * DH, w.wave, w.nw, w.lane);
}

// LDS of a workgroup of nw waves, and how many waves fit (one always does)
size_t split_lds(int dh, int size, int nw, int N, int slice) {
    return split_image(dh, size) + (size_t)nw * (split_region(dh, size) + 512) + ((size_t)(N + 31) / 32 * 32 + slice) * 4;
}
int split_waves(int dh, int size, int N, int slice, int most) {
    const int nt = ceil_div(N, 32);
    int nw = nt < most ? nt : most;
    while (nw > 1 && split_lds(dh, size, nw, N, slice) > 160 * 1024) --nw;
    return nw;
}

template <int DH>
int launch_split(const RelSplitArgs& a, const vit_rel_pos* pos, int batch, int dtype, int most, hipStream_t stream) {
    const int slice = rel_slice_max(pos->grid_h, pos->grid_w, 32);
    const int size = dtype == VIT_F32 ? 4 : 2, nw = split_waves(DH, size, a.N, slice, most);
    const size_t lds = split_lds(DH, size, nw, a.N, slice);
    const void* kern = dtype == VIT_BF16 ? (const void*)attention_rel_split_bf16_kernel<DH> : (const void*)attention_rel_split_f32_kernel<DH>;
    static PerDeviceInt attr_set[2];
    std::atomic<int>* as = attr_set[dtype].slot();
    if (!as || !as->load(std::memory_order_relaxed)) {
        VIT_CHECK_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        if (as) as->store(1, std::memory_order_relaxed);
    }
    const dim3 grid(batch * a.H, ceil_div(a.N, 32));
    if (dtype == VIT_BF16) hipLaunchKernelGGL(attention_rel_split_bf16_kernel<DH>, grid, dim3(nw * 64), lds, stream, a);
    else hipLaunchKernelGGL(attention_rel_split_f32_kernel<DH>, grid, dim3(nw * 64), lds, stream, a);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

}  // namespace

bool attention_rel_split_eligible(const vit_rel_pos* pos, int batch, int heads, int dtype, int ncu) {
    if (dtype == VIT_F32) return true;
    const int N = pos->prefix + pos->grid_h * pos->grid_w;
    return N > 32 && (int64_t)batch * heads * ceil_div(N, 32) <= (int64_t)4 * ncu;
}

int launch_attention_rel_split(const vit_rel_pos* pos, const RelGeo& geo, const void* qkv, const int* lengths, void* out, float* lse, int batch, int heads,
                               int kv_heads, int head_dim, float scale, int dtype, int ncu, hipStream_t stream) {
    RelSplitArgs a{};
    a.qkv = qkv;
    a.out = out;
    a.lse = lse;
    a.lengths = lengths;
    a.geo = geo;
    a.N = pos->prefix + pos->grid_h * pos->grid_w;
    a.H = heads;
    a.HK = kv_heads;
    a.scale_log2e = scale * LOG2E;
    const int most = (int64_t)batch * heads * ceil_div(a.N, 32) > ncu ? 4 : 8;
#define SPLIT_CASE(DHV) \
    case DHV: return launch_split<DHV>(a, pos, batch, dtype, most, stream);
    switch (head_dim) {
        SPLIT_CASE(16) SPLIT_CASE(32) SPLIT_CASE(48) SPLIT_CASE(64) SPLIT_CASE(80) SPLIT_CASE(96) SPLIT_CASE(112) SPLIT_CASE(128)
    }
#undef SPLIT_CASE
    return vit_set_error(VIT_E_INVALID, "attention_rel: unsupported head_dim %d", head_dim);
}
