// Norm of every query / key head and the rotary position rotation in one pass over the packed projection output
// [tokens, (H + 2 Hk) dh] (q heads | k heads | v heads), and its gradient.
//
//   xh = (x - mu) r,  r = 1 / sqrt(mean((x - mu)^2) + eps)      (mu = 0: RMS norm; mu = mean(x): LayerNorm)
//   y  = xh * w (+ b);   out = R y, R the rotation of the token's position on the first rot_dim values of the head
// backward, g_out the gradient of out:
//   t  = R^T g_out;  db = sum t;  dw = sum t * xh;  g = t * w;  dx = r (g - mean(g) [LayerNorm] - xh mean(g * xh))
//
// Bound by HBM: a forward reads and writes the packed rows once (queries, keys; values are copied unless the call is in
// place), a backward also reads the queries and keys. So one wave takes a token at a time and runs over its heads: a lane
// holds 8 values of a head (16 bytes of bf16), dh / 8 lanes (padded to a power of two) a head, and the cosines, sines and
// weights of those 8 values are loaded once per token / once per wave. Row sums are DPP adds inside 2..16 lanes, the
// rotation's partner values come from a lane of the same head.
//
// 256 x 197 tokens, 12 + 12 heads of 64, bf16, RMS: forward 87 us for 464 MB (5.3 TB/s, what a large copy reaches), backward 117 us for
// 620 MB (5.3 TB/s); 9 x 331 tokens, 12 + 4 heads of 96, LayerNorm, positions: 9.2 us, of which 4.4 are its bytes: the loads' chain of one
// token a wave (heads before weights: 15.2 us the other way round); fp32 backward of 3 x 1025 tokens, 16 + 16 heads of 80: 30 us for 126 MB
// that come from HBM, 26 us where an earlier call left them in the caches. The parameters' sums are fp32 (in a fixed order).
#include "vit_common.h"
#include <math.h>

namespace {

constexpr int U = 5;  // heads a lane has in flight

struct QkArgs {
    const void* x;    // packed projection output
    const void* g;    // backward: gradient of the output
    void* out;        // forward: output; backward: gradient of x
    const float* w[2];     // q, k weights [dh]
    const float* b[2];     // q, k biases [dh] or null
    const float2* rope;    // [rope_len, rot_dim / 2] (cos, sin)
    const int* positions;  // [pos_count] or null (= token % seq)
    float* part;           // backward: [blocks][4][dh] partial sums (dwq, dwk, dbq, dbk)
    int tokens, seq, pos_count, heads, kv_heads, dh, rot_dim, rope_len;
    float eps;
};

template <typename T> struct Raw8;
template <> struct Raw8<bf16_t> {
    bf16x8 v;
    __device__ void load(const bf16_t* p) { v = *(const bf16x8*)p; }
    __device__ void zero() {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (bf16_t)0.f;
    }
    __device__ float get(int e) const { return (float)v[e]; }
    static __device__ void store(bf16_t* p, const float (&y)[8]) {
        bf16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (bf16_t)y[e];
        *(bf16x8*)p = o;
    }
};
template <> struct Raw8<float> {
    f32x4 a, c;
    __device__ void load(const float* p) { a = *(const f32x4*)p; c = *(const f32x4*)(p + 4); }
    __device__ void zero() { a = f32x4{0.f, 0.f, 0.f, 0.f}; c = a; }
    __device__ float get(int e) const { return e < 4 ? a[e & 3] : c[e & 3]; }
    static __device__ void store(float* p, const float (&y)[8]) {
        *(f32x4*)p = f32x4{y[0], y[1], y[2], y[3]};
        *(f32x4*)(p + 4) = f32x4{y[4], y[5], y[6], y[7]};
    }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over the GL lanes of a head, the same bits in each of them
template <int GL>
__device__ __forceinline__ float head_sum(float v) {
    v = dpp_add<0xB1>(v);                            // quad_perm 1,0,3,2
    if constexpr (GL >= 4) v = dpp_add<0x4E>(v);     // quad_perm 2,3,0,1
    if constexpr (GL >= 8) v = dpp_add<0x141>(v);    // row_half_mirror
    if constexpr (GL >= 16) v = dpp_add<0x140>(v);   // row_mirror
    return v;
}

// a product that is 0 where a factor is, whatever the other one (for finite factors the ordinary one)
__device__ __forceinline__ float mul_or_zero(float a, float b) {
    float r;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// what a lane needs to turn its 8 values: cosines and sines of their pairs, and the lane that holds their partners.
template <int GL, bool IL>
struct Turn {
    static constexpr int NC = IL ? 4 : 8;  // (neighbours share theirs)
    float c[NC], s[NC];
    int partner;  // half-split pairs: lane of the partner values (itself outside the rotated part)
    int other;    // that lane, itself for a token that is not turned: what is not turned meets no other value, not even times 0 (it may be
                  // NaN). Neighbours: the multiplication whose product with 0 is 0, whatever the other factor
    __device__ void place(int lane, int chunk, int rot_dim) {
        const int hc = rot_dim >> 4;  // chunks in half the rotated part
        partner = lane;
        if (!IL && chunk < 2 * hc) partner = chunk < hc ? lane + hc : lane - hc;
    }
    __device__ void load(const QkArgs& a, int tok, int chunk) {
#pragma unroll
        for (int e = 0; e < NC; ++e) { c[e] = 1.f; s[e] = 0.f; }
        other = (int)(threadIdx.x & 63);
        if (chunk * 8 >= a.rot_dim) return;
        const int i = tok % a.pos_count;
        const int pos = a.positions ? a.positions[i] : i;
        if (pos < 0 || pos >= a.rope_len) return;  // not turned
        other = partner;
        const float2* row = a.rope + (size_t)pos * (a.rot_dim >> 1);
        if constexpr (IL) {
            row += chunk * 4;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float2 v = row[p];
                c[p] = v.x;
                s[p] = v.y;
            }
        } else {
            const int half = a.rot_dim >> 1;
            const bool second = chunk * 8 >= half;
            row += chunk * 8 - (second ? half : 0);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float4 v = *(const float4*)(row + e);
                c[e] = v.x;
                s[e] = second ? v.y : -v.y;
                c[e + 1] = v.z;
                s[e + 1] = second ? v.w : -v.w;
            }
        }
    }
    // sign +1: R y, -1: R^T y (the angle's sign). All lanes call it together.
    template <int SIGN>
    __device__ void apply(float (&y)[8]) const {
        if constexpr (IL) {
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float a = y[2 * p], b = y[2 * p + 1], v = SIGN > 0 ? s[p] : -s[p];
                y[2 * p] = fmaf(a, c[p], -mul_or_zero(v, b));
                y[2 * p + 1] = fmaf(b, c[p], mul_or_zero(v, a));
            }
        } else {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __shfl(y[e], other, 64);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = fmaf(SIGN > 0 ? s[e] : -s[e], o[e], y[e] * c[e]);
        }
    }
};

// a head's 8 weights of a lane's chunk (any 4-byte alignment); lanes past the head take the first chunk's, which meet zeros
__device__ __forceinline__ void load8(float (&w)[8], const float* p, int chunk, bool on) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const f32x4u* v = (const f32x4u*)(p + (on ? chunk * 8 : 0));
    const f32x4u lo = v[0], hi = v[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) { w[e] = lo[e]; w[4 + e] = hi[e]; }
}

// mean, 1 / deviation and the normalised values of a head; lanes past the head hold zeros and stay out of the sums
template <int GL, bool LAYER>
__device__ __forceinline__ float normalise(float (&x)[8], bool on, float inv_dh, float eps) {
    if constexpr (LAYER) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m += x[e];
        m = head_sum<GL>(m) * inv_dh;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = on ? x[e] - m : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) q = fmaf(x[e], x[e], q);
    const float r = 1.0f / sqrtf(fmaf(head_sum<GL>(q), inv_dh, eps));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= r;
    return r;
}

template <typename T, int GL, bool LAYER, bool IL>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const QkArgs a) {
    constexpr int HS = 64 / GL;  // heads side by side in a wave
    const int lane = threadIdx.x & 63, slot = lane / GL, chunk = lane % GL;
    const int wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = gridDim.x * 4;
    const bool on = chunk * 8 < a.dh;
    const int nh = a.heads + a.kv_heads;
    const int all = a.out != a.x ? nh + a.kv_heads : nh;  // out of place the values pass through, as heads behind the keys
    const size_t row = (size_t)(nh + a.kv_heads) * a.dh;
    const float inv_dh = 1.0f / (float)a.dh;
    Raw8<T> raw[U];
    auto load_heads = [&](int tok, int h0) {
        const T* xr = (const T*)a.x + (size_t)tok * row + chunk * 8;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * HS + slot;
            if (on && h < all) raw[u].load(xr + (size_t)h * a.dh); else raw[u].zero();
        }
    };
    if (wave < a.tokens) load_heads(wave, 0);  // (ahead of the weights: a small call is one token a wave)
    float w[2][8], b[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        load8(w[k], a.w[k], chunk, on);
        if constexpr (LAYER) {
            if (a.b[k]) {
                load8(b[k], a.b[k], chunk, on);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) b[k][e] = 0.f;
            }
        }
    }
    Turn<GL, IL> turn;
    turn.place(lane, chunk, a.rot_dim);
    for (int tok = wave; tok < a.tokens; tok += waves) {
        T* yr = (T*)a.out + (size_t)tok * row + chunk * 8;
        turn.load(a, tok, chunk);
        for (int h0 = 0; h0 < all; h0 += HS * U) {
            if (h0 > 0) load_heads(tok, h0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (h0 + u * HS >= all) break;
                int h = h0 + u * HS + slot;
                asm volatile("" : "+v"(h));  // (opaque: the weights chosen for each of the heads would be kept in registers)
                const bool isk = h >= a.heads;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = raw[u].get(e);
                if (h0 + u * HS < nh) {  // (uniform: some head of the group is a query or a key)
                    normalise<GL, LAYER>(y, on, inv_dh, a.eps);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float we = isk ? w[1][e] : w[0][e];
                        if constexpr (LAYER) y[e] = fmaf(y[e], we, isk ? b[1][e] : b[0][e]); else y[e] *= we;
                    }
                    turn.template apply<1>(y);
                }
                if (on && h < nh) Raw8<T>::store(yr + (size_t)h * a.dh, y);
                else if (on && h < all) *(Raw8<T>*)(yr + (size_t)h * a.dh) = raw[u];
            }
        }
        if (tok + waves < a.tokens) load_heads(tok + waves, 0);
    }
}

template <typename T, int GL, bool LAYER, bool IL>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void qk_norm_rope_bwd_kernel(const QkArgs a) {
    constexpr int HS = 64 / GL, UB = 2;
    constexpr int NS = LAYER ? 4 : 2;  // sums kept: dw of q, k (and db of q, k)
    __shared__ float part[4][4][128];
    const int lane = threadIdx.x & 63, slot = lane / GL, chunk = lane % GL;
    const int wib = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = blockIdx.x * 4 + wib, waves = gridDim.x * 4;
    const bool on = chunk * 8 < a.dh;
    const int nh = a.heads + a.kv_heads;
    const size_t row = (size_t)(nh + a.kv_heads) * a.dh;
    const float inv_dh = 1.0f / (float)a.dh;
    Raw8<T> rx[UB], rg[UB];
    auto load_heads = [&](int tok, int h0) {
        const T* xr = (const T*)a.x + (size_t)tok * row + chunk * 8;
        const T* gr = (const T*)a.g + (size_t)tok * row + chunk * 8;
#pragma unroll
        for (int u = 0; u < UB; ++u) {
            const int h = h0 + u * HS + slot;
            if (on && h < nh) {
                rx[u].load(xr + (size_t)h * a.dh);
                rg[u].load(gr + (size_t)h * a.dh);
            } else {
                rx[u].zero();
                rg[u].zero();
            }
        }
    };
    if (wave < a.tokens) load_heads(wave, 0);  // (ahead of the weights: a small call is one token a wave)
    float w[2][8], sum[NS][8];
    load8(w[0], a.w[0], chunk, on);
    load8(w[1], a.w[1], chunk, on);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int k = 0; k < NS; ++k) sum[k][e] = 0.f;
    Turn<GL, IL> turn;
    turn.place(lane, chunk, a.rot_dim);
    for (int tok = wave; tok < a.tokens; tok += waves) {
        T* dr = (T*)a.out + (size_t)tok * row + chunk * 8;
        turn.load(a, tok, chunk);
        for (int h0 = 0; h0 < nh; h0 += HS * UB) {
            if (h0 > 0) load_heads(tok, h0);
#pragma unroll
            for (int u = 0; u < UB; ++u) {
                if (h0 + u * HS >= nh) break;
                int h = h0 + u * HS + slot;
                asm volatile("" : "+v"(h));  // (opaque: the weights chosen for each of the heads would be kept in registers)
                const bool isk = h >= a.heads;
                float x[8], t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) { x[e] = rx[u].get(e); t[e] = rg[u].get(e); }
                const float r = normalise<GL, LAYER>(x, on, inv_dh, a.eps);
                turn.template apply<-1>(t);
                float sg = 0.f, sgx = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float tx = t[e] * x[e];
                    // (chosen, not times 0 or 1: what is not finite stays with its own sums)
                    sum[0][e] += isk ? 0.f : tx;
                    sum[1][e] += isk ? tx : 0.f;
                    if constexpr (LAYER) {
                        sum[2][e] += isk ? 0.f : t[e];
                        sum[3][e] += isk ? t[e] : 0.f;
                    }
                    t[e] *= isk ? w[1][e] : w[0][e];
                    sg += t[e];
                    sgx = fmaf(t[e], x[e], sgx);
                }
                const float mgx = head_sum<GL>(sgx) * inv_dh;
                const float mg = LAYER ? head_sum<GL>(sg) * inv_dh : 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = r * (t[e] - mg - x[e] * mgx);
                if (on && h < nh) Raw8<T>::store(dr + (size_t)h * a.dh, t);
            }
        }
        if (a.out != a.g) {
            const int nv = a.kv_heads * a.dh / 8;
            const size_t v0 = (size_t)tok * row + (size_t)nh * a.dh;
            for (int i = lane; i < nv; i += 64) {
                Raw8<T> v;
                v.load((const T*)a.g + v0 + i * 8);
                *(Raw8<T>*)((T*)a.out + v0 + i * 8) = v;
            }
        }
        if (tok + waves < a.tokens) load_heads(tok + waves, 0);
    }
    // heads side by side, then the block's four waves; fixed order
#pragma unroll
    for (int k = 0; k < NS; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = sum[k][e];
#pragma unroll
            for (int o = GL; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
            if (slot == 0 && on) part[wib][k][chunk * 8 + e] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < NS * a.dh; i += 256) {
        const int k = i / a.dh, d = i - k * a.dh;
        a.part[(size_t)blockIdx.x * NS * a.dh + i] = (part[0][k][d] + part[1][k][d]) + (part[2][k][d] + part[3][k][d]);
    }
}

// column sums of the blocks' partial rows [blocks][ns * dh]: 16 columns a block, 64 row groups with their loads in flight
// together, joined in a fixed order
__global__ __launch_bounds__(1024) void qk_norm_rope_sum_kernel(const float* __restrict__ part, int blocks, int dh, int ns, float* dwq,
                                                                float* dwk, float* dbq, float* dbk) {
    __shared__ float red[64][17];
    const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + c, cols = ns * dh;  // dh is a multiple of 16: every column exists
    float s = 0.f;
    for (int i0 = 0; i0 < blocks; i0 += 64 * 16) {
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int i = i0 + k * 64 + g;
            v[k] = i < blocks ? part[(size_t)i * cols + col] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) s += v[k];
    }
    red[g][c] = s;
    __syncthreads();
    if (g < 8) {
        s = red[g][c];
#pragma unroll
        for (int k = 1; k < 8; ++k) s += red[g + 8 * k][c];
        red[g][c] = s;  // (each of these rows is read by its own thread alone above)
    }
    __syncthreads();
    if (g == 0) {
        float v = red[0][c];
#pragma unroll
        for (int k = 1; k < 8; ++k) v += red[k][c];
        const int which = col / dh, d = col - which * dh;
        float* dst = which == 0 ? dwq : which == 1 ? dwk : which == 2 ? dbq : dbk;
        if (dst) dst[d] = v;
    }
}

constexpr int kBwdBlocksPerCu = 4;

int check_cfg(const char* who, const vit_qk_norm_config* c, const void* rope) {
    VIT_REQUIRE(c, "%s: null config", who);
    VIT_REQUIRE(c->batch > 0 && c->seq > 0 && c->heads > 0 && c->kv_heads > 0, "%s: empty problem", who);
    VIT_REQUIRE(c->heads % c->kv_heads == 0, "%s: heads %d is not a multiple of kv_heads %d", who, c->heads, c->kv_heads);
    VIT_REQUIRE(c->head_dim % 16 == 0 && c->head_dim >= 16 && c->head_dim <= 128,
                "%s: head_dim must be a multiple of 16 in [16,128], got %d", who, c->head_dim);
    VIT_REQUIRE(c->rot_dim % 16 == 0 && c->rot_dim >= 0 && c->rot_dim <= c->head_dim,
                "%s: rot_dim must be a multiple of 16 in [0, head_dim], got %d", who, c->rot_dim);
    VIT_REQUIRE(c->norm == VIT_NORM_RMS || c->norm == VIT_NORM_LAYER, "%s: bad norm %d", who, c->norm);
    VIT_REQUIRE(c->dtype == VIT_BF16 || c->dtype == VIT_F32, "%s: bad dtype %d", who, c->dtype);
    VIT_REQUIRE(c->eps > 0.f && c->eps < INFINITY, "%s: eps must be positive and finite", who);
    VIT_REQUIRE(c->rot_dim == 0 || (rope && c->rope_len > 0), "%s: rot_dim %d without a rope table", who, c->rot_dim);
    // (a wave's next token, up to 32768 further on, is counted in 32 bits too)
    VIT_REQUIRE((int64_t)c->batch * c->seq < (1LL << 31) - (1 << 16), "%s: too many tokens", who);
    return VIT_OK;
}
bool overlaps(const void* a, const void* b, size_t bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + bytes && y < x + bytes;
}
bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

QkArgs make_args(const vit_qk_norm_config* c, const float* qw, const float* kw, const float* rope, const int32_t* positions) {
    QkArgs a{};
    a.w[0] = qw;
    a.w[1] = kw;
    a.rope = (const float2*)rope;
    a.positions = positions;
    a.tokens = c->batch * c->seq;
    a.seq = c->seq;
    a.pos_count = (positions && c->positions_per_sample) ? a.tokens : c->seq;
    a.heads = c->heads;
    a.kv_heads = c->kv_heads;
    a.dh = c->head_dim;
    a.rot_dim = c->rot_dim;
    a.rope_len = c->rope_len;
    a.eps = c->eps;
    return a;
}

template <bool BWD, typename T, int GL, bool LAYER>
void launch_il(const QkArgs& a, bool il, int grid, hipStream_t s) {
    if constexpr (BWD) {
        if (il) hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, GL, LAYER, true>), dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<T, GL, LAYER, false>), dim3(grid), dim3(256), 0, s, a);
    } else {
        if (il) hipLaunchKernelGGL((qk_norm_rope_kernel<T, GL, LAYER, true>), dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((qk_norm_rope_kernel<T, GL, LAYER, false>), dim3(grid), dim3(256), 0, s, a);
    }
}
template <bool BWD, typename T>
void launch_t(const QkArgs& a, bool layer, bool il, int grid, hipStream_t s) {
    // lanes per head: dh / 8, up to a power of two
    if (a.dh <= 16) layer ? launch_il<BWD, T, 2, true>(a, il, grid, s) : launch_il<BWD, T, 2, false>(a, il, grid, s);
    else if (a.dh <= 32) layer ? launch_il<BWD, T, 4, true>(a, il, grid, s) : launch_il<BWD, T, 4, false>(a, il, grid, s);
    else if (a.dh <= 64) layer ? launch_il<BWD, T, 8, true>(a, il, grid, s) : launch_il<BWD, T, 8, false>(a, il, grid, s);
    else layer ? launch_il<BWD, T, 16, true>(a, il, grid, s) : launch_il<BWD, T, 16, false>(a, il, grid, s);
}
template <bool BWD>
void launch_any(const QkArgs& a, const vit_qk_norm_config* c, int grid, hipStream_t s) {
    const bool layer = c->norm == VIT_NORM_LAYER, il = c->interleaved != 0;
    if (c->dtype == VIT_BF16) launch_t<BWD, bf16_t>(a, layer, il, grid, s);
    else launch_t<BWD, float>(a, layer, il, grid, s);
}
int bwd_blocks(const vit_qk_norm_config* c, int* blocks) {
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    const int want = (int)(((int64_t)c->batch * c->seq + 3) / 4);
    *blocks = want < ncu * kBwdBlocksPerCu ? want : ncu * kBwdBlocksPerCu;
    return VIT_OK;
}

}  // namespace

extern "C" int vit_qk_norm_rope_fwd(const vit_qk_norm_config* cfg, const void* qkv, const float* q_weight, const float* k_weight,
                                    const float* q_bias, const float* k_bias, const float* rope, const int32_t* positions,
                                    void* out, void* stream) {
    VIT_TRY_RC(check_cfg("vit_qk_norm_rope_fwd", cfg, rope));
    VIT_REQUIRE(qkv && out && q_weight && k_weight, "vit_qk_norm_rope_fwd: null argument");
    VIT_REQUIRE(cfg->norm == VIT_NORM_LAYER || (!q_bias && !k_bias), "vit_qk_norm_rope_fwd: the RMS norm takes no bias");
    VIT_REQUIRE(!misaligned(qkv) && !misaligned(out) && !misaligned(rope), "vit_qk_norm_rope_fwd: tensors must be 16-byte aligned");
    const size_t bytes = (size_t)cfg->batch * cfg->seq * (cfg->heads + 2 * cfg->kv_heads) * cfg->head_dim * (cfg->dtype == VIT_BF16 ? 2 : 4);
    VIT_REQUIRE(out == qkv || !overlaps(qkv, out, bytes), "vit_qk_norm_rope_fwd: out overlaps qkv without being it");
    QkArgs a = make_args(cfg, q_weight, k_weight, rope, positions);
    a.x = qkv;
    a.out = out;
    a.b[0] = q_bias;
    a.b[1] = k_bias;
    int ncu = 0;
    VIT_TRY_RC(vit_cu_count(&ncu));
    const int64_t want = ((int64_t)a.tokens + 3) / 4;
    const int grid = want < ncu * 8 ? (int)want : ncu * 8;
    launch_any<false>(a, cfg, grid, (hipStream_t)stream);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}

extern "C" size_t vit_qk_norm_rope_bwd_workspace_bytes(const vit_qk_norm_config* cfg) {
    int blocks = 0;
    if (!cfg || cfg->batch <= 0 || cfg->seq <= 0 || cfg->head_dim <= 0 || bwd_blocks(cfg, &blocks) != VIT_OK) return 0;
    return (size_t)blocks * 4 * cfg->head_dim * sizeof(float);
}

extern "C" int vit_qk_norm_rope_bwd(const vit_qk_norm_config* cfg, const void* qkv, const void* d_out, const float* q_weight,
                                    const float* k_weight, const float* rope, const int32_t* positions, void* dqkv,
                                    float* dq_weight, float* dk_weight, float* dq_bias, float* dk_bias, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    VIT_TRY_RC(check_cfg("vit_qk_norm_rope_bwd", cfg, rope));
    VIT_REQUIRE(qkv && d_out && q_weight && k_weight && dqkv && dq_weight && dk_weight && workspace, "vit_qk_norm_rope_bwd: null argument");
    VIT_REQUIRE(cfg->norm == VIT_NORM_LAYER || (!dq_bias && !dk_bias), "vit_qk_norm_rope_bwd: the RMS norm has no bias");
    VIT_REQUIRE(!misaligned(qkv) && !misaligned(d_out) && !misaligned(dqkv) && !misaligned(rope) && !misaligned(workspace),
                "vit_qk_norm_rope_bwd: tensors must be 16-byte aligned");
    const size_t bytes = (size_t)cfg->batch * cfg->seq * (cfg->heads + 2 * cfg->kv_heads) * cfg->head_dim * (cfg->dtype == VIT_BF16 ? 2 : 4);
    VIT_REQUIRE(!overlaps(qkv, dqkv, bytes) && (dqkv == d_out || !overlaps(d_out, dqkv, bytes)),
                "vit_qk_norm_rope_bwd: dqkv overlaps qkv, or d_out without being it");
    int blocks = 0;
    VIT_TRY_RC(bwd_blocks(cfg, &blocks));
    const size_t need = (size_t)blocks * 4 * cfg->head_dim * sizeof(float);
    if (workspace_bytes < need)
        return vit_set_error(VIT_E_NOMEM, "vit_qk_norm_rope_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    QkArgs a = make_args(cfg, q_weight, k_weight, rope, positions);
    a.x = qkv;
    a.g = d_out;
    a.out = dqkv;
    a.part = (float*)workspace;
    launch_any<true>(a, cfg, blocks, (hipStream_t)stream);
    VIT_CHECK_HIP(hipGetLastError());
    const int ns = cfg->norm == VIT_NORM_LAYER ? 4 : 2;
    hipLaunchKernelGGL(qk_norm_rope_sum_kernel, dim3(ns * cfg->head_dim / 16), dim3(1024), 0, (hipStream_t)stream, a.part, blocks,
                       cfg->head_dim, ns, dq_weight, dk_weight, dq_bias, dk_bias);
    VIT_CHECK_HIP(hipGetLastError());
    return VIT_OK;
}
