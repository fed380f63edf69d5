// Rows of one head (DH bf16 values each) as an LDS image filled by LDS-DMA: 16-byte chunks, a wave instruction writes 64 of them
// lane-linear. Conflict-free for ds_read_b128 of one chunk column over 16 consecutive rows:
//  * 8, 16 or 32 chunks a row (bf16 head_dim 64, 128; fp32 rows of twice the width): unpadded, chunk c of row r sits at position c ^ swizzle(r). For 8 chunks the swizzle is
//    the bit reversal of (r >> 1) & 7, with which ds_read_b64_tr_b16 of 8 consecutive rows x 64 bytes is conflict-free too (rows r and
//    r + 2 differ in the position's highest bit), so one image serves row reads and transposed reads.
//  * other widths: one chunk of padding a row (an odd number of chunks); the lanes on the padding re-read the row's last chunk.
#pragma once
#include "vit_common.h"

template <int DH>
struct LdsImage {
    static constexpr int CH = DH / 8;                       // 16-byte chunks of a row
    static constexpr bool SWZ = CH == 8 || CH == 16 || CH == 32;
    static constexpr int PCH = SWZ ? CH : CH + 1;           // chunks a row takes in LDS
    static constexpr int ROW = PCH * 16;                    // bytes
    static constexpr int RPI = 64 / PCH;                    // rows a wave instruction fills
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (CH == 8) return ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3);
        else if constexpr (SWZ) return row & 15;
        else return 0;
    }
    // byte offset of chunk c of a row
    static __device__ __forceinline__ int at(int row, int c) { return row * ROW + ((c ^ swizzle(row)) << 4); }
    // the same row's chunk 2 k further on, from the address of an even or odd chunk 0 / 1 (an image starts at a multiple of 256 bytes)
    static __device__ __forceinline__ int step(int addr, int k) { return SWZ ? addr ^ (k * 32) : addr + k * 32; }
    // One wave instruction: rows [r0, r0 + RPI) of the image at `dst`, from rows src_row0 + .. of the resource (row pitch `pitch`
    // bytes); rows past src_last re-read it; rows >= rows of the image are not written (nothing behind the image is).
    static __device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int r0, int rows, int src_row0, int src_last,
                                               int pitch, int lane) {
        const int rr = lane / PCH, pos = lane - rr * PCH, row = r0 + rr;
        int c = SWZ ? pos ^ swizzle(row) : pos < CH ? pos : CH - 1;
        int src = src_row0 + row;
        src = src < src_last ? src : src_last;
        if (lane < RPI * PCH && row < rows)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, LDS_PTR(dst + r0 * ROW), 16, src * pitch + c * 16, 0, 0, 0);
    }
};
// The same for whole chunks in a loop: what a lane adds to a piece's address is made once; a chunk that ends before the sample does
// needs no more per instruction than a scalar offset.
template <int DH>
struct LdsFill {
    using I = LdsImage<DH>;
    int rr, c16;  // the lane's row of a piece, its chunk's byte in the row
    __device__ __forceinline__ LdsFill(int lane) {
        const int pos = lane - lane / I::PCH * I::PCH;
        rr = lane / I::PCH;
        c16 = (I::SWZ ? pos ^ I::swizzle(rr) : pos < I::CH ? pos : I::CH - 1) << 4;
    }
    // pieces first, first + step .. of an image of `rows` rows
    __device__ __forceinline__ void chunk(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int rows, int first, int step, int src_row0, int src_last,
                                          int pitch) const {
        if (src_row0 + rows - 1 <= src_last) {
            const int lane_off = rr * pitch + (I::SWZ ? 0 : c16);
            for (int i = first * I::RPI; i < rows; i += step * I::RPI) {
                const int off = I::SWZ ? lane_off + (c16 ^ (I::swizzle(i) << 4)) : lane_off;  // (a piece's row and a lane's have no bit in common)
                if (rr < (rows - i < I::RPI ? rows - i : I::RPI))
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, LDS_PTR(dst + i * I::ROW), 16, off, (src_row0 + i) * pitch, 0, 0);
            }
        } else {
            for (int i = first * I::RPI; i < rows; i += step * I::RPI) {
                const int off = I::SWZ ? c16 ^ (I::swizzle(i) << 4) : c16;
                int src = src_row0 + i + rr;
                src = src < src_last ? src : src_last;
                if (rr < (rows - i < I::RPI ? rows - i : I::RPI))
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, LDS_PTR(dst + i * I::ROW), 16, src * pitch + off, 0, 0, 0);
            }
        }
    }
};
// 16 bytes at an LDS address
__device__ __forceinline__ bf16x8 lds_chunk(int addr) { return *(__attribute__((address_space(3))) const bf16x8*)(uintptr_t)addr; }
// buffer resource over `rows` rows of one head, `pitch` bytes apart
template <int DH>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_resource(const void* base, int rows, int pitch) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (unsigned)(rows - 1) * (unsigned)pitch + (unsigned)(DH * 2), 0x00020000);
}

// 16 rows x 2 steps of an image read transposed (ds_read_b64_tr_b16): A fragments [step][32-value block] of rows row0 .. row0 + 31, for
// products that sum over rows. The wait is in the same statement: the compiler holds its outputs as written when it ends. (Through the
// builtin every such read would also wait for all LDS-DMA under way.)
template <int DH>
struct TrRead {
    using I = LdsImage<DH>;
    static constexpr int DB = (DH + 31) / 32;
    unsigned base;  // lane address of rows 0..7 of the first value block, from the image (16 rows on have the same swizzle)
    __device__ __forceinline__ TrRead(int lane) {
        const int g = lane >> 4, i16 = lane & 15;
        base = (unsigned)(I::at(4 * (g >> 1) + (i16 >> 2), (g & 1) * 2 + ((i16 & 3) >> 1)) + (i16 & 1) * 8);
    }
    // the other addresses are made where they are used, not kept in registers: value block d, rows 8..15 (half)
    __device__ __forceinline__ void addresses(unsigned (&at)[DB][2], unsigned img) const {
        unsigned a0 = base + img;
        asm volatile("" : "+v"(a0));
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if constexpr (I::SWZ) at[d][half] = (a0 ^ (unsigned)((d * 64) ^ (half * (I::CH == 8 ? 16 : 128)))) + half * 8 * I::ROW;
                else at[d][half] = a0 + (unsigned)((d * 4 < I::CH ? d * 64 : 0) + half * 8 * I::ROW);
            }
    }
    // (values behind the head's, where DH is no multiple of 32, are others of the image: those accumulator rows are not stored)
    __device__ __forceinline__ void read(bf16x8 (&f)[2][DB], unsigned img) const {
        unsigned at[DB][2];
        addresses(at, img);
        short4v v[4 * DB];
        if constexpr (DB == 1)
            asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5\n\t"
                         "ds_read_b64_tr_b16 %2, %4 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                         : "v"(at[0][0]), "v"(at[0][1]), "n"(16 * I::ROW)
                         : "memory");
        else if constexpr (DB == 2)
            asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\t"
                         "ds_read_b64_tr_b16 %2, %8 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %11\n\t"
                         "ds_read_b64_tr_b16 %6, %10 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                         : "v"(at[0][0]), "v"(at[0][1]), "v"(at[1][0]), "v"(at[1][1]), "n"(16 * I::ROW)
                         : "memory");
        else if constexpr (DB == 3)
            asm volatile("ds_read_b64_tr_b16 %0, %12\n\tds_read_b64_tr_b16 %1, %13\n\t"
                         "ds_read_b64_tr_b16 %2, %12 offset:%18\n\tds_read_b64_tr_b16 %3, %13 offset:%18\n\t"
                         "ds_read_b64_tr_b16 %4, %14\n\tds_read_b64_tr_b16 %5, %15\n\t"
                         "ds_read_b64_tr_b16 %6, %14 offset:%18\n\tds_read_b64_tr_b16 %7, %15 offset:%18\n\t"
                         "ds_read_b64_tr_b16 %8, %16\n\tds_read_b64_tr_b16 %9, %17\n\t"
                         "ds_read_b64_tr_b16 %10, %16 offset:%18\n\tds_read_b64_tr_b16 %11, %17 offset:%18\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]), "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11])
                         : "v"(at[0][0]), "v"(at[0][1]), "v"(at[1][0]), "v"(at[1][1]), "v"(at[2][0]), "v"(at[2][1]), "n"(16 * I::ROW)
                         : "memory");
        else if constexpr (DB == 4)
            asm volatile("ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %17\n\t"
                         "ds_read_b64_tr_b16 %2, %16 offset:%24\n\tds_read_b64_tr_b16 %3, %17 offset:%24\n\t"
                         "ds_read_b64_tr_b16 %4, %18\n\tds_read_b64_tr_b16 %5, %19\n\t"
                         "ds_read_b64_tr_b16 %6, %18 offset:%24\n\tds_read_b64_tr_b16 %7, %19 offset:%24\n\t"
                         "ds_read_b64_tr_b16 %8, %20\n\tds_read_b64_tr_b16 %9, %21\n\t"
                         "ds_read_b64_tr_b16 %10, %20 offset:%24\n\tds_read_b64_tr_b16 %11, %21 offset:%24\n\t"
                         "ds_read_b64_tr_b16 %12, %22\n\tds_read_b64_tr_b16 %13, %23\n\t"
                         "ds_read_b64_tr_b16 %14, %22 offset:%24\n\tds_read_b64_tr_b16 %15, %23 offset:%24\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]), "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]), "=&v"(v[14]), "=&v"(v[15])
                         : "v"(at[0][0]), "v"(at[0][1]), "v"(at[1][0]), "v"(at[1][1]), "v"(at[2][0]), "v"(at[2][1]), "v"(at[3][0]), "v"(at[3][1]), "n"(16 * I::ROW)
                         : "memory");
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                f[k][d] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v[4 * d + 2 * k], v[4 * d + 2 * k + 1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // one step of it: half the registers at a time
    template <int STEP>
    __device__ __forceinline__ void read_step(bf16x8 (&f)[DB], unsigned img) const {
        unsigned at[DB][2];
        addresses(at, img);
        short4v v[2 * DB];
        if constexpr (DB == 1)
            asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%4\n\tds_read_b64_tr_b16 %1, %3 offset:%4\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1])
                         : "v"(at[0][0]), "v"(at[0][1]), "n"(STEP * 16 * I::ROW)
                         : "memory");
        else if constexpr (DB == 2)
            asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%8\n\t"
                         "ds_read_b64_tr_b16 %2, %6 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                         : "v"(at[0][0]), "v"(at[0][1]), "v"(at[1][0]), "v"(at[1][1]), "n"(STEP * 16 * I::ROW)
                         : "memory");
        else if constexpr (DB == 3)
            asm volatile("ds_read_b64_tr_b16 %0, %6 offset:%12\n\tds_read_b64_tr_b16 %1, %7 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %2, %8 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5])
                         : "v"(at[0][0]), "v"(at[0][1]), "v"(at[1][0]), "v"(at[1][1]), "v"(at[2][0]), "v"(at[2][1]), "n"(STEP * 16 * I::ROW)
                         : "memory");
        else if constexpr (DB == 4)
            asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
                         "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
                         "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
                         "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                         : "v"(at[0][0]), "v"(at[0][1]), "v"(at[1][0]), "v"(at[1][1]), "v"(at[2][0]), "v"(at[2][1]), "v"(at[3][0]), "v"(at[3][1]), "n"(STEP * 16 * I::ROW)
                         : "memory");
#pragma unroll
        for (int d = 0; d < DB; ++d) f[d] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v[2 * d], v[2 * d + 1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
};
