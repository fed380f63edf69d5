// Rows of one head (DH bf16 values each) as an LDS image filled by LDS-DMA: 16-byte chunks, a wave instruction writes 64 of them
// lane-linear. Conflict-free for ds_read_b128 of one chunk column over 16 consecutive rows:
//  * 8 or 16 chunks a row (head_dim 64, 128): unpadded, chunk c of row r sits at position c ^ swizzle(r). For 8 chunks the swizzle is
//    the bit reversal of (r >> 1) & 7, with which ds_read_b64_tr_b16 of 8 consecutive rows x 64 bytes is conflict-free too (rows r and
//    r + 2 differ in the position's highest bit), so one image serves row reads and transposed reads.
//  * other widths: one chunk of padding a row (an odd number of chunks); the lanes on the padding re-read the row's last chunk.
#pragma once
#include "vit_common.h"

template <int DH>
struct LdsImage {
    static constexpr int CH = DH / 8;                       // 16-byte chunks of a row
    static constexpr bool SWZ = CH == 8 || CH == 16;
    static constexpr int PCH = SWZ ? CH : CH + 1;           // chunks a row takes in LDS
    static constexpr int ROW = PCH * 16;                    // bytes
    static constexpr int RPI = 64 / PCH;                    // rows a wave instruction fills
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (CH == 8) return ((row & 2) << 1) | ((row & 4) >> 1) | ((row & 8) >> 3);
        else if constexpr (CH == 16) return row & 15;
        else return 0;
    }
    // byte offset of chunk c of a row
    static __device__ __forceinline__ int at(int row, int c) { return row * ROW + ((c ^ swizzle(row)) << 4); }
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
// buffer resource over `rows` rows of one head, `pitch` bytes apart
template <int DH>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_resource(const void* base, int rows, int pitch) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (unsigned)(rows - 1) * (unsigned)pitch + (unsigned)(DH * 2), 0x00020000);
}
