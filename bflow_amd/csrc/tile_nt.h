// The product of two row-contiguous operands, C[i][j] = sum_k A[i][k] B[j][k], as a tile of one workgroup (gfx950: wave64, LDS-DMA, MFMA).
// Shared by the 8-bit product (int8_gemm.hip) and by the Newton-Schulz products on fp16 pairs (newton_schulz.hip).
//
// Both see an operand as rows of 128-byte CHUNKS, the unit of the k loop:
//   8-bit integers   128 consecutive k of a row
//   fp16 pairs       32 consecutive k of a row: 32 hi halves, then 32 lo halves (value = hi + lo * 2^-11, common.h)
// so one loader and one LDS image serve both.  A stage holds one chunk of BM rows of A and BN rows of B; it is filled by LDS-DMA, 16 bytes a
// lane: a wave instruction moves 8 rows of 128 bytes.  The DMA writes LDS linearly, so the bank swizzle is applied to the SOURCE address:
// the 16-byte segment s of row r lands at segment s ^ ((r >> 1) & 7).  LDS has 64 banks, two rows; 16 rows of a fragment read (ds_read_b128) then
// take each bank once.  (With r & 7, rows r and r + 8 met: half of all LDS cycles were conflicts.)
// Two stages alternate; the next chunk is in flight while the current one is multiplied, one barrier per chunk.
#pragma once
#include "common.h"

namespace bflow {
namespace nt {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lptr_t;
typedef __amdgpu_buffer_rsrc_t rsrc_t;

constexpr int CHUNK = 128;   // bytes

// Rows [0, rows) of `base`, `ld` bytes apart, `row_bytes` of each readable (a multiple of 16).  Reads behind the last row give zeros.
__device__ __forceinline__ rsrc_t rows_rsrc(const void* base, int rows, long long ld, long long row_bytes) {
    const long long n = rows > 0 ? (rows - 1) * ld + row_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(n > 0x7fffffffLL ? 0x7fffffffLL : n), 0x00020000);
}

// A wave's 8-row piece of a stage: lane_offset() + the piece's first row * ld in `voff`, the bytes along the row in `soff`.  The bounds check takes
// soff off the descriptor's size before it compares voff, so what may lie outside (rows behind the last one, OUTSIDE for a whole piece) goes into
// voff, and soff stays below the length of a row.
constexpr int OUTSIDE = (int)0x80000000u;
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }
// `piece`: the piece's number in the LDS image (its parity counts: eight rows are half a period of the swizzle)
__device__ __forceinline__ int lane_segment(int lane, int piece) { return (lane & 7) ^ swizzle((piece & 1) * 8 + (lane >> 3)); }
__device__ __forceinline__ int lane_offset(int lane, int ld, int piece) { return (lane >> 3) * ld + (lane_segment(lane, piece) << 4); }
__device__ __forceinline__ void dma_piece(rsrc_t r, char* lds_piece, int voff, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr_t)lds_piece, 16, voff, soff, 0, 0);
}

// 16 bytes of the fragment of row block `rows` (32 rows, LDS image): lane l reads row l % 32, segment 2 * sub + l / 32.
__device__ __forceinline__ i32x4 frag(const char* rows, int lane, int sub) {
    const int seg = (2 * sub + (lane >> 5)) ^ swizzle(lane & 31);
    return *reinterpret_cast<const i32x4*>(rows + (lane & 31) * CHUNK + seg * 16);
}

// Before the barrier that ends a chunk: this wave's part of the next chunk has landed (vmcnt), and its reads of the current one have returned
// (lgkmcnt): behind the barrier another wave's DMA may overwrite them.
__device__ __forceinline__ void wait_chunk() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

}  // namespace nt
}  // namespace bflow
