// Rows of keys and values held in 4 bits: the format that cache_q4.cu writes, lays out and moves and attention_q4.cu reads.
//
// A layer's pool is bytes [n_pages][2 (K, V)][nkv][P * (hd / 2 + 4)]: of a page, plane and head P rows of hd / 2 bytes of codes, then
// P pairs (scale, mid) of bfloat16.  A row x is held as
//
//   scale = bf16((max / 2 - min / 2) / 7.5)   mid = bf16(min / 2 + max / 2)   code = clamp(floor((x - mid) / scale) + 8, 0, 15)
//
// and stands for mid + scale * (code - 7.5): sixteen cells of one width around the middle of the row's range, each read as its centre,
// so an element is off by at most half a cell and what the two factors' rounding to bfloat16 adds (at most 2^-8 of 7.5 cells and of mid).
// A row of equal values has scale 0 and is read as mid; a row that holds a value that is not finite has a scale that is not a number, and so
// has everything read from it.
// One pair of factors per token and key/value head: a row is written once, by the step that has it, and never again (factors that several
// tokens share would have to be revised when the next token comes).  bfloat16 has float32's range, so no row is too small, nor too large up to 3.38e38
// (a factor of a row of larger values may round to infinity, or the row be read beyond float32's range).
// The factors of a page lie together behind its codes: rows of hd / 2 bytes keep the alignment of 16-byte loads and bulk copies (hd / 2 + 4
// would not), and of a whole page codes and factors are one run.
// Of the eight values of a little-endian 32-bit word value 2 i lies in nibble i and value 2 i + 1 in nibble i + 4: one shift and one mask
// give two consecutive values in the two halves of a register.
#pragma once

#include "common.cuh"

#define Q4_FACTOR_BYTES 4   // of a row

__host__ __device__ __forceinline__ int q4_row_bytes(int hd) { return hd / 2 + Q4_FACTOR_BYTES; }
__host__ __device__ __forceinline__ bool q4_head_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }

// Start of the bytes of (page, plane, head): codes, and P * hd / 2 further on the factors.
__device__ __forceinline__ size_t q4_place(int page, int plane, int head, int nkv, int P, int hd) {
    return ((static_cast<size_t>(page) * 2 + plane) * nkv + head) * static_cast<size_t>(P) * q4_row_bytes(hd);
}

__device__ __forceinline__ uint32_t q4_factors(float scale, float mid) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(scale, mid);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float q4_scale(uint32_t f) { return __uint_as_float(f << 16); }
__device__ __forceinline__ float q4_mid(uint32_t f) { return __uint_as_float(f & 0xffff0000u); }

// place of value d (0 .. 7) in its word
__host__ __device__ __forceinline__ constexpr int q4_shift(int d) { return 16 * (d & 1) + 4 * (d >> 1); }

// eight values of a row in the model's type
__device__ __forceinline__ void load8(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16* p, float* v) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
