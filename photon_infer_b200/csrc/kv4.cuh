// A paged cache whose keys and values have 4 bits a number.
//
// A head's d numbers (a multiple of 32) lie in G = d / 32 groups.  A group has one scale, an unsigned number with 5 bits of exponent and 3 of
// mantissa: the byte that follows the sign in a 16-bit float, so byte << 7 is that float's bits.  scale = the nearest such number to max|x| / 7, at most 61,440; code =
// x / scale to the nearest whole number (halves to the even one) in -7 .. 7, plus 8.  scale and code have 4 bits each, so what is read back is exact in bfloat16.  A
// group with a number that is not finite has the scale 255, a NaN, and so has what is read back.
//
// A page of a head is page_size rows of d / 2 bytes, then page_size rows of G scales: one piece of page_size * 17 * G bytes, a multiple of 16.  Rows are ordered
// for the reader's registers.  Keys in words of 8 numbers: word t * G + j holds numbers 32 j + 8 t .. (t < 4), so that the 4 lanes that share a key in a matrix
// instruction's first operand read one run each and get 8 numbers of every group.  Values in half words of 4: half word g * G + j holds numbers 32 j + 4 g .. (g < 8), so that the
// 8 lanes that share the rows of a product's result read one run each and get 4 numbers of every group.
#pragma once
#include "common.cuh"
#include "limits.cuh"
#include <cuda_fp16.h>
#include <math.h>

__host__ __device__ __forceinline__ long kv4_page_bytes(int page_size, int d) { return (long)page_size * (d / 32) * 17; }
static inline bool kv4_sizes_ok(int page_size, int d) { return d > 0 && d % 32 == 0 && d <= 256 && page_size > 0 && (long)page_size * d % 512 == 0; }

__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __half2float(__ushort_as_half((unsigned short)(byte << 7))); }
// Nibble i of a word, less 8: 2^23 + code is exact, and so is what is left.
__device__ __forceinline__ float kv4_code(uint32_t word, int i) { return __uint_as_float(((word >> (4 * i)) & 15u) | 0x4B000000u) - 8388616.f; }

// A query's number.  One that is not finite makes every score of its row NaN: infinity and keys of one sign give scores of minus infinity, as if the row saw nothing.
// x + 0 x is x or NaN.
template <typename T>
__device__ __forceinline__ float kv4_query(T x) {
  const float y = to_f32(x);
  return __fmaf_rn(y, 0.f, y);
}
__device__ __forceinline__ uint32_t kv4_query2(uint32_t x) {      // two bfloat16 numbers likewise
  const __nv_bfloat162 v = *(const __nv_bfloat162*)&x, y = __hfma2(v, __float2bfloat162_rn(0.f), v);
  return *(const uint32_t*)&y;
}
