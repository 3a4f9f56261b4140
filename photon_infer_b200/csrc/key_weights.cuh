// What the kernels of key_weights*.cu share: their arguments, numbers of keys, scores, and the join of the runs' maxima and sums.
#pragma once
#include "kv4.cuh"
#include <math.h>

#define KX_KEYS 128              // of a tile

struct KeyWeightsMmaArgs {
  const bf16* q; float* weights; const void* k; const int* table; const int* cu_tokens; const int* context_lens; const int* held; const float* sinks; const float* lse;
  float* scratch; int* err;
  long q_stride;
  float* scores;                 // [T * n_q][width] in powers of two, or null
  long width;
  int max_pages, S, n_q, n_kv, page_size, num_pages, window;
  int parts, each;               // runs of a request, and tiles of 128 keys in a run
  int room;                      // for query rows: a multiple of 16
  float scale, softcap;
};

__device__ __forceinline__ float kx_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kx_scaled(uint32_t word, int shift, __nv_bfloat162 scale) {      // codes at `shift` and 16 bits behind it, as numbers
  const uint32_t x = (word >> shift & 0x000F000Fu) | 0x43004300u;                                     // 128 + c
  const __nv_bfloat162 y = __hmul2(__hsub2(*(const __nv_bfloat162*)&x, __float2bfloat162_rn(136.f)), scale);
  return *(const uint32_t*)&y;
}

__device__ __forceinline__ float key_score(float x, float scale, float softcap) {      // in powers of two
  constexpr float LOG2E = 1.4426950408889634f;
  return softcap > 0.f ? softcap * tanhf(x * scale / softcap) * LOG2E : x * (scale * LOG2E);
}

__device__ __forceinline__ uint4 kx_queries(uint4 x) { return make_uint4(kv4_query2(x.x), kv4_query2(x.y), kv4_query2(x.z), kv4_query2(x.w)); }

// Numbers 8 x .. 8 x + 7 of a key's row in its own order.
template <typename C>
__device__ __forceinline__ void key_numbers(const C* row, int x, float* c) {
  if constexpr (sizeof(C) == 2) {
    const uint4 u = ((const uint4*)row)[x];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[2 * i] = __uint_as_float(w[i] << 16); c[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  } else {
    const float4 a = ((const float4*)row)[2 * x], b = ((const float4*)row)[2 * x + 1];
    c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w; c[4] = b.x; c[5] = b.y; c[6] = b.z; c[7] = b.w;
  }
}

// A warp joins the maxima and sums of one (token, head).
static __global__ void __launch_bounds__(128)
key_weights_lse_kernel(const KeyWeightsMmaArgs a, float* __restrict__ lse) {
  pdl_wait();
  const int seq = blockIdx.y, lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, i = at / a.n_q, h = at - i * a.n_q;
  if (i >= n) return;
  const int parts = a.parts;
  const long of = (long)(first + i) * a.n_q + h;
  const float2* ml = (const float2*)(a.scratch + of * a.parts * 2);
  float m = a.sinks != nullptr && lane == 0 ? a.sinks[h] * 1.4426950408889634f : -INFINITY, l = m == -INFINITY ? 0.f : 1.f;
  for (int p = lane; p < parts; p += 32) {
    const float2 x = ml[p];
    if (x.y == 0.f) continue;
    const float top = fmaxf(m, x.x);
    l = (m == -INFINITY ? l : l * exp2f(m - top)) + (x.x == -INFINITY ? x.y : x.y * exp2f(x.x - top));
    m = top;
  }
  const float top = warp_max(m);
  l = warp_sum(m == -INFINITY ? l : l * exp2f(m - top));
  if (lane == 0) lse[of] = l == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(l)) * 0.6931471805599453f;
}

