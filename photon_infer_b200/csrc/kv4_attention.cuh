// What kv4_attention.cu and kv4_attention_rows.cu share: their arguments, a score, and the join of the shares of the keys.
#pragma once
#include "kv4.cuh"
#include <math.h>

struct Kv4Args {
  const void* q; void* out; const uint8_t* k; const uint8_t* v;
  const int* table; const int* cu_tokens; const int* context_lens; const float* sinks; float* lse; float* scratch; int* err;
  long q_stride, out_stride;
  int max_pages, n_q, n_kv, groups, page_size, num_pages, window, parts;
  float scale, softcap;
  int max_rows;                 // requests with more are left to another kernel
};

__device__ __forceinline__ float kv4_bounded(float x, float scale, float softcap) {      // a score in powers of two
  constexpr float LOG2E = 1.4426950408889634f;
  return softcap > 0.f ? softcap * tanhf(x * scale / softcap) * LOG2E : x * (scale * LOG2E);
}

// One (token, head): the shares' results in ascending order.
template <typename T>
static __global__ void __launch_bounds__(256)
kv4_join_kernel(const Kv4Args a, int S) {
  pdl_wait();
  const int seq = blockIdx.y, d = a.groups * 32, G = a.n_q / a.n_kv, head = blockIdx.x % a.n_q, i = blockIdx.x / a.n_q;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first;
  if (i >= n || n * G > a.max_rows) return;
  const long token = first + i, of = token * a.n_q + head;
  const float* part = a.scratch + of * a.parts * (d + 2);
  float m = a.sinks != nullptr ? a.sinks[head] * 1.4426950408889634f : -INFINITY;
  const float sink = m;
  for (int p = 0; p < a.parts; ++p) m = fmaxf(m, part[p * (d + 2) + d]);
  const float ref = m == -INFINITY ? 0.f : m;
  float total = a.sinks != nullptr ? exp2f(sink - ref) : 0.f, sum = 0.f;
  const int at = threadIdx.x;
  for (int p = 0; p < a.parts; ++p) {
    const float pm = part[p * (d + 2) + d], pl = part[p * (d + 2) + d + 1];
    if (pl == 0.f) continue;                          // a share of which the row sees nothing
    const float f = pm == -INFINITY ? 1.f : exp2f(pm - ref);      // no maximum and yet a sum: it is no number
    total += pl * f;
    if (at < d) sum += part[p * (d + 2) + at] * f;
  }
  if (at == 0 && a.lse != nullptr) a.lse[of] = total == 0.f ? -INFINITY : (m + log2f(total)) * 0.6931471805599453f;
  if (at < d) ((T*)a.out)[token * a.out_stride + head * d + at] = from_f32<T>(total == 0.f ? 0.f : sum / total);
}
