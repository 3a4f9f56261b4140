// Which drafted tokens of a tree a request keeps.
//
// Node 0 is the request's last token.  From it on: y = the token that the node's logits give (the first largest one, or with a
// temperature T the first i with e^((x_0 - max) / T) + .. + e^((x_i - max) / T) >= u sum); the first child whose token is y is the next node; where there
// is none the walk ends.  The tokens y are what the request generates, one for every node on the path.
//
// A block a request; only the logits of the nodes on the path are read.
#include "common.cuh"
#include <math.h>

#define TA_THREADS 1024

__device__ __forceinline__ void ta_better(float& v, int& i, float ov, int oi) {
  if (ov > v || (ov == v && oi < i)) { v = ov; i = oi; }
}

// The token that a row of logits gives; every thread gets it.
__device__ int ta_token(const float* row, int V, float temperature, float u) {
  __shared__ float sv[32];
  __shared__ int si[32];
  __shared__ float span_sum[TA_THREADS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float best = -INFINITY;
  int at = 0x7fffffff;
  for (int i = threadIdx.x; i < V; i += TA_THREADS) ta_better(best, at, row[i], i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ta_better(best, at, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  __syncthreads();
  if (lane == 0) { sv[warp] = best; si[warp] = at; }
  __syncthreads();
  best = sv[lane]; at = si[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ta_better(best, at, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, at, o));
  if (at == 0x7fffffff) at = 0;
  if (!(temperature > 0.f)) return at;
  const int span = (V + TA_THREADS - 1) / TA_THREADS, lo = threadIdx.x * span, hi = min(V, lo + span);
  float s = 0.f;
  for (int i = lo; i < hi; ++i) s += expf((row[i] - best) / temperature);
  span_sum[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float total = 0.f;
    for (int i = 0; i < TA_THREADS; ++i) total += span_sum[i];
    const float target = u * total;
    float cum = 0.f;
    int pick = -1;
    for (int c = 0; c < TA_THREADS && pick < 0; ++c) {
      if (cum + span_sum[c] >= target && span_sum[c] > 0.f) {
        for (int i = c * span; i < min(V, (c + 1) * span); ++i) {
          cum += expf((row[i] - best) / temperature);
          if (cum >= target) { pick = i; break; }
        }
      } else {
        cum += span_sum[c];
      }
    }
    si[0] = pick < 0 ? at : pick;
  }
  __syncthreads();
  const int got = si[0];
  __syncthreads();
  return got;
}

__global__ void __launch_bounds__(TA_THREADS)
tree_accept_kernel(const float* __restrict__ logits, long ld, const int* __restrict__ tokens, const int* __restrict__ parents,
                   const int* __restrict__ cu_tokens, int T, int V, const float* __restrict__ temperature, const float* __restrict__ uniforms,
                   int* __restrict__ path, int* __restrict__ counts, int* __restrict__ sampled, int D, int most) {
  __shared__ int next;
  const int seq = blockIdx.x;
  const int t0 = max(0, min(cu_tokens[seq], T)), n = max(0, min(min(cu_tokens[seq + 1], T) - t0, most));
  int node = 0, count = 0;
  while (count < D && node < n) {
    const int y = ta_token(logits + (size_t)(t0 + node) * ld, V, temperature ? temperature[seq] : 0.f, temperature ? uniforms[t0 + node] : 0.f);
    if (threadIdx.x == 0) { path[(size_t)seq * D + count] = node; sampled[(size_t)seq * D + count] = y; next = n; }
    ++count;
    __syncthreads();
    for (int i = node + 1 + threadIdx.x; i < n; i += TA_THREADS)
      if (parents[t0 + i] == node && tokens[t0 + i] == y) atomicMin(&next, i);
    __syncthreads();
    node = next;
    __syncthreads();
  }
  for (int i = count + threadIdx.x; i < D; i += TA_THREADS) { path[(size_t)seq * D + i] = -1; sampled[(size_t)seq * D + i] = -1; }
  if (threadIdx.x == 0) counts[seq] = count;
}

PHOTON_API int photon_tree_accept(const float* logits, long ld, const int* tokens, const int* parents, const int* cu_tokens, int S, int T,
                                  int max_tokens_per_seq, int V, const float* temperature, const float* uniforms, int* path, int* counts,
                                  int* sampled, int D, cudaStream_t stream) {
  if (S <= 0) return 0;
  if (V <= 0 || T < 0 || D <= 0 || max_tokens_per_seq <= 0 || (temperature != nullptr && uniforms == nullptr)) return PHOTON_ERR_ARGUMENT;
  tree_accept_kernel<<<S, TA_THREADS, 0, stream>>>(logits, ld, tokens, parents, cu_tokens, T, V, temperature, uniforms, path, counts, sampled, D,
                                                   max_tokens_per_seq);
  return launch_status();
}
