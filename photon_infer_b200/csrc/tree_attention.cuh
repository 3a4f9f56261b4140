// What the kernels of tree attention share: the sizes of a call, and which keys a node of a drafted tree sees.
//
// A request's nodes are its last tokens: with n nodes and a context of L tokens (the nodes counted), node i is key base + i, base =
// L - n.  Node t sees the cached keys j < base with j > pos(t) - window, and the nodes i whose bit is set in its mask and whose
// place on their path, pos(i), is within the window.  A bit at or behind n says nothing.
#pragma once
#include "common.cuh"

struct TreeParams {
  const void* q; long q_stride;                    // [T, n_q * d] view
  void* out; long out_stride;                      // [T, n_q * d]
  const void* k_cache; const void* v_cache;        // [num_pages, n_kv, page_size, d]
  const int* block_table; int max_pages;           // [S, max_pages]
  const int* cu_tokens;                            // [S + 1] first node of each request
  const int* context_lens;                         // [S] keys of each request, its nodes counted
  const int* positions;                            // [T]
  const int* tree_mask; int mask_words;            // [T, mask_words]: bit i of a row: the node sees node i of its request
  int S, T, max_tokens, n_q, n_kv, group, d, page_size, num_pages, window;
  float scale;
  const float* sinks;                              // [n_q] or null
  float softcap;                                   // 0: off
  int* err;
};

// The request's node range and first key that is a node, kept inside the call's arrays whatever the tables say.
struct TreeRequest { int tok0, n, base; };
__device__ __forceinline__ TreeRequest tree_request(const TreeParams& P, int s) {
  TreeRequest r;
  const int a = P.cu_tokens[s], b = P.cu_tokens[s + 1];
  r.tok0 = max(0, min(a, P.T));
  r.n = max(0, min(min(b, P.T) - r.tok0, P.max_tokens));
  r.base = max(0, P.context_lens[s] - r.n);
  return r;
}

// 32 keys from `key0` on, as bits: those that the node at row `t` of the step may see.  lo: first cached key inside its window.
__device__ __forceinline__ uint32_t tree_visible32(const TreeParams& P, const TreeRequest& r, int t, int key0, int lo) {
  const int i0 = key0 - r.base;                    // place of the first of them among the nodes
  uint32_t bits = 0;
  if (i0 < 0) {                                    // cached keys: lo <= key < base
    const int past = min(32, -i0), skip = max(0, min(lo - key0, past));
    bits = (past >= 32 ? 0xffffffffu : (1u << past) - 1u);
    bits &= skip >= 32 ? 0u : (0xffffffffu << skip);
  }
  if (i0 > -32 && i0 < r.n) {                      // nodes
    const int* row = P.tree_mask + (size_t)t * P.mask_words;
    uint32_t m;
    if (i0 < 0) {
      m = (uint32_t)row[0] << (-i0);
      if (r.n + (-i0) < 32) m &= (1u << (r.n - i0)) - 1u;
    } else {
      const int w = i0 >> 5, sh = i0 & 31;
      const uint32_t a = w < P.mask_words ? (uint32_t)row[w] : 0u, b = w + 1 < P.mask_words ? (uint32_t)row[w + 1] : 0u;
      m = __funnelshift_r(a, b, sh);
      if (r.n - i0 < 32) m &= (1u << (r.n - i0)) - 1u;
    }
    // Nodes stand at base or behind, so a window that begins before base cuts none of them.
    const int pos = P.window > 0 ? P.positions[t] : 0;
    if (P.window > 0 && pos - P.window >= r.base) {
      for (uint32_t left = m; left != 0; left &= left - 1) {
        const int u = __ffs(left) - 1;
        if (P.positions[r.tok0 + i0 + u] <= pos - P.window) m &= ~(1u << u);
      }
    }
    bits |= m;
  }
  return bits;
}

// tanh(y) for |y| <= 1/2 by its series up to y^11: off by less than 21844 / 6081075 y^13 < 5e-7.  Scores far below their bound need no exponential and no division.
__device__ __forceinline__ float tree_tanh_half(float y) {
  const float z = y * y;
  return y * fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1382.f / 155925.f, 62.f / 2835.f), -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
}

// A partial result of a row that sees none of its keys: it has no part in the row, whatever lies in its place.  One whose weights are merely too small beside the
// others' has, so that a value that is not finite shows wherever the keys are cut.  In a list of factors it is marked.
__device__ __forceinline__ bool tree_nothing(float maximum, float sum) { return maximum == -INFINITY && sum == 0.f; }       // the sum of scores that are NaN is one
#define TREE_NOTHING (-1.f)

// The cache row (of d numbers) of a key, or -1 where its page is missing, which is recorded.
__device__ __forceinline__ long long tree_row(const TreeParams& P, const int* table, int g, int key, int tok0) {
  const int pidx = key / P.page_size;
  const int page = pidx < P.max_pages ? table[pidx] : -1;
  if (page < 0 || page >= P.num_pages) {
    report_error(P.err, PHOTON_DEV_BAD_PAGE, tok0, key, page);
    return -1;
  }
  return ((long long)page * P.n_kv + g) * P.page_size + (key - pidx * P.page_size);
}

// Dynamic shared memory of a kernel, asked for once a device.
static int tree_smem_limit(const void* kernel, int bytes, bool (&ready)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64 || !ready[dev])) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) ready[dev] = true;
  }
  return (int)e;
}

// The call's arguments as the kernels take them; 0 or the error that refuses them.
static int tree_params(const photon_tree_call* c, TreeParams& P) {
  if (c->softcap < 0.f || c->mask_words < 1 || c->page_size <= 0 || c->num_pages <= 0 || c->max_pages <= 0 || c->parts < 1) return PHOTON_ERR_ARGUMENT;
  if (c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) return PHOTON_ERR_ARGUMENT;
  if (c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->d <= 0 || c->d > 256 || !(c->scale > 0.f)) return PHOTON_ERR_UNSUPPORTED;
  P.q = c->q; P.q_stride = c->q_stride; P.out = c->out; P.out_stride = c->out_stride; P.k_cache = c->k_cache; P.v_cache = c->v_cache;
  P.block_table = c->block_table; P.max_pages = c->max_pages; P.cu_tokens = c->cu_tokens; P.context_lens = c->context_lens;
  P.positions = c->positions; P.tree_mask = c->tree_mask; P.mask_words = c->mask_words; P.S = c->S; P.T = c->T; P.max_tokens = c->max_tokens_per_seq;
  P.n_q = c->n_q; P.n_kv = c->n_kv; P.group = c->n_q / c->n_kv; P.d = c->d; P.page_size = c->page_size; P.num_pages = c->num_pages;
  P.window = c->window > 0 ? c->window : 0; P.scale = c->scale; P.sinks = c->sinks; P.softcap = c->softcap; P.err = c->err;
  return 0;
}

// Blocks of a cluster read one another's shared memory.
__device__ __forceinline__ void tree_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float tree_peer(const float* p, int rank) {        // the float at the same place in another block of the cluster
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 tree_peer4(const float* p, int rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

template <typename... KArgs, typename... Args>
static inline int tree_launch_clusters(void (*kernel)(KArgs...), long blocks, int cluster, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks); cfg.blockDim = dim3((unsigned)threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = photon_pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
