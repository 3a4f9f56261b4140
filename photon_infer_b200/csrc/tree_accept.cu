// Which drafted tokens of a tree a request keeps.
//
// Node 0 is the request's last token.  From it on: y = the token that the node's logits give (the first largest one, or with a temperature T the first i of any
// probability with e^((x_0 - max) / T) + .. + e^((x_i - max) / T) >= u sum); the first child whose token is y is the next node; where there is none the walk
// ends.  The tokens y are what the request generates, one for every node on the path.
//
// A row of logits is a cluster of blocks' work: a block takes a run of the vocabulary, up to 32 numbers a thread in registers (longer runs are read again), and the blocks'
// maxima and sums meet in each other's shared memory.  Sums are in 32 bits, added up in an order that the sizes alone give.
//
// Two ways.  A cluster for every request walks its tree, and reads the logits of the nodes on the path alone, one after the other.  Few logits in all that tokens are
// drawn from: a cluster for every node at once, and a second kernel walks the trees.
// A step of a walk is latency: 2.1 us greedily (a row from memory, the warps' and the blocks' maxima, one exchange), 5.6 us with a temperature (weights, sums, and
// a second exchange, which tells all blocks what one of them has chosen).  128,256 tokens: one request of 8 nodes 4.4 us greedily, sampled 13 as a walk and 7.5 at once; 32 requests of 64
// nodes, half of them sampled, walk in 52 us (all 1.05 GB of logits would take 268 and more), the paths' 65 MB at the copy rate 10.
#include "common.cuh"
#include <math.h>

#define TA_THREADS 512
#define TA_VALUES 32                               // numbers of a row that a thread keeps
#define TA_MAX_CLUSTER 8

struct TaParams {
  const float* logits; long ld;
  const int* tokens; const int* parents; const int* cu_tokens;
  const float* temperature; const float* uniforms;
  int* path; int* counts; int* sampled;
  int* given;                                      // [T]: the token that every node's logits give, where all of them are asked
  int* err;
  int S, T, V, D, most, cluster, vectors;          // vectors: rows begin on 16-byte boundaries
};

struct TaShared {
  float4 x[2][TA_MAX_CLUSTER];                     // what the cluster's blocks have found, (value, index, sum, -), twice in turn
  uint64_t bar[2];                                 // all of them are there
  // of each warp: its largest number's key and place, twice in turn (greedily nothing holds a warp back until all have read them), and the sum of its weights
  uint32_t key[2][TA_THREADS / 32]; int at[2][TA_THREADS / 32];
  float wsum[TA_THREADS / 32];
  int chosen;
};
// Where a block is in the exchanges: how many there were, and whether the cluster has begun.
// `late`: a wait for the others ran out; the thread sends nothing from then on.
struct TaTurn { int count; bool met, late; };

__device__ __forceinline__ float ta_scan(float v) {         // the sum up to this lane
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float a = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += a;
  }
  return v;
}
__device__ __forceinline__ float ta_exp2(float x) {        // 2^x, to 2^-22 of itself; 0 at -inf
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t ta_peer(const void* p, int rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t ta_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// The blocks of a cluster tell each other that their barriers stand; the wait for it is in the first exchange.
__device__ __forceinline__ void ta_begin(TaShared& sh) {
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(ta_smem(&sh.bar[b])));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
// Every block of the cluster hands (v, i, s) to all of them, itself too; behind it each has all in the half of sh.x that is returned.  Called by all threads.  The stores carry
// their own signal: what is sent in one exchange is read before its reader sends in the next, so the half is free again two exchanges on.
__device__ __forceinline__ const float4* ta_exchange(TaShared& sh, TaTurn& turn, int rank, int cluster, float v, int i, float s) {
  const int half = turn.count & 1, parity = (turn.count >> 1) & 1;
  if (!turn.met) { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); turn.met = true; }
  const uint32_t bar = ta_smem(&sh.bar[half]);
  if (threadIdx.x == 0)
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(cluster * 16) : "memory");
  if (threadIdx.x < cluster && !turn.late)
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(ta_peer(&sh.x[half][rank], threadIdx.x)), "r"(__float_as_uint(v)), "r"(i), "r"(__float_as_uint(s)), "r"(0),
                 "r"(ta_peer(&sh.bar[half], threadIdx.x)) : "memory");
  uint32_t there = 0;
  for (int k = 0; k < (1 << 20) && !there && !turn.late; ++k)
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(there) : "r"(bar), "r"(parity) : "memory");
  turn.late |= !there;
  ++turn.count;
  return sh.x[half];
}

// Order-preserving whole numbers for the warp's reductions: a larger number has a larger key.
__device__ __forceinline__ uint32_t ta_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);     // -0 as 0
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// The token that a row of logits gives; every thread of the cluster gets it.  A warp takes a run of neighbouring numbers, 128 at a time.
template <bool KEEP>
__device__ int ta_token(const TaParams& P, TaShared& sh, const float* row, int rank, float temperature, float u, TaTurn& turn) {
  constexpr int UNROLL = KEEP ? TA_VALUES / 4 : 1, WARPS = TA_THREADS / 32;
  constexpr unsigned ALL = 0xffffffffu;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, C = P.cluster;
  const int span = ((P.V + C - 1) / C + 3) & ~3, lo = min(P.V, rank * span), hi = min(P.V, lo + span);
  const int runs = KEEP ? UNROLL : (span + WARPS * 128 - 1) / (WARPS * 128);
  const int w0 = lo + warp * runs * 128;
  auto read = [&](int j, float* x) {               // this thread's four numbers of run j; behind the block's part -inf
    const int at = w0 + j * 128 + lane * 4;
    if (P.vectors && at + 4 <= hi) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(row + at));
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = at + e < hi ? __ldg(row + at + e) : -INFINITY;
    }
  };
  float kept[KEEP ? TA_VALUES : 4];
  if (KEEP) {
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) read(j, kept + 4 * j);
  }
  // the largest number (a NaN never is), then its first place
  float best = -INFINITY;
#pragma unroll UNROLL
  for (int j = 0; j < runs; ++j) {
    if (!KEEP) read(j, kept);
#pragma unroll
    for (int e = 0; e < 4; ++e) best = fmaxf(best, kept[KEEP ? 4 * j + e : e]);
  }
  const float mine = best;
  const uint32_t key = __reduce_max_sync(ALL, ta_key(best));
  int at = 0x7fffffff;
  if (ta_key(mine) == key) {
#pragma unroll UNROLL
    for (int j = runs - 1; j >= 0; --j) {
      if (!KEEP) read(j, kept);
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        const int i = w0 + j * 128 + lane * 4 + e;
        if (i < hi && kept[KEEP ? 4 * j + e : e] == mine) at = i;
      }
    }
  }
  at = __reduce_min_sync(ALL, (unsigned)at);
  const int half = turn.count & 1;
  if (lane == 0) { sh.key[half][warp] = key; sh.at[half][warp] = at; }
  __syncthreads();
  // every warp: the block's
  {
    const uint32_t k = lane < WARPS ? sh.key[half][lane] : 0u, top = __reduce_max_sync(ALL, k);
    at = (int)__reduce_min_sync(ALL, lane < WARPS && k == top ? (unsigned)sh.at[half][lane] : 0x7fffffffu);
    best = __uint_as_float(top ^ ((top >> 31) ? 0x80000000u : 0xffffffffu));
  }
  // With a temperature the warps' sums of weights relative to the block's largest number go along.
  const bool draw = temperature > 0.f;
  const float scale = 1.4426950408889634f / temperature, own = best == -INFINITY ? 0.f : best;
  auto weight = [&](float x) { return ta_exp2((x - own) * scale); };
  float part = 0.f, upto = 0.f, sum = 0.f;         // lane w: warp w's sum, the sum up to it; the block's
  if (draw) {
    float s = 0.f;
#pragma unroll UNROLL
    for (int j = 0; j < runs; ++j) {
      if (!KEEP) read(j, kept);
#pragma unroll
      for (int e = 0; e < 4; ++e) s += weight(kept[KEEP ? 4 * j + e : e]);
    }
    s = warp_sum(s);
    if (lane == 0) sh.wsum[warp] = s;
    __syncthreads();
    part = lane < WARPS ? sh.wsum[lane] : 0.f;
    upto = ta_scan(part);
    sum = __shfl_sync(ALL, upto, 31);
  }
  const float4* all = ta_exchange(sh, turn, rank, C, best, at, sum);
  const float4 other = lane < C ? all[lane] : make_float4(-INFINITY, __int_as_float(0x7fffffff), 0.f, 0.f);
  const uint32_t top_key = __reduce_max_sync(ALL, ta_key(other.x));
  at = (int)__reduce_min_sync(ALL, ta_key(other.x) == top_key ? __float_as_uint(other.y) : 0x7fffffffu);
  if (at == 0x7fffffff) at = 0;                    // nothing but NaN
  if (!draw) return at;

  // the block in whose part the target lies
  const float top = __uint_as_float(top_key ^ ((top_key >> 31) ? 0x80000000u : 0xffffffffu));
  const float share = other.x == -INFINITY ? 0.f : other.z * ta_exp2((other.x - top) * scale), run = ta_scan(share);
  const float total = __shfl_sync(ALL, run, 31), target = u * total;
  if (!(total > 0.f)) return at;                   // weights that are not numbers
  const unsigned some = __ballot_sync(ALL, share > 0.f), hit = __ballot_sync(ALL, share > 0.f && run >= target);
  const int owner = hit != 0 ? __ffs(hit) - 1 : 31 - __clz(some);              // rounding left the sums below the target: the last one with weight
  const float before = __shfl_sync(ALL, run - share, owner);
  if (rank == owner) {
    // what is left of the target, relative to this block's largest number; in the block the warp, in the warp the run, in the run the lane, in the lane the number: the first
    // of any weight whose sum reaches the target, or else the last of any weight
    // (a block some 90 temperatures below the row's largest number has a share of so few bits that its weights' factor is infinite: the target's part of the share then)
    const float factor = ta_exp2((top - own) * scale), left = target - before;
    float want = hit == 0 ? INFINITY : isfinite(factor) ? left * factor : left / __shfl_sync(ALL, share, owner) * sum;
    const unsigned with = __ballot_sync(ALL, part > 0.f), reach = __ballot_sync(ALL, part > 0.f && upto >= want);
    const int w = reach != 0 ? __ffs(reach) - 1 : 31 - __clz(with);
    if (warp == w) {
      want = reach != 0 ? want - __shfl_sync(ALL, upto - part, w) : INFINITY;
      float x[4], p[4], passed = 0.f, rest = want;
      int in = -1, full = 0;
#pragma unroll UNROLL
      for (int j = 0; j < runs; ++j) {
        if (!KEEP) read(j, kept);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s += weight(kept[KEEP ? 4 * j + e : e]);
        s = warp_sum(s);
        if (s > 0.f) {
          if (in < 0 && passed + s >= want) { in = j; rest = want - passed; }
          full = j;
        }
        passed += s;
      }
      if (in < 0) { in = full; rest = INFINITY; }
      if (KEEP) {
#pragma unroll
        for (int j = 0; j < UNROLL; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) if (j == in) x[e] = kept[KEEP ? 4 * j + e : e];
      } else {
        read(in, x);
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) { p[e] = weight(x[e]); s += p[e]; }
      const float to = ta_scan(s);
      const unsigned any = __ballot_sync(ALL, s > 0.f), at_last = __ballot_sync(ALL, s > 0.f && to >= rest);
      const int l = at_last != 0 ? __ffs(at_last) - 1 : 31 - __clz(any);
      if (lane == l) {
        float a = to - s;
        int pick = -1, end = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a += p[e];
          if (p[e] > 0.f) {
            if (pick < 0 && a >= rest) pick = e;
            end = e;
          }
        }
        sh.chosen = w0 + in * 128 + lane * 4 + (pick >= 0 ? pick : end);
      }
    }
  }
  __syncthreads();                                 // the number is chosen; all warps have read the exchange before
  return __float_as_int(ta_exchange(sh, turn, rank, C, 0.f, rank == owner ? sh.chosen : 0, 0.f)[owner].y);
}

// The first child of a node with a token; n where there is none.  Warp-wide; parents and tokens of the first 64 nodes are in the lanes.
struct TaNodes { int parent[2], token[2]; };
__device__ __forceinline__ TaNodes ta_nodes(const TaParams& P, int t0, int n) {
  TaNodes q;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = (threadIdx.x & 31) + 32 * k;
    q.parent[k] = i < n ? P.parents[t0 + i] : -1;
    q.token[k] = i < n ? P.tokens[t0 + i] : -1;
  }
  return q;
}
__device__ __forceinline__ int ta_child(const TaParams& P, const TaNodes& q, int t0, int n, int node, int y) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = lane + 32 * k;
    const unsigned hit = __ballot_sync(0xffffffffu, i > node && i < n && q.parent[k] == node && q.token[k] == y);
    if (hit != 0) return 32 * k + __ffs(hit) - 1;
  }
  for (int i0 = max(64, node + 1); i0 < n; i0 += 32) {
    const int i = i0 + lane;
    const unsigned hit = __ballot_sync(0xffffffffu, i < n && P.parents[t0 + i] == node && P.tokens[t0 + i] == y);
    if (hit != 0) return i0 + __ffs(hit) - 1;
  }
  return n;
}
__device__ __forceinline__ void ta_range(const TaParams& P, int seq, int& t0, int& n) {
  t0 = max(0, min(P.cu_tokens[seq], P.T));
  n = max(0, min(min(P.cu_tokens[seq + 1], P.T) - t0, P.most));
}

// What is sent to a block is read by it before it ends, so no block has to wait for another here; one that exchanged nothing still takes the wait it has begun.
__device__ __forceinline__ void ta_end(const TaParams& P, TaShared& sh, const TaTurn& turn, int seq) {
  if (!turn.met) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if (threadIdx.x == 0 && turn.late) report_error(P.err, PHOTON_DEV_WAIT_TIMEOUT, seq, turn.count, 0);
}

// A cluster a request: the walk itself.
template <bool KEEP>
__global__ void __launch_bounds__(TA_THREADS, 2)
tree_accept_kernel(const TaParams P) {
  __shared__ TaShared sh;
  TaTurn turn = {0, false, false};
  ta_begin(sh);
  pdl_wait();
  const int rank = blockIdx.x % P.cluster, seq = blockIdx.x / P.cluster;
  int t0, n, node = 0, count = 0;
  ta_range(P, seq, t0, n);
  const TaNodes nodes = ta_nodes(P, t0, n);
  const float temperature = P.temperature ? P.temperature[seq] : 0.f;
  while (count < P.D && node < n) {
    const int y = ta_token<KEEP>(P, sh, P.logits + (size_t)(t0 + node) * P.ld, rank, temperature, temperature > 0.f ? P.uniforms[t0 + node] : 0.f, turn);
    if (rank == 0 && threadIdx.x == 0) { P.path[(size_t)seq * P.D + count] = node; P.sampled[(size_t)seq * P.D + count] = y; }
    ++count;
    node = ta_child(P, nodes, t0, n, node, y);
    if (turn.late) break;
  }
  if (rank == 0) {
    for (int i = count + threadIdx.x; i < P.D; i += TA_THREADS) { P.path[(size_t)seq * P.D + i] = -1; P.sampled[(size_t)seq * P.D + i] = -1; }
    if (threadIdx.x == 0) P.counts[seq] = count;
  }
  ta_end(P, sh, turn, seq);
}

// A cluster a node: what its logits give.
template <bool KEEP>
__global__ void __launch_bounds__(TA_THREADS, 2)
tree_tokens_kernel(const TaParams P) {
  __shared__ TaShared sh;
  TaTurn turn = {0, false, false};
  ta_begin(sh);
  pdl_wait();
  const int rank = blockIdx.x % P.cluster, unit = blockIdx.x / P.cluster, seq = unit / P.most, node = unit % P.most;
  int t0, n;
  ta_range(P, seq, t0, n);
  if (node >= n) { ta_end(P, sh, turn, seq); return; }         // the whole cluster
  const float temperature = P.temperature ? P.temperature[seq] : 0.f;
  const int y = ta_token<KEEP>(P, sh, P.logits + (size_t)(t0 + node) * P.ld, rank, temperature, temperature > 0.f ? P.uniforms[t0 + node] : 0.f, turn);
  if (rank == 0 && threadIdx.x == 0) P.given[t0 + node] = y;
  pdl_launch_dependents();
  ta_end(P, sh, turn, seq);
}

// A warp a request.
__global__ void __launch_bounds__(32)
tree_walk_kernel(const TaParams P) {
  pdl_wait();
  const int seq = blockIdx.x, lane = threadIdx.x;
  int t0, n, node = 0, count = 0;
  ta_range(P, seq, t0, n);
  const TaNodes nodes = ta_nodes(P, t0, n);
  while (count < P.D && node < n) {
    const int y = P.given[t0 + node];
    if (lane == 0) { P.path[(size_t)seq * P.D + count] = node; P.sampled[(size_t)seq * P.D + count] = y; }
    ++count;
    node = ta_child(P, nodes, t0, n, node, y);
  }
  for (int i = count + lane; i < P.D; i += 32) { P.path[(size_t)seq * P.D + i] = -1; P.sampled[(size_t)seq * P.D + i] = -1; }
  if (lane == 0) P.counts[seq] = count;
}

template <typename K>
static int ta_launch(K kernel, long clusters, const TaParams& P, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * P.cluster)); cfg.blockDim = dim3(TA_THREADS); cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = P.cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = photon_pdl_enabled() ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

PHOTON_API int photon_tree_accept(const photon_accept_call* c, cudaStream_t stream) {
  if (c->S <= 0) return 0;
  if (c->V <= 0 || c->T < 0 || c->D <= 0 || c->max_tokens_per_seq <= 0 || (c->temperature != nullptr && c->uniforms == nullptr)) return PHOTON_ERR_ARGUMENT;
  TaParams P;
  P.logits = c->logits; P.ld = c->ld; P.tokens = c->tokens; P.parents = c->parents; P.cu_tokens = c->cu_tokens; P.temperature = c->temperature;
  P.uniforms = c->uniforms; P.path = c->path; P.counts = c->counts; P.sampled = c->sampled; P.given = c->given; P.err = c->err;
  P.S = c->S; P.T = c->T; P.V = c->V; P.D = c->D; P.most = c->max_tokens_per_seq;
  P.cluster = 1;
  while (P.cluster < TA_MAX_CLUSTER && P.V > P.cluster * TA_THREADS * TA_VALUES) P.cluster *= 2;
  P.vectors = (uintptr_t)c->logits % 16 == 0 && c->ld % 4 == 0;
  const int span = ((P.V + P.cluster - 1) / P.cluster + 3) & ~3;
  const bool keep = span <= TA_THREADS * TA_VALUES;
  const long nodes = (long)P.S * P.most;
  if ((P.given != nullptr ? nodes : P.S) * P.cluster > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  if (P.given == nullptr) return keep ? ta_launch(tree_accept_kernel<true>, P.S, P, stream) : ta_launch(tree_accept_kernel<false>, P.S, P, stream);
  const int st = keep ? ta_launch(tree_tokens_kernel<true>, nodes, P, stream) : ta_launch(tree_tokens_kernel<false>, nodes, P, stream);
  if (st != 0) return st;
  return launch_pdl(tree_walk_kernel, dim3((unsigned)P.S), dim3(32), 0, stream, P);
}
