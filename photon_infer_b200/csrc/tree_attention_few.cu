// Attention for small trees of drafted tokens: bfloat16, heads of 64 or 128 numbers, up to 64 rows (nodes x query heads per key/value head) a request.
//
// A cluster of blocks has one (request, key/value head): its tiles of 64 keys are dealt to the blocks in equal runs, a block's four warps
// take MT tiles of 16 rows times 4 / MT parts of a key tile.  Keys and values come by cp.async, two tiles ahead, the block table followed row by row (any page
// size); scores and weighted sums are mma.m16n8k16 with 32-bit sums, the softmax is a running one in 32 bits, weights are rounded to bfloat16 as the values are.
// At the end the warps' partial results lie in shared memory, and the blocks of the cluster join them there, each for its share of the outputs: one
// launch, no scratch, the same order of sums in every run.
//
// What bounds it: latency.  5 nodes behind 640 keys (32/8 heads of 64): 6.5 us, where the bytes take 0.2; 1 node behind 100: 5.5; 2 requests of 8 behind 1,000 (32/8
// heads of 128): 11.1 (bytes: 1.3).  A launch, the request's range and its pages, the first keys, two tiles of work and the join follow one another; in the
// kernel's wait counters memory, barriers and instructions that are not there yet have like parts.  A second kernel for the join took 15.8 us for the first of
// these.  Each step below half a microsecond: a row's factors once for all its outputs, short tables read beside the request's range, the shorter run for the block
// whose tiles masks cut, a key's row in the cache found once for all its pieces.
//
// Which keys a row sees: tree_attention.cuh.  In tiles where some row's mask cuts, values that are not finite are set to zero in shared memory before the
// products (0 times them would not be 0), and rows that see them get them back at the end from the cache.
#include "tree_attention.cuh"
#include <math.h>

#define TF_KT 64
#define TF_THREADS 128
#define TF_TABLE 512                               // block-table entries of the block's keys that are kept in shared memory
#define TF_LOG2E 1.4426950408889634f

struct TfParams {
  TreeParams t;
  float scale_log2, cap_in;
  int cluster, page_shift;
};

__device__ __forceinline__ uint32_t tf_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void tf_copy16(void* dst, const void* src, bool there) {       // not there: the bytes become zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tf_smem(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void tf_ld4(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(tf_smem(p)));
}
__device__ __forceinline__ void tf_ld4t(uint32_t* r, const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(tf_smem(p)));
}
__device__ __forceinline__ void tf_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float tf_exp2(float x) {         // 2^x; 0 at -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t tf_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <int D, int MT> struct Tf {
  static constexpr int KG = 4 / MT;                // warps that share a row tile, each with a part of every key tile
  static constexpr int NT = TF_KT / KG / 8;        // a warp's n-tiles of keys
  static constexpr int LD = D + 8;                 // padded row: conflict-free ldmatrix
  static constexpr int ROWS = 16 * MT;
  static constexpr int STAGES = D == 64 ? 3 : 2;   // three blocks an SM with heads of 64, two with heads of 128
  static constexpr int STAGE = 2 * TF_KT * LD;     // elements: a K tile, then a V tile
  static constexpr int LO = D + 4;                 // row of the joined partial results (floats)
  static constexpr int RING = (ROWS * LD + STAGES * STAGE) * 2;
  static constexpr int PART = 4 * 16 * LO * 4;     // every warp's 16 rows
  static constexpr int SMEM = RING > PART ? RING : PART;
};

template <int D, int MT>
__global__ void __launch_bounds__(TF_THREADS, D == 64 ? 3 : 2)
tree_attention_few_kernel(const TfParams P) {
  using C = Tf<D, MT>;
  extern __shared__ __align__(16) unsigned char tf_dyn[];
  bf16* qs = reinterpret_cast<bf16*>(tf_dyn);
  bf16* ring = qs + C::ROWS * C::LD;
  __shared__ int table_s[TF_TABLE];
  constexpr int SLOTS = C::STAGES + 1;
  __shared__ long long row_s[SLOTS][TF_KT];        // the cache rows of a tile's keys, found a tile before they are asked for; -1: none
  __shared__ uint32_t gone_s[SLOTS][2];            // its keys whose page is missing
  __shared__ int poison;                           // 1: some value of a tile where a mask cuts was not finite
  __shared__ float ml_s[2][4][16];                 // [maximum, sum][warp][row]
  __shared__ float factor_s[C::ROWS][32 / MT];     // of each partial result of a row
  const TreeParams& t = P.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % P.cluster, unit = blockIdx.x / P.cluster, g = unit % t.n_kv, seq = unit / t.n_kv;
  if (tid == 0) poison = 0;
  pdl_wait();
  // The request's pages: a short table is read whole, beside the request's range; of a long one the entries of the block's keys, once they are known.
  const int* table = t.block_table + (size_t)seq * t.max_pages;
  const bool whole = t.max_pages <= TF_TABLE;
  int entry[TF_TABLE / TF_THREADS];
#pragma unroll
  for (int k = 0; k < TF_TABLE / TF_THREADS; ++k) entry[k] = whole && k * TF_THREADS + tid < t.max_pages ? table[k * TF_THREADS + tid] : -1;
  const TreeRequest R = tree_request(t, seq);
  const int G = t.group, rows = min(R.n * G, C::ROWS);
  const int key_end = R.base + R.n, key_lo = t.window > 0 ? max(0, R.base - t.window + 1) : 0;
  const int cut_lo = t.window > 0 ? key_end - t.window : -1;      // no row's window begins behind this key
  const int tile_lo = key_lo / TF_KT, all = rows > 0 ? (key_end + TF_KT - 1) / TF_KT - tile_lo : 0;
  // the last block, whose tiles masks cut, has one that is no longer than the others'
  const int first = (all * rank + P.cluster - 1) / P.cluster, ntiles = (all * (rank + 1) + P.cluster - 1) / P.cluster - first, tile0 = tile_lo + first;
  auto page_of = [&](int key) { return P.page_shift >= 0 ? key >> P.page_shift : key / t.page_size; };
  const int from = page_of(tile0 * TF_KT), pages = ntiles > 0 ? page_of(min(key_end, (tile0 + ntiles) * TF_KT) - 1) - from + 1 : 0;
  const int page0 = whole ? 0 : from;
  const bool kept = whole || pages <= TF_TABLE;
  if (whole) {
#pragma unroll
    for (int k = 0; k < TF_TABLE / TF_THREADS; ++k) table_s[k * TF_THREADS + tid] = entry[k];
  } else if (kept) {
    for (int i = tid; i < pages; i += TF_THREADS) table_s[i] = page0 + i < t.max_pages ? table[page0 + i] : -1;
  }
  // Q, zeros behind the rows
  {
    const bf16* q = (const bf16*)t.q;
    for (int c = tid; c < C::ROWS * (D / 8); c += TF_THREADS) {
      const int r = c / (D / 8), j = c % (D / 8) * 8;
      const bool there = r < rows;
      const int node = there ? r / G : 0, h = there ? r - node * G : 0;
      tf_copy16(qs + r * C::LD + j, q + (size_t)(R.tok0 + node) * t.q_stride + (size_t)(g * G + h) * D + j, there);
    }
  }
  __syncthreads();
  auto find = [&](int i, int x) {                  // key x of tile i of the block; by whole warps
    const int key = (tile0 + i) * TF_KT + x;
    long long row = -1;
    bool bad = false;
    if (i < ntiles && key >= key_lo && key < key_end) {
      const int pidx = page_of(key), page = pidx >= t.max_pages ? -1 : kept ? table_s[pidx - page0] : table[pidx];
      bad = page < 0 || page >= t.num_pages;
      if (bad) report_error(t.err, PHOTON_DEV_BAD_PAGE, R.tok0, key, page);
      else row = ((long long)page * t.n_kv + g) * t.page_size + (key - pidx * t.page_size);
    }
    const uint32_t gone = __ballot_sync(0xffffffffu, bad);
    row_s[i % SLOTS][x] = row;
    if (lane == 0) gone_s[i % SLOTS][x >> 5] = gone;
  };
  auto load = [&](int i) {                         // tile i of the block into its stage
    bf16* ks = ring + i % C::STAGES * C::STAGE;
    bf16* vs = ks + TF_KT * C::LD;
    constexpr int CPR = D / 8, STEP = TF_THREADS / CPR;           // 16-byte pieces of a row; rows that the block copies at a time
    const int j = tid % CPR * 8;
#pragma unroll
    for (int r = tid / CPR; r < TF_KT; r += STEP) {
      const long long row = row_s[i % SLOTS][r];
      const size_t at = row >= 0 ? (size_t)row * D + j : 0;
      tf_copy16(ks + r * C::LD + j, (const bf16*)t.k_cache + at, row >= 0);
      tf_copy16(vs + r * C::LD + j, (const bf16*)t.v_cache + at, row >= 0);
    }
  };
  for (int i = tid / TF_KT; i < min(C::STAGES, ntiles); i += TF_THREADS / TF_KT) find(i, tid % TF_KT);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C::STAGES - 1; ++i) {
    if (i < ntiles) load(i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const int rt = warp / C::KG, kg = warp % C::KG;  // the warp's row tile and its part of the keys
  const int krow = kg * (TF_KT / C::KG);
  const int c2 = (lane & 3) * 2;
  int tok[2], lo[2];                               // of the lane's rows lane / 4 and lane / 4 + 8; -1: no such row
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = rt * 16 + (lane >> 2) + h * 8;
    tok[h] = r < rows ? R.tok0 + r / G : -1;
    lo[h] = tok[h] >= 0 && t.window > 0 ? max(0, t.positions[tok[h]] - t.window + 1) : 0;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  uint32_t qa[D / 16][4];

  for (int i = 0; i < ntiles; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncthreads();                               // tile i is there for all; the tile before is read
    if (i + C::STAGES - 1 < ntiles) load(i + C::STAGES - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const int st = i % C::STAGES, key_base = (tile0 + i) * TF_KT;
    const bf16* ks = ring + st * C::STAGE;
    bf16* vs = ring + st * C::STAGE + TF_KT * C::LD;
    if (i == 0) {
#pragma unroll
      for (int kd = 0; kd < D / 16; ++kd) tf_ld4(qa[kd], qs + (rt * 16 + (lane & 15)) * C::LD + kd * 16 + ((lane >> 4) << 3));
    }
    const uint64_t gone = (uint64_t)gone_s[i % SLOTS][1] << 32 | gone_s[i % SLOTS][0];
    if (tid < TF_KT && i + C::STAGES < ntiles) find(i + C::STAGES, tid);
    const bool cut = key_base + TF_KT > R.base || key_base <= cut_lo;           // some row's mask cuts; rows of a missing page are zeros
    if (cut) {
      bool found = false;
      for (int c = tid; c < TF_KT * (D / 8); c += TF_THREADS) {
        uint4* at = reinterpret_cast<uint4*>(vs + c / (D / 8) * C::LD + c % (D / 8) * 8);
        const uint4 x = *at;
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        bool bad = false;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if ((w[u] & 0x7f80u) == 0x7f80u) { w[u] &= 0xffff0000u; bad = true; }
          if ((w[u] & 0x7f800000u) == 0x7f800000u) { w[u] &= 0xffffu; bad = true; }
        }
        if (bad) { *at = make_uint4(w[0], w[1], w[2], w[3]); found = true; }
      }
      if (found) poison = 1;
      __syncthreads();
    }
    float s[C::NT][4];
#pragma unroll
    for (int j = 0; j < C::NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kd = 0; kd < D / 16; ++kd) {
#pragma unroll
      for (int j = 0; j < C::NT; j += 2) {
        uint32_t b[4];
        tf_ld4(b, ks + (krow + j * 8 + (lane & 7) + ((lane >> 4) << 3)) * C::LD + kd * 16 + (((lane >> 3) & 1) << 3));
        tf_mma(s[j], qa[kd], b[0], b[1]);
        tf_mma(s[j + 1], qa[kd], b[2], b[3]);
      }
    }
    if (t.softcap > 0.f) {
      bool small = true;
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) small = small && fabsf(s[j][u]) * P.cap_in <= 0.5f;
      if (__all_sync(0xffffffffu, small)) {
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u) s[j][u] = t.softcap * tree_tanh_half(s[j][u] * P.cap_in);
      } else {
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u)              // tanh(x) = 1 - 2 / (2^(2 x log2 e) + 1)
            s[j][u] = t.softcap - __fdividef(2.0f * t.softcap, tf_exp2(s[j][u] * P.cap_in * 2.8853900817779268f) + 1.0f);
      }
    }
    if (cut || gone != 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint64_t bits = 0;
        if (tok[h] >= 0)
          bits = (uint64_t)tree_visible32(t, R, tok[h], key_base, lo[h]) | (uint64_t)tree_visible32(t, R, tok[h], key_base + 32, lo[h]) << 32;
        bits &= ~gone;
        bits >>= krow + c2;
#pragma unroll
        for (int j = 0; j < C::NT; ++j) {
          if (!((bits >> (8 * j)) & 1)) s[j][2 * h] = -INFINITY;
          if (!((bits >> (8 * j + 1)) & 1)) s[j][2 * h + 1] = -INFINITY;
        }
      }
    }
    float sub[2], keep[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < C::NT; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * h], s[j][2 * h + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[h], mx * P.scale_log2);
      sub[h] = mn == -INFINITY ? 0.f : mn;
      keep[h] = tf_exp2(m[h] - sub[h]);
      m[h] = mn;
      l[h] *= keep[h];
    }
    uint32_t pa[C::NT / 2][4];
#pragma unroll
    for (int j = 0; j < C::NT; ++j) {
      const float p0 = tf_exp2(fmaf(s[j][0], P.scale_log2, -sub[0])), p1 = tf_exp2(fmaf(s[j][1], P.scale_log2, -sub[0]));
      const float p2 = tf_exp2(fmaf(s[j][2], P.scale_log2, -sub[1])), p3 = tf_exp2(fmaf(s[j][3], P.scale_log2, -sub[1]));
      l[0] += p0 + p1; l[1] += p2 + p3;            // the lane's part of the sum; the quad is added up at the end
      pa[j >> 1][(j & 1) * 2] = tf_pack(p0, p1);
      pa[j >> 1][(j & 1) * 2 + 1] = tf_pack(p2, p3);
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) { o[n][0] *= keep[0]; o[n][1] *= keep[0]; o[n][2] *= keep[1]; o[n][3] *= keep[1]; }
#pragma unroll
    for (int kk = 0; kk < C::NT / 2; ++kk) {
#pragma unroll
      for (int n = 0; n < D / 8; n += 2) {
        uint32_t b[4];
        tf_ld4t(b, vs + (krow + kk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3)) * C::LD + n * 8 + ((lane >> 4) << 3));
        tf_mma(o[n], pa[kk], b[0], b[1]);
        tf_mma(o[n + 1], pa[kk], b[2], b[3]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  pdl_launch_dependents();
  __syncthreads();                                 // the ring is read; poison is known
  if (poison) {
    // what was not finite, for the rows that see it: each warp the keys of its own part, whose weights its sum has
    for (int i = 0; i < ntiles; ++i) {
      const int key_base = (tile0 + i) * TF_KT;
      if (!(key_base + TF_KT > R.base || key_base <= cut_lo)) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint64_t bits = 0;
        if (tok[h] >= 0)
          bits = (uint64_t)tree_visible32(t, R, tok[h], key_base, lo[h]) | (uint64_t)tree_visible32(t, R, tok[h], key_base + 32, lo[h]) << 32;
        if (C::KG > 1) bits &= ((1ull << (TF_KT / C::KG & 63)) - 1ull) << krow;
        for (; bits != 0; bits &= bits - 1) {
          const int key = key_base + __ffsll(bits) - 1, pidx = page_of(key);
          const int page = pidx < t.max_pages ? table[pidx] : -1;
          if (page < 0 || page >= t.num_pages) continue;
          const bf16* vr = (const bf16*)t.v_cache + (((size_t)page * t.n_kv + g) * t.page_size + (key - pidx * t.page_size)) * D + c2;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const float y0 = to_f32(vr[n * 8]), y1 = to_f32(vr[n * 8 + 1]);
            if (!isfinite(y0)) o[n][2 * h] += y0;
            if (!isfinite(y1)) o[n][2 * h + 1] += y1;
          }
        }
      }
    }
  }
  // ---- the warps' results into shared memory
  float* po = reinterpret_cast<float*>(tf_dyn);    // [warp][16][LO]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int r = (lane >> 2) + h * 8;
    if ((lane & 3) == 0) { ml_s[0][warp][r] = m[h]; ml_s[1][warp][r] = l[h]; }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(po + (warp * 16 + r) * C::LO + n * 8 + c2) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
  }
  tree_cluster_sync();
  // ---- every block joins its share of the rows' numbers: over the blocks in their order, over a block's warps in theirs
  {
    constexpr int W = TF_THREADS / (16 * MT);      // threads a row, four of its results each
    const int r = tid / W, n = P.cluster * C::KG, w0 = r / 16 * C::KG, rr = r & 15;
    const float sink = t.sinks && r < rows ? t.sinks[g * G + r % G] * TF_LOG2E : -INFINITY;
    float f[4], s[4], top = sink, sum = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = tid % W + W * u;
      f[u] = w < n ? tree_peer(&ml_s[0][w0 + w % C::KG][rr], w / C::KG) : -INFINITY;
      s[u] = w < n ? tree_peer(&ml_s[1][w0 + w % C::KG][rr], w / C::KG) : 0.f;
      top = fmaxf(top, f[u]);
    }
#pragma unroll
    for (int w = W / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float sub = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool none = tree_nothing(f[u], s[u]);
      f[u] = tf_exp2(f[u] - sub);                  // 0 for what is not there
      sum += s[u] * f[u];
      s[u] = none ? TREE_NOTHING : 0.f;
    }
#pragma unroll
    for (int w = W / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    sum += tf_exp2(sink - sub);
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (tid % W + W * u < n) factor_s[r][tid % W + W * u] = s[u] == TREE_NOTHING ? TREE_NOTHING : f[u] * inv;
  }
  __syncthreads();
  const int pieces = rows * (D / 4), last = pieces * (rank + 1) / P.cluster;
  for (int e = pieces * rank / P.cluster + tid; e < last; e += TF_THREADS) {
    const int r = e / (D / 4), j = e % (D / 4) * 4, w0 = r / 16 * C::KG, rr = r & 15;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int B = 8 / C::KG;                   // blocks whose results are on their way at a time
    for (int b0 = 0; b0 < P.cluster; b0 += B) {
      float4 x[B][C::KG];
      float w[B][C::KG];
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int k = 0; k < C::KG; ++k) {
          w[b][k] = b0 + b < P.cluster ? factor_s[r][(b0 + b) * C::KG + k] : TREE_NOTHING;
          x[b][k] = tree_peer4(po + ((w0 + k) * 16 + rr) * C::LO + j, min(b0 + b, P.cluster - 1));
        }
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int k = 0; k < C::KG; ++k)
          if (!(w[b][k] < 0.f)) {
            a.x = fmaf(w[b][k], x[b][k].x, a.x); a.y = fmaf(w[b][k], x[b][k].y, a.y); a.z = fmaf(w[b][k], x[b][k].z, a.z); a.w = fmaf(w[b][k], x[b][k].w, a.w);
          }
    }
    uint2 v;
    v.x = tf_pack(a.x, a.y); v.y = tf_pack(a.z, a.w);
    *reinterpret_cast<uint2*>((bf16*)t.out + (size_t)(R.tok0 + r / G) * t.out_stride + (size_t)(g * G + r % G) * D + j) = v;
  }
  tree_cluster_sync();                               // the others have read this block's results
}

template <int D, int MT>
static int tf_launch(const TfParams& P, cudaStream_t stream) {
  static bool ready[64] = {};
  int st = tree_smem_limit((const void*)tree_attention_few_kernel<D, MT>, Tf<D, MT>::SMEM, ready);
  if (st != 0) return st;
  return tree_launch_clusters(tree_attention_few_kernel<D, MT>, (long)P.t.S * P.t.n_kv * P.cluster, P.cluster, TF_THREADS, Tf<D, MT>::SMEM, stream, P);
}

PHOTON_API int photon_tree_attention_few(const photon_tree_call* call, cudaStream_t stream) {
  if (call->S <= 0 || call->T <= 0 || call->max_tokens_per_seq <= 0) return 0;
  TfParams P;
  TreeParams& t = P.t;
  const int st = tree_params(call, t);
  if (st != 0) return st;
  const long rows = (long)t.max_tokens * t.group;
  if (call->dtype != PHOTON_BF16 || (t.d != 64 && t.d != 128) || rows > 64) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)t.q & 15) || (t.q_stride & 7) || ((uintptr_t)t.k_cache & 15) || ((uintptr_t)t.v_cache & 15) || ((uintptr_t)t.out & 7) || (t.out_stride & 3))
    return PHOTON_ERR_UNSUPPORTED;
  P.cluster = call->parts;
  if (P.cluster < 1 || P.cluster > 8) return PHOTON_ERR_ARGUMENT;
  if ((long)t.S * t.n_kv * P.cluster > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  P.page_shift = -1;
  for (int sh = 0; sh < 20; ++sh) if ((1 << sh) == t.page_size) P.page_shift = sh;
  P.scale_log2 = t.scale * TF_LOG2E; P.cap_in = 0.f;
  if (t.softcap > 0.f) { P.cap_in = t.scale / t.softcap; P.scale_log2 = TF_LOG2E; }
  if (t.d == 64) return rows <= 16 ? tf_launch<64, 1>(P, stream) : rows <= 32 ? tf_launch<64, 2>(P, stream) : tf_launch<64, 4>(P, stream);
  return rows <= 16 ? tf_launch<128, 1>(P, stream) : rows <= 32 ? tf_launch<128, 2>(P, stream) : tf_launch<128, 4>(P, stream);
}
