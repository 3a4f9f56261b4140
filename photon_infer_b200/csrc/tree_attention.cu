// Attention for trees of drafted tokens over a paged cache, for either type and heads of up to 256 numbers.
//
//   out[t, h] = sum_j w_j v_j / (sum_j w_j + e^(sink_h - m)),  w_j = e^(x_j - m),  x_j = scale q[t, h] . k_j
//
// (bounded scores: x_j = softcap tanh(scale q . k_j / softcap); m the largest of the scores and the sink) over the keys that node t sees
// (tree_attention.cuh); a row that sees nothing is zero.  Scores, weights, sums and outputs are held in 32 bits.
//
// A block takes up to 32 rows, (node, query head) pairs that share a key/value head, and a share of the request's keys, in tiles of 64; a warp has 16 of the rows and a half, a
// quarter or an eighth of a tile's keys (tree_choose).  A thread holds the scores of four rows with up to four keys, then those rows' outputs for D / 8 numbers, and a
// lane's neighbours read the same operands, so that a product costs a quarter of a word of shared memory; products go in pairs (fma.rn.f32x2).  Each warp has its own
// maxima and sums; the weights pass through shared memory inside the warp.  The warps' results, and those of a cluster of up to eight blocks that share a row tile's
// keys, are joined in shared memory in their order; where more blocks share them, by a second kernel.
//
// What bounds it: 32-bit products, and for small calls their latency.  4 requests of 13 nodes behind up to 700 keys (32/8 heads of 64): 19 us, 1 us of it for the bytes; 8 of
// 32 behind up to 2,000: 89 us = 17 TFLOP/s of products that are needed; 1 of 8 behind 640: 14; 3 of 5 behind up to 36: 7.5.  A tile ahead in shared memory left two
// blocks an SM and was slower (32 and 25 us, 132 and 108); tiles of 32 keys 23 and 118; the sums of products in one number after the other, 32 keys a
// tile, 36 and 334.
//
// A key that a row does not see has weight 0, and 0 times a value that is not finite would not be: in tiles where masks cut and such values lie, products with keys that
// a row does not see are left out, and so are shares of which it sees nothing; rows behind the last key or of a missing page are zeros.
#include "tree_attention.cuh"
#include <math.h>
#include <type_traits>

#define TG_KEYS 64

// How a block's warps share a tile: GROUPS of 16 rows, SHARES of the keys.
template <int GROUPS, int SHARES> struct Tg {
  static constexpr int ROWS = 16 * GROUPS, THREADS = 32 * GROUPS * SHARES;
  static constexpr int MINE = TG_KEYS / SHARES;    // a warp's keys
  static constexpr int PS = MINE + 4;              // row stride of a warp's weights, [16][MINE]
};

struct TreeShares {
  float* part_o;                                   // [T * n_q, splits, d]
  float* part_ml;                                  // [T * n_q, splits, 2]: maximum (-inf: nothing is seen) and sum of a share
  int splits, cluster, row_tiles;                  // cluster: the shares of a row tile are a cluster's blocks, which join them; else 1
};

// Four neighbouring numbers of a row in shared memory, in 32 bits.
__device__ __forceinline__ float4 tg_four(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 tg_four(const bf16* p) {
  const uint2 u = *(const uint2*)p;
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
}

// 16 bytes into shared memory, without waiting; zeros where nothing is to be read.
__device__ __forceinline__ void tg_copy16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Keys and values of a tile into shared memory; rows that are not there and the columns behind d are zeros.
template <typename T, int D, int KS, int THREADS>
__device__ __forceinline__ void tg_load_tile(const TreeParams& P, const long long* krow, T* ks, T* vs, bool wide, int tid) {
  const T* kc = (const T*)P.k_cache;
  const T* vc = (const T*)P.v_cache;
  constexpr int E = 16 / (int)sizeof(T), PIECES = D / E;
  if (wide) {
#pragma unroll
    for (int e = tid; e < TG_KEYS * PIECES; e += THREADS) {
      const int r = e / PIECES, j = e % PIECES * E;
      const long long at = krow[r];
      const bool there = at >= 0 && j < P.d;
      const size_t from = there ? (size_t)at * P.d + j : 0;
      tg_copy16(ks + r * KS + j, kc + from, there);
      tg_copy16(vs + r * D + j, vc + from, there);
    }
  } else {                                         // rows that do not begin at 16 bytes
    for (int e = tid; e < TG_KEYS * D; e += THREADS) {
      const int r = e / D, j = e % D;
      const long long at = krow[r];
      const bool there = at >= 0 && j < P.d;
      ks[r * KS + j] = there ? kc[at * P.d + j] : from_f32<T>(0.f);
      vs[r * D + j] = there ? vc[at * P.d + j] : from_f32<T>(0.f);
    }
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

template <typename T, int D, int GROUPS, int SHARES>
constexpr size_t tg_smem_bytes() {
  using C = Tg<GROUPS, SHARES>;
  const size_t tile = TG_KEYS * (D + 16 / sizeof(T) + D) * sizeof(T), results = SHARES * C::ROWS * (D + 4) * sizeof(float);
  return (size_t)(C::ROWS * (D + 4) + GROUPS * SHARES * 16 * C::PS) * sizeof(float) + (tile > results ? tile : results);
}

// Two products and sums at once, each rounded like fmaf.
__device__ __forceinline__ void tg_fma2(float2& acc, const float2 a, const float2 b) {
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%0, %1};\n\tfma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}" : "+f"(acc.x), "+f"(acc.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

template <typename T, int D, int GROUPS, int SHARES>
__global__ void __launch_bounds__(32 * GROUPS * SHARES)
tree_attention_kernel(const TreeParams P, const TreeShares H) {
  using Y = Tg<GROUPS, SHARES>;
  constexpr int ROWS = Y::ROWS, THREADS = Y::THREADS, MINE = Y::MINE, PS = Y::PS;
  constexpr int S = D + 4, C = D / 32, U = MINE / 8;             // row stride of the queries; groups of four output numbers a thread has
  constexpr int KS = D + 16 / (int)sizeof(T);         // row stride of the keys
  extern __shared__ __align__(16) float tg_smem[];
  float* qs = tg_smem;                             // [ROWS][S]
  float* ps = qs + ROWS * S;                       // per warp [16][PS]
  T* ks = (T*)(ps + GROUPS * SHARES * 16 * PS);               // [TG_KEYS][KS]
  T* vs = ks + TG_KEYS * KS;                       // [TG_KEYS][D]
  __shared__ long long krow[TG_KEYS], qrow[32];
  __shared__ float ml_s[2][SHARES][ROWS], factor[ROWS][8 * SHARES];
  __shared__ uint32_t seen[2][2][32];   // a warp may be at work on the tile before when the next one's are found
  pdl_wait();
  int b = blockIdx.x;
  const int split = b % H.splits; b /= H.splits;
  const int g = b % P.n_kv; b /= P.n_kv;
  const int rt = b % H.row_tiles, seq = b / H.row_tiles;
  const TreeRequest R = tree_request(P, seq);
  const int G = P.group, d = P.d, rows = R.n * G, row0 = rt * ROWS;
  if (row0 >= rows) return;
  const int nrows = min(ROWS, rows - row0);
  const int* table = P.block_table + (size_t)seq * P.max_pages;
  const int tid = threadIdx.x, lane = tid & 31, rw = (tid >> 5) % GROUPS, kw = (tid >> 5) / GROUPS;
  const int lr = lane >> 3, lc = lane & 7;         // rows 16 rw + lr + 4 i; keys MINE kw + lc + 8 u; columns 4 lc + 32 c

  // the first cached key that any of the rows sees
  int key_lo = 0;
  if (P.window > 0) {
    int first = 0x7fffffff;
    for (int r = 0; r < nrows; r += G) first = min(first, P.positions[R.tok0 + (row0 + r) / G]);
    first = min(first, P.positions[R.tok0 + (row0 + nrows - 1) / G]);
    key_lo = max(0, min(first - P.window + 1, R.base));
  }
  const int key_end = R.base + R.n;
  const int tile0 = key_lo / TG_KEYS, tiles = (key_end + TG_KEYS - 1) / TG_KEYS - tile0;
  // the last share, whose tiles masks cut, is no longer than the others
  const int begin = tile0 + (int)(((long long)tiles * split + H.splits - 1) / H.splits);
  const int end = tile0 + (int)(((long long)tiles * (split + 1) + H.splits - 1) / H.splits);
  // what threads r and r + 32 know of row r; rows that are none see every key, so that they cut no tile
  const int my_t = tid < TG_KEYS && lane < nrows ? R.tok0 + (row0 + lane) / G : -1;
  const int my_lo = my_t >= 0 && P.window > 0 ? max(0, P.positions[my_t] - P.window + 1) : 0;
  // Table entries are read a tile before the rows they lead to.
  int pidx = 0;                                    // of this thread's key in the next tile
  auto entry = [&](int tile) {
    const int key = tile * TG_KEYS + tid;
    if (tid >= TG_KEYS || tile >= end || key < key_lo || key >= key_end) return -1;
    pidx = key / P.page_size;
    return pidx < P.max_pages ? table[pidx] : -1;
  };
  auto find = [&](int tile, int page) {            // a tile's rows, and which of them are seen
    if (tid < TG_KEYS) {
      const int key = tile * TG_KEYS + tid;
      long long at = -1;
      if (key >= key_lo && key < key_end) {
        if (page >= 0 && page < P.num_pages) at = ((long long)page * P.n_kv + g) * P.page_size + (key - pidx * P.page_size);
        else report_error(P.err, PHOTON_DEV_BAD_PAGE, R.tok0, key, page);
      }
      krow[tid] = at;
      const unsigned there = __ballot_sync(0xffffffffu, at >= 0);
      seen[tile & 1][tid >> 5][lane] = my_t >= 0 ? tree_visible32(P, R, my_t, key - lane, my_lo) & there : there;
    }
  };
  int page = entry(begin);
  if (tid < 32) qrow[tid] = tid < nrows ? (long long)my_t * P.q_stride + (long long)(g * G + row0 + tid - (my_t - R.tok0) * G) * d : -1;
  __syncthreads();
  const T* q = (const T*)P.q;
  if (d % 4 == 0 && P.q_stride % 4 == 0 && (uintptr_t)q % (4 * sizeof(T)) == 0) {
#pragma unroll 8
    for (int e = tid; e < ROWS * (D / 4); e += THREADS) {
      const int r = e / (D / 4), j = e % (D / 4) * 4;
      const long long at = qrow[r];
      *(float4*)(qs + r * S + j) = at >= 0 && j < d ? tg_four(q + at + j) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
#pragma unroll 8
    for (int e = tid; e < ROWS * D; e += THREADS) {
      const int r = e / D, j = e % D;
      const long long at = qrow[r];
      qs[r * S + j] = at >= 0 && j < d ? to_f32(q[at + j]) : 0.f;
    }
  }

  float m[4], l[4];                                // l: of this thread's keys
  float2 o[4][C * 2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < C * 2; ++j) o[i][j] = make_float2(0.f, 0.f);
  }
  const float* my_q = qs + (16 * rw + lr) * S;
  const T* my_k = ks + (MINE * kw + lc) * KS;
  const T* my_v = vs + MINE * kw * D + lc * 4;
  float* my_p = ps + (tid >> 5) * 16 * PS;
  const bool wide = (size_t)d * sizeof(T) % 16 == 0 && ((((uintptr_t)P.k_cache | (uintptr_t)P.v_cache) & 15) == 0);
  for (int tile = begin; tile < end; ++tile) {
    find(tile, page);
    page = entry(tile + 1);
    __syncthreads();                               // the rows are known; the tile before is read
    tg_load_tile<T, D, KS, THREADS>(P, krow, ks, vs, wide, tid);
    __syncthreads();
    constexpr uint32_t KEYS = MINE < 32 ? (1u << (MINE & 31)) - 1u : 0xffffffffu;
    uint32_t see[4], all = 0xffffffffu, any = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      see[i] = seen[tile & 1][MINE * kw >> 5][16 * rw + lr + 4 * i] >> (MINE * kw & 31);
      all &= see[i] | ~KEYS;
      any |= see[i] & KEYS;
    }
    if (16 * rw >= nrows || !__any_sync(0xffffffffu, any != 0)) continue;            // none of the warp's rows sees one of its keys
    float2 s[4][U];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int u = 0; u < U; ++u) s[i][u] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < D; j += 4) {
      float4 k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) k[u] = tg_four(my_k + u * 8 * KS + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 a = *(const float4*)(my_q + i * 4 * S + j);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          tg_fma2(s[i][u], make_float2(a.x, a.y), make_float2(k[u].x, k[u].y));
          tg_fma2(s[i][u], make_float2(a.z, a.w), make_float2(k[u].z, k[u].w));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[U], mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = (s[i][u].x + s[i][u].y) * P.scale;
        if (P.softcap > 0.f) x[u] = P.softcap * tanhf(x[u] / P.softcap);
        x[u] = (see[i] >> (lc + 8 * u)) & 1u ? x[u] : -INFINITY;
        mx = fmaxf(mx, x[u]);
      }
#pragma unroll
      for (int w = 4; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx), sub = mn == -INFINITY ? 0.f : mn;
      const float keep = expf(m[i] - sub);         // e^-inf = 0 before the first key
      m[i] = mn;
      l[i] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = expf(x[u] - sub);
        l[i] += p;
        my_p[(lr + 4 * i) * PS + lc + 8 * u] = p;
      }
#pragma unroll
      for (int j = 0; j < C * 2; ++j) { o[i][j].x *= keep; o[i][j].y *= keep; }
    }
    __syncwarp();
    // A mask cuts: is there a value that a weight of 0 must not meet?
    bool odd = false;
    if (__any_sync(0xffffffffu, all != 0xffffffffu)) {
      for (int e = lane; e < MINE * (D / 4); e += 32) {
        const float4 v = tg_four(vs + MINE * kw * D + e * 4);
        odd |= !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w));
      }
    }
    if (__any_sync(0xffffffffu, odd)) {
      for (int k = 0; k < MINE; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = my_p[(lr + 4 * i) * PS + k];
          if ((see[i] >> k) & 1u) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
              const float4 v = tg_four(my_v + k * D + c * 32);
              tg_fma2(o[i][2 * c], make_float2(p, p), make_float2(v.x, v.y));
              tg_fma2(o[i][2 * c + 1], make_float2(p, p), make_float2(v.z, v.w));
            }
          }
        }
      }
    } else {
#pragma unroll 2
      for (int k = 0; k < MINE; k += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *(const float4*)(my_p + (lr + 4 * i) * PS + k);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float4 v = tg_four(my_v + (k + u) * D + c * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
              tg_fma2(o[i][2 * c], make_float2(w, w), make_float2(v.x, v.y));
              tg_fma2(o[i][2 * c + 1], make_float2(w, w), make_float2(v.z, v.w));
            }
          }
        }
      }
    }
    __syncwarp();
  }
  pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int w = 4; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);

  // The warps of a row's keys, and the blocks of a cluster, leave their results where the tiles were.
  float* po = (float*)ks;                          // [SHARES][ROWS][S]
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 16 * rw + lr + 4 * i;
#pragma unroll
    for (int c = 0; c < C; ++c)
      *(float4*)(po + (kw * ROWS + r) * S + c * 32 + lc * 4) = make_float4(o[i][2 * c].x, o[i][2 * c].y, o[i][2 * c + 1].x, o[i][2 * c + 1].y);
    if (lc == 0) { ml_s[0][kw][r] = m[i]; ml_s[1][kw][r] = l[i]; }
  }
  const int rank = H.cluster > 1 ? split : 0;
  if (H.cluster > 1) tree_cluster_sync();
  else __syncthreads();
  const bool last = H.cluster == H.splits;         // else: a share of several
  // Each result's factor: 2 SHARES threads a row, four results each.
  {
    constexpr int W = 2 * SHARES;
    const int r = tid / W, n = SHARES * H.cluster;
    float mx[4], l4[4], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int w = tid % W + W * u;
      mx[u] = w < n ? tree_peer(&ml_s[0][w % SHARES][r], w / SHARES) : -INFINITY;
      l4[u] = w < n ? tree_peer(&ml_s[1][w % SHARES][r], w / SHARES) : 0.f;
      top = fmaxf(top, mx[u]);
    }
#pragma unroll
    for (int w = W / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float sink = last && P.sinks && r < nrows ? P.sinks[g * G + (row0 + r) % G] : -INFINITY;
    const float most = fmaxf(top, sink), sub = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool none = tree_nothing(mx[u], l4[u]);
      mx[u] = expf(mx[u] - sub);                   // 0 for what is not there
      sum += l4[u] * mx[u];
      l4[u] = none ? TREE_NOTHING : 0.f;
    }
#pragma unroll
    for (int w = W / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    const float total = sum + (sink == -INFINITY ? 0.f : expf(sink - sub)), inv = !last ? 1.f : sum != 0.f ? 1.f / total : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (tid % W + W * u < n) factor[r][tid % W + W * u] = l4[u] == TREE_NOTHING ? TREE_NOTHING : mx[u] * inv;
    if (!last && tid % W == 0 && r < nrows) {
      const size_t slot = ((size_t)(R.tok0 + (row0 + r) / G) * P.n_q + g * G + (row0 + r) % G) * H.splits + split;
      H.part_ml[slot * 2] = top; H.part_ml[slot * 2 + 1] = sum;         // -inf: a share that the row sees nothing of
    }
  }
  __syncthreads();
  const int fours = nrows * (D / 4), stop = fours * (rank + 1) / H.cluster;
  for (int e = fours * rank / H.cluster + tid; e < stop; e += THREADS) {
    const int r = e / (D / 4), j = e % (D / 4) * 4, row = row0 + r, t = R.tok0 + row / G, head = g * G + row % G;
    if (j >= d) continue;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < H.cluster; ++c) {
#pragma unroll
      for (int k = 0; k < SHARES; ++k) {
        const float w = factor[r][SHARES * c + k];
        const float4 x = tree_peer4(po + (k * ROWS + r) * S + j, c);
        if (!(w < 0.f)) { a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y); a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w); }
      }
    }
    const float v[4] = {a.x, a.y, a.z, a.w};
    if (last) {
      T* dst = (T*)P.out + (size_t)t * P.out_stride + (size_t)head * d + j;
#pragma unroll
      for (int u = 0; u < 4; ++u) if (j + u < d) dst[u] = from_f32<T>(v[u]);
    } else {
      float* dst = H.part_o + (((size_t)t * P.n_q + head) * H.splits + split) * d + j;
#pragma unroll
      for (int u = 0; u < 4; ++u) if (j + u < d) dst[u] = v[u];
    }
  }
  if (H.cluster > 1) tree_cluster_sync();          // the others have read this block's results
}

// Joins the shares of a row in their order: a warp a row.
template <typename T>
__global__ void __launch_bounds__(128)
tree_join_kernel(const TreeParams P, const TreeShares H) {
  pdl_wait();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= P.T * P.n_q || row / P.n_q < P.cu_tokens[0] || row / P.n_q >= P.cu_tokens[P.S]) return;   // rows of no request
  const float* ml = H.part_ml + (size_t)row * H.splits * 2;
  const float* po = H.part_o + (size_t)row * H.splits * P.d;
  const int head = row % P.n_q;
  const float sink = P.sinks ? P.sinks[head] : -INFINITY;
  float top = sink;
  for (int s = 0; s < H.splits; ++s) top = fmaxf(top, ml[2 * s]);
  const float sub = top == -INFINITY ? 0.f : top;
  float total = 0.f;
  for (int s = 0; s < H.splits; ++s) total += ml[2 * s + 1] * expf(ml[2 * s] - sub);
  if (P.sinks) total += expf(sink - sub);
  const float inv = total != 0.f ? 1.f / total : 0.f;
  T* dst = (T*)P.out + (size_t)(row / P.n_q) * P.out_stride + (size_t)head * P.d;
  for (int j = lane; j < P.d; j += 32) {
    float a = 0.f;
    for (int s = 0; s < H.splits; ++s) {
      const float w = expf(ml[2 * s] - sub);
      if (!tree_nothing(ml[2 * s], ml[2 * s + 1])) a = fmaf(w, po[(size_t)s * P.d + j], a);
    }
    dst[j] = from_f32<T>(a * inv);
  }
}

template <typename T, int D, int GROUPS, int SHARES>
static int tree_launch(const TreeParams& P, const TreeShares& H, long blocks, cudaStream_t stream) {
  constexpr int THREADS = Tg<GROUPS, SHARES>::THREADS;
  const size_t smem = tg_smem_bytes<T, D, GROUPS, SHARES>();
  static bool ready[64] = {};                      // the limit is set once a device
  const int set = tree_smem_limit((const void*)tree_attention_kernel<T, D, GROUPS, SHARES>, (int)smem, ready);
  if (set != 0) return set;
  if (H.cluster > 1) return tree_launch_clusters(tree_attention_kernel<T, D, GROUPS, SHARES>, blocks, H.cluster, THREADS, smem, stream, P, H);
  const int st = launch_pdl(tree_attention_kernel<T, D, GROUPS, SHARES>, dim3((unsigned)blocks), dim3(THREADS), smem, stream, P, H);
  if (st != 0 || H.splits == 1) return st;
  return launch_pdl(tree_join_kernel<T>, dim3((unsigned)(((long)P.T * P.n_q + 3) / 4)), dim3(128), 0, stream, P, H);
}

template <typename T>
static int tree_choose(const TreeParams& P, TreeShares& H, cudaStream_t stream) {
  const long rows = (long)P.max_tokens * P.group;
  H.row_tiles = (int)((rows + 31) / 32);
  const long blocks = (long)P.S * H.row_tiles * P.n_kv * H.splits;
  if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  // Four warps a block, so that several blocks share an SM; eight where every block has an SM to itself (32-bit, four and eight warps, us: 1 request of 8 x 4 rows behind
  // 640 keys 17.2 and 16.0; 8 of 32 x 4 behind up to 2,000: 104 and 116).  Up to 16 rows: no warps for others (3 of 4 x 4 behind up to 187, heads of 128: 25.4
  // with half of four warps idle, 17.6 with eight at work; 8 of 4 x 4 behind up to 2,000: 67 and, with four at work, 58).
  const bool alone = blocks <= photon_sm_count();
  auto launch = [&](auto head) {
    constexpr int D = decltype(head)::value;
    if (rows <= 16) return alone ? tree_launch<T, D, 1, 8>(P, H, blocks, stream) : tree_launch<T, D, 1, 4>(P, H, blocks, stream);
    return alone ? tree_launch<T, D, 2, 4>(P, H, blocks, stream) : tree_launch<T, D, 2, 2>(P, H, blocks, stream);
  };
  return P.d <= 64 ? launch(std::integral_constant<int, 64>()) : P.d <= 128 ? launch(std::integral_constant<int, 128>())
                                                                           : tree_launch<T, 256, 2, 2>(P, H, blocks, stream);
}

PHOTON_API int photon_tree_attention(const photon_tree_call* call, cudaStream_t stream) {
  if (call->S <= 0 || call->T <= 0 || call->max_tokens_per_seq <= 0) return 0;
  TreeParams P;
  const int st = tree_params(call, P);
  if (st != 0) return st;
  const long rows = (long)P.T * P.n_q * call->parts;
  const bool clusters = call->parts > 1 && call->parts <= 8;
  if (call->parts > 1 && !clusters && (call->scratch == nullptr || call->scratch_floats < rows * (P.d + 2))) return PHOTON_ERR_ARGUMENT;
  TreeShares H;
  H.part_o = call->scratch; H.part_ml = call->scratch + rows * P.d; H.splits = call->parts; H.cluster = clusters ? call->parts : 1;
  return call->dtype == PHOTON_F32 ? tree_choose<float>(P, H, stream) : tree_choose<bf16>(P, H, stream);
}
