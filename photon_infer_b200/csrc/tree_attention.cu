// Attention for trees of drafted tokens over a paged cache, for either type and heads of up to 256 numbers.
//
//   out[t, h] = sum_j w_j v_j / (sum_j w_j + e^(sink_h - m)),  w_j = e^(x_j - m),  x_j = scale q[t, h] . k_j
//
// (bounded scores: x_j = softcap tanh(scale q . k_j / softcap); m the largest of the scores and the sink) over the keys that node t sees
// (tree_attention.cuh); a row that sees nothing is zero.  Scores, weights, sums and outputs are held in 32 bits.
//
// A block takes 32 rows, (node, query head) pairs that share a key/value head, and a share of the request's keys, in tiles of 32.  A thread holds the scores
// of four rows with two keys, then the outputs of those rows for D / 16 numbers; its rows' other scores lie with the 15 threads beside it, so
// maxima and sums are butterflies inside half a warp and the weights pass through shared memory between the lanes of one warp.
// Shares are joined in their order by a second kernel.
//
// A key that a row does not see has weight 0, and 0 times a value that is not finite would not be: in tiles where masks cut, products with a weight of 0
// are left out, and rows behind the last key or of a missing page are zeros.
#include "tree_attention.cuh"
#include <math.h>

#define TG_ROWS 32
#define TG_KEYS 32
#define TG_THREADS 128
#define TG_PS (TG_KEYS + 4)

struct TreeShares {
  float* part_o;                                   // [T * n_q, splits, d]
  float* part_ml;                                  // [T * n_q, splits, 2]: maximum and sum of a share
  int splits, row_tiles;
};

template <typename T, int D>
__global__ void __launch_bounds__(TG_THREADS)
tree_attention_kernel(const TreeParams P, const TreeShares H) {
  constexpr int S = D + 4, C4 = D / 64;            // row stride in shared memory; groups of four output numbers a thread has
  extern __shared__ __align__(16) float tg_smem[];
  float* qs = tg_smem;                             // [TG_ROWS][S]
  float* ks = qs + TG_ROWS * S;                    // [TG_KEYS][S]
  float* vs = ks + TG_KEYS * S;                    // [TG_KEYS][D]
  float* ps = vs + TG_KEYS * D;                    // [TG_ROWS][TG_PS]
  __shared__ long long krow[TG_KEYS];
  __shared__ uint32_t seen[TG_ROWS];
  pdl_wait();
  int b = blockIdx.x;
  const int split = b % H.splits; b /= H.splits;
  const int g = b % P.n_kv; b /= P.n_kv;
  const int rt = b % H.row_tiles, seq = b / H.row_tiles;
  const TreeRequest R = tree_request(P, seq);
  const int G = P.group, d = P.d, rows = R.n * G, row0 = rt * TG_ROWS;
  if (row0 >= rows) return;
  const int nrows = min(TG_ROWS, rows - row0);
  const int* table = P.block_table + (size_t)seq * P.max_pages;
  const int tid = threadIdx.x, tr = tid >> 4, tc = tid & 15;     // rows tr + 8 i; keys tc, tc + 16; columns 4 tc + 64 j

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
  const int per = (tiles + H.splits - 1) / H.splits;
  const int begin = tile0 + split * per, end = min(tile0 + tiles, begin + per);

  const T* q = (const T*)P.q;
  for (int e = tid; e < TG_ROWS * D; e += TG_THREADS) {
    const int r = e / D, j = e % D, row = row0 + r;
    qs[r * S + j] = r < nrows && j < d ? to_f32(q[(size_t)(R.tok0 + row / G) * P.q_stride + (size_t)(g * G + row % G) * d + j]) : 0.f;
  }
  // what thread r < 32 knows of row r
  const int my_t = tid < nrows ? R.tok0 + (row0 + tid) / G : -1;
  const int my_lo = my_t >= 0 && P.window > 0 ? max(0, P.positions[my_t] - P.window + 1) : 0;

  float m[4], l[4], o[4][C4 * 4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < C4 * 4; ++j) o[i][j] = 0.f;
  }
  const T* kc = (const T*)P.k_cache;
  const T* vc = (const T*)P.v_cache;
  for (int tile = begin; tile < end; ++tile) {
    const int key0 = tile * TG_KEYS;
    __syncthreads();                               // the tile before is read
    if (tid < TG_KEYS) {
      const int key = key0 + tid;
      const long long at = key < key_end && key >= key_lo ? tree_row(P, table, g, key, R.tok0) : -1;
      krow[tid] = at;
      const unsigned there = __ballot_sync(0xffffffffu, at >= 0);
      seen[tid] = my_t >= 0 ? tree_visible32(P, R, my_t, key0, my_lo) & there : 0u;
    }
    __syncthreads();
    for (int e = tid; e < TG_KEYS * D; e += TG_THREADS) {
      const int r = e / D, j = e % D;
      const long long at = krow[r];
      const bool ok = at >= 0 && j < d;
      ks[r * S + j] = ok ? to_f32(kc[at * d + j]) : 0.f;
      vs[r * D + j] = ok ? to_f32(vc[at * d + j]) : 0.f;
    }
    __syncthreads();
    float s[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = 0.f;
#pragma unroll 4
    for (int j = 0; j < D; j += 4) {
      const float4 k0 = *(const float4*)(ks + tc * S + j), k1 = *(const float4*)(ks + (tc + 16) * S + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 a = *(const float4*)(qs + (tr + 8 * i) * S + j);
        s[i][0] = fmaf(a.x, k0.x, s[i][0]); s[i][0] = fmaf(a.y, k0.y, s[i][0]);
        s[i][0] = fmaf(a.z, k0.z, s[i][0]); s[i][0] = fmaf(a.w, k0.w, s[i][0]);
        s[i][1] = fmaf(a.x, k1.x, s[i][1]); s[i][1] = fmaf(a.y, k1.y, s[i][1]);
        s[i][1] = fmaf(a.z, k1.z, s[i][1]); s[i][1] = fmaf(a.w, k1.w, s[i][1]);
      }
    }
    bool cut = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t see = seen[tr + 8 * i];
      cut |= see != 0xffffffffu;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float x = s[i][u] * P.scale;
        if (P.softcap > 0.f) x = P.softcap * tanhf(x / P.softcap);
        s[i][u] = (see >> (tc + 16 * u)) & 1u ? x : -INFINITY;
      }
      float mx = fmaxf(s[i][0], s[i][1]);
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx), sub = mn == -INFINITY ? 0.f : mn;
      const float keep = expf(m[i] - sub);         // e^-inf = 0 before the first key
      const float p0 = expf(s[i][0] - sub), p1 = expf(s[i][1] - sub);
      float sum = p0 + p1;
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      m[i] = mn;
      l[i] = l[i] * keep + sum;
#pragma unroll
      for (int j = 0; j < C4 * 4; ++j) o[i][j] *= keep;
      ps[(tr + 8 * i) * TG_PS + tc] = p0;
      ps[(tr + 8 * i) * TG_PS + tc + 16] = p1;
    }
    __syncwarp();                                  // a row's weights come from the lanes of this warp
    if (cut) {
      for (int k = 0; k < TG_KEYS; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = ps[(tr + 8 * i) * TG_PS + k];
          if (p != 0.f) {                          // a NaN is not 0
#pragma unroll
            for (int c = 0; c < C4; ++c) {
              const float4 v = *(const float4*)(vs + k * D + c * 64 + tc * 4);
              o[i][c * 4] = fmaf(p, v.x, o[i][c * 4]); o[i][c * 4 + 1] = fmaf(p, v.y, o[i][c * 4 + 1]);
              o[i][c * 4 + 2] = fmaf(p, v.z, o[i][c * 4 + 2]); o[i][c * 4 + 3] = fmaf(p, v.w, o[i][c * 4 + 3]);
            }
          }
        }
      }
    } else {
#pragma unroll 2
      for (int k = 0; k < TG_KEYS; k += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *(const float4*)(ps + (tr + 8 * i) * TG_PS + k);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
          for (int c = 0; c < C4; ++c) {
            const float4 v = *(const float4*)(vs + (k + u) * D + c * 64 + tc * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
              o[i][c * 4] = fmaf(w, v.x, o[i][c * 4]); o[i][c * 4 + 1] = fmaf(w, v.y, o[i][c * 4 + 1]);
              o[i][c * 4 + 2] = fmaf(w, v.z, o[i][c * 4 + 2]); o[i][c * 4 + 3] = fmaf(w, v.w, o[i][c * 4 + 3]);
            }
          }
        }
      }
    }
    __syncwarp();
  }
  pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = tr + 8 * i, row = row0 + r;
    if (r >= nrows) continue;
    const int t = R.tok0 + row / G, head = g * G + row % G;
    if (H.splits == 1) {
      float total = l[i], scale = 1.f;
      if (P.sinks) {                               // relative to the larger of the two maxima
        const float top = fmaxf(m[i], P.sinks[head]), sub = top == -INFINITY ? 0.f : top;
        scale = expf(m[i] - sub);
        total = l[i] * scale + expf(P.sinks[head] - sub);
      }
      const float inv = total != 0.f ? scale / total : 0.f;
      T* dst = (T*)P.out + (size_t)t * P.out_stride + (size_t)head * d;
#pragma unroll
      for (int c = 0; c < C4 * 4; ++c) {
        const int j = (c >> 2) * 64 + tc * 4 + (c & 3);
        if (j < d) dst[j] = from_f32<T>(l[i] != 0.f ? o[i][c] * inv : 0.f);
      }
    } else {
      const size_t slot = ((size_t)t * P.n_q + head) * H.splits + split;
#pragma unroll
      for (int c = 0; c < C4 * 4; ++c) {
        const int j = (c >> 2) * 64 + tc * 4 + (c & 3);
        if (j < d) H.part_o[slot * d + j] = o[i][c];
      }
      if (tc == 0) { H.part_ml[slot * 2] = m[i]; H.part_ml[slot * 2 + 1] = l[i]; }
    }
  }
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
  const float keys = total;
  if (P.sinks) total += expf(sink - sub);
  const float inv = total != 0.f ? 1.f / total : 0.f;
  T* dst = (T*)P.out + (size_t)(row / P.n_q) * P.out_stride + (size_t)head * P.d;
  for (int j = lane; j < P.d; j += 32) {
    float a = 0.f;
    for (int s = 0; s < H.splits; ++s) {
      const float w = expf(ml[2 * s] - sub);
      if (w != 0.f) a = fmaf(w, po[(size_t)s * P.d + j], a);
    }
    dst[j] = from_f32<T>(keys != 0.f ? a * inv : 0.f);
  }
}

template <typename T, int D>
static int tree_launch(const TreeParams& P, const TreeShares& H, long blocks, cudaStream_t stream) {
  const size_t smem = (size_t)(TG_ROWS * (D + 4) + TG_KEYS * (D + 4) + TG_KEYS * D + TG_ROWS * TG_PS) * sizeof(float);
  static bool ready[64] = {};                      // the limit is set once a device
  const int set = tree_smem_limit((const void*)tree_attention_kernel<T, D>, (int)smem, ready);
  if (set != 0) return set;
  int st = launch_pdl(tree_attention_kernel<T, D>, dim3((unsigned)blocks), dim3(TG_THREADS), smem, stream, P, H);
  if (st != 0 || H.splits == 1) return st;
  return launch_pdl(tree_join_kernel<T>, dim3((unsigned)(((long)P.T * P.n_q + 3) / 4)), dim3(128), 0, stream, P, H);
}

PHOTON_API int photon_tree_attention(const photon_tree_call* call, cudaStream_t stream) {
  if (call->S <= 0 || call->T <= 0 || call->max_tokens_per_seq <= 0) return 0;
  TreeParams P;
  const int st = tree_params(call, P);
  if (st != 0) return st;
  const long rows = (long)P.T * P.n_q * call->parts;
  if (call->parts > 1 && (call->scratch == nullptr || call->scratch_floats < rows * (P.d + 2))) return PHOTON_ERR_ARGUMENT;
  TreeShares H;
  H.part_o = call->scratch; H.part_ml = call->scratch + rows * P.d; H.splits = call->parts;
  H.row_tiles = (int)(((long)P.max_tokens * P.group + TG_ROWS - 1) / TG_ROWS);
  const long blocks = (long)P.S * H.row_tiles * P.n_kv * H.splits;
  if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  if (call->dtype == PHOTON_F32)
    return P.d <= 64 ? tree_launch<float, 64>(P, H, blocks, stream) : P.d <= 128 ? tree_launch<float, 128>(P, H, blocks, stream)
                                                                                : tree_launch<float, 256>(P, H, blocks, stream);
  return P.d <= 64 ? tree_launch<bf16, 64>(P, H, blocks, stream) : P.d <= 128 ? tree_launch<bf16, 128>(P, H, blocks, stream)
                                                                              : tree_launch<bf16, 256>(P, H, blocks, stream);
}
