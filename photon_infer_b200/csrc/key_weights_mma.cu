// What each cached key got of the softmax of a request's query rows (key_weights.cu) on the tensor cores: bfloat16 queries, heads of 64 or 128, a plain bfloat16 cache or one in
// 4 bits (kv4.cuh), whose numbers bfloat16 holds exactly.
//
// A block has 128 keys of a request and head in shared memory, the cache's own rows or what their codes stand for, and up to 128 rows (tokens x query heads of the key/value
// head) at a time, 16 for a warp; with fewer rows the warps share the keys out too.  The keys are the first operand: a score's row is a key, so what is not finite stays
// with its key, and a key's sum over the rows lies in the lanes of one row.  Every key is one block's: no atomics, the same bits every time.
// Without the rows' logarithms a first kernel leaves each 128 keys' maxima and sums, a second one joins them, and then the keys are read again.
#include "kv4.cuh"
#include <math.h>

#define KX_KEYS 128
#define KX_THREADS 256
#define KX_WARPS 8
#define KX_ROWS 128              // query rows in shared memory at a time, at most

struct KeyWeightsMmaArgs {
  const bf16* q; float* weights; const void* k; const int* table; const int* cu_tokens; const int* context_lens; const int* held; const float* sinks; const float* lse;
  float* scratch; int* err;
  long q_stride;
  int max_pages, S, n_q, n_kv, page_size, num_pages, window, parts;
  int room;                      // for query rows: a multiple of 16
  float scale, softcap;
};

__device__ __forceinline__ float kx_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void kx_matrices(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void kx_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t kx_scaled(uint32_t word, int shift, __nv_bfloat162 scale) {      // codes at `shift` and 16 bits behind it, as numbers
  const uint32_t x = (word >> shift & 0x000F000Fu) | 0x43004300u;                                     // 128 + c
  const __nv_bfloat162 y = __hmul2(__hsub2(*(const __nv_bfloat162*)&x, __float2bfloat162_rn(136.f)), scale);
  return *(const uint32_t*)&y;
}

// FINAL: the weights; else the maxima and sums of the block's keys.
template <int D, bool PACKED, bool FINAL>
__global__ void __launch_bounds__(KX_THREADS, 2)
key_weights_mma_kernel(const KeyWeightsMmaArgs a) {
  constexpr int PITCH = 2 * D + 16, GROUPS = D / 32, STEPS = D / 16;
  extern __shared__ __align__(16) uint8_t kx_smem[];
  uint8_t* k_s = kx_smem;                             // [KX_KEYS] rows
  uint8_t* q_s = k_s + KX_KEYS * PITCH;               // [room] rows
  __shared__ float sum_s[KX_WARPS][KX_KEYS], lse_s[KX_ROWS], ml_s[KX_WARPS][16][2];
  __shared__ uint32_t there_s[4];                     // keys that are there
  __shared__ int slot_s[KX_KEYS];
  __shared__ long page_s[KX_KEYS];                    // page and head
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y, key0 = blockIdx.x * KX_KEYS;
  const int ctx = a.context_lens[seq];
  if (key0 >= ctx) return;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, G = a.n_q / a.n_kv, rows = n * G, base = ctx - n, last_place = ctx - 1;
  if (n <= 0) return;
  const int known = a.held != nullptr ? a.held[seq] : base, keys = min(KX_KEYS, ctx - key0);
  const bool unseen = a.window > 0 && key0 + keys - 1 <= base - a.window;      // by any row
  if (unseen && (!FINAL || key0 + keys <= known)) {
    if (!FINAL) {
      for (int r = tid; r < rows; r += KX_THREADS) {
        float* to = a.scratch + ((long)(first + r / G) * a.n_q + head * G + r % G) * a.parts * 2 + 2 * blockIdx.x;
        to[0] = -INFINITY;
        to[1] = 0.f;
      }
    }
    return;
  }
  // ---- the first threads' keys: their places, their sums so far
  int page = -1, slot = 0;
  float before = 0.f;
  if (tid < KX_KEYS) {
    const int mine = key0 + tid, pidx = mine / a.page_size;
    slot = mine - pidx * a.page_size;
    if (mine < ctx) {
      page = pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1;
      if (page < 0 || page >= a.num_pages) {
        if (FINAL) report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, mine, page);
        page = -1;
      }
    }
    const uint32_t votes = __ballot_sync(0xffffffffu, page >= 0);
    if (lane == 0) there_s[warp] = votes;
    page_s[tid] = (long)max(page, 0) * a.n_kv + head;  // some page of the pool where it is not there: what is read is not used
    slot_s[tid] = slot;
    if (FINAL && page >= 0 && mine < known) before = a.weights[page_s[tid] * a.page_size + slot];
  }
  const bool all_there = __syncthreads_and(tid >= KX_KEYS || page >= 0);      // of 128 keys
  if constexpr (PACKED) {
    // 16 bytes of a row's codes at a time: words t GROUPS + j
    constexpr int PIECES = D / 32, EACH = KX_KEYS * PIECES / KX_THREADS;
    uint4 u[EACH];
    uint32_t scales[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int x = i * KX_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
      const uint8_t* at = (const uint8_t*)a.k + page_s[key] * kv4_page_bytes(a.page_size, D);
      const uint8_t* sc = at + (long)a.page_size * (D / 2) + slot_s[key] * GROUPS;
      u[i] = *(const uint4*)(at + (long)slot_s[key] * (D / 2) + 16 * piece);
      scales[i] = GROUPS == 4 ? *(const uint32_t*)sc : *(const uint16_t*)sc;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int x = i * KX_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int word = 4 * piece + c, tt = word / GROUPS, j = word - tt * GROUPS;
        const __nv_bfloat162 s = __float2bfloat162_rn(kv4_scale(scales[i] >> (8 * j) & 255u));
        // numbers 0 and 4, 1 and 5, 2 and 6, 3 and 7
        const uint32_t y0 = kx_scaled(w[c], 0, s), y1 = kx_scaled(w[c], 4, s), y2 = kx_scaled(w[c], 8, s), y3 = kx_scaled(w[c], 12, s);
        *(uint4*)(k_s + key * PITCH + 64 * j + 16 * tt) =
            make_uint4(__byte_perm(y0, y1, 0x5410), __byte_perm(y2, y3, 0x5410), __byte_perm(y0, y1, 0x7632), __byte_perm(y2, y3, 0x7632));
      }
    }
  } else {
    constexpr int PIECES = D / 8;                     // of 16 bytes
#pragma unroll
    for (int i = 0; i < KX_KEYS * PIECES / KX_THREADS; ++i) {
      const int x = i * KX_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
      const long at = page_s[key] * a.page_size + slot_s[key];
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(k_s + key * PITCH + 16 * piece)), "l"((const bf16*)a.k + at * D + 8 * piece)
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  if (FINAL) for (int i = tid; i < KX_WARPS * KX_KEYS; i += KX_THREADS) sum_s[i / KX_KEYS][i % KX_KEYS] = 0.f;
  // warps by rows and by keys
  const int some = min(rows, a.room), wr = some > 64 ? 8 : some > 32 ? 4 : some > 16 ? 2 : 1, wk = KX_WARPS / wr, my_r = warp % wr, my_k = warp / wr;
  const float scale2 = a.scale * 1.4426950408889634f, cap_in = 2.f * 1.4426950408889634f * a.scale / a.softcap, cap_out = a.softcap * 1.4426950408889634f;
  const bool clear = all_there && key0 + KX_KEYS - 1 <= base && (a.window <= 0 || key0 > last_place - a.window);      // all rows see all keys
  const uint32_t k_at = (uint32_t)__cvta_generic_to_shared(k_s) + (lane & 15) * PITCH + (lane >> 4) * 16;
  const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(q_s) + (my_r * 16 + (lane & 7) + (lane >> 4) * 8) * PITCH + (lane >> 3 & 1) * 16;
  for (int r0 = 0; r0 < rows; r0 += a.room) {
    const int now = min(a.room, rows - r0);
    __syncthreads();                                  // the rows in front of these are done with
    for (int x = tid; x < (now + 15) / 16 * 16 * (D / 8); x += KX_THREADS) {
      const int r = x / (D / 8), piece = x - r * (D / 8), row = r0 + r;
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows) u = *(const uint4*)(a.q + (first + row / G) * a.q_stride + (long)(head * G + row % G) * D + 8 * piece);
      *(uint4*)(q_s + r * PITCH + 16 * piece) = u;
    }
    if (FINAL && tid < KX_ROWS) {
      const int row = r0 + tid;
      lse_s[tid] = row < rows ? a.lse[(long)(first + row / G) * a.n_q + head * G + row % G] * 1.4426950408889634f : INFINITY;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // with fewer rows than the warps have room for, some have none
    const bool busy = my_r * 16 < now, two = my_r * 16 + 8 < now;      // rows in its first eight, in its second
    uint32_t b[STEPS][4];                             // rows 0 to 7: [0], [1]; 8 to 15: [2], [3]
#pragma unroll
    for (int i = 0; i < STEPS; ++i) if (busy) kx_matrices(b[i], q_at + 32 * i);
    float ref[4], m[4], l[4];
    int at_place[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {                     // rows 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t
      const int r = my_r * 16 + (c >> 1) * 8 + 2 * t + (c & 1);
      ref[c] = FINAL && busy ? lse_s[r] : 0.f;
      at_place[c] = r0 + r < rows ? base + (r0 + r) / G : -1;
      m[c] = -INFINITY;
      l[c] = 0.f;
    }
    for (int tile = my_k; tile < KX_KEYS / 16; tile += wk) {
      if (tile * 16 >= keys || !busy) break;
      float d[2][4] = {};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        uint32_t k4[4];
        kx_matrices(k4, k_at + tile * 16 * PITCH + 32 * i);
        kx_mma(d[0], k4, b[i][0], b[i][1]);
        if (two) kx_mma(d[1], k4, b[i][2], b[i][3]);
      }
      float x[4][2];                                  // rows as above, keys g and 8 + g
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float y = d[c >> 1][2 * h + (c & 1)];
          x[c][h] = a.softcap > 0.f ? cap_out * (1.f - __fdividef(2.f, 1.f + kx_exp2(y * cap_in))) : y * scale2;
        }
      if (!clear) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = tile * 16 + 8 * h + g, key = key0 + k;
          const bool there = there_s[k >> 5] >> (k & 31) & 1u;
#pragma unroll
          for (int c = 0; c < 4; ++c) if (!(there && key <= at_place[c] && (a.window <= 0 || key > at_place[c] - a.window))) x[c][h] = -INFINITY;
        }
      }
      if constexpr (FINAL) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float sum = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) if (c < 2 || two) sum += x[c][h] == -INFINITY ? 0.f : kx_exp2(x[c][h] - ref[c]);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (t == 0) sum_s[my_r][tile * 16 + 8 * h + g] += sum;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c >= 2 && !two) continue;
          const float top = fmaxf(m[c], fmaxf(x[c][0], x[c][1])), zero = top == -INFINITY ? 0.f : top;
          l[c] = (m[c] == -INFINITY ? l[c] : l[c] * kx_exp2(m[c] - zero)) + kx_exp2(x[c][0] - zero) + kx_exp2(x[c][1] - zero);
          m[c] = top;
        }
      }
    }
    if constexpr (!FINAL) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float top = m[c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float zero = top == -INFINITY ? 0.f : top;
        float sum = m[c] == -INFINITY ? l[c] : l[c] * kx_exp2(m[c] - zero);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (g == 0) {
          const int r = (c >> 1) * 8 + 2 * t + (c & 1);
          ml_s[warp][r][0] = top;
          ml_s[warp][r][1] = sum;
        }
      }
      __syncthreads();
      if (tid < now) {                                // the warps that share the row's keys
        const int of = tid >> 4, r = tid & 15, row = r0 + tid;
        float top = -INFINITY, sum = 0.f;
        for (int w = 0; w < wk; ++w) top = fmaxf(top, ml_s[w * wr + of][r][0]);
        const float zero = top == -INFINITY ? 0.f : top;
        for (int w = 0; w < wk; ++w) {
          const float pm = ml_s[w * wr + of][r][0], pl = ml_s[w * wr + of][r][1];
          if (pl != 0.f) sum += pm == -INFINITY ? pl : pl * exp2f(pm - zero);
        }
        float* to = a.scratch + ((long)(first + row / G) * a.n_q + head * G + row % G) * a.parts * 2 + 2 * blockIdx.x;
        to[0] = top;
        to[1] = sum;
      }
    }
  }
  if constexpr (FINAL) {
    __syncthreads();
    if (page >= 0) {
      float sum = before;
      for (int w = 0; w < wr; ++w) sum += sum_s[w][tid];
      a.weights[page_s[tid] * a.page_size + slot] = sum;
    }
  }
}

// A warp joins the maxima and sums of one (token, head).
__global__ void __launch_bounds__(128)
key_weights_lse_kernel(const KeyWeightsMmaArgs a, float* __restrict__ lse) {
  pdl_wait();
  const int seq = blockIdx.y, lane = threadIdx.x & 31, at = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, i = at / a.n_q, h = at - i * a.n_q;
  if (i >= n) return;
  const int parts = min(a.parts, (a.context_lens[seq] + KX_KEYS - 1) / KX_KEYS);
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

template <int D, bool PACKED, bool FINAL>
static int kx_launch(const KeyWeightsMmaArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr size_t most = (KX_KEYS + KX_ROWS) * (2 * D + 16);
  const size_t smem = (KX_KEYS + a.room) * (2 * D + 16);
  static bool set = false;
  if (!set) {
    cudaError_t e = cudaFuncSetAttribute(key_weights_mma_kernel<D, PACKED, FINAL>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(key_weights_mma_kernel<D, PACKED, FINAL>, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e != cudaSuccess) return (int)e;
    set = true;
  }
  return launch_pdl(key_weights_mma_kernel<D, PACKED, FINAL>, grid, dim3(KX_THREADS), smem, stream, a);
}

PHOTON_API int photon_key_weights_mma(const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_keys <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0) return PHOTON_ERR_ARGUMENT;
  if ((c->d != 64 && c->d != 128) || c->num_pages <= 0 || c->page_size <= 0 || (c->packed && !kv4_sizes_ok(c->page_size, c->d))) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)c->q | (uintptr_t)c->k_cache) % 16 || c->q_stride % 8) return PHOTON_ERR_UNSUPPORTED;
  if (c->S > 65535 || c->n_kv > 65535 || c->scale <= 0.f) return PHOTON_ERR_UNSUPPORTED;
  const int parts = (c->max_keys + KX_KEYS - 1) / KX_KEYS;
  if (c->parts != parts || (c->lse == nullptr && c->scratch == nullptr)) return PHOTON_ERR_ARGUMENT;
  const long rows = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv);
  const int room = rows >= KX_ROWS ? KX_ROWS : (int)(rows + 15) / 16 * 16;
  KeyWeightsMmaArgs a = {(const bf16*)c->q, c->weights, c->k_cache, c->block_table, c->cu_tokens, c->context_lens, c->held, c->sinks, c->lse, c->scratch, c->err, c->q_stride,
                         c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, parts, room, c->scale, c->softcap};
  const dim3 grid(parts, c->n_kv, c->S);
#define WEIGH(FINAL) (c->d == 64 ? c->packed ? kx_launch<64, true, FINAL>(a, grid, stream) : kx_launch<64, false, FINAL>(a, grid, stream) \
                                 : c->packed ? kx_launch<128, true, FINAL>(a, grid, stream) : kx_launch<128, false, FINAL>(a, grid, stream))
  if (c->lse == nullptr) {
    int status = WEIGH(false);
    if (status != 0) return status;
    float* lse = c->scratch + c->scratch_rows * c->n_q * parts * 2;
    const long blocks = ((long)c->max_tokens_per_seq * c->n_q + 3) / 4;
    if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
    status = launch_pdl(key_weights_lse_kernel, dim3((unsigned)blocks, c->S), dim3(128), 0, stream, a, lse);
    if (status != 0) return status;
    a.lse = lse;
  }
  return WEIGH(true);
#undef WEIGH
}
