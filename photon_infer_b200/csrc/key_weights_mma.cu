// What each cached key got of the softmax of a request's query rows (key_weights.cu) on the tensor cores: bfloat16 queries, heads of 64 or 128, a plain bfloat16 cache or one in
// 4 bits (kv4.cuh), whose numbers bfloat16 holds exactly.
//
// A block walks a run of a request's keys, 128 at a time, for one head: the cache's own rows or what their codes stand for in shared memory, the next ones on their way; beside
// them up to 32 rows (tokens x query heads of the key/value head), 16 for a warp, and the warps share the keys out.  The keys are the first operand: a score's row is a key, so what is not finite stays
// with its key, and a key's sum over the rows lies in the lanes of one row.  Every key is one block's: no atomics, the same bits every time.
// Without the rows' logarithms a first kernel leaves each run's maxima and sums and a second one joins them.  Up to 16 rows' scores are kept as well, 4 bytes for 2 d of a key's
// row, and a third kernel turns them into weights; for more rows the keys are read again.
//
// What bounds it: a token of 32 requests beside 8,000 keys, 32 query heads on 8, heads of 128: 160 us, 524 MB of keys, 0.5 of the copy rate (runs end at different times, scores are written and
// read once); of 8 beside 4,000: 29 us.  With the keys read twice and no scores kept the 32 requests took twice the bytes.  More than 32 rows are key_weights_tc.cu's, which is the faster.
#include "key_weights.cuh"
#include <type_traits>

#define KX_THREADS 256
#define KX_WARPS 8
#define KX_ROWS 32               // query rows, at most

__device__ __forceinline__ void kx_matrices(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void kx_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// FINAL: the weights; else the maxima and sums of the run.
template <int D, bool PACKED, bool FINAL>
__global__ void __launch_bounds__(KX_THREADS, 2)
key_weights_mma_kernel(const KeyWeightsMmaArgs a) {
  constexpr int PITCH = 2 * D + 16, GROUPS = D / 32, STEPS = D / 16, PIECES = PACKED ? D / 32 : D / 8, EACH = KX_KEYS * PIECES / KX_THREADS;      // of 16 bytes
  extern __shared__ __align__(16) uint8_t kx_smem[];
  uint8_t* k_s = kx_smem;                             // twice [KX_KEYS] rows
  uint8_t* q_s = k_s + 2 * KX_KEYS * PITCH;           // [room] rows
  __shared__ float sum_s[KX_ROWS / 16][KX_KEYS], lse_s[KX_ROWS], ml_s[KX_WARPS][16][2];
  __shared__ uint32_t there_s[2][4];                  // keys that are there
  __shared__ long row_s[2][KX_KEYS];                  // (page, head, slot) of a key, counted through
  __shared__ int slot_s[2][KX_KEYS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq], G = a.n_q / a.n_kv, rows = min(n * G, a.room), base = ctx - n, last_place = ctx - 1;
  if (n <= 0 || ctx <= 0) return;
  const int known = a.held != nullptr ? a.held[seq] : base;
  // keys that no row sees and that have a sum already are left out
  int low = a.window > 0 ? max(0, base - a.window + 1) : 0;
  if (FINAL) low = max(0, min(low, known));
  const int tile0 = max((int)blockIdx.x * a.each, low / KX_KEYS), tile1 = min(((int)blockIdx.x + 1) * a.each, (ctx + KX_KEYS - 1) / KX_KEYS);
  const int wr = rows > 16 ? 2 : 1, wk = KX_WARPS / wr, my_r = warp % wr, my_k = warp / wr;
  if (tile0 >= tile1) {
    if (!FINAL)
      for (int r = tid; r < rows; r += KX_THREADS) {
        float* to = a.scratch + ((long)(first + r / G) * a.n_q + head * G + r % G) * a.parts * 2 + 2 * blockIdx.x;
        to[0] = -INFINITY;
        to[1] = 0.f;
      }
    return;
  }
  // ---- places: thread `tid` has key `tid` of a tile, and the block table's entry of the next one
  auto entry_of = [&](int tile) {
    const int key = tile * KX_KEYS + tid, pidx = key / a.page_size;
    return tid < KX_KEYS && tile < tile1 && key >= low && key < ctx ? (pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1) : -2;      // -2: not asked for
  };
  auto settle = [&](int tile, int entry) {             // the tile's places, from its entries
    if (tid < KX_KEYS) {
      const int key = tile * KX_KEYS + tid, slot = key - key / a.page_size * a.page_size;
      const bool good = entry >= 0 && entry < a.num_pages;
      if (FINAL && !good && entry != -2) report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, key, entry);
      const uint32_t votes = __ballot_sync(0xffffffffu, good);
      if (lane == 0) there_s[tile & 1][warp] = votes;
      row_s[tile & 1][tid] = ((long)(good ? entry : 0) * a.n_kv + head) * a.page_size + (good ? slot : 0);      // else some row of the pool: what is read is not used
      slot_s[tile & 1][tid] = good ? slot : 0;
    }
  };
  uint4 u[PACKED ? EACH : 1];
  uint32_t scales[PACKED ? EACH : 1];
  auto ask = [&](int tile) {
    const long* row = row_s[tile & 1];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int x = i * KX_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
      if constexpr (PACKED) {
        const int slot = slot_s[tile & 1][key];
        const uint8_t* at = (const uint8_t*)a.k + (row[key] - slot) * (GROUPS * 17);
        const uint8_t* sc = at + (long)a.page_size * (D / 2) + slot * GROUPS;
        u[i] = *(const uint4*)(at + (long)slot * (D / 2) + 16 * piece);
        scales[i] = GROUPS == 4 ? *(const uint32_t*)sc : *(const uint16_t*)sc;
      } else {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(k_s + ((tile & 1) * KX_KEYS + key) * PITCH + 16 * piece)),
                     "l"((const bf16*)a.k + row[key] * D + 8 * piece)
                     : "memory");
      }
    }
    if constexpr (!PACKED) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto put = [&](int tile) {                           // what was asked for, as numbers
    if constexpr (PACKED) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int x = i * KX_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {                  // words t GROUPS + j
          const int word = 4 * piece + c, tt = word / GROUPS, j = word - tt * GROUPS;
          const __nv_bfloat162 s = __float2bfloat162_rn(kv4_scale(scales[i] >> (8 * j) & 255u));
          // numbers 0 and 4, 1 and 5, 2 and 6, 3 and 7
          const uint32_t y0 = kx_scaled(w[c], 0, s), y1 = kx_scaled(w[c], 4, s), y2 = kx_scaled(w[c], 8, s), y3 = kx_scaled(w[c], 12, s);
          *(uint4*)(k_s + ((tile & 1) * KX_KEYS + key) * PITCH + 64 * j + 16 * tt) =
              make_uint4(__byte_perm(y0, y1, 0x5410), __byte_perm(y2, y3, 0x5410), __byte_perm(y0, y1, 0x7632), __byte_perm(y2, y3, 0x7632));
        }
      }
    }
  };
  const float scale2 = a.scale * 1.4426950408889634f, cap_in = 2.f * 1.4426950408889634f * a.scale / a.softcap, cap_out = a.softcap * 1.4426950408889634f;
  const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(q_s) + (my_r * 16 + (lane & 7) + (lane >> 4) * 8) * PITCH + (lane >> 3 & 1) * 16;
  uint32_t b[STEPS][4];                                // rows 0 to 7: [0], [1]; 8 to 15: [2], [3]
  float ref[4], m[4], l[4];
  int at_place[4];
  // ---- the rows, into shared memory and into the second operand
  int entry = entry_of(tile0);
  for (int x = tid; x < wr * 16 * (D / 8); x += KX_THREADS) {
    const int r = x / (D / 8), piece = x - r * (D / 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows) v = kx_queries(*(const uint4*)(a.q + (first + r / G) * a.q_stride + (long)(head * G + r % G) * D + 8 * piece));
    *(uint4*)(q_s + r * PITCH + 16 * piece) = v;
  }
  if (FINAL && tid < KX_ROWS) lse_s[tid] = tid < rows ? a.lse[(long)(first + tid / G) * a.n_q + head * G + tid % G] * 1.4426950408889634f : INFINITY;
  __syncthreads();
  const bool two = my_r * 16 + 8 < rows;               // rows in the warp's second eight
#pragma unroll
  for (int i = 0; i < STEPS; ++i) kx_matrices(b[i], q_at + 32 * i);
#pragma unroll
  for (int c = 0; c < 4; ++c) {                        // rows 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t
    const int r = my_r * 16 + (c >> 1) * 8 + 2 * t + (c & 1);
    ref[c] = FINAL ? lse_s[r] : 0.f;
    at_place[c] = r < rows ? base + r / G : -1;
    m[c] = -INFINITY;
    l[c] = 0.f;
  }
  settle(tile0, entry);
  entry = entry_of(tile0 + 1);
  __syncthreads();
  ask(tile0);
  put(tile0);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int key0 = tile * KX_KEYS, keys = min(KX_KEYS, ctx - key0);
    const bool more = tile + 1 < tile1;
    float before = 0.f;
    const bool mine = FINAL && tid < KX_KEYS && (there_s[tile & 1][warp & 3] >> lane & 1u);
    if (mine && key0 + tid < known) before = a.weights[row_s[tile & 1][tid]];
    if (more) {
      settle(tile + 1, entry);
      entry = entry_of(tile + 2);
    }
    __syncthreads();                                 // the tile in front of this one is done with, the next one's places are known
    if (more) ask(tile + 1);
    if constexpr (!PACKED) {
      if (more) asm volatile("cp.async.wait_group 1;" ::: "memory");
      else asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
    }
    const uint32_t* there = there_s[tile & 1];
    const bool clear = (there[0] & there[1] & there[2] & there[3]) == 0xffffffffu && key0 + KX_KEYS - 1 <= base && (a.window <= 0 || key0 > last_place - a.window);      // all rows see all
    const uint32_t k_at = (uint32_t)__cvta_generic_to_shared(k_s) + ((tile & 1) * KX_KEYS + (lane & 15)) * PITCH + (lane >> 4) * 16;
    // 16 keys, or twice 16 side by side: the second ones' products fill the first ones' waits
    auto work = [&](auto several, int part0) {
      constexpr int P = decltype(several)::value;
      float d[P][2][4] = {};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        uint32_t k4[P][4];
#pragma unroll
        for (int p = 0; p < P; ++p) kx_matrices(k4[p], k_at + (part0 + p * wk) * 16 * PITCH + 32 * i);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          kx_mma(d[p][0], k4[p], b[i][0], b[i][1]);
          if (two) kx_mma(d[p][1], k4[p], b[i][2], b[i][3]);
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int part = part0 + p * wk;
        float x[4][2];                               // rows as above, keys g and 8 + g
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) x[c][h] = d[p][c >> 1][2 * h + (c & 1)];
        if (a.softcap > 0.f) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[c][h] = cap_out * (1.f - __fdividef(2.f, 1.f + kx_exp2(x[c][h] * cap_in)));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[c][h] *= scale2;
        }
        if (!clear) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = part * 16 + 8 * h + g, key = key0 + k;
            const bool is = there[k >> 5] >> (k & 31) & 1u;
#pragma unroll
            for (int c = 0; c < 4; ++c) if (!(is && key <= at_place[c] && (a.window <= 0 || key > at_place[c] - a.window))) x[c][h] = -INFINITY;
          }
        }
        if constexpr (FINAL) {
          float sum[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sum[h] = 0.f;
            // a hidden key's weight is 0 whatever the row's logarithm is
#pragma unroll
            for (int c = 0; c < 4; ++c) if (c < 2 || two) sum[h] += !clear && x[c][h] == -INFINITY ? 0.f : kx_exp2(x[c][h] - ref[c]);
          }
          // the four lanes with a key's rows: an even lane has key g in the end, an odd one key 8 + g
          const float y = (t & 1 ? sum[1] : sum[0]) + __shfl_xor_sync(0xffffffffu, t & 1 ? sum[0] : sum[1], 1), z = y + __shfl_xor_sync(0xffffffffu, y, 2);
          if (t < 2) sum_s[my_r][part * 16 + 8 * t + g] = z;
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c >= 2 && !two) continue;
            const float top = fmaxf(m[c], fmaxf(x[c][0], x[c][1])), zero = top == -INFINITY ? 0.f : top;
            l[c] = (m[c] == -INFINITY ? l[c] : l[c] * kx_exp2(m[c] - zero)) + kx_exp2(x[c][0] - zero) + kx_exp2(x[c][1] - zero);
            m[c] = top;
          }
          if (a.scores != nullptr) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int row = my_r * 16 + (c >> 1) * 8 + 2 * t + (c & 1);
              if (row >= rows) continue;
              float* to = a.scores + ((long)(first + row / G) * a.n_q + head * G + row % G) * a.width + key0 + part * 16 + g;
#pragma unroll
              for (int h = 0; h < 2; ++h) if (part * 16 + 8 * h + g < keys && key0 + part * 16 + 8 * h + g < a.width) to[8 * h] = x[c][h];
            }
          }
        }
      }
    };
    int part = my_k;
    for (; (part + wk) * 16 < keys; part += 2 * wk) work(std::integral_constant<int, 2>(), part);
    if (part * 16 < keys) work(std::integral_constant<int, 1>(), part);
    if (more) put(tile + 1);
    if constexpr (FINAL) {
      __syncthreads();
      if (mine) {
        float sum = before;
        for (int w = 0; w < wr; ++w) sum += sum_s[w][tid];
        a.weights[row_s[tile & 1][tid]] = sum;
      }
    }
    __syncthreads();                                 // the tile, its places and its sums are done with
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
    if (tid < rows) {                                // the warps that share the row's keys
      const int of = tid >> 4, r = tid & 15;
      float top = -INFINITY, sum = 0.f;
      for (int w = 0; w < wk; ++w) top = fmaxf(top, ml_s[w * wr + of][r][0]);
      const float zero = top == -INFINITY ? 0.f : top;
      for (int w = 0; w < wk; ++w) {
        const float pm = ml_s[w * wr + of][r][0], pl = ml_s[w * wr + of][r][1];
        if (pl != 0.f) sum += pm == -INFINITY ? pl : pl * exp2f(pm - zero);
      }
      float* to = a.scratch + ((long)(first + tid / G) * a.n_q + head * G + tid % G) * a.parts * 2 + 2 * blockIdx.x;
      to[0] = top;
      to[1] = sum;
    }
  }
}

// The weights from the scores of up to 16 rows: a thread has a key.
__global__ void __launch_bounds__(KX_THREADS)
key_weights_scores_kernel(const KeyWeightsMmaArgs a) {
  __shared__ float lse_s[16];
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y, key = blockIdx.x * KX_THREADS + threadIdx.x;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq], G = a.n_q / a.n_kv, rows = min(n * G, 16), base = ctx - n;
  if (n <= 0 || (int)(blockIdx.x * KX_THREADS) >= ctx) return;
  if (threadIdx.x < rows) lse_s[threadIdx.x] = a.lse[(long)(first + threadIdx.x / G) * a.n_q + head * G + threadIdx.x % G] * 1.4426950408889634f;
  __syncthreads();
  if (key >= ctx || key >= a.width) return;
  const int known = a.held != nullptr ? a.held[seq] : base, low = a.window > 0 ? max(0, base - a.window + 1) : 0;
  if (key < min(low, known)) return;                  // no row sees it, and it has a sum
  const int pidx = key / a.page_size, page = pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1;
  if (page < 0 || page >= a.num_pages) {
    report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, key, page);
    return;
  }
  float* w = a.weights + ((long)page * a.n_kv + head) * a.page_size + (key - pidx * a.page_size);
  float sum = key < known ? *w : 0.f;
  if (key >= low)                                     // else there are no scores
    for (int r = 0; r < rows; ++r) {
      const float x = a.scores[((long)(first + r / G) * a.n_q + head * G + r % G) * a.width + key];
      if (x != -INFINITY) sum += kx_exp2(x - lse_s[r]);
    }
  *w = sum;
}

template <int D, bool PACKED, bool FINAL>
static int kx_launch(const KeyWeightsMmaArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr size_t most = (2 * KX_KEYS + KX_ROWS) * (2 * D + 16);
  const size_t smem = (2 * KX_KEYS + a.room) * (2 * D + 16);
  static bool ready[64] = {};
  const int limit = smem_limit((const void*)key_weights_mma_kernel<D, PACKED, FINAL>, (int)most, true, ready);
  if (limit != 0) return limit;
  return launch_pdl(key_weights_mma_kernel<D, PACKED, FINAL>, grid, dim3(KX_THREADS), smem, stream, a);
}

PHOTON_API int photon_key_weights_mma(const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_keys <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0) return PHOTON_ERR_ARGUMENT;
  if ((c->d != 64 && c->d != 128) || c->num_pages <= 0 || c->page_size <= 0 || (c->packed && !kv4_sizes_ok(c->page_size, c->d))) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)c->q | (uintptr_t)c->k_cache) % 16 || c->q_stride % 8) return PHOTON_ERR_UNSUPPORTED;
  const long rows = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv), all_rows = c->scratch_rows * c->n_q;
  if (c->S > 65535 || c->n_kv > 65535 || c->scale <= 0.f || rows > KX_ROWS) return PHOTON_ERR_UNSUPPORTED;
  if (c->parts < 1 || (c->lse == nullptr && c->scratch == nullptr)) return PHOTON_ERR_ARGUMENT;
  const int room = (int)(rows + 15) / 16 * 16, tiles = (c->max_keys + KX_KEYS - 1) / KX_KEYS, each = (tiles + c->parts - 1) / c->parts;
  KeyWeightsMmaArgs a = {(const bf16*)c->q, c->weights, c->k_cache, c->block_table, c->cu_tokens, c->context_lens, c->held, c->sinks, c->lse, c->scratch, c->err, c->q_stride,
                         nullptr, 0, c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, c->parts, each, room, c->scale, c->softcap};
  const dim3 grid(c->parts, c->n_kv, c->S);
#define WEIGH(FINAL) (c->d == 64 ? c->packed ? kx_launch<64, true, FINAL>(a, grid, stream) : kx_launch<64, false, FINAL>(a, grid, stream) \
                                 : c->packed ? kx_launch<128, true, FINAL>(a, grid, stream) : kx_launch<128, false, FINAL>(a, grid, stream))
  if (c->lse != nullptr) return WEIGH(true);
  float* lse = c->scratch + all_rows * c->parts * 2;
  if (c->keep_scores) {
    if (rows > 16) return PHOTON_ERR_ARGUMENT;
    a.scores = lse + all_rows;
    a.width = c->max_keys;
  }
  int status = WEIGH(false);
  if (status != 0) return status;
  const long blocks = ((long)c->max_tokens_per_seq * c->n_q + 3) / 4;
  if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  status = launch_pdl(key_weights_lse_kernel, dim3((unsigned)blocks, c->S), dim3(128), 0, stream, a, lse);
  if (status != 0) return status;
  a.lse = lse;
  if (!c->keep_scores) return WEIGH(true);
  return launch_pdl(key_weights_scores_kernel, dim3((c->max_keys + KX_THREADS - 1) / KX_THREADS, c->n_kv, c->S), dim3(KX_THREADS), 0, stream, a);
#undef WEIGH
}
