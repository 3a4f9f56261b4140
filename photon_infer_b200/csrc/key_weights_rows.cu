// What each cached key got of the softmax of a request's query rows (key_weights.cu), for more than 8 rows, with products in 32 bits: any type, head and page.
//
// A block has 128 keys and 16 R rows at a time, 32 numbers of each in shared memory in 32 bits, the next ones on their way in registers; a thread has the products of 8 keys and R
// rows, so that a number from shared memory is used R or 8 times.  Lanes read neighbouring numbers of a row and turn four keys' over on the way.  R is 1 up to 16 rows, else 4.
// What bounds it: the products, 4 d for a score without the logarithms, at 0.2 of the rate of 32-bit sums; short runs of tiles with a chain of latencies in front take most of the
// rest.  Two requests of 32 tokens beside 4,000 keys, 32 query heads on 8, heads of 128, 32 bits: 188 us, where key_weights.cu takes 640; 4 of 8 beside 2,000, heads of 64: 62 and
// 103; 1 of 4 beside 1,000: 23 and 53; of 1 token (4 rows) beside 4,000: 35 and 30.
#include "key_weights.cuh"

#define KW_THREADS 256
#define KW_PIECE 32              // numbers of a row in shared memory at a time
#define KW_KEY_PITCH 132

struct KeyWeightsArgs {
  KeyWeightsMmaArgs s;           // what all forms have; q behind its own type
  const void* q;
  int d;
};

// T: the queries' type, C: the cache's; FINAL: the weights, else the shares' maxima and sums.
template <typename T, typename C, int R, bool FINAL>
__global__ void __launch_bounds__(KW_THREADS, 2)
key_weights_rows_kernel(const KeyWeightsArgs w) {
  constexpr int ROWS = 16 * R, PITCH = ROWS + 4, PER = ROWS * KW_PIECE / KW_THREADS;
  constexpr bool PACKED = sizeof(C) == 1;
  __shared__ __align__(16) float k_s[KW_PIECE * KW_KEY_PITCH], q_s[KW_PIECE * PITCH];
  __shared__ __align__(16) int there_s[KX_KEYS];
  __shared__ float lse_s[ROWS], sums_s[KW_THREADS / 32][KX_KEYS];
  __shared__ int place_s[ROWS], slot_s[KX_KEYS];
  __shared__ long row_s[KX_KEYS];                     // (page, head, slot) of a key, counted through
  const KeyWeightsMmaArgs& a = w.s;
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y % a.n_kv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kt = lane & 15, rt = 2 * warp + (lane >> 4);
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq];
  const int G = a.n_q / a.n_kv, rows = n * G, d = w.d, groups = d / 32, base = ctx - n, known = a.held != nullptr ? a.held[seq] : base;
  const int low = a.window > 0 ? min(base - a.window + 1, known) : 0;      // keys in front of it no row sees, and they have a sum
  const int tiles = (max(ctx, 0) + KX_KEYS - 1) / KX_KEYS, per = (tiles + a.parts - 1) / a.parts, tile0 = (int)blockIdx.x * per, tile1 = min(tile0 + per, tiles);
  if (n <= 0) return;
  auto settle = [&](int tile) {                       // thread `tid` finds key `tid` of the tile
    if (tid >= KX_KEYS) return;
    const int key = tile * KX_KEYS + tid, pidx = key / a.page_size, slot = key - pidx * a.page_size;
    int page = -1;
    if (key >= low && key < ctx) {
      page = pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1;
      if (page < 0 || page >= a.num_pages) {
        if (FINAL) report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, key, page);
        page = -1;
      }
    }
    there_s[tid] = page >= 0;
    slot_s[tid] = slot;
    row_s[tid] = ((long)page * a.n_kv + head) * a.page_size + slot;
  };
  auto settle_rows = [&](int r0) {
    if (tid >= ROWS) return;
    const int row = r0 + tid;
    place_s[tid] = row < rows ? base + row / G : -1;
    lse_s[tid] = FINAL && row < rows ? a.lse[(long)(first + row / G) * a.n_q + head * G + row % G] * 1.4426950408889634f : 0.f;
  };
  float acc[R][8];                                    // of rows rt R .. and keys 4 kt .., 64 + 4 kt ..
  auto products = [&](int r0) {
    const int p = tid & 7, g = tid >> 3;              // numbers 4 p .. of keys 4 g ..; number `lane` of rows PER warp ..
    float k[4][4];
    T x[PER];                                         // as they come: whoever looks at one waits for it
    auto load = [&](int c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 4 * g + i, at = KW_PIECE * c + 4 * p;
#pragma unroll
        for (int j = 0; j < 4; ++j) k[i][j] = 0.f;
        if (there_s[key] == 0 || at >= d) continue;
        if constexpr (PACKED) {                       // word t groups + c has numbers 8 t .. of the group
          const int slot = slot_s[key];
          const uint8_t* page = (const uint8_t*)a.k + (row_s[key] - slot) * (groups * 17);
          const float scale = kv4_scale(page[(long)a.page_size * (d / 2) + slot * groups + c]);
          const uint32_t word = ((const uint32_t*)(page + (long)slot * (d / 2)))[(p >> 1) * groups + c];
#pragma unroll
          for (int j = 0; j < 4; ++j) k[i][j] = kv4_code(word >> (16 * (p & 1)), j) * scale;
        } else if constexpr (sizeof(C) == 2) {
          const uint2 u = *(const uint2*)((const C*)a.k + row_s[key] * d + at);
          k[i][0] = __uint_as_float(u.x << 16); k[i][1] = __uint_as_float(u.x & 0xffff0000u);
          k[i][2] = __uint_as_float(u.y << 16); k[i][3] = __uint_as_float(u.y & 0xffff0000u);
        } else {
          const float4 u = *(const float4*)((const C*)a.k + row_s[key] * d + at);
          k[i][0] = u.x; k[i][1] = u.y; k[i][2] = u.z; k[i][3] = u.w;
        }
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int row = r0 + PER * warp + i, at = KW_PIECE * c + lane;
        x[i] = row < rows && at < d ? ((const T*)w.q)[(first + row / G) * a.q_stride + (long)(head * G + row % G) * d + at] : from_f32<T>(0.f);
      }
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] = 0.f;
    load(0);
    for (int c = 0; c * KW_PIECE < d; ++c) {
      __syncthreads();                                // the piece in front of this one is done with
#pragma unroll
      for (int j = 0; j < 4; ++j) *(float4*)&k_s[(4 * p + j) * KW_KEY_PITCH + 4 * g] = make_float4(k[0][j], k[1][j], k[2][j], k[3][j]);
      if constexpr (R == 4) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) *(float4*)&q_s[lane * PITCH + PER * warp + i] = make_float4(kv4_query(x[i]), kv4_query(x[i + 1]), kv4_query(x[i + 2]), kv4_query(x[i + 3]));
      } else {
        *(float2*)&q_s[lane * PITCH + PER * warp] = make_float2(kv4_query(x[0]), kv4_query(x[1]));
      }
      __syncthreads();
      if ((c + 1) * KW_PIECE < d) load(c + 1);
#pragma unroll 8
      for (int i = 0; i < KW_PIECE; ++i) {
        const float4 u = *(const float4*)&k_s[i * KW_KEY_PITCH + 4 * kt], v = *(const float4*)&k_s[i * KW_KEY_PITCH + 64 + 4 * kt];
        const float b[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        float y[R];
        if constexpr (R == 4) {
          const float4 z = *(const float4*)&q_s[i * PITCH + 4 * rt];
          y[0] = z.x; y[1] = z.y; y[2] = z.z; y[3] = z.w;
        } else {
          y[0] = q_s[i * PITCH + rt];
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(b[e], y[r], acc[r][e]);
      }
    }
  };
  auto key_at = [&](int e) { return e < 4 ? 4 * kt + e : 60 + 4 * kt + e; };
  auto sees = [&](int tile, int r, int e) {
    const int key = tile * KX_KEYS + key_at(e), place = place_s[rt * R + r];
    return there_s[key_at(e)] != 0 && key <= place && (a.window <= 0 || key > place - a.window);
  };
  if constexpr (FINAL) {
    for (int tile = tile0; tile < tile1; ++tile) {
      settle(tile);
      float sum[8] = {};
      for (int r0 = 0; r0 < rows; r0 += ROWS) {
        __syncthreads();                              // the rows in front of these are done with, the keys are known
        settle_rows(r0);
        products(r0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float lse = lse_s[rt * R + r];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (sees(tile, r, e)) sum[e] += exp2f(key_score(acc[r][e], a.scale, a.softcap) - lse);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 16);
        if (lane < 16) sums_s[warp][key_at(e)] = sum[e];
      }
      __syncthreads();
      if (tid < KX_KEYS && there_s[tid]) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < KW_THREADS / 32; ++i) total += sums_s[i][tid];
        float* to = a.weights + row_s[tid];
        *to = tile * KX_KEYS + tid < known ? *to + total : total;
      }
    }
  } else {
    for (int r0 = (int)(blockIdx.y / a.n_kv) * ROWS; r0 < rows; r0 += (int)(gridDim.y / a.n_kv) * ROWS) {
      float m[R], l[R];
#pragma unroll
      for (int r = 0; r < R; ++r) { m[r] = -INFINITY; l[r] = 0.f; }
      __syncthreads();
      settle_rows(r0);
      for (int tile = tile0; tile < tile1; ++tile) {
        __syncthreads();
        settle(tile);
        __syncthreads();
        products(r0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float x[8], top = m[r];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = sees(tile, r, e) ? key_score(acc[r][e], a.scale, a.softcap) : -INFINITY;
            top = fmaxf(top, x[e]);
          }
          const float ref = top == -INFINITY ? 0.f : top;
          l[r] = l[r] == 0.f ? 0.f : l[r] * (m[r] == -INFINITY ? 1.f : exp2f(m[r] - ref));
#pragma unroll
          for (int e = 0; e < 8; ++e) l[r] += exp2f(x[e] - ref);
          m[r] = top;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float total = l[r] == 0.f ? 0.f : l[r] * (m[r] == -INFINITY ? 1.f : exp2f(m[r] - top));
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const int row = r0 + rt * R + r;
        if (kt == 0 && row < rows) {
          float* to = a.scratch + ((long)(first + row / G) * a.n_q + head * G + row % G) * a.parts * 2 + 2 * blockIdx.x;
          to[0] = top;
          to[1] = total;
        }
      }
    }
  }
}

template <typename T, typename C, int R>
static int kw_launch(KeyWeightsArgs w, const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->lse == nullptr) {
    const long rows = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv), levels = (rows + 16 * R - 1) / (16 * R), most = 65535 / c->n_kv;
    const long blocks = ((long)c->max_tokens_per_seq * c->n_q + 3) / 4;
    if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
    int status = launch_pdl(key_weights_rows_kernel<T, C, R, false>, dim3(c->parts, (unsigned)(c->n_kv * (levels < most ? levels : most)), c->S), dim3(KW_THREADS), 0, stream, w);
    if (status != 0) return status;
    float* lse = c->scratch + c->scratch_rows * c->n_q * c->parts * 2;
    status = launch_pdl(key_weights_lse_kernel, dim3((unsigned)blocks, c->S), dim3(128), 0, stream, w.s, lse);
    if (status != 0) return status;
    w.s.lse = lse;
  }
  return launch_pdl(key_weights_rows_kernel<T, C, R, true>, dim3(c->parts, c->n_kv, c->S), dim3(KW_THREADS), 0, stream, w);
}

PHOTON_API int photon_key_weights_rows(const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_keys <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (c->packed ? !kv4_sizes_ok(c->page_size, c->d) : (c->page_size <= 0 || c->d <= 0 || c->d > 256 || c->d % 8 != 0)) return PHOTON_ERR_UNSUPPORTED;
  if (c->parts < 1 || (c->lse == nullptr && c->scratch == nullptr) || c->keep_scores) return PHOTON_ERR_ARGUMENT;
  if (c->S > 65535 || c->n_kv > 65535 || c->scale <= 0.f) return PHOTON_ERR_UNSUPPORTED;
  const KeyWeightsArgs w = {{nullptr, c->weights, c->k_cache, c->block_table, c->cu_tokens, c->context_lens, c->held, c->sinks, c->lse, c->scratch, c->err, c->q_stride,
                             nullptr, 0, c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, c->parts, 0, 0, c->scale, c->softcap}, c->q, c->d};
  const bool few = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv) <= 16;
#define WEIGH(T, C) (few ? kw_launch<T, C, 1>(w, c, stream) : kw_launch<T, C, 4>(w, c, stream))
  if (c->packed) return c->dtype == PHOTON_F32 ? WEIGH(float, uint8_t) : WEIGH(bf16, uint8_t);
  return c->dtype == PHOTON_F32 ? WEIGH(float, float) : WEIGH(bf16, bf16);
#undef WEIGH
}
