// What each cached key got of the softmax of a request's query rows, added to a sum beside the key.
//
// weights [pages][n_kv][page_size]: for the rows (tokens x query heads of a key/value head) of the request, w[key] += sum over rows of exp(score - lse[row]); keys from
// held[seq] on have no sum yet and get this one.  lse [T, n_q]: the natural logarithm of each row's sum of exponentials; where there is none, a first kernel leaves
// the maximum and the sum of every share of the keys, and the second joins them.  Every key is one thread's: no sums over blocks, no atomics.
// The cache: 4 bits (kv4.cuh), bfloat16 or 32 bits.
//
// For up to 8 rows, in 32 bits: what bounds it is the reading, since a thread has a key and reads its row by itself, and every number meets 8 rows' whether they are there or not.  4
// rows beside 4,000 keys, 8 heads of 128, 32 bits: 30 us; key_weights_rows.cu takes 35 for them and from 9 rows on less.
#include "key_weights.cuh"

#define KW_THREADS 128
#define KW_ROWS 8

struct KeyWeightsArgs {
  const void* q; float* weights; const void* k; const int* table; const int* cu_tokens; const int* context_lens; const int* held; const float* sinks; const float* lse;
  float* scratch; int* err;
  long q_stride;
  int max_pages, n_q, n_kv, d, page_size, num_pages, window, parts;
  float scale, softcap;
};

// T: the queries' type, C: the cache's; FINAL: the weights, else the shares' maxima and sums.
template <typename T, typename C, bool FINAL>
__global__ void __launch_bounds__(KW_THREADS)
key_weights_kernel(const KeyWeightsArgs a) {
  extern __shared__ __align__(16) float qs[];                        // KW_ROWS * d
  __shared__ float lse_s[KW_ROWS], red[32];
  constexpr bool PACKED = sizeof(C) == 1;
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq];
  const int G = a.n_q / a.n_kv, rows = min(n * G, KW_ROWS), d = a.d, groups = d / 32, words = d / 8, base = ctx - n;
  const int tiles = (max(ctx, 0) + KW_THREADS - 1) / KW_THREADS, per = (tiles + a.parts - 1) / a.parts;
  if (n <= 0) return;
  const int known = a.held != nullptr ? a.held[seq] : base, low = a.window > 0 ? min(base - a.window + 1, known) : 0;      // keys in front of it no row sees, and they have a sum
  for (int i = tid; i < KW_ROWS * d; i += KW_THREADS) {
    const int r = i / d, p = i - r * d, x = p / 8, t = PACKED ? x / groups : 0, at = PACKED ? 32 * (x - t * groups) + 8 * t + p % 8 : p;
    qs[r * d + p] = r < rows ? kv4_query(((const T*)a.q)[(first + r / G) * a.q_stride + (head * G + r % G) * d + at]) : 0.f;
  }
  if (FINAL && tid < rows) {
    const int h = head * G + tid % G;
    const long of = (long)(first + tid / G) * a.n_q + h;
    float v;
    if (a.lse != nullptr) {
      v = a.lse[of] * 1.4426950408889634f;
    } else {
      const float* part_ml = a.scratch + of * a.parts * 2;
      float m = a.sinks != nullptr ? a.sinks[h] * 1.4426950408889634f : -INFINITY;
      const float sink = m;
      for (int p = 0; p < a.parts; ++p) m = fmaxf(m, part_ml[2 * p]);
      const float ref = m == -INFINITY ? 0.f : m;
      float total = a.sinks != nullptr ? exp2f(sink - ref) : 0.f;
      for (int p = 0; p < a.parts; ++p) {
        const float pm = part_ml[2 * p], pl = part_ml[2 * p + 1];
        if (pl != 0.f) total += pl * (pm == -INFINITY ? 1.f : exp2f(pm - ref));
      }
      v = total == 0.f ? -INFINITY : ref + log2f(total);
    }
    lse_s[tid] = v;
  }
  __syncthreads();
  float m[KW_ROWS], l[KW_ROWS];
#pragma unroll
  for (int r = 0; r < KW_ROWS; ++r) { m[r] = -INFINITY; l[r] = 0.f; }
  for (int tile = part * per; tile < min((part + 1) * per, tiles); ++tile) {
    const int key = tile * KW_THREADS + tid, pidx = key / a.page_size, slot = key - pidx * a.page_size;
    int page = -1;
    if (key >= low && key < ctx) {
      page = pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1;
      if (page < 0 || page >= a.num_pages) {
        if (FINAL) report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, key, page);
        page = -1;
      }
    }
    float s[KW_ROWS];
#pragma unroll
    for (int r = 0; r < KW_ROWS; ++r) s[r] = 0.f;
    if (page >= 0) {
      const uint8_t* at = PACKED ? (const uint8_t*)a.k + ((long)page * a.n_kv + head) * kv4_page_bytes(a.page_size, d) : nullptr;
      const uint32_t* codes = PACKED ? (const uint32_t*)(at + (long)slot * (d / 2)) : nullptr;
      const uint8_t* scales = PACKED ? at + (long)a.page_size * (d / 2) + slot * groups : nullptr;
      const C* row = (const C*)a.k + (((long)page * a.n_kv + head) * a.page_size + slot) * d;
      for (int x = 0; x < words; ++x) {
        float c[8];
        if constexpr (PACKED) {
          const uint32_t word = codes[x];
          const float scale = kv4_scale(scales[x % groups]);
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = kv4_code(word, i) * scale;
        } else {
          key_numbers<C>(row, x, c);
        }
#pragma unroll
        for (int r = 0; r < KW_ROWS; ++r) {
          const float4 u = *(const float4*)&qs[r * d + x * 8], v = *(const float4*)&qs[r * d + x * 8 + 4];
          s[r] += c[0] * u.x + c[1] * u.y + c[2] * u.z + c[3] * u.w + c[4] * v.x + c[5] * v.y + c[6] * v.z + c[7] * v.w;
        }
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < KW_ROWS; ++r) {
      const int place = base + r / G;
      if (page < 0 || r >= rows || key > place || (a.window > 0 && key <= place - a.window)) continue;
      const float x = key_score(s[r], a.scale, a.softcap);
      if (FINAL) {
        sum += exp2f(x - lse_s[r]);
      } else {
        const float top = fmaxf(m[r], x);
        const float ref = top == -INFINITY ? 0.f : top;
        l[r] = l[r] * (m[r] == -INFINITY ? 1.f : exp2f(m[r] - ref)) + exp2f(x - ref);
        m[r] = top;
      }
    }
    if (FINAL && page >= 0) {
      float* w = a.weights + ((long)page * a.n_kv + head) * a.page_size + slot;
      *w = key < known ? *w + sum : sum;
    }
  }
  if (!FINAL) {
#pragma unroll
    for (int r = 0; r < KW_ROWS; ++r) {
      __syncthreads();
      const float top = warp_max(m[r]);
      if (lane == 0) red[warp] = top;
      __syncthreads();
      const float all = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), ref = all == -INFINITY ? 0.f : all;
      const float total = block_sum(l[r] == 0.f ? 0.f : l[r] * (m[r] == -INFINITY ? 1.f : exp2f(m[r] - ref)), red);
      if (tid == 0 && r < rows) {
        float* to = a.scratch + ((long)(first + r / G) * a.n_q + head * G + r % G) * a.parts * 2 + 2 * part;
        to[0] = all;
        to[1] = total;
      }
    }
  }
}

PHOTON_API int photon_key_weights(const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_keys <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (c->packed ? !kv4_sizes_ok(c->page_size, c->d) : (c->page_size <= 0 || c->d <= 0 || c->d > 256 || c->d % 8 != 0)) return PHOTON_ERR_UNSUPPORTED;
  if (c->parts < 1 || (c->lse == nullptr && c->scratch == nullptr)) return PHOTON_ERR_ARGUMENT;
  if (c->S > 65535 || c->n_kv > 65535 || c->scale <= 0.f || (long)c->max_tokens_per_seq * (c->n_q / c->n_kv) > KW_ROWS) return PHOTON_ERR_UNSUPPORTED;
  const KeyWeightsArgs a = {c->q, c->weights, c->k_cache, c->block_table, c->cu_tokens, c->context_lens, c->held, c->sinks, c->lse, c->scratch, c->err, c->q_stride,
                            c->max_pages, c->n_q, c->n_kv, c->d, c->page_size, c->num_pages, c->window, c->parts, c->scale, c->softcap};
  const dim3 grid(c->parts, c->n_kv, c->S);
  const size_t smem = KW_ROWS * c->d * sizeof(float);
#define WEIGH(T, C) ((c->lse == nullptr && (status = launch_pdl(key_weights_kernel<T, C, false>, grid, dim3(KW_THREADS), smem, stream, a)) != 0) ? status \
                     : launch_pdl(key_weights_kernel<T, C, true>, grid, dim3(KW_THREADS), smem, stream, a))
  int status = 0;
  if (c->packed) return c->dtype == PHOTON_F32 ? WEIGH(float, uint8_t) : WEIGH(bf16, uint8_t);
  return c->dtype == PHOTON_F32 ? WEIGH(float, float) : WEIGH(bf16, bf16);
#undef WEIGH
}
