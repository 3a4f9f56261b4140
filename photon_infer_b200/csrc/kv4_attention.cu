// Attention over a paged cache in 4 bits (the format: kv4.cuh): the general kernel, for either type, any head of up to 256 numbers, any page.
//
// A block has a tile of ROWS rows (tokens x query heads of one key/value head) of a request and a share of its keys, 128 at a time: every thread
// works out one key's scores from the row it reads, then every thread has 8 numbers of the result (a word of a value's row) over a part of the keys.  32-bit sums, a
// running maximum; shares are joined by a second kernel in ascending order.
//
// A row at place p of the request (its tokens of the step are the last ones) sees keys p - window + 1 .. p.  A row that sees nothing is zero.  A key that a row does not
// see has the weight -0: where a value is not finite, the sign says that it is no part of the row.
//
// What bounds it: the products in 32 bits, and with few requests the chain of a block (range, page, rows, join).  32 query heads on 8, 32 bits: 4 requests of a token behind up to
// 2,001 keys, heads of 64, 23 us; 8 behind 4,000, heads of 128, 74; 8 of 3 tokens behind 2,000, 135.  From 25 rows on kv4_attention_rows.cu is the faster where there is work for
// many blocks.  Shares of the keys: as many as give four blocks an SM, of 128 keys at least, since each has a row's maximum, sum and result to leave and to be read again.
#include "kv4_attention.cuh"

#define KA_KEYS 128
#define KA_THREADS 128

template <typename T, int ROWS>
__global__ void __launch_bounds__(KA_THREADS)
kv4_attention_kernel(const Kv4Args a) {
  __shared__ __align__(16) float qs[ROWS * 256];
  __shared__ __align__(16) float ps[ROWS * KA_KEYS];
  __shared__ float red[KA_THREADS * 8];
  __shared__ float m_s[ROWS], l_s[ROWS], alpha_s[ROWS], top_s[ROWS * 4];
  __shared__ int page_s[KA_KEYS];
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y % a.n_kv, tile = blockIdx.y / a.n_kv, part = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq];
  const int G = a.n_q / a.n_kv, all = n * G, row0 = tile * ROWS;
  if (row0 >= all || all > a.max_rows) return;
  const int rows = min(ROWS, all - row0), d = a.groups * 32, words = d / 8, base = ctx - n;
  const int last_place = base + (row0 + rows - 1) / G, first_place = base + row0 / G;
  const int lo = a.window > 0 ? max(0, first_place - a.window + 1) : 0, hi = max(lo, last_place + 1);
  const int tiles = (hi - lo + KA_KEYS - 1) / KA_KEYS, per = (tiles + a.parts - 1) / a.parts;
  const int from = lo + min(part * per, tiles) * KA_KEYS, to = min(hi, lo + min((part + 1) * per, tiles) * KA_KEYS);
  for (int i = tid; i < ROWS * d; i += KA_THREADS) {                 // the query rows, in the order of a key's row
    const int r = i / d, p = i - r * d, w = p / 8, t = w / a.groups, j = w - t * a.groups;
    const int row = row0 + r, token = first + row / G, h = head * G + row % G;
    qs[r * 256 + p] = r < rows ? kv4_query(((const T*)a.q)[token * a.q_stride + h * d + 32 * j + 8 * t + p % 8]) : 0.f;
  }
  if (tid < ROWS) m_s[tid] = -INFINITY;
  const int subsets = KA_THREADS / words, sub = tid / words, w = tid - sub * words;      // the second half's share: word w, keys sub, sub + subsets ..
  const int ja = (2 * w) % a.groups, jb = (2 * w + 1) % a.groups;
  float acc[ROWS][8], l[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[r][i] = 0.f;
  }
  const long bytes = kv4_page_bytes(a.page_size, d);
  for (int k0 = from; k0 < to; k0 += KA_KEYS) {
    const int key = k0 + tid, pidx = key / a.page_size, slot = key - pidx * a.page_size;
    int page = -1;
    if (key < to) {
      page = pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1;
      if (page < 0 || page >= a.num_pages) {
        report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, key, page);
        page = -1;
      }
    }
    __syncthreads();                                                 // the last tile's weights are done with
    page_s[tid] = page;
    float s[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[r] = 0.f;
    if (page >= 0) {
      const uint8_t* at = a.k + ((long)page * a.n_kv + head) * bytes;
      const uint8_t* scales = at + (long)a.page_size * (d / 2) + slot * a.groups;
      const uint32_t* row = (const uint32_t*)(at + (long)slot * (d / 2));
      for (int x = 0; x < words; ++x) {
        const uint32_t word = row[x];
        const float scale = kv4_scale(scales[x % a.groups]);
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = kv4_code(word, i) * scale;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float4 u = *(const float4*)&qs[r * 256 + x * 8], v = *(const float4*)&qs[r * 256 + x * 8 + 4];
          s[r] += c[0] * u.x + c[1] * u.y + c[2] * u.z + c[3] * u.w + c[4] * v.x + c[5] * v.y + c[6] * v.z + c[7] * v.w;
        }
      }
    }
    bool seen[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int place = base + (row0 + r) / G;
      seen[r] = page >= 0 && r < rows && key <= place && (a.window <= 0 || key > place - a.window);
      s[r] = seen[r] ? kv4_bounded(s[r], a.scale, a.softcap) : -INFINITY;
      const float top = warp_max(s[r]);
      if (lane == 0) top_s[r * 4 + warp] = top;
    }
    __syncthreads();
    if (tid < ROWS) {
      const float top = fmaxf(fmaxf(fmaxf(top_s[tid * 4], top_s[tid * 4 + 1]), fmaxf(top_s[tid * 4 + 2], top_s[tid * 4 + 3])), m_s[tid]);
      alpha_s[tid] = m_s[tid] == -INFINITY ? 1.f : exp2f(m_s[tid] - top);       // nothing but what is not a number can have been added yet
      m_s[tid] = top;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float top = m_s[r], p = seen[r] ? exp2f(s[r] - (top == -INFINITY ? 0.f : top)) : -0.f;
      ps[r * KA_KEYS + tid] = p;
      l[r] = l[r] * alpha_s[r] + p;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[r][i] *= alpha_s[r];
    if (sub < subsets) {
      const int here = min(KA_KEYS, to - k0);
      for (int x = sub; x < here; x += subsets) {
        const int pg = page_s[x];
        if (pg < 0) continue;
        const int sl = (k0 + x) % a.page_size;
        const uint8_t* at = a.v + ((long)pg * a.n_kv + head) * bytes;
        const uint8_t* scales = at + (long)a.page_size * (d / 2) + sl * a.groups;
        const uint32_t word = ((const uint32_t*)(at + (long)sl * (d / 2)))[w];
        const float sa = kv4_scale(scales[ja]), sb = kv4_scale(scales[jb]);
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = kv4_code(word, i) * (i < 4 ? sa : sb);
        const bool odd = !isfinite(sa) || !isfinite(sb);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float p = ps[r * KA_KEYS + x];
          if (odd && signbit(p)) continue;
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r][i] += p * c[i];
        }
      }
    }
  }
  // the threads' parts of every row, in the order of the threads
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float sum = block_sum(l[r], top_s);
    if (tid == 0) l_s[r] = sum;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) red[tid * 8 + i] = acc[r][i];
    __syncthreads();
    if (r < rows) {
      const int row = row0 + r, h = head * G + row % G;
      const long token = first + row / G, of = token * a.n_q + h;
      float m = m_s[r], total = l_s[r], mul = 1.f;
      if (a.parts == 1) {
        if (a.sinks != nullptr) {
          const float sink = a.sinks[h] * 1.4426950408889634f, top = fmaxf(m, sink);
          mul = m == -INFINITY ? 1.f : exp2f(m - top);
          if (sink != -INFINITY) total = total * mul + exp2f(sink - top);
          m = top;
        }
        if (tid == 0 && a.lse != nullptr) a.lse[of] = total == 0.f ? -INFINITY : (m + log2f(total)) * 0.6931471805599453f;
        mul = total == 0.f ? 0.f : mul / total;
      }
      for (int p = tid; p < d; p += KA_THREADS) {
        float sum = 0.f;
        for (int x = 0; x < subsets; ++x) sum += red[(x * words) * 8 + p];
        const int hw = p / 4, g = hw / a.groups, j = hw - g * a.groups, at = 32 * j + 4 * g + p % 4;
        if (a.parts == 1) ((T*)a.out)[token * a.out_stride + h * d + at] = from_f32<T>(mul == 0.f ? 0.f : sum * mul);
        else a.scratch[(of * a.parts + part) * (d + 2) + at] = sum;
      }
      if (a.parts > 1 && tid == 0) {
        a.scratch[(of * a.parts + part) * (d + 2) + d] = m;
        a.scratch[(of * a.parts + part) * (d + 2) + d + 1] = total;
      }
    }
    __syncthreads();
  }
}

PHOTON_API int photon_kv4_attention(const photon_kv4_attention_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_UNSUPPORTED;
  if (c->parts < 1 || (c->parts > 1 && c->scratch == nullptr)) return PHOTON_ERR_ARGUMENT;
  Kv4Args a = {c->q, c->out, (const uint8_t*)c->k_cache, (const uint8_t*)c->v_cache, c->block_table, c->cu_tokens, c->context_lens, c->sinks, c->lse, c->scratch, c->err,
               c->q_stride, c->out_stride, c->max_pages, c->n_q, c->n_kv, c->d / 32, c->page_size, c->num_pages, c->window, c->parts, c->scale, c->softcap, c->max_rows};
  const long rows = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv);
  const int R = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8;
  const long y = (rows + R - 1) / R * c->n_kv;
  if (c->S > 65535 || y > 65535 || c->scale <= 0.f) return PHOTON_ERR_UNSUPPORTED;
  const dim3 grid(c->parts, (unsigned)y, c->S);
#define ATTEND(T, R) launch_pdl(kv4_attention_kernel<T, R>, grid, dim3(KA_THREADS), 0, stream, a)
  int status = c->dtype == PHOTON_F32 ? (R == 1 ? ATTEND(float, 1) : R == 2 ? ATTEND(float, 2) : R == 4 ? ATTEND(float, 4) : ATTEND(float, 8))
                                      : (R == 1 ? ATTEND(bf16, 1) : R == 2 ? ATTEND(bf16, 2) : R == 4 ? ATTEND(bf16, 4) : ATTEND(bf16, 8));
#undef ATTEND
  if (status != 0 || c->parts == 1) return status;
  const long x = (long)c->max_tokens_per_seq * c->n_q;
  if (x > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  const dim3 join((unsigned)x, c->S), threads((c->d + 31) / 32 * 32);
  return c->dtype == PHOTON_F32 ? launch_pdl(kv4_join_kernel<float>, join, threads, 0, stream, a, c->S) : launch_pdl(kv4_join_kernel<bf16>, join, threads, 0, stream, a, c->S);
}
