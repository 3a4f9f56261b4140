// Attention over a paged cache in 4 bits (the format: kv4.cuh) for many rows (tokens x query heads of a key/value head) a request, with products in 32 bits: either type, any head
// of up to 256 numbers, any page.  Rows, masks and what is not finite: as in kv4_attention.cu.
//
// A block has 64 rows and a share of their keys, 128 at a time.  Scores: 32 numbers of the rows and of the keys at a time in shared memory, in 32 bits, the next ones on their way in
// registers; a thread has the products of 4 rows and 8 keys, and 16 lanes have a row's.  Weights, turned over in shared memory, meet the values a few keys at a time: a thread has
// 4 rows and 4 NV numbers of the result.  A value that is not finite lies there as zero, since a weight of 0 would make it a NaN in rows that do not see it; a tile with such a value
// is looked through once more for the rows that do.
//
// What bounds it: the products, at 0.3 of the rate of 32-bit sums: three 16-byte reads of shared memory for 32 of them, barriers between pieces, and blocks of which some SMs have two and
// some one.  32 query heads on 8, 32 bits: 200 tokens behind 4,000, heads of 128, 733 us (kv4_attention.cu 1,004; the framework's kernel for plain caches, with pages laid out, 1,094);
// 256 of 2 requests behind 8,192, heads of 64, 1,648 (2,890; 1,503).
#include "kv4_attention.cuh"

#define KR_THREADS 256
#define KR_ROWS 64
#define KR_KEYS 128
#define KR_PIECE 32              // numbers of rows and keys in shared memory at a time
#define KR_KEY_PITCH 132
#define KR_PITCH 68

// NV: heads of up to 64 NV numbers.
template <typename T, int NV>
__global__ void __launch_bounds__(KR_THREADS, NV == 4 ? 1 : 2)
kv4_attention_rows_kernel(const Kv4Args a) {
  constexpr int W = 64 * NV, SOME = NV == 4 ? 16 : 32, WORDS = SOME * (W / 8) / KR_THREADS;      // keys whose values are in shared memory at a time; a thread's words of them
  extern __shared__ __align__(16) float kr_smem[];
  float *p_s = kr_smem, *k_s = p_s + KR_KEYS * KR_PITCH, *q_s = k_s + KR_PIECE * KR_KEY_PITCH, *v_s = k_s;
  static_assert(SOME * W <= KR_PIECE * (KR_KEY_PITCH + KR_PITCH), "values lie where rows and keys were");
  __shared__ int place_s[KR_ROWS], there_s[KR_KEYS], slot_s[KR_KEYS], odd_s;
  __shared__ long page_s[KR_KEYS];                    // (page, head) of a key, counted through
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y % a.n_kv, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kt = lane & 15, rt = 2 * warp + (lane >> 4);
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq];
  const int G = a.n_q / a.n_kv, all = n * G, row0 = (int)(blockIdx.y / a.n_kv) * KR_ROWS;
  if (row0 >= all || all > a.max_rows) return;
  const int groups = a.groups, rows = min(KR_ROWS, all - row0), d = groups * 32, base = ctx - n;
  const int last_place = base + (row0 + rows - 1) / G, first_place = base + row0 / G;
  const int lo = a.window > 0 ? max(0, first_place - a.window + 1) : 0, hi = max(lo, last_place + 1);
  const int tiles = (hi - lo + KR_KEYS - 1) / KR_KEYS, per = (tiles + a.parts - 1) / a.parts;
  const int from = lo + min(part * per, tiles) * KR_KEYS, to = min(hi, lo + min((part + 1) * per, tiles) * KR_KEYS);
  const long bytes = kv4_page_bytes(a.page_size, d);
  if (tid < KR_ROWS) place_s[tid] = tid < rows ? base + (row0 + tid) / G : -1;
  float m[4], l[4], out[4][4 * NV];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) out[r][i] = 0.f;
  }
  auto key_at = [&](int e) { return e < 4 ? 4 * kt + e : 60 + 4 * kt + e; };
  for (int k0 = from; k0 < to; k0 += KR_KEYS) {
    __syncthreads();                                  // the tile in front of this one is done with
    if (tid < KR_KEYS) {
      const int key = k0 + tid, pidx = key / a.page_size;
      int page = -1;
      if (key < to) {
        page = pidx < a.max_pages ? a.table[(long)seq * a.max_pages + pidx] : -1;
        if (page < 0 || page >= a.num_pages) {
          report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, key, page);
          page = -1;
        }
      }
      there_s[tid] = page >= 0;
      slot_s[tid] = key - pidx * a.page_size;
      page_s[tid] = (long)page * a.n_kv + head;
    }
    if (tid == 0) odd_s = 0;
    __syncthreads();
    // ---- products of rows and keys
    float acc[4][8];
    {
      const int p = tid & 7, g = tid >> 3;            // numbers 4 p .. of keys 4 g ..; number `lane` of rows 8 warp ..
      float k[4][4];
      T x[8];                                         // as they come: whoever looks at one waits for it
      auto load = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 4 * g + i;
#pragma unroll
          for (int j = 0; j < 4; ++j) k[i][j] = 0.f;
          if (there_s[key] == 0) continue;
          const int slot = slot_s[key];               // word t groups + c has numbers 8 t .. of the group
          const uint8_t* page = a.k + page_s[key] * bytes;
          const float scale = kv4_scale(page[(long)a.page_size * (d / 2) + slot * groups + c]);
          const uint32_t word = ((const uint32_t*)(page + (long)slot * (d / 2)))[(p >> 1) * groups + c];
#pragma unroll
          for (int j = 0; j < 4; ++j) k[i][j] = kv4_code(word >> (16 * (p & 1)), j) * scale;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 8 * warp + i, row = row0 + min(r, rows - 1), token = row / G;
          x[i] = r < rows ? ((const T*)a.q)[(first + token) * a.q_stride + (long)(head * G + row - token * G) * d + KR_PIECE * c + lane] : from_f32<T>(0.f);
        }
      };
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[r][e] = 0.f;
      load(0);
      for (int c = 0; c < groups; ++c) {
        __syncthreads();                              // the piece in front of this one is done with
#pragma unroll
        for (int j = 0; j < 4; ++j) *(float4*)&k_s[(4 * p + j) * KR_KEY_PITCH + 4 * g] = make_float4(k[0][j], k[1][j], k[2][j], k[3][j]);
#pragma unroll
        for (int i = 0; i < 8; i += 4) *(float4*)&q_s[lane * KR_PITCH + 8 * warp + i] = make_float4(kv4_query(x[i]), kv4_query(x[i + 1]), kv4_query(x[i + 2]), kv4_query(x[i + 3]));
        __syncthreads();
        if (c + 1 < groups) load(c + 1);
#pragma unroll 8
        for (int i = 0; i < KR_PIECE; ++i) {
          const float4 u = *(const float4*)&k_s[i * KR_KEY_PITCH + 4 * kt], v = *(const float4*)&k_s[i * KR_KEY_PITCH + 64 + 4 * kt], z = *(const float4*)&q_s[i * KR_PITCH + 4 * rt];
          const float b[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w}, y[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(b[e], y[r], acc[r][e]);
        }
      }
    }
    // ---- weights
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int place = place_s[4 * rt + r];
      float top = -INFINITY;
      bool seen[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = k0 + key_at(e);
        seen[e] = there_s[key_at(e)] != 0 && key <= place && (a.window <= 0 || key > place - a.window);
        acc[r][e] = seen[e] ? kv4_bounded(acc[r][e], a.scale, a.softcap) : -INFINITY;
        top = fmaxf(top, acc[r][e]);
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmaxf(top, m[r]);
      const float alpha = m[r] == -INFINITY ? 1.f : exp2f(m[r] - top), ref = top == -INFINITY ? 0.f : top;      // nothing but what is no number can have been added yet
      m[r] = top;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        acc[r][e] = seen[e] ? exp2f(acc[r][e] - ref) : 0.f;
        sum += acc[r][e];
      }
      l[r] = l[r] * alpha + sum;
#pragma unroll
      for (int i = 0; i < 4 * NV; ++i) out[r][i] *= alpha;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) *(float4*)&p_s[key_at(e) * KR_PITCH + 4 * rt] = make_float4(acc[0][e], acc[1][e], acc[2][e], acc[3][e]);
    // ---- weights by values
    const int here = min(KR_KEYS, to - k0);
    uint32_t words[WORDS], scales[WORDS];             // two half words of 4 numbers, and their scales
    auto ask = [&](int x0) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const int at = i * KR_THREADS + tid, key = x0 + at / (W / 8), w = at % (W / 8);
        words[i] = 0x88888888u;
        scales[i] = 0u;
        if (8 * w >= d || there_s[key] == 0) continue;
        const int slot = slot_s[key];
        const uint8_t* page = a.v + page_s[key] * bytes;
        const uint8_t* sc = page + (long)a.page_size * (d / 2) + slot * groups;
        words[i] = ((const uint32_t*)(page + (long)slot * (d / 2)))[w];
        scales[i] = sc[2 * w % groups] | (uint32_t)sc[(2 * w + 1) % groups] << 8;
      }
    };
    ask(0);
    for (int x0 = 0; x0 < here; x0 += SOME) {
      __syncthreads();                                // weights are there; keys, or the values in front of these, are done with
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        const int at = i * KR_THREADS + tid, w = at % (W / 8);
        float* to_s = v_s + at / (W / 8) * W;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int hw = 2 * w + h, g = hw / groups, j = hw - g * groups;
          const uint32_t byte = scales[i] >> (8 * h) & 255u;
          const bool odd = byte >= 248u;
          if (odd) odd_s = 1;
          const float scale = odd ? 0.f : kv4_scale(byte);
          float4 v;
          v.x = kv4_code(words[i], 4 * h) * scale;
          v.y = kv4_code(words[i], 4 * h + 1) * scale;
          v.z = kv4_code(words[i], 4 * h + 2) * scale;
          v.w = kv4_code(words[i], 4 * h + 3) * scale;
          *(float4*)&to_s[8 * w < d ? 32 * j + 4 * g : 8 * w + 4 * h] = v;
        }
      }
      __syncthreads();
      if (x0 + SOME < here) ask(x0 + SOME);
#pragma unroll 8
      for (int x = 0; x < SOME; ++x) {
        const float4 z = *(const float4*)&p_s[(x0 + x) * KR_PITCH + 4 * rt];
        const float y[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const float4 u = *(const float4*)&v_s[x * W + 64 * i + 4 * kt];
          const float b[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) out[r][4 * i + j] = fmaf(y[r], b[j], out[r][4 * i + j]);
        }
      }
    }
    if (odd_s != 0) {
      for (int x = 0; x < here; ++x) {
        if (there_s[x] == 0) continue;
        const uint8_t* sc = a.v + page_s[x] * bytes + (long)a.page_size * (d / 2) + slot_s[x] * groups;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (64 * i + 4 * kt >= d || sc[(64 * i + 4 * kt) / 32] < 248) continue;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int place = place_s[4 * rt + r];
            if (k0 + x > place || (a.window > 0 && k0 + x <= place - a.window)) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) out[r][4 * i + j] = NAN;
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float total = l[r], top = m[r], mul = 1.f;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (4 * rt + r >= rows) continue;
    const int row = row0 + 4 * rt + r, h = head * G + row % G;
    const long token = first + row / G, of = token * a.n_q + h;
    if (a.parts == 1) {
      if (a.sinks != nullptr) {
        const float sink = a.sinks[h] * 1.4426950408889634f, both = fmaxf(top, sink);
        mul = top == -INFINITY ? 1.f : exp2f(top - both);
        if (sink != -INFINITY) total = total * mul + exp2f(sink - both);
        top = both;
      }
      if (kt == 0 && a.lse != nullptr) a.lse[of] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
      mul = total == 0.f ? 0.f : mul / total;
    } else if (kt == 0) {
      a.scratch[(of * a.parts + part) * (d + 2) + d] = top;
      a.scratch[(of * a.parts + part) * (d + 2) + d + 1] = total;
    }
#pragma unroll
    for (int i = 0; i < 4 * NV; ++i) {
      const int at = 64 * (i / 4) + 4 * kt + i % 4;
      if (at >= d) continue;
      if (a.parts == 1) ((T*)a.out)[token * a.out_stride + h * d + at] = from_f32<T>(mul == 0.f ? 0.f : out[r][i] * mul);
      else a.scratch[(of * a.parts + part) * (d + 2) + at] = out[r][i];
    }
  }
}

template <typename T, int NV>
static int kr_launch(const Kv4Args& a, dim3 grid, cudaStream_t stream) {
  constexpr size_t smem = (KR_KEYS * KR_PITCH + KR_PIECE * (KR_KEY_PITCH + KR_PITCH)) * sizeof(float);
  static bool ready[64] = {};
  const int limit = smem_limit((const void*)kv4_attention_rows_kernel<T, NV>, (int)smem, false, ready);
  if (limit != 0) return limit;
  return launch_pdl(kv4_attention_rows_kernel<T, NV>, grid, dim3(KR_THREADS), smem, stream, a);
}

PHOTON_API int photon_kv4_attention_rows(const photon_kv4_attention_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_UNSUPPORTED;
  if (c->parts < 1 || (c->parts > 1 && c->scratch == nullptr)) return PHOTON_ERR_ARGUMENT;
  const Kv4Args a = {c->q, c->out, (const uint8_t*)c->k_cache, (const uint8_t*)c->v_cache, c->block_table, c->cu_tokens, c->context_lens, c->sinks, c->lse, c->scratch, c->err,
                     c->q_stride, c->out_stride, c->max_pages, c->n_q, c->n_kv, c->d / 32, c->page_size, c->num_pages, c->window, c->parts, c->scale, c->softcap, c->max_rows};
  const long rows = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv), y = (rows + KR_ROWS - 1) / KR_ROWS * c->n_kv, x = (long)c->max_tokens_per_seq * c->n_q;
  if (c->S > 65535 || y > 65535 || x > 0x7fffffffL || c->scale <= 0.f) return PHOTON_ERR_UNSUPPORTED;
  const dim3 grid(c->parts, (unsigned)y, c->S);
#define ATTEND(T) (c->d <= 64 ? kr_launch<T, 1>(a, grid, stream) : c->d <= 128 ? kr_launch<T, 2>(a, grid, stream) : kr_launch<T, 4>(a, grid, stream))
  const int status = c->dtype == PHOTON_F32 ? ATTEND(float) : ATTEND(bf16);
#undef ATTEND
  if (status != 0 || c->parts == 1) return status;
  const dim3 join((unsigned)x, c->S), threads((c->d + 31) / 32 * 32);
  return c->dtype == PHOTON_F32 ? launch_pdl(kv4_join_kernel<float>, join, threads, 0, stream, a, c->S) : launch_pdl(kv4_join_kernel<bf16>, join, threads, 0, stream, a, c->S);
}
