// Rows of keys and values rounded to 4 bits into the paged cache, and pages of it read back (the format: kv4.cuh).
//
// kv4_write: four lanes have a group of 32 numbers, 8 each; two exchanges give its largest magnitude.  The rounding is the definition's, to the last tie: max / 7 is cut
// to 24 bits with its last bit set where something was cut off, which rounds to 4 bits as the whole quotient would; a number's multiple comes from a product with 1 /
// scale and is put right by what is left over, x - n scale, which is exact.
// kv4_unpack: a thread reads 8 numbers and writes them where they belong.
#include "kv4.cuh"

#define KV4_THREADS 256

// The scale of a group whose largest magnitude is `top`, finite.
__device__ __forceinline__ float kv4_scale_of(float top) {
  float q = __fdiv_rz(top, 7.f);
  if (fmaf(-q, 7.f, top) != 0.f) q = __uint_as_float(__float_as_uint(q) | 1u);
  q = fminf(q, 61440.f);
  const uint32_t e = max(__float_as_uint(q) >> 23, 113u);          // the exponent, 2^-14 at least: steps of 2^-17
  const float magic = __uint_as_float((e + 20u) << 23 | 0x400000u);
  return __fsub_rn(__fadd_rn(q, magic), magic);
}

// x / scale to the nearest whole number, halves to the even one, in -7 .. 7; scale > 0.
__device__ __forceinline__ int kv4_round(float x, float scale, float inv, float half) {
  float n = rintf(fminf(fmaxf(__fmul_rn(x, inv), -8.f), 8.f));
  const float left = fmaf(-n, scale, x), away = fabsf(left);       // exact: x and n scale are as near as that
  const bool odd = (int)n & 1;
  if (away > half || (away == half && odd)) n += left > 0.f ? 1.f : -1.f;
  return (int)fminf(fmaxf(n, -7.f), 7.f) + 8;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint4 u = *(const uint4*)p;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  } else if constexpr (VEC) {
    const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(KV4_THREADS)
kv4_write_kernel(const T* __restrict__ k, long k_stride, const T* __restrict__ v, long v_stride, const int* __restrict__ slot_mapping, uint8_t* __restrict__ k_cache,
                 uint8_t* __restrict__ v_cache, long items, int n_kv, int groups, int page_size, long num_slots, int* err) {
  pdl_wait();
  pdl_launch_dependents();
  const long at = (long)blockIdx.x * (KV4_THREADS / 4) + threadIdx.x / 4;      // (token, plane, head, group)
  const int t = threadIdx.x & 3;
  const bool live = at < items;                      // a warp's lanes stay together for the exchanges
  const long of = live ? at : items - 1;
  const int j = (int)(of % groups);
  const long row = of / groups;
  const int h = (int)(row % n_kv), plane = (int)(row / n_kv % 2);
  const long token = row / n_kv / 2;
  long slot = slot_mapping[token];
  if (slot >= num_slots || slot < -1) {
    if (live && t == 0 && j == 0 && h == 0 && plane == 0) report_error(err, PHOTON_DEV_BAD_SLOT, (int)token, (int)slot, (int)min(num_slots, 0x7fffffffL));
    slot = -1;
  }
  float x[8];
  load8<T, VEC>((plane ? v + token * v_stride : k + token * k_stride) + (h * groups + j) * 32 + 8 * t, x);
  uint32_t top = 0;                                  // magnitudes as whole numbers: a NaN is the largest
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  uint32_t word = 0x88888888u, byte = 255;
  if (top < 0x7f800000u) {
    const float scale = kv4_scale_of(__uint_as_float(top));
    byte = __half_as_ushort(__float2half_rn(scale)) >> 7;
    if (scale > 0.f) {
      const float inv = __frcp_rn(scale), half = 0.5f * scale;
      word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) word |= (uint32_t)kv4_round(x[i], scale, inv, half) << (4 * i);
    }
  }
  if (!live || slot < 0) return;
  const long page = slot / page_size;
  const int place = (int)(slot - page * page_size), d2 = groups * 16;
  uint8_t* base = (plane ? v_cache : k_cache) + (page * n_kv + h) * kv4_page_bytes(page_size, groups * 32);
  uint8_t* codes = base + (long)place * d2;
  if (plane == 0) {
    *(uint32_t*)(codes + 4 * (t * groups + j)) = word;
  } else {
    *(uint16_t*)(codes + 2 * (2 * t * groups + j)) = (uint16_t)word;
    *(uint16_t*)(codes + 2 * ((2 * t + 1) * groups + j)) = (uint16_t)(word >> 16);
  }
  if (t == 0) base[(long)page_size * d2 + place * groups + j] = (uint8_t)byte;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {      // 16-byte aligned
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *(const uint32_t*)&b;
    }
    *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    ((float4*)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    ((float4*)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// Page i of the outputs is page table[i / per * stride + i % per] of the caches.  With cu_tokens: i / per is a request, and only the requests with more than min_rows
// rows (tokens x group) and their pages below context_lens count, and what lies behind their keys is zero; new_table (per wide) gets the outputs' page, or -1;
// positions gets every token's place in its request.  A value that is not finite is laid out as zero then (a weight of 0 would make it a NaN in rows that do not see it), and
// flags [S * per * parts] tells where there was one: kv4_spoil_kernel gives it to the rows that see it.
template <typename T>
__global__ void __launch_bounds__(KV4_THREADS)
kv4_unpack_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int* __restrict__ table, int per, long stride, T* __restrict__ k_out,
                  T* __restrict__ v_out, int n_kv, int groups, int page_size, int num_pages, int parts, const int* __restrict__ cu_tokens,
                  const int* __restrict__ context_lens, int group, int min_rows, int* __restrict__ new_table, int* __restrict__ positions,
                  int* __restrict__ flags, int* err) {
  pdl_wait();
  pdl_launch_dependents();
  const long i = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - i * parts), s = (int)(i / per), p = (int)(i - (long)s * per);
  int end = 0x7fffffff;                              // keys of the request
  if (cu_tokens != nullptr) {
    const int first = cu_tokens[s], n = cu_tokens[s + 1] - first;
    end = context_lens[s];
    if (positions != nullptr && p == 0 && part == 0)
      for (int x = threadIdx.x; x < n; x += KV4_THREADS) positions[first + x] = end - n + x;
    if ((long)n * group <= min_rows || (long)p * page_size >= end) {
      if (new_table != nullptr && part == 0 && threadIdx.x == 0) new_table[i] = -1;
      return;
    }
  }
  const int page = table[s * stride + p];
  const bool bad = page < 0 || page >= num_pages;
  if (part == 0 && threadIdx.x == 0) {
    if (new_table != nullptr) new_table[i] = bad ? -1 : (int)i;
    if (bad) report_error(err, PHOTON_DEV_BAD_PAGE, s, p, page);
  }
  if (bad) return;
  const int words = groups * 4, rows = n_kv * page_size, d = groups * 32;
  const long bytes = kv4_page_bytes(page_size, d);
  const int unit = part * KV4_THREADS + threadIdx.x;            // (plane, head and slot, word)
  const bool live = unit < 2 * rows * words;
  const int plane = live && unit >= rows * words, at = live ? unit - plane * rows * words : 0, row = at / words, w = at - row * words;
  const int h = row / page_size, slot = row - h * page_size;
  const uint8_t* base = (plane ? v_cache : k_cache) + ((long)page * n_kv + h) * bytes;
  const uint8_t* codes = base + (long)slot * groups * 16;
  const int t = w / groups, j = w - t * groups;
  const uint32_t word = plane == 0 ? *(const uint32_t*)(codes + 4 * w)
                                   : *(const uint16_t*)(codes + 2 * (2 * t * groups + j)) | (uint32_t)*(const uint16_t*)(codes + 2 * ((2 * t + 1) * groups + j)) << 16;
  const float scale = kv4_scale(base[(long)page_size * groups * 16 + slot * groups + j]);
  float x[8];
#pragma unroll
  for (int b = 0; b < 8; ++b) x[b] = (long)p * page_size + slot < end ? kv4_code(word, b) * scale : 0.f;
  if (flags != nullptr) {
    const bool odd = live && plane && (long)p * page_size + slot < end && !isfinite(scale);
#pragma unroll
    for (int b = 0; b < 8; ++b) if (odd) x[b] = 0.f;
    const int any = __syncthreads_or(odd);
    if (threadIdx.x == 0) flags[blockIdx.x] = any;
  }
  if (live) store8((plane ? v_out : k_out) + ((i * n_kv + h) * page_size + slot) * d + 32 * j + 8 * t, x);
}

// The rows of the requests with more than min_rows rows that see a value which is not finite: its group's numbers are none either.  One block for each (request, head), which has
// nothing to do but read the flags as a rule.
__global__ void __launch_bounds__(1024)
kv4_spoil_kernel(const uint8_t* __restrict__ v_cache, const int* __restrict__ table, int per, long stride, int n_kv, int groups, int page_size, int num_pages, int parts,
                 const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, int group, int min_rows, const int* __restrict__ flags, bf16* __restrict__ out,
                 long out_stride, int window) {
  pdl_wait();
  const int head = blockIdx.x, s = blockIdx.y, first = cu_tokens[s], n = cu_tokens[s + 1] - first, len = context_lens[s], base = len - n;
  if ((long)n * group <= min_rows) return;
  const int pages = min(per, (len + page_size - 1) / page_size);
  int any = 0;
  for (int i = threadIdx.x; i < pages * parts; i += 1024) any |= flags[(long)s * per * parts + i];
  if (!__syncthreads_or(any)) return;
  for (int key = threadIdx.x; key < min(len, pages * page_size); key += 1024) {
    const int page = table[s * stride + key / page_size];
    if (page < 0 || page >= num_pages) continue;
    const uint8_t* scales = v_cache + ((long)page * n_kv + head) * kv4_page_bytes(page_size, groups * 32) + (long)page_size * groups * 16 + key % page_size * groups;
    for (int j = 0; j < groups; ++j) {
      if (scales[j] < 248) continue;
      const int last = window > 0 && window < n + base - key ? key + window - 1 - base : n - 1;
      for (int i = max(0, key - base); i <= last; ++i)
        for (int x = 0; x < group * 32; ++x)
          out[(first + i) * out_stride + (head * group + x / 32) * groups * 32 + 32 * j + x % 32] = __float2bfloat16_rn(__int_as_float(0x7fc00000));
    }
  }
}

PHOTON_API int photon_kv4_write(const photon_kv4_write_call* c, cudaStream_t stream) {
  if (c->T <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_UNSUPPORTED;
  const int groups = c->d / 32, size = c->dtype == PHOTON_F32 ? 4 : 2;
  const long items = (long)c->T * 2 * c->n_kv * groups, blocks = (items + KV4_THREADS / 4 - 1) / (KV4_THREADS / 4);
  if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  const bool vec = ((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)(c->k_stride * size) | (uintptr_t)(c->v_stride * size)) % 16 == 0;
#define WRITE(T, VEC) launch_pdl(kv4_write_kernel<T, VEC>, dim3((unsigned)blocks), dim3(KV4_THREADS), 0, stream, (const T*)c->k, c->k_stride, (const T*)c->v, c->v_stride, \
                                 c->slot_mapping, (uint8_t*)c->k_cache, (uint8_t*)c->v_cache, items, c->n_kv, groups, c->page_size, (long)c->num_pages * c->page_size, c->err)
  if (c->dtype == PHOTON_F32) return vec ? WRITE(float, true) : WRITE(float, false);
  return vec ? WRITE(bf16, true) : WRITE(bf16, false);
#undef WRITE
}

PHOTON_API int photon_kv4_unpack(const photon_kv4_unpack_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->per <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)c->k_out | (uintptr_t)c->v_out) % 16) return PHOTON_ERR_ARGUMENT;
  const long units = 2L * c->n_kv * c->page_size * (c->d / 8), parts = (units + KV4_THREADS - 1) / KV4_THREADS, blocks = parts * c->S * c->per;
  if (units > 0x7fffffffL || blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
#define UNPACK(T) launch_pdl(kv4_unpack_kernel<T>, dim3((unsigned)blocks), dim3(KV4_THREADS), 0, stream, (const uint8_t*)c->k_cache, (const uint8_t*)c->v_cache, c->table, \
                             c->per, c->stride, (T*)c->k_out, (T*)c->v_out, c->n_kv, c->d / 32, c->page_size, c->num_pages, (int)parts, c->cu_tokens, c->context_lens, \
                             c->group, c->min_rows, c->new_table, c->positions, c->cu_tokens != nullptr ? c->flags : nullptr, c->err)
  return c->dtype == PHOTON_F32 ? UNPACK(float) : UNPACK(bf16);
#undef UNPACK
}

PHOTON_API int photon_kv4_spoil(const photon_kv4_unpack_call* c, void* out, long out_stride, int window, cudaStream_t stream) {
  if (c->S <= 0 || c->per <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->flags == nullptr || c->cu_tokens == nullptr || !kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_ARGUMENT;
  if (c->S > 65535) return PHOTON_ERR_UNSUPPORTED;
  const long units = 2L * c->n_kv * c->page_size * (c->d / 8), parts = (units + KV4_THREADS - 1) / KV4_THREADS;
  return launch_pdl(kv4_spoil_kernel, dim3(c->n_kv, c->S), dim3(1024), 0, stream, (const uint8_t*)c->v_cache, c->table, c->per, c->stride, c->n_kv, c->d / 32, c->page_size,
                    c->num_pages, (int)parts, c->cu_tokens, c->context_lens, c->group, c->min_rows, (const int*)c->flags, (bf16*)out, out_stride, window);
}
