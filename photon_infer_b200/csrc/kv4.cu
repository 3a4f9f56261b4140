// Rows of keys and values rounded to 4 bits into the paged cache, and pages of it read back (the format: kv4.cuh).
//
// kv4_write: two lanes have a group of 32 numbers, 16 each; an exchange gives its largest magnitude.  The rounding is the definition's, to the last tie.  In 32 bits max / 7 is
// cut to 24 bits with its last bit set where something was cut off, which rounds to 4 bits as the whole quotient would.  A bfloat16 number's quotient by the scale, 8 bits by 4, is a
// half and something or at least 2^-10 away from one: x / scale rounded to multiples of 2^-12 lies where the quotient lies, and a half on the half (max / 7 likewise, to 2^-9 of a
// step, where 2^-6 is the least).  For 32 bits the multiple from that product is put right by what is left over, x - n scale, which is exact.
// kv4_unpack: a thread reads a quarter of a row, 8 numbers of every group, and writes them where they belong.
//
// What bounds it: the instructions of the rounding.  8,191 rows of keys and values, 8 heads of 128, written, and their pages read back: 21 us, 85 MB, 0.6 of the copy rate (in 32 bits 42 us); one row of 8
// heads of 64 and its page: 3.2 us, launches and rounds of latencies.  With one thread for a group and quotients by division it was 57 us.  Pages of 6,144 keys laid out for the tcgen05 kernel: 12 us
// of a portion's 187.
#include "kv4.cuh"

#define KV4_THREADS 256
#define KV4_SPOIL_TOKENS 64      // of a block: two of a lane

// The scale of a group whose largest magnitude is `top`, finite.
template <typename T>
__device__ __forceinline__ float kv4_scale_of(float top) {
  float q;
  if constexpr (sizeof(T) == 2) {
    q = __fmul_rn(top, 0.14285714924335479736328125f);
  } else {
    q = __fdiv_rz(top, 7.f);
    if (fmaf(-q, 7.f, top) != 0.f) q = __uint_as_float(__float_as_uint(q) | 1u);
  }
  q = fminf(q, 61440.f);
  const uint32_t e = max(__float_as_uint(q) >> 23, 113u);          // the exponent, 2^-14 at least: steps of 2^-17
  const float magic = __uint_as_float((e + 20u) << 23 | 0x400000u);
  if constexpr (sizeof(T) == 2) {                                   // to 2^-9 of a step first
    const float fine = __uint_as_float((e + 11u) << 23 | 0x400000u);
    q = __fsub_rn(__fadd_rn(q, fine), fine);
  }
  return __fsub_rn(__fadd_rn(q, magic), magic);
}

// x / scale to the nearest whole number, halves to the even one, -7 to 7, plus 8, as a number; scale > 0, inv = 1 / scale.
template <typename T>
__device__ __forceinline__ float kv4_round(float x, float scale, float inv) {
  constexpr float WHOLE = 12582912.f;                              // 1.5 * 2^23: its last bit is 1
  if constexpr (sizeof(T) == 2) {
    constexpr float FINE = 1.5f * 2048.f;                          // its last bit is 2^-12
    const float y = __fsub_rn(__fmaf_rn(x, inv, FINE), FINE);
    return __fsub_rn(__fadd_rn(fminf(fmaxf(y, -7.f), 7.f), WHOLE), WHOLE - 8.f);
  } else {
    float n = __fsub_rn(__fadd_rn(fminf(fmaxf(__fmul_rn(x, inv), -8.f), 8.f), WHOLE), WHOLE);
    const float left = fmaf(-n, scale, x), away = fabsf(left), half = 0.5f * scale;      // exact: x and n scale are as near as that
    if (away > half || (away == half && ((int)n & 1))) n += left > 0.f ? 1.f : -1.f;
    return fminf(fmaxf(n, -7.f), 7.f) + 8.f;
  }
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

// A token's items: (plane, head, group, half of the group); `tokens` of them a block.
template <typename T, bool VEC, int GROUPS>
__global__ void __launch_bounds__(KV4_THREADS)
kv4_write_kernel(const T* __restrict__ k, long k_stride, const T* __restrict__ v, long v_stride, const int* __restrict__ slot_mapping, uint8_t* __restrict__ k_cache,
                 uint8_t* __restrict__ v_cache, int T_all, int n_kv, int page_size, int page_shift, long num_slots, int per_token, int* err) {
  pdl_wait();
  pdl_launch_dependents();
  // several tokens a block (threadIdx.y), or a token's items in rounds of the block's threads (blockIdx.y)
  const int token = blockIdx.x * blockDim.y + threadIdx.y, item = blockIdx.y * blockDim.x + threadIdx.x;
  const bool there = token < T_all;
  long slot = there ? slot_mapping[token] : -1;
  if (slot >= num_slots || slot < -1) {
    if (item == 0) report_error(err, PHOTON_DEV_BAD_SLOT, token, (int)slot, (int)min(num_slots, 0x7fffffffL));
    slot = -1;
  }
  const bool live = there && item < per_token;         // a warp's lanes stay together for the exchanges
  const int half = item & 1, j = (item >> 1) % GROUPS, row = (item >> 1) / GROUPS, plane = row >= n_kv, h = row - plane * n_kv;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  if (live) {
    const T* from = (plane ? v + token * v_stride : k + token * k_stride) + (h * GROUPS + j) * 32 + 16 * half;
    load8<T, VEC>(from, x);
    load8<T, VEC>(from + 8, x + 8);
  }
  uint32_t top = 0;                                  // magnitudes as whole numbers: a NaN is the largest
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  uint32_t word[2] = {0x88888888u, 0x88888888u}, byte = 255;
  if (top < 0x7f800000u) {
    const float scale = kv4_scale_of<T>(__uint_as_float(top));
    byte = __half_as_ushort(__float2half_rn(scale)) >> 7;
    if (scale > 0.f) {
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        uint32_t part[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {                  // four codes as one whole number below 2^16
          const float* y = x + 8 * w + 4 * q;
          float sum = kv4_round<T>(y[3], scale, inv);
#pragma unroll
          for (int i = 2; i >= 0; --i) sum = __fmaf_rn(sum, 16.f, kv4_round<T>(y[i], scale, inv));
          part[q] = __float_as_uint(__fadd_rn(sum, 8388608.f));
        }
        word[w] = __byte_perm(part[0], part[1], 0x5410);
      }
    }
  }
  uint8_t *base = nullptr, *codes = nullptr;
  const int d2 = GROUPS * 16;
  int place = 0;
  if (live && slot >= 0) {
    const int at = (int)slot, page = page_shift >= 0 ? at >> page_shift : at / page_size;
    place = at - page * page_size;
    base = (plane ? v_cache : k_cache) + ((long)page * n_kv + h) * ((long)page_size * GROUPS * 17);
    codes = base + place * d2;
  }
  if constexpr (GROUPS % 2 == 0) {
    // the neighbouring group's half words beside this one's: the even group has the values' first two eights, the odd one the others
    // half words of g = 4 half + 0, 1 | 2, 3: word[0] has 0 and 1, word[1] has 2 and 3
    const uint32_t other = __shfl_xor_sync(0xffffffffu, j & 1 ? word[0] : word[1], 2);
    if (codes != nullptr) {
      if (plane == 0) {
        *(uint32_t*)(codes + 4 * (2 * half * GROUPS + j)) = word[0];
        *(uint32_t*)(codes + 4 * ((2 * half + 1) * GROUPS + j)) = word[1];
      } else {
        const uint32_t a = j & 1 ? other : word[0], b = j & 1 ? word[1] : other;      // of the even group, of the odd one
        const int g = 4 * half + 2 * (j & 1);
        *(uint32_t*)(codes + 2 * (g * GROUPS + (j & ~1))) = __byte_perm(a, b, 0x5410);
        *(uint32_t*)(codes + 2 * ((g + 1) * GROUPS + (j & ~1))) = __byte_perm(a, b, 0x7632);
      }
    }
  } else if (codes != nullptr) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int t = 2 * half + w;
      if (plane == 0) {
        *(uint32_t*)(codes + 4 * (t * GROUPS + j)) = word[w];
      } else {
        *(uint16_t*)(codes + 2 * (2 * t * GROUPS + j)) = (uint16_t)word[w];
        *(uint16_t*)(codes + 2 * ((2 * t + 1) * GROUPS + j)) = (uint16_t)(word[w] >> 16);
      }
    }
  }
  if (codes != nullptr && half == 0) base[(long)page_size * d2 + place * GROUPS + j] = (uint8_t)byte;
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

// Page blockIdx.x of the outputs is page table[i / per * stride + i % per] of the caches; blockIdx.y has a part of its (plane, head, slot, t).  With cu_tokens: i / per is a request, and
// only the requests with more than min_rows rows (tokens x group) and their pages below context_lens and, with a window, not wholly in front of the first token's count, and what lies behind their keys is zero; new_table (per wide) gets the
// outputs' page, or -1; positions gets every token's place in its request.  A value that is not finite is laid out as zero then (a weight of 0 would make it a NaN in rows that
// do not see it), and flags [S * per * gridDim.y] tells where there was one: kv4_spoil_kernel gives it to the rows that see it.
template <typename T, int GROUPS>
__global__ void __launch_bounds__(KV4_THREADS)
kv4_unpack_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, const int* __restrict__ table, int per, long stride, T* __restrict__ k_out,
                  T* __restrict__ v_out, int n_kv, int page_size, int page_shift, int num_pages, const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, int group,
                  int min_rows, int window, int* __restrict__ new_table, int* __restrict__ positions, int* __restrict__ flags, int* err) {
  constexpr int D = GROUPS * 32;
  pdl_wait();
  pdl_launch_dependents();
  const int i = blockIdx.x, s = per == (int)gridDim.x ? 0 : i / per, p = i - s * per;
  int end = 0x7fffffff;                              // keys of the request
  if (cu_tokens != nullptr) {
    const int first = cu_tokens[s], n = cu_tokens[s + 1] - first;
    end = context_lens[s];
    if (positions != nullptr && p == 0 && blockIdx.y == 0)
      for (int x = threadIdx.x; x < n; x += KV4_THREADS) positions[first + x] = end - n + x;
    // pages in front of the window are not asked for: they may have been given back
    if ((long)n * group <= min_rows || (long)p * page_size >= end || (window > 0 && (p + 1L) * page_size <= (long)end - n - window + 1)) {
      if (new_table != nullptr && blockIdx.y == 0 && threadIdx.x == 0) new_table[i] = -1;
      return;
    }
  }
  const int page = table[s * stride + p];
  const bool bad = page < 0 || page >= num_pages;
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    if (new_table != nullptr) new_table[i] = bad ? -1 : i;
    if (bad) report_error(err, PHOTON_DEV_BAD_PAGE, s, p, page);
  }
  if (bad) {
    if (flags != nullptr && threadIdx.x == 0) flags[(long)i * gridDim.y + blockIdx.y] = 0;
    return;
  }
  // lane t of four has bytes 4 t GROUPS .. of a row: 8 numbers of every group, whichever plane
  const int unit = blockIdx.y * KV4_THREADS + threadIdx.x, t = unit & 3, row = unit >> 2, ph = page_shift >= 0 ? row >> page_shift : row / page_size, slot = row - ph * page_size;
  bool odd = false;
  if (ph < 2 * n_kv) {
    const bool plane = ph >= n_kv;
    const int h = plane ? ph - n_kv : ph;
    const uint8_t* base = (plane ? v_cache : k_cache) + ((long)page * n_kv + h) * ((long)page_size * GROUPS * 17);
    const uint8_t* codes = base + (long)slot * (GROUPS * 16) + 4 * GROUPS * t;
    const uint8_t* scales = base + (long)page_size * GROUPS * 16 + slot * GROUPS;
    T* out = (plane ? v_out : k_out) + (((long)i * n_kv + h) * page_size + slot) * D + 8 * t;
    uint32_t w[GROUPS];
    uint8_t b[GROUPS];
    if constexpr (GROUPS % 4 == 0) {
#pragma unroll
      for (int j = 0; j < GROUPS; j += 4) {
        const uint4 u = *(const uint4*)(codes + 4 * j);
        w[j] = u.x; w[j + 1] = u.y; w[j + 2] = u.z; w[j + 3] = u.w;
        const uint32_t x = *(const uint32_t*)(scales + j);
#pragma unroll
        for (int c = 0; c < 4; ++c) b[j + c] = (uint8_t)(x >> (8 * c));
      }
    } else if constexpr (GROUPS == 2) {
      const uint2 u = *(const uint2*)codes;
      w[0] = u.x; w[1] = u.y;
      const uint16_t x = *(const uint16_t*)scales;
      b[0] = (uint8_t)x; b[1] = (uint8_t)(x >> 8);
    } else {
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) { w[j] = *(const uint32_t*)(codes + 4 * j); b[j] = scales[j]; }
    }
    const bool behind = (long)p * page_size + slot >= end;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      uint32_t word = w[j];
      if (plane) {                                   // half word j of the first half, half word j of the second
        const uint32_t lo = w[j / 2] >> (16 * (j & 1)), hi = w[(GROUPS + j) / 2] >> (16 * ((GROUPS + j) & 1));
        word = __byte_perm(lo, hi, 0x5410);
      }
      const float scale = kv4_scale(b[j]);
      const bool none = flags != nullptr && plane && !behind && !isfinite(scale);
      odd |= none;
      float y[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) y[c] = behind || none ? 0.f : kv4_code(word, c) * scale;
      store8(out + 32 * j, y);
    }
  }
  if (flags != nullptr) {
    const int any = __syncthreads_or(odd);
    if (threadIdx.x == 0) flags[(long)i * gridDim.y + blockIdx.y] = any;
  }
}

// The rows of the requests with more than min_rows rows that see a value which is not finite: its group's numbers are none either.  Rows whose query is not finite, too, if they see a key, and
// else none: where all their scores are minus infinity they are zero now, else NaN, which is what is looked for; where scores are bounded they can be any number, so that all queries are looked at.
// A block has 64 tokens of a (request, head), and nothing to do but read its keys' flags and the rows' first numbers as a rule: 5 of the 187 us of 2,048 tokens behind 6,144 keys.  Else it finds, for every group and
// token, the last broken key at or before the token's place, which decides for any window, and writes each number once.
__global__ void __launch_bounds__(KV4_THREADS)
kv4_spoil_kernel(const uint8_t* __restrict__ v_cache, const int* __restrict__ table, int per, long stride, int n_kv, int groups, int page_size, int num_pages,
                 const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, int group, int min_rows, int parts, const int* __restrict__ flags, bf16* out,
                 long out_stride, const bf16* __restrict__ q, long q_stride, int window, bool bounded) {
  __shared__ int last_s[8][KV4_SPOIL_TOKENS];
  __shared__ uint32_t odd_s[KV4_SPOIL_TOKENS * 128 / 32];      // rows (tokens x query heads, at most 128) whose query is not finite
  pdl_wait();
  const int head = blockIdx.x, s = blockIdx.y, first = cu_tokens[s], n = cu_tokens[s + 1] - first, len = context_lens[s], base = len - n, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((long)n * group <= min_rows) return;
  const int pages = min(per, (max(len, 0) + page_size - 1) / page_size);
  for (int t0 = blockIdx.z * KV4_SPOIL_TOKENS; t0 < n; t0 += gridDim.z * KV4_SPOIL_TOKENS) {
    const int tokens = min(KV4_SPOIL_TOKENS, n - t0), place0 = base + t0, place1 = place0 + tokens - 1;
    if (place1 < 0) continue;
    const int low = window > 0 ? max(0, place0 - window + 1) : 0, page0 = low / page_size, page1 = min(pages, place1 / page_size + 1);
    for (int i = tid; i < (tokens * group + 31) / 32; i += KV4_THREADS) odd_s[i] = 0;
    __syncthreads();
    int any = 0;
    for (int row = tid; row < tokens * group; row += KV4_THREADS) {
      const int t = row / group, h = head * group + row - t * group;
      if (!bounded) {
        const uint4 u = *(const uint4*)(out + (first + t0 + t) * out_stride + (long)h * groups * 32);
        if (((u.x | u.y | u.z | u.w) & 0x7fff7fffu) != 0 && (u.x & 0x7fffu) <= 0x7f80u) continue;
      }
      const uint4* query = (const uint4*)(q + (first + t0 + t) * q_stride + (long)h * groups * 32);
      uint32_t carry = 0;                              // the exponent's bits all set: one more of them carries into the bit in front of them, which the mask has cleared
#pragma unroll 4
      for (int i = 0; i < groups * 4; ++i) {
        const uint4 u = query[i];
        carry |= ((u.x & 0x7f807f80u) + 0x00800080u) | ((u.y & 0x7f807f80u) + 0x00800080u) | ((u.z & 0x7f807f80u) + 0x00800080u) | ((u.w & 0x7f807f80u) + 0x00800080u);
      }
      if ((carry & 0x80008000u) == 0) continue;
      atomicOr(&odd_s[row >> 5], 1u << (row & 31));
      any = 1;
    }
    for (long i = ((long)s * per + page0) * parts + tid; i < ((long)s * per + page1) * parts; i += KV4_THREADS) any |= flags[i];
    if (!__syncthreads_or(any)) continue;
    for (int i = tid; i < groups * KV4_SPOIL_TOKENS; i += KV4_THREADS) last_s[i / KV4_SPOIL_TOKENS][i % KV4_SPOIL_TOKENS] = -1;
    __syncthreads();
    for (int key = low + tid; key <= place1 && key / page_size < page1; key += KV4_THREADS) {
      const int page = table[s * stride + key / page_size];
      if (page < 0 || page >= num_pages) continue;
      const uint8_t* scales = v_cache + ((long)page * n_kv + head) * kv4_page_bytes(page_size, groups * 32) + (long)page_size * groups * 16 + key % page_size * groups;
      for (int j = 0; j < groups; ++j) if (scales[j] >= 248) atomicMax(&last_s[j][max(0, key - place0)], key);
    }
    __syncthreads();
    if (warp < groups) {                               // the largest up to every token: a lane has two
      const int a = last_s[warp][2 * lane], b = max(a, last_s[warp][2 * lane + 1]);
      int upto = b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto = max(upto, x);
      }
      const int before = __shfl_up_sync(0xffffffffu, upto, 1);
      last_s[warp][2 * lane] = lane > 0 ? max(a, before) : a;
      last_s[warp][2 * lane + 1] = upto;
    }
    __syncthreads();
    for (int i = tid; i < tokens * group * groups * 4; i += KV4_THREADS) {      // 8 numbers of a (token, query head, group)
      const int at = i >> 2, j = at % groups, row = at / groups, t = row / group, last = last_s[j][t], place = place0 + t;
      uint32_t is = 0x7fc07fc0u;
      if (odd_s[row >> 5] >> (row & 31) & 1u) {
        bool sees = false;                             // a key that is there
        for (int p = place < 0 ? -1 : min(place / page_size, pages - 1); !sees && p >= (window > 0 ? max(0, place - window + 1) : 0) / page_size; --p) {
          const int page = table[s * stride + p];
          sees = page >= 0 && page < num_pages;
        }
        if (!sees) is = 0u;
      } else if (last < 0 || (window > 0 && last <= place - window)) {
        continue;
      }
      *(uint4*)(out + (first + t0 + t) * out_stride + ((long)(head * group + row - t * group) * groups + j) * 32 + 8 * (i & 3)) = make_uint4(is, is, is, is);
    }
    __syncthreads();                                   // what was found is done with
  }
}

PHOTON_API int photon_kv4_write(const photon_kv4_write_call* c, cudaStream_t stream) {
  if (c->T <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_UNSUPPORTED;
  const int groups = c->d / 32, size = c->dtype == PHOTON_F32 ? 4 : 2, per_token = 4 * c->n_kv * groups, tokens = per_token <= KV4_THREADS / 2 && c->T > 1 ? KV4_THREADS / 32 * 32 / per_token : 1;
  const long slots = (long)c->num_pages * c->page_size;
  if (c->n_kv > 65536 || slots > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  const bool vec = ((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)(c->k_stride * size) | (uintptr_t)(c->v_stride * size)) % 16 == 0;
  const dim3 grid((c->T + tokens - 1) / tokens, tokens > 1 ? 1 : (per_token + KV4_THREADS - 1) / KV4_THREADS), block(tokens > 1 ? per_token : KV4_THREADS, tokens);
  int shift = -1;
  for (int i = 0; i < 31; ++i) if (c->page_size == 1 << i) shift = i;
#define WRITE(TYPE, VEC, G) launch_pdl(kv4_write_kernel<TYPE, VEC, G>, grid, block, 0, stream, (const TYPE*)c->k, c->k_stride, (const TYPE*)c->v, c->v_stride, c->slot_mapping, \
                                    (uint8_t*)c->k_cache, (uint8_t*)c->v_cache, c->T, c->n_kv, c->page_size, shift, slots, per_token, c->err)
#define WRITE_OF(G) (c->dtype == PHOTON_F32 ? vec ? WRITE(float, true, G) : WRITE(float, false, G) : vec ? WRITE(bf16, true, G) : WRITE(bf16, false, G))
  switch (groups) {
    case 1: return WRITE_OF(1);
    case 2: return WRITE_OF(2);
    case 3: return WRITE_OF(3);
    case 4: return WRITE_OF(4);
    case 5: return WRITE_OF(5);
    case 6: return WRITE_OF(6);
    case 7: return WRITE_OF(7);
    default: return WRITE_OF(8);
  }
#undef WRITE_OF
#undef WRITE
}

// Blocks of a page.
static int kv4_unpack_parts(const photon_kv4_unpack_call* c) { return (int)((8L * c->n_kv * c->page_size + KV4_THREADS - 1) / KV4_THREADS); }

PHOTON_API int photon_kv4_unpack(const photon_kv4_unpack_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->per <= 0) return 0;
  if ((c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) || c->n_kv <= 0 || c->num_pages < 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)c->k_out | (uintptr_t)c->v_out) % 16) return PHOTON_ERR_ARGUMENT;
  if ((long)c->S * c->per > 0x7fffffffL || 8L * c->n_kv * c->page_size > 65535L * KV4_THREADS) return PHOTON_ERR_UNSUPPORTED;
  const dim3 grid(c->S * c->per, kv4_unpack_parts(c));
  int shift = -1;
  for (int i = 0; i < 31; ++i) if (c->page_size == 1 << i) shift = i;
#define UNPACK(T, G) launch_pdl(kv4_unpack_kernel<T, G>, grid, dim3(KV4_THREADS), 0, stream, (const uint8_t*)c->k_cache, (const uint8_t*)c->v_cache, c->table, c->per, c->stride, \
                                (T*)c->k_out, (T*)c->v_out, c->n_kv, c->page_size, shift, c->num_pages, c->cu_tokens, c->context_lens, c->group, c->min_rows, c->window, c->new_table, \
                                c->positions, c->cu_tokens != nullptr ? c->flags : nullptr, c->err)
#define UNPACK_OF(G) (c->dtype == PHOTON_F32 ? UNPACK(float, G) : UNPACK(bf16, G))
  switch (c->d / 32) {
    case 1: return UNPACK_OF(1);
    case 2: return UNPACK_OF(2);
    case 3: return UNPACK_OF(3);
    case 4: return UNPACK_OF(4);
    case 5: return UNPACK_OF(5);
    case 6: return UNPACK_OF(6);
    case 7: return UNPACK_OF(7);
    default: return UNPACK_OF(8);
  }
#undef UNPACK_OF
#undef UNPACK
}

PHOTON_API int photon_kv4_spoil(const photon_kv4_unpack_call* c, void* out, long out_stride, const void* q, long q_stride, int max_tokens, int bounded, cudaStream_t stream) {
  if (c->S <= 0 || c->per <= 0 || max_tokens <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->flags == nullptr || c->cu_tokens == nullptr || c->n_kv <= 0 || c->group <= 0 || !kv4_sizes_ok(c->page_size, c->d)) return PHOTON_ERR_ARGUMENT;
  if (c->S > 65535 || c->group > 128 || ((uintptr_t)out | (uintptr_t)q) % 16 || out_stride % 8 || q_stride % 8) return PHOTON_ERR_UNSUPPORTED;
  const int chunks = (max_tokens + KV4_SPOIL_TOKENS - 1) / KV4_SPOIL_TOKENS;
  return launch_pdl(kv4_spoil_kernel, dim3(c->n_kv, c->S, chunks < 65535 ? chunks : 65535), dim3(KV4_THREADS), 0, stream, (const uint8_t*)c->v_cache, c->table, c->per, c->stride, c->n_kv,
                    c->d / 32, c->page_size, c->num_pages, c->cu_tokens, c->context_lens, c->group, c->min_rows, kv4_unpack_parts(c), (const int*)c->flags, (bf16*)out, out_stride,
                    (const bf16*)q, q_stride, c->window, bounded != 0);
}
