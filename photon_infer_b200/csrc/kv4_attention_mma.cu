// Attention of decoded tokens over a paged cache in 4 bits (the format: kv4.cuh): bfloat16, heads of 64 or 128 numbers.
//
// The codes go to the tensor cores as they are: a byte under a mask, two codes c0 + 16 c1, is the 16-bit float (c0 + 16 c1) 2^-24, and its upper half under a mask is 16 c1
// 2^-24, both below the normal numbers and exact.  Four instructions make eight numbers of an operand so (four ANDs and a shift, with every code by itself: five), and what
// those cost bounds the kernel: they run at half the rate of others.  The pairs are taken apart where it costs nothing: a key's by the queries they meet,
//   c0 q0 + c1 q1 = (c0 + 16 c1) q0 + 16 c1 (q1 / 16 - q0),
// where the last factor has two parts, two 16-bit floats, in neighbouring columns of the second operand, so that four rows (tokens x query heads of a key/value head) fill its
// eight columns; a value's behind the sum, since two rows of the result are the sums over c0 + 16 c1 and 16 c1.
//   score[key][row] = factor[row] sum over groups  scale[key][group] (sum over the group  c q  -  8 sum over the group  q),
// the last sum being what the product's result begins with.  The weights, as 16-bit floats, are turned over in registers and multiplied by the values' scales,
//   out[number][row] = sum over keys  c (p scale)[key][group(number)][row]  -  8 sum over keys (p scale)[key][group][row],
// where the last sums of all groups are one more product, with ones in a row of the first operand for each group.  Weights are lifted by 2^15, and the scales of a group
// whose largest so far is 2 or more, or below 2^-7, by the power of two that brings it to [1, 2).  All sums and the softmax are in 32 bits.
//
// Every warp walks keys of its own, 32 at a time, straight from the cache into registers, the next keys' codes asked for as soon as these are in the operands.  All
// blocks have equal runs of the requests' tiles of 128 keys; results of a unit (request, head, 4 or 8 rows) that lies in one block are written, others are joined by a
// second kernel in ascending order.
#include "kv4.cuh"
#include <math.h>

#define KM_THREADS 128
#define KM_KEYS 128              // of a block's step, 32 a warp
#define KM_MAX_SEQS 1024

struct Kv4MmaArgs {
  const bf16* q; bf16* out; const uint8_t* k; const uint8_t* v;
  const int* table; const int* cu_tokens; const int* context_lens; const float* sinks; float* lse; float* scratch; int* err;
  long q_stride, out_stride;
  int max_pages, S, n_q, n_kv, page_size, num_pages, window;
  float scale, softcap;
  int min_rows, max_rows, q_vec;      // q_vec: rows of q on 16-byte boundaries
};

// d += a b: 16 x 16 and 16 x 8 numbers of 16 bits.
__device__ __forceinline__ void km_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t km_turn(uint32_t x) {      // an 8 x 8 matrix of 16-bit numbers, rows for columns
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float km_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float km_power(int e) { return __int_as_float((127 + e) << 23); }      // 2^e, -126 <= e <= 127
__device__ __forceinline__ float km_scaled(float x, int e) { return x * km_power(e / 2) * km_power(e - e / 2); }
__device__ __forceinline__ uint32_t km_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *(const uint32_t*)&h;
}
__device__ __forceinline__ uint32_t km_mul2(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*(const __half2*)&a, *(const __half2*)&b);
  return *(const uint32_t*)&h;
}
// Bytes of two words by a selector's nibbles; 8 + i: eight times byte i's first bit.
__device__ __forceinline__ uint32_t km_bytes(uint32_t a, uint32_t b, uint32_t selector) {
  uint32_t y;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(selector));
  return y;
}
template <int WORDS>
__device__ __forceinline__ void km_load(uint32_t* x, const uint8_t* p) {      // read once: not kept in the first cache
  if constexpr (WORDS == 4) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "l"(p));
  else if constexpr (WORDS == 2) asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "l"(p));
  else asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(x[0]) : "l"(p));
}
__device__ __forceinline__ uint32_t km_load16(const uint8_t* p) {
  uint16_t x;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(x) : "l"(p));
  return x;
}

// A request's place in the work: rows, row tiles, keys from..to (from a multiple of 8), steps of 128 keys.
struct KmRequest { int first, n, ctx, rows, row_tiles, from, steps; };
template <int RT>
__device__ __forceinline__ KmRequest km_request(const Kv4MmaArgs& a, int s) {
  KmRequest r;
  r.first = a.cu_tokens[s];
  r.n = a.cu_tokens[s + 1] - r.first;
  r.ctx = a.context_lens[s];
  r.rows = r.n * (a.n_q / a.n_kv);
  if (r.rows <= a.min_rows || r.rows > a.max_rows) r.rows = 0;
  r.row_tiles = (r.rows + RT - 1) / RT;
  const int lo = a.window > 0 ? max(0, r.ctx - r.n - a.window + 1) : 0;
  r.from = lo & ~7;
  r.steps = r.rows > 0 ? max(1, (r.ctx - r.from + KM_KEYS - 1) / KM_KEYS) : 0;
  return r;
}

// GROUPS: of 32 numbers of a head (2 or 4); NT: tiles of 4 rows; CAP: bounded scores.
template <int GROUPS, int NT, bool CAP>
__global__ void __launch_bounds__(KM_THREADS, (GROUPS == 4 ? 3 : 4) - (NT - 1))
kv4_mma_kernel(const Kv4MmaArgs a) {
  constexpr int D = GROUPS * 32, RT = 4 * NT, KW = GROUPS, VW = GROUPS / 2;      // words of a key's and of a value's piece
  extern __shared__ __align__(16) float smem[];
  float* o_s = smem;                                  // [4][RT][D]
  float* m_s = o_s + 4 * RT * D;                      // [4][RT]
  float* l_s = m_s + 4 * RT;
  int* before_s = (int*)(l_s + 4 * RT);               // [S + 1] units' steps in front of a request
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  pdl_wait();
  if (warp == 0) {
    int sum = 0;
    for (int s0 = 0; s0 < a.S; s0 += 32) {
      int x = 0;
      if (s0 + lane < a.S) { const KmRequest r = km_request<RT>(a, s0 + lane); x = r.steps * r.row_tiles * a.n_kv; }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (s0 + lane < a.S) before_s[s0 + lane + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) before_s[0] = 0;
  }
  __syncthreads();
  const int total = before_s[a.S], N = gridDim.x;
  const int begin = (int)((long)total * blockIdx.x / N), end = (int)((long)total * (blockIdx.x + 1) / N);
  if (begin >= end) return;
  int s = 0;
  {                                                   // the request of the first step: the last one that begins at or before it
    int lo = 0, hi = a.S;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (before_s[mid] <= begin) lo = mid; else hi = mid; }
    s = lo;
  }
  const int G = a.n_q / a.n_kv;
  const long page_bytes = (long)a.page_size * GROUPS * 17;
  const float cap_in = 2.f * 1.4426950408889634f / a.softcap, cap_out = a.softcap * 1.4426950408889634f;
  uint32_t one[GROUPS];                               // row j of the first operand: ones
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) one[j] = g == j ? 0x3C003C00u : 0u;
  for (int pos = begin; pos < end;) {
    while (before_s[s + 1] <= pos) ++s;
    const KmRequest R = km_request<RT>(a, s);
    const int at = pos - before_s[s], unit = at / R.steps, step0 = at - unit * R.steps, step1 = min(R.steps, step0 + end - pos);
    const int head = unit / R.row_tiles, row0 = (unit - head * R.row_tiles) * RT, rows = min(RT, R.rows - row0), base = R.ctx - R.n;
    const int first_place = base + row0 / G, last_place = base + (row0 + rows - 1) / G;
    const int low = a.window > 0 ? max(0, first_place - a.window + 1) : 0;                            // keys from here to last_place some row sees
    const int clear_from = a.window > 0 ? last_place - a.window + 1 : 0, clear_to = first_place;      // keys that all rows see

    // ---- where the keys are: lane 4 i + o has the 8 keys o of the warp's 32 of step i, 8 steps at a time
    const int key_w = R.from + warp * 32;
    // off: where the 8 keys' codes begin, in 16 bytes; sc: where their scales do
    uint32_t off = 0, off_next = 0, sc16 = 0, sc16_next = 0, ok = 0, ok_next = 0;
    auto find = [&](int step, uint32_t& to, uint32_t& scales, uint32_t& mask) {
      const int i = step + (lane >> 2), key = key_w + i * KM_KEYS + (lane & 3) * 8;
      const int pidx = key / a.page_size;
      int page = -1, sl = key - pidx * a.page_size;
      if (i < step1 && key <= last_place) {
        page = pidx < a.max_pages ? a.table[(long)s * a.max_pages + pidx] : -1;
        if (page < 0 || page >= a.num_pages) { report_error(a.err, PHOTON_DEV_BAD_PAGE, s, key, page); page = -1; }
      }
      const bool good = page >= 0;
      if (!good) page = sl = 0;                       // some page of the pool: what is read there is not used
      const uint32_t begin16 = ((uint32_t)page * a.n_kv + head) * (uint32_t)(page_bytes >> 4);
      to = begin16 + sl * (D / 32);
      scales = begin16 + a.page_size * (D / 32) + sl * GROUPS / 16;
      mask = __ballot_sync(0xffffffffu, good);
    };
    find(step0, off, sc16, ok);
    // keys 8 o + g and values 8 o + 2 t, + 1; the scales of keys 8 o + g and of values 8 o + 2 t, + 1 for o = 2 u + (g & 1)
    uint32_t kw[4][KW], vw[4][2][VW], ks[4], vs[2][2];
    const uint8_t* k_codes = a.k + g * (D / 2) + 4 * GROUPS * t;
    const uint8_t* v_codes = a.v + 2 * t * (D / 2) + 2 * GROUPS * g;
    auto load_k = [&](int i) {                         // i: the step's place among the 8 that are known
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        km_load<KW>(kw[o], k_codes + __shfl_sync(0xffffffffu, off, 4 * i + o) * 16ull);
        const uint8_t* p = a.k + g * GROUPS + __shfl_sync(0xffffffffu, sc16, 4 * i + o) * 16ull;
        if constexpr (GROUPS == 4) km_load<1>(&ks[o], p); else ks[o] = km_load16(p);
      }
    };
    auto load_v = [&](int i) {
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        const uint8_t* p = v_codes + __shfl_sync(0xffffffffu, off, 4 * i + o) * 16ull;
        km_load<VW>(vw[o][0], p);
        km_load<VW>(vw[o][1], p + D / 2);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint8_t* p = a.v + 2 * t * GROUPS + __shfl_sync(0xffffffffu, sc16, 4 * i + 2 * u + (g & 1)) * 16ull;
        if constexpr (GROUPS == 4) km_load<2>(vs[u], p);
        else { uint32_t both; km_load<1>(&both, p); vs[u][0] = both & 0xffffu; vs[u][1] = both >> 16; }
      }
    };
    load_k(0);
    load_v(0);

    // ---- the queries: column g of the second operand is part g & 1 of row 4 x + g / 2
    uint32_t qb[NT][GROUPS][4];
    float init[NT][GROUPS], factor[NT];
    int place[NT];                                     // of row 4 x + t
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int r = 4 * x + (g >> 1), row = row0 + r;
      const bool there = r < rows, second = g & 1;
      const bf16* q = a.q + (there ? (R.first + row / G) * a.q_stride + (long)(head * G + row % G) * D : 0) + 8 * t;
      float v[GROUPS][8];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        if (a.q_vec) {
          const uint4 u = *(const uint4*)(q + 32 * j);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) { v[j][2 * i] = __uint_as_float(w[i] << 16); v[j][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = __bfloat162float(q[32 * j + i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!there) v[j][i] = 0.f;
          top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
        }
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool odd = top >= 0x7f800000u;
      const int e = top == 0 || odd ? 0 : max((int)(top >> 23), 1) - 127;
      const float up1 = km_power((14 - e) / 2), up2 = km_power(14 - e - (14 - e) / 2);      // the largest number to [2^14, 2^15)
      const float f = odd ? NAN : fmaxf(km_scaled(a.scale * (CAP ? 1.f : 1.4426950408889634f), e - 14 + 24), 1e-37f);
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        float sum = 0.f, y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = v[j][i] * up1 * up2;
          if (!(i & 1)) y[i] = __half2float(__float2half_rn(y[i]));      // exact from 2^-14 on
          sum += y[i];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {                  // numbers 0, 1, 4, 5, then 2, 3, 6, 7
          const float w0 = y[2 * h + 1] * 0.0625f - y[2 * h], w1 = y[2 * h + 5] * 0.0625f - y[2 * h + 4];
          const uint32_t p1 = km_half2(w0, w1);
          const float2 b1 = __half22float2(*(const __half2*)&p1);
          qb[x][j][2 * h] = second ? 0u : km_half2(y[2 * h], y[2 * h + 4]);
          qb[x][j][2 * h + 1] = second ? km_half2(w0 - b1.x, w1 - b1.y) : p1;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        init[x][j] = __shfl_sync(0xffffffffu, sum, 8 * t) * (-8.f / 16777216.f);
      }
      factor[x] = __shfl_sync(0xffffffffu, f, 8 * t);
      place[x] = 4 * x + t < rows ? base + (row0 + 4 * x + t) / G : -1;
    }
    float acc[NT][GROUPS][2][4], ones[NT][4], m[NT], l[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ones[x][i] = 0.f;
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) acc[x][j][0][i] = acc[x][j][1][i] = 0.f;
      }
    }
    uint32_t bad[NT] = {};                             // bit j: row 4 x + g / 2 sees a value of group j that is no number
    int top_e[GROUPS];                                 // the exponent of the largest scale so far: 15 is that of 1
    uint32_t room = 0;                                 // what makes a byte with a larger exponent set its first bit, where that matters
    bool lifted = false;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) top_e[j] = 1;

    for (int step = step0; step < step1; ++step) {
      const int i8 = (step - step0) & 7;
      const uint32_t here = ok >> (4 * i8) & 15u;
      if (i8 == 0) find(step + 8, off_next, sc16_next, ok_next);
      const int key0 = key_w + step * KM_KEYS;
      // ---- scores of the keys 8 o + g for row 4 x + t
      float sc[NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int jj = 0; jj < GROUPS; jj += 2) {
          // two groups' scales of the keys g and 8 + g of this half
          const uint32_t h0 = __byte_perm(ks[2 * i], 0, jj ? 0x3424 : 0x1404) >> 1, h1 = __byte_perm(ks[2 * i + 1], 0, jj ? 0x3424 : 0x1404) >> 1;
          const float2 s0 = __half22float2(*(const __half2*)&h0), s1 = __half22float2(*(const __half2*)&h1);
#pragma unroll
          for (int jx = 0; jx < 2; ++jx) {
            const int j = jj + jx;
            const uint32_t w0 = kw[2 * i][j], w1 = kw[2 * i + 1][j];
            const uint32_t u0 = __byte_perm(w0, 0, 0x4341), u1 = __byte_perm(w1, 0, 0x4341);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              float d[4] = {init[x][j], 0.f, init[x][j], 0.f};
              km_mma(d, w0 & 0x00FF00FFu, w1 & 0x00FF00FFu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qb[x][j][0], qb[x][j][1]);
              km_mma(d, u0, u1, u0 & 0x00F000F0u, u1 & 0x00F000F0u, qb[x][j][2], qb[x][j][3]);
              const float d0 = d[0] + d[1], d1 = d[2] + d[3];
              sc[x][2 * i] = j == 0 ? (jx ? s0.y : s0.x) * d0 : fmaf(jx ? s0.y : s0.x, d0, sc[x][2 * i]);
              sc[x][2 * i + 1] = j == 0 ? (jx ? s1.y : s1.x) * d1 : fmaf(jx ? s1.y : s1.x, d1, sc[x][2 * i + 1]);
            }
          }
        }
      }
      const bool more = step + 1 < step1;
      const bool turn = i8 == 7;
      if (more) {
        if (turn) { off = off_next; sc16 = sc16_next; }
        load_k((i8 + 1) & 7);
      }
      // ---- the softmax
      const bool masked = here != 15u || key0 < clear_from || key0 + 31 > clear_to;
      if constexpr (CAP) {                              // tanh y = 1 - 2 / (1 + e^2y); the factor is in it then
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int o = 0; o < 4; ++o) {
            const float y = km_exp2(sc[x][o] * (factor[x] * cap_in));
            sc[x][o] = fmaf(-cap_out, __fdividef(2.f, 1.f + y), cap_out);
          }
      }
      if (masked) {
#pragma unroll
        for (int o = 0; o < 4; ++o)
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            const int key = key0 + 8 * o + g;
            if (!((here >> o & 1u) && key <= place[x] && (a.window <= 0 || key > place[x] - a.window))) sc[x][o] = -INFINITY;
          }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int o = 2 * u + (g & 1), key = key0 + 8 * o + 2 * t + b;
            if (!(here >> o & 1u) || key > last_place || key < low) vs[u][b] = 0;      // whatever lies there
          }
      }
      float alpha[NT], ref[NT];
      bool grown = false;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        float top = fmaxf(fmaxf(sc[x][0], sc[x][1]), fmaxf(sc[x][2], sc[x][3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        if constexpr (!CAP) top *= factor[x];
        top = fmaxf(top, m[x]);
        alpha[x] = m[x] == -INFINITY ? 1.f : km_exp2(m[x] - top);
        grown |= top > m[x];
        m[x] = top;
        ref[x] = top == -INFINITY ? 0.f : top - 15.f;
      }
      // scales that call for another power of two, or no numbers
      const uint32_t high = ((vs[0][0] + room) | vs[0][0] | (vs[0][1] + room) | vs[0][1] | (vs[1][0] + room) | vs[1][0] | (vs[1][1] + room) | vs[1][1]) &
                            (GROUPS == 4 ? 0x80808080u : 0x8080u);
      const bool rare = __any_sync(0xffffffffu, high != 0 || step == step0);
      bool odd_scales = false;
      if (rare) {
        room = 0;
        lifted = false;
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
          int most = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int byte = vs[w >> 1][w & 1] >> (8 * j) & 255;
            if (byte < 248) most = max(most, byte); else odd_scales = true;
          }
          most = __reduce_max_sync(0xffffffffu, most) >> 3;
          const int was = top_e[j], to = max(was, most), old_lift = was > 15 || was < 8 ? 15 - was : 0, new_lift = to > 15 || to < 8 ? 15 - to : 0;
          top_e[j] = to;
          if (new_lift != old_lift) {
            const float f = km_power(new_lift - old_lift);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
              for (int i = 0; i < 4; ++i) { acc[x][j][0][i] *= f; acc[x][j][1][i] *= f; }
              if (g == j) { ones[x][0] *= f; ones[x][1] *= f; }
            }
          }
          lifted |= new_lift != 0;
          if (to < 8) room |= (uint32_t)(0x7F - (8 * to + 7)) << (8 * j);
        }
        odd_scales = __any_sync(0xffffffffu, odd_scales);
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          l[x] *= alpha[x];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ones[x][i] *= alpha[x];
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) { acc[x][j][0][i] *= alpha[x]; acc[x][j][1][i] *= alpha[x]; }
          }
        }
      }
      uint32_t p2[NT][2];                              // weights of the keys g and 8 + g, 16 + g and 24 + g
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        float p[4];
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          p[o] = km_exp2(CAP ? sc[x][o] - ref[x] : fmaf(sc[x][o], factor[x], -ref[x]));
          l[x] += p[o];
        }
        p2[x][0] = km_half2(p[0], p[1]);
        p2[x][1] = km_half2(p[2], p[3]);
      }
      // ---- the values.  Column g of the second operand has the weights of row 4 x + g / 2 for the 8 keys 2 u + (g & 1), and nothing for the 8 beside them
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t pe[NT], po[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const uint32_t y = km_turn(p2[x][u]);
          pe[x] = g & 1 ? 0u : y;
          po[x] = g & 1 ? y : 0u;
        }
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) {
          // the scales of its keys 2 t and 2 t + 1; the bytes between are a scale's first bit, 0 below 2
          uint32_t s2 = km_bytes(vs[u][0], vs[u][1], j == 0 ? 0x4C08 : j == 1 ? 0x5D19 : j == 2 ? 0x6E2A : 0x7F3B) >> 1;
          if (rare || lifted) {
            s2 &= 0x7F807F80u;
            if (odd_scales) {                          // no number goes into the sums, where it would meet the zeros beside the ones: who sees it is noted
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if ((s2 >> (16 * h) & 0x7fffu) >= 0x7c00u) {
                  s2 &= h ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
                  for (int x = 0; x < NT; ++x) {
                    const int r = 4 * x + (g >> 1), key = key0 + 16 * u + 8 * (g & 1) + 2 * t + h, at_place = base + (row0 + r) / G;
                    if (r < rows && key <= at_place && (a.window <= 0 || key > at_place - a.window)) bad[x] |= 1u << j;
                  }
                }
            }
            const float f = km_power(top_e[j] > 15 || top_e[j] < 8 ? 15 - top_e[j] : 0);
            s2 = km_mul2(s2, km_half2(f, f));
          }
          const uint32_t r0 = __byte_perm(vw[2 * u][0][j / 2], vw[2 * u][1][j / 2], j & 1 ? 0x7632 : 0x5410);
          const uint32_t r1 = __byte_perm(vw[2 * u + 1][0][j / 2], vw[2 * u + 1][1][j / 2], j & 1 ? 0x7632 : 0x5410);
          const uint32_t t0 = __byte_perm(r0, 0, 0x4341), t1 = __byte_perm(r1, 0, 0x4341);
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            const uint32_t b0 = km_mul2(pe[x], s2), b1 = km_mul2(po[x], s2);
            km_mma(acc[x][j][0], r0 & 0x00FF00FFu, r0 & 0x00F000F0u, r1 & 0x00FF00FFu, r1 & 0x00F000F0u, b0, b1);
            km_mma(acc[x][j][1], t0, t0 & 0x00F000F0u, t1, t1 & 0x00F000F0u, b0, b1);
            km_mma(ones[x], one[j], 0u, one[j], 0u, b0, b1);
          }
        }
      }
      if (more) {
        load_v((i8 + 1) & 7);
        if (turn) ok = ok_next;
      }
    }
    // ---- the warps' results side by side
    __syncthreads();
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
      bad[x] = __reduce_or_sync(0xffffffffu, bad[x] << (8 * (g >> 1))) >> (8 * t);
      const int row = 4 * x + t;
      if (g == 0) { m_s[warp * RT + row] = m[x]; l_s[warp * RT + row] = l[x]; }
      const float both = ones[x][0] + ones[x][1];
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        const float eight = 8.f * __shfl_sync(0xffffffffu, both, 4 * j + t), f = bad[x] >> j & 1u ? NAN : km_power(top_e[j] > 15 || top_e[j] < 8 ? top_e[j] - 15 : 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float* c = acc[x][j][h];
          const float c1 = c[2] + c[3], c0 = c[0] + c[1] - c1;
          *(float2*)&o_s[(warp * RT + row) * D + 32 * j + 4 * g + 2 * h] = make_float2((c0 * 16777216.f - eight) * f, (c1 * 1048576.f - eight) * f);
        }
      }
    }
    __syncthreads();
    const bool whole = step0 == 0 && step1 == R.steps;
    const long part = 2L * blockIdx.x + (pos == begin ? 0 : 1);
    float* part_o = a.scratch + part * RT * D;
    float* part_ml = a.scratch + 2L * N * RT * D + part * RT * 2;
    for (int i = tid; i < rows * (D / 4); i += KM_THREADS) {
      const int r = i / (D / 4), d4 = i - r * (D / 4), row = row0 + r, h = head * G + row % G;
      const long token = R.first + row / G;
      const float m0 = fmaxf(fmaxf(m_s[r], m_s[RT + r]), fmaxf(m_s[2 * RT + r], m_s[3 * RT + r]));
      float top = m0;
      if (whole && a.sinks != nullptr) top = fmaxf(top, a.sinks[h] * 1.4426950408889634f);
      const float zero = top == -INFINITY ? 0.f : top;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float total_l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float lw = l_s[w * RT + r];
        if (lw == 0.f) continue;
        const float f = m_s[w * RT + r] == -INFINITY ? 1.f : exp2f(m_s[w * RT + r] - zero);
        const float4 o = *(const float4*)&o_s[(w * RT + r) * D + 4 * d4];
        total_l += lw * f;
        sum.x += o.x * f; sum.y += o.y * f; sum.z += o.z * f; sum.w += o.w * f;
      }
      if (whole) {
        if (a.sinks != nullptr) total_l += exp2f(a.sinks[h] * 1.4426950408889634f - zero + 15.f);
        if (d4 == 0 && a.lse != nullptr) a.lse[token * a.n_q + h] = total_l == 0.f ? -INFINITY : (zero - 15.f + log2f(total_l)) * 0.6931471805599453f;
        const float f = total_l == 0.f ? 0.f : 1.f / total_l;
        bf16* to = a.out + token * a.out_stride + (long)h * D + 4 * d4;
        to[0] = __float2bfloat16_rn(sum.x * f);
        to[1] = __float2bfloat16_rn(sum.y * f);
        to[2] = __float2bfloat16_rn(sum.z * f);
        to[3] = __float2bfloat16_rn(sum.w * f);
      } else {
        *(float4*)&part_o[r * D + 4 * d4] = sum;
        if (d4 == 0) { part_ml[2 * r] = top; part_ml[2 * r + 1] = total_l; }
      }
    }
    pos += step1 - step0;
    __syncthreads();
  }
}

// Units that lie in several blocks.  A block has one row of a unit's tile.
template <int GROUPS, int NT>
__global__ void __launch_bounds__(GROUPS * 32)
kv4_mma_join_kernel(const Kv4MmaArgs a, int N) {
  constexpr int D = GROUPS * 32, RT = 4 * NT;
  __shared__ int sums[2][GROUPS];
  pdl_wait();
  const int s = blockIdx.z, head = blockIdx.y, row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const KmRequest R = km_request<RT>(a, s);
  if (row >= R.rows) return;
  int before = 0, total = 0;
  for (int i = tid; i < a.S; i += D) {
    const KmRequest r = km_request<RT>(a, i);
    const int x = r.steps * r.row_tiles * a.n_kv;
    total += x;
    if (i < s) before += x;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  total = __reduce_add_sync(0xffffffffu, total);
  if (lane == 0) { sums[0][warp] = before; sums[1][warp] = total; }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) { before += sums[0][i]; total += sums[1][i]; }
  const int from = before + (head * R.row_tiles + row / RT) * R.steps, to = from + R.steps;
  // the block that has step x: the last one that begins at or before it
  auto block_of = [&](int x) {
    int b = (int)((long)x * N / total);
    while (b + 1 < N && (long)total * (b + 1) / N <= x) ++b;
    while ((long)total * b / N > x) --b;
    return b;
  };
  const int b0 = block_of(from), b1 = block_of(to - 1);
  if (b0 == b1) return;
  const int r = row % RT, G = a.n_q / a.n_kv, h = head * G + row % G;
  const float* part_ml = a.scratch + 2L * N * RT * D;
  const float sink = a.sinks != nullptr ? a.sinks[h] * 1.4426950408889634f : -INFINITY;
  auto part_of = [&](int b) { return 2L * b + ((long)total * b / N >= from ? 0 : 1); };
  float m = sink;
  for (int b = b0; b <= b1; ++b) if ((long)total * b / N < (long)total * (b + 1) / N) m = fmaxf(m, part_ml[(part_of(b) * RT + r) * 2]);
  const float zero = m == -INFINITY ? 0.f : m;
  float l = a.sinks != nullptr ? exp2f(sink - zero + 15.f) : 0.f, sum = 0.f;
  for (int b = b0; b <= b1; ++b) {
    if ((long)total * b / N >= (long)total * (b + 1) / N) continue;
    const long part = part_of(b);
    const float pm = part_ml[(part * RT + r) * 2], pl = part_ml[(part * RT + r) * 2 + 1], o = a.scratch[(part * RT + r) * D + tid];
    if (pl == 0.f) continue;
    const float f = pm == -INFINITY ? 1.f : exp2f(pm - zero);
    l += pl * f;
    sum += o * f;
  }
  const long token = R.first + row / G;
  if (tid == 0 && a.lse != nullptr) a.lse[token * a.n_q + h] = l == 0.f ? -INFINITY : (zero - 15.f + log2f(l)) * 0.6931471805599453f;
  a.out[token * a.out_stride + (long)h * D + tid] = __float2bfloat16_rn(l == 0.f ? 0.f : sum / l);
}

template <int GROUPS, int NT, bool CAP>
static int km_launch(const Kv4MmaArgs& a, int N, int max_rows, cudaStream_t stream) {
  constexpr int RT = 4 * NT;
  const size_t smem = (4 * RT * GROUPS * 32 + 8 * RT) * sizeof(float) + (a.S + 1) * sizeof(int);
  static bool set = false;
  if (!set) {
    const cudaError_t e = cudaFuncSetAttribute(kv4_mma_kernel<GROUPS, NT, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (4 * RT * GROUPS * 32 + 8 * RT) * 4 + (KM_MAX_SEQS + 1) * 4);
    if (e != cudaSuccess) return (int)e;
    set = true;
  }
  int status = launch_pdl(kv4_mma_kernel<GROUPS, NT, CAP>, dim3(N), dim3(KM_THREADS), smem, stream, a);
  if (status != 0) return status;
  return launch_pdl(kv4_mma_join_kernel<GROUPS, NT>, dim3(max_rows, a.n_kv, a.S), dim3(GROUPS * 32), 0, stream, a, N);
}

// parts: blocks; scratch: 2 * parts * RT * (d + 2) floats, RT = 4 for up to 4 rows, else 8.
PHOTON_API int photon_kv4_attention_mma(const photon_kv4_attention_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d) || (c->d != 64 && c->d != 128) || c->page_size % 8 || c->num_pages <= 0) return PHOTON_ERR_UNSUPPORTED;
  if (c->S > KM_MAX_SEQS || c->n_kv > 65535 || c->scale <= 0.f || ((uintptr_t)c->k_cache | (uintptr_t)c->v_cache) % 16) return PHOTON_ERR_UNSUPPORTED;
  if (kv4_page_bytes(c->page_size, c->d) / 16 * c->num_pages * c->n_kv > 0xffffffffL) return PHOTON_ERR_UNSUPPORTED;      // a key's place in 16 bytes: 32 bits
  if (c->parts < 1 || c->scratch == nullptr) return PHOTON_ERR_ARGUMENT;
  const int rows = c->max_tokens_per_seq * (c->n_q / c->n_kv), most = rows < c->max_rows ? rows : c->max_rows;
  const Kv4MmaArgs a = {(const bf16*)c->q, (bf16*)c->out, (const uint8_t*)c->k_cache, (const uint8_t*)c->v_cache, c->block_table, c->cu_tokens, c->context_lens, c->sinks, c->lse,
                        c->scratch, c->err, c->q_stride, c->out_stride, c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, c->scale, c->softcap, c->min_rows,
                        c->max_rows, (uintptr_t)c->q % 16 == 0 && c->q_stride % 8 == 0};
#define ATTEND(GROUPS, NT) (c->softcap > 0.f ? km_launch<GROUPS, NT, true>(a, c->parts, most, stream) : km_launch<GROUPS, NT, false>(a, c->parts, most, stream))
  if (c->d == 64) return most <= 4 ? ATTEND(2, 1) : ATTEND(2, 2);
  return most <= 4 ? ATTEND(4, 1) : ATTEND(4, 2);
#undef ATTEND
}
