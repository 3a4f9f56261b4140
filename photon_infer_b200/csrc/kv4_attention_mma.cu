// Attention of decoded tokens over a paged cache in 4 bits (the format: kv4.cuh): bfloat16, heads of 64 or 128 numbers.
//
// The codes go to the tensor cores as they are: a byte under a mask, two codes c0 + 16 c1, is the 16-bit float (c0 + 16 c1) 2^-24, and its upper half under a mask is 16 c1
// 2^-24, both below the normal numbers and exact.  Four instructions make eight numbers of an operand so (four ANDs and a shift, with every code by itself: five), which
// run at half the rate of others.  The pairs are taken apart where it costs nothing: a key's by the queries they meet,
//   c0 q0 + c1 q1 = (c0 + 16 c1) q0 + 16 c1 (q1 / 16 - q0),
// where the last factor has two parts, two 16-bit floats, in neighbouring columns of the second operand, so that four rows (tokens x query heads of a key/value head) fill its
// eight columns; a value's behind the sum, since two rows of the result are the sums over c0 + 16 c1 and 16 c1.
//   score[key][row] = factor[row] sum over groups  scale[key][group] (sum over the group  c q  -  8 sum over the group  q),
// the last sum known beforehand.  The weights, as 16-bit floats, are turned over in registers and multiplied by the values' scales,
//   out[number][row] = sum over keys  (c - 8) (p scale)[key][group(number)][row],
// where pairs of codes under the mask get the exponent of 1,024 with it and 1,024 and the eights are taken off by an addition, which is exact.  Weights are lifted by 2^15, and scales of 2
// or more, or below 2^-9, meet them by themselves, lifted by a power of two.  All sums and the softmax are in 32 bits (an exponential is off by 2^-22).
// A query has 22 bits, a weight and its product with a scale 11 each, since they meet the values as 16-bit floats: a row is off by 0.0017 of its size, which the result's own rounding to 8 bits
// gives with weights in 32 bits, too.  The first number of a pair is the difference of two sums and so off
// by some 2^-20 of the second one's, where its own rounding to 4 bits was off by half a scale.
//
// All warps have equal runs of the requests' tiles of 32 keys, wherever units (a request, a head, 4 or 8 rows) begin and end, and nothing to do with one another: a tile's
// bytes come through three stages of the warp's own in shared memory, two of them on their way.  Results of a unit that lies in one warp are written, the others' parts are joined by a
// second kernel, in the same order every time.
//
// What bounds it: latency, with three warps a scheduler.  64 requests of up to 6,000 keys (24 query heads on 8 of 128; 253 MB) take 69 us, 0.56 of the copy rate: 68,000 instructions a scheduler are
// 36 us of them if each cycle had one, and neither the issue slots (61 %) nor a pipe (54 % of the one that takes codes apart, 22 % of the tensor cores) is full; for each instruction issued a warp waits
// one for the last one's result, 0.6 for that pipe and 0.7 for the others' turn.  A sum's registers (160 a thread) leave room for no fourth warp.  20 us of the 69 are begin, end and join.  Two requests of
// 100,003 keys, 32 on 8: 63 us, 0.52.  One of 640, heads of 64: 7.7 us, a chain of latencies.  Equal runs instead of a block for each share of a request: 94 to 79 us for the 64.  8-bit
// products were slower.  Values' scales all in another band take 86 us instead of the 69, one in 100 in another 119.
#include "kv4.cuh"
#include <math.h>

#pragma nv_diag_suppress 128      // what keys got has no use for the second half of the loop

#define KM_THREADS 128
#define KM_KEYS 32               // of a warp's step
#define KM_MAX_SEQS 1024
// Blocks an SM: what their registers leave room for.
#define KM_BLOCKS(GROUPS, NT) ((GROUPS == 4 ? 4 : 5) - NT)
#define KM_STAGES 3              // of a warp's 32 keys and values in shared memory
#define KM_MOST 0x7fffffffu      // steps of a call: so many or more are counted as this, and not taken

struct Kv4MmaArgs {
  const bf16* q; bf16* out; const uint8_t* k; const uint8_t* v;
  const int* table; const int* cu_tokens; const int* context_lens; const float* sinks; float* lse; float* scratch; int* before; int* err;      // before [S + 1]: behind the scratch
  long q_stride, out_stride;
  int max_pages, S, n_q, n_kv, page_size, num_pages, window;
  float scale, softcap;
  int page_shift;                // of page_size / 8, or -1
  float* weights; const int* held;      // the second use: what keys got, beside them
  int max_rows, q_vec, out_vec;      // rows of q on 16-byte boundaries, of out on 8-byte ones
};

// d += a b: 16 x 16 and 16 x 8 numbers of 16 bits; and d = a b.
__device__ __forceinline__ void km_mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void km_mma0(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
__device__ __forceinline__ void km_copy(uint32_t to, const uint8_t* from) {      // 16 bytes to shared memory
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint32_t km_add2(uint32_t a, uint32_t b) {
  const __half2 h = __hadd2(*(const __half2*)&a, *(const __half2*)&b);
  return *(const uint32_t*)&h;
}
template <int WORDS>
__device__ __forceinline__ void km_read(uint32_t* x, uint32_t at) {
  if constexpr (WORDS == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
  else if constexpr (WORDS == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at));
  else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x[0]) : "r"(at));
}
__device__ __forceinline__ uint32_t km_read16(uint32_t at) {
  uint16_t x;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(at));
  return x;
}
__device__ __forceinline__ const uint8_t* km_at(const uint8_t* base, uint32_t sixteens) {
  const uint8_t* p;
  asm("mad.wide.u32 %0, %1, 16, %2;" : "=l"(p) : "r"(sixteens), "l"(base));
  return p;
}
// Where 16 bytes `c` of row r of 8 rows lie in a stage: no two of the lanes that read together, 8 rows' pieces by turns (keys) or every other row's (values), meet in a bank.
template <int GROUPS>
__device__ __forceinline__ int km_place(int r, int c) {
  if constexpr (GROUPS == 4) return (r ^ (r >> 1 & 1)) * 64 + ((c ^ (r >> 2 & 1) << 1) * 16);
  else return (r & 1 ? 4 + (r >> 1 ^ 2) : r >> 1) * 32 + c * 16;
}

// A request's place in the work: rows, row tiles, keys from..to (from a multiple of 8), steps of 32 keys.
struct KmRequest { int first, n, ctx, rows, row_tiles, from, steps; };
template <int RT, bool WEIGH>
__device__ __forceinline__ KmRequest km_request(const Kv4MmaArgs& a, int s) {
  KmRequest r;
  r.first = a.cu_tokens[s];
  r.n = a.cu_tokens[s + 1] - r.first;
  r.ctx = a.context_lens[s];
  r.rows = r.n * (a.n_q / a.n_kv);
  if (r.rows > a.max_rows) r.rows = 0;
  r.row_tiles = (r.rows + RT - 1) / RT;
  int lo = a.window > 0 ? max(0, r.ctx - r.n - a.window + 1) : 0;
  if (WEIGH) lo = max(0, min(lo, a.held != nullptr ? a.held[s] : r.ctx - r.n));      // keys without a sum get one
  r.from = lo & ~7;
  r.steps = r.rows <= 0 ? 0 : r.ctx <= r.from ? 1 : (int)(((unsigned)(r.ctx - r.from) + KM_KEYS - 1) / KM_KEYS);
  return r;
}

// Steps in equal runs, the first ones a step longer.
struct KmRuns {
  int each, longer;
  __device__ __forceinline__ KmRuns(int total, int warps) : each(total / warps), longer(total - total / warps * warps) {}
  __device__ __forceinline__ int begin(int w) const { return w * each + min(w, longer); }
  __device__ __forceinline__ int warp_of(int step) const {
    const int first = longer * (each + 1);
    return step < first ? step / (each + 1) : longer + (step - first) / each;
  }
};

// GROUPS: of 32 numbers of a head (2 or 4); NT: tiles of 4 rows; CAP: bounded scores.
// WEIGH: no values.  With every row's logarithm known, a key's sum over the rows is added to the one beside it: lane (g, t) has key 8 t + g of a step.
template <int GROUPS, int NT, bool CAP, bool WEIGH>
__global__ void __launch_bounds__(KM_THREADS, WEIGH ? 4 : KM_BLOCKS(GROUPS, NT))
kv4_mma_kernel(const Kv4MmaArgs a) {
  constexpr int D = GROUPS * 32, RT = 4 * NT, KW = GROUPS, VW = GROUPS / 2;      // words of a key's and of a value's piece
  constexpr int ROW = D / 2, CODES = (WEIGH ? 32 : 64) * ROW, STAGE = CODES + CODES / 16;      // codes of 32 keys, of 32 values, their scales
  extern __shared__ __align__(16) uint8_t smem[];     // the four warps' stages
  int* before_s = (int*)(smem + 4 * KM_STAGES * STAGE);      // [S + 1] units' steps in front of a request
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  pdl_wait();
  if (warp == 0) {
    uint32_t sum = 0;                                 // a sum of two such counts fits 32 bits
    for (int s0 = 0; s0 < a.S; s0 += 32) {
      uint32_t x = 0;
      if (s0 + lane < a.S) {
        const KmRequest r = km_request<RT, WEIGH>(a, s0 + lane);
        x = (uint32_t)min((unsigned long long)r.steps * (uint32_t)(r.row_tiles * a.n_kv), (unsigned long long)KM_MOST);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x = min(x + y, KM_MOST);
      }
      if (s0 + lane < a.S) before_s[s0 + lane + 1] = (int)min(sum + x, KM_MOST);
      sum = min(sum + __shfl_sync(0xffffffffu, x, 31), KM_MOST);
    }
    if (lane == 0) before_s[0] = 0;
    if (!WEIGH && blockIdx.x == 0) {                  // for the second kernel
      __syncwarp();
      for (int i = lane; i <= a.S; i += 32) a.before[i] = before_s[i];
    }
  }
  __syncthreads();
  pdl_launch_dependents();
  const int total = before_s[a.S], N = gridDim.x * 4, me = blockIdx.x * 4 + warp;
  if ((uint32_t)total == KM_MOST) {                   // lengths that the call's limits do not cover: the host gives no such call to this kernel
    if (blockIdx.x == 0 && threadIdx.x == 0) report_error(a.err, PHOTON_DEV_TOO_LONG, a.S, a.n_kv, 0);
    return;
  }
  const KmRuns runs(total, N);
  const int begin = runs.begin(me), end = runs.begin(me + 1);
  if (begin >= end) return;
  int s = 0;
  {                                                   // the request of the first step: the last one that begins at or before it
    int lo = 0, hi = a.S;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (before_s[mid] <= begin) lo = mid; else hi = mid; }
    s = lo;
  }
  const int G = a.n_q / a.n_kv;
  const uint32_t page16 = (uint32_t)a.page_size * GROUPS * 17 / 16;
  const float cap_in = 2.f * 1.4426950408889634f / a.softcap, cap_out = a.softcap * 1.4426950408889634f;
  // constants that stay in registers: two of them in one instruction do not fit, and the compiler would make them again for each
  uint32_t c_1024, c_64, c_both, c_high;
  asm volatile("mov.u32 %0, 0x64006400;" : "=r"(c_1024));
  asm volatile("mov.u32 %0, 0x64646464;" : "=r"(c_64));
  asm volatile("mov.u32 %0, 0xE488E488;" : "=r"(c_both));      // -1160 twice
  asm volatile("mov.u32 %0, 0xE480E480;" : "=r"(c_high));      // -1152 twice
  for (int pos = begin; pos < end;) {
    while (before_s[s + 1] <= pos) ++s;
    const KmRequest R = km_request<RT, WEIGH>(a, s);
    const int at = pos - before_s[s], unit = at / R.steps, step0 = at - unit * R.steps, step1 = min(R.steps, step0 + end - pos);
    const int head = unit / R.row_tiles, row0 = (unit - head * R.row_tiles) * RT, rows = min(RT, R.rows - row0), base = R.ctx - R.n;
    const int first_place = base + row0 / G, last_place = base + (row0 + rows - 1) / G;
    const int low = a.window > 0 ? max(0, first_place - a.window + 1) : 0;                            // keys from here to last_place some row sees
    const int clear_from = a.window > 0 ? last_place - a.window + 1 : 0, clear_to = first_place;      // keys that all rows see

    // ---- where the keys are: lane 4 i + o has the 8 keys o of step i's 32, 8 steps at a time
    // off: where the 8 keys' codes begin, in 16 bytes; sc: where their scales do
    uint32_t off = 0, sc16 = 0, ok = 0, w8 = 0;       // w8: where the 8 keys' sums are, in eights
    int entry = -1, place8 = 0;                       // the block table's entry and which 8 of the page
    const int eight0 = (R.from >> 3) + lane;
    auto look = [&](int step) {
      const int eight = eight0 + step * 4;
      const int pidx = a.page_shift >= 0 ? eight >> a.page_shift : eight / (a.page_size >> 3);
      place8 = eight - pidx * (a.page_size >> 3);
      entry = -2;                                     // not asked for
      if (step + (lane >> 2) < step1 && eight * 8 <= last_place) entry = pidx < a.max_pages ? a.table[(long)s * a.max_pages + pidx] : -1;
    };
    auto found = [&](int step) {
      const bool good = entry >= 0 && entry < a.num_pages;
      ok = __ballot_sync(0xffffffffu, good);
      if (!good && entry != -2) report_error(a.err, PHOTON_DEV_BAD_PAGE, s, (eight0 + step * 4) * 8, entry);
      const uint32_t begin16 = ((uint32_t)(good ? entry : 0) * a.n_kv + head) * page16;      // else some page of the pool: what is read there is not used
      off = begin16 + place8 * (D / 4);
      sc16 = begin16 + a.page_size * (D / 32) + place8 * GROUPS / 2;
      if (WEIGH) w8 = ((uint32_t)(good ? entry : 0) * a.n_kv + head) * (uint32_t)(a.page_size >> 3) + place8;
    };
    const int known = WEIGH ? (a.held != nullptr ? a.held[s] : base) : 0;
    float old_a = 0.f, old_b = 0.f, old_c = 0.f;       // the sums so far of this lane's key: of this step, the next and the one behind it
    float *at_a = nullptr, *at_b = nullptr, *at_c = nullptr;
    look(step0);
    uint32_t ok_use = 0;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (KM_STAGES * STAGE);
    int given = 0;                                     // steps asked for, stages in turn
    uint32_t give_to = ring;
    auto ask = [&]() {
      if (step0 + given < step1) {
        if ((given & 7) == 0) {
          found(step0 + given);
          look(step0 + given + 8);
        }
        const int i = given & 7;
        if constexpr (GROUPS == 4) {
          const uint32_t to = give_to + km_place<4>(lane >> 2, lane & 3);
#pragma unroll
          for (int o = 0; o < 4; ++o) {
            const uint32_t x = __shfl_sync(0xffffffffu, off, 4 * i + o) + lane;
            km_copy(to + o * 512, km_at(a.k, x));
            if (!WEIGH) km_copy(to + 2048 + o * 512, km_at(a.v, x));
          }
          const uint32_t x = __shfl_sync(0xffffffffu, sc16, 4 * i + (lane >> 1 & 3)) + (lane & 1);
          if (lane < (WEIGH ? 8 : 16)) km_copy(give_to + CODES + lane * 16, km_at(lane < 8 ? a.k : a.v, x));
        } else {
          const uint32_t to = give_to + (lane >> 4) * 256 + km_place<2>(lane >> 1 & 7, lane & 1);
#pragma unroll
          for (int o = 0; o < 4; o += 2) {
            const uint32_t x = __shfl_sync(0xffffffffu, off, 4 * i + o + (lane >> 4)) + (lane & 15);
            km_copy(to + o * 256, km_at(a.k, x));
            if (!WEIGH) km_copy(to + 1024 + o * 256, km_at(a.v, x));
          }
          const uint32_t x = __shfl_sync(0xffffffffu, sc16, 4 * i + (lane & 3));
          if (lane < (WEIGH ? 4 : 8)) km_copy(give_to + CODES + lane * 16, km_at(lane < 4 ? a.k : a.v, x));
        }
        if constexpr (WEIGH) {
          const int key = R.from + (step0 + given) * KM_KEYS + 8 * t + g;
          float* p = a.weights + __shfl_sync(0xffffffffu, w8, 4 * i + t) * 8ull + g;
          at_c = (ok >> (4 * i + t) & 1u) && key < R.ctx ? p : nullptr;
          old_c = at_c != nullptr && key < known ? *p : 0.f;
        }
        ++given;
        give_to = give_to == ring + (KM_STAGES - 1) * STAGE ? ring : give_to + STAGE;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // ---- the queries: column g of the second operand is part g & 1 of row 4 x + g / 2
    uint4 raw[NT][GROUPS];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int r = 4 * x + (g >> 1), row = row0 + r;
      const bf16* q = a.q + (R.first + row / G) * a.q_stride + (long)(head * G + row % G) * D + 8 * t;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        raw[x][j] = make_uint4(0u, 0u, 0u, 0u);
        if (r >= rows) continue;
        if (a.q_vec) {
          raw[x][j] = *(const uint4*)(q + 32 * j);
        } else {
          uint32_t w[4];
          const uint16_t* p = (const uint16_t*)(q + 32 * j);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
          raw[x][j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < KM_STAGES - 1; ++i) {
      ask();
      if (i == 0) { at_a = at_c; old_a = old_c; } else { at_b = at_c; old_b = old_c; }
    }

    uint32_t qb[NT][GROUPS][4];
    float init[NT][GROUPS], factor[NT];
    int place[NT];                                     // of row 4 x + t
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const bool second = g & 1;
      float v[GROUPS][8];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        const uint32_t w[4] = {raw[x][j].x, raw[x][j].y, raw[x][j].z, raw[x][j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[j][2 * i] = __uint_as_float(w[i] << 16); v[j][2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const bool odd = top >= 0x7f800000u;
      const int e = top == 0 || odd ? 0 : max((int)(top >> 23), 1) - 127;
      const float up1 = km_power((14 - e) / 2), up2 = km_power(14 - e - (14 - e) / 2);      // the largest number to [2^14, 2^15)
      // where no 32 bits hold it, the largest that they do: scores stay as far apart as a softmax can tell
      const float f = fminf(fmaxf(km_scaled(a.scale * (CAP ? 1.f : 1.4426950408889634f), e - 14 + 24), 1e-37f), 3e38f);
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
        // a query that is not finite: no score is a number, but for those that a mask takes out behind this
        init[x][j] = __shfl_sync(0xffffffffu, odd ? NAN : sum, 8 * t) * (-8.f / 16777216.f);
      }
      factor[x] = __shfl_sync(0xffffffffu, f, 8 * t);
      place[x] = 4 * x + t < rows ? base + (row0 + 4 * x + t) / G : -1;
    }
    float acc[NT][GROUPS][2][4], m[NT], l[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) acc[x][j][0][i] = acc[x][j][1][i] = 0.f;
      }
    }
    float lse2[NT];                                    // WEIGH: of row 4 x + t, in powers of two
    if constexpr (WEIGH) {
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        const int row = 4 * x + t;
        lse2[x] = INFINITY;
        if (row < rows) lse2[x] = a.lse[(long)(R.first + row / G) * a.n_q + head * G + row % G] * 1.4426950408889634f;
        if (lse2[x] == -INFINITY) lse2[x] = INFINITY;   // a row that sees nothing
      }
    }
    uint32_t bad[NT] = {};                             // bit j: row 4 x + g / 2 sees a value of group j that is no number
    int held = 0;                                      // the sums in acc are multiplied by 2^held

    uint32_t stage = ring;
    const uint32_t k_at = km_place<GROUPS>(g, GROUPS == 4 ? t : t >> 1) + (GROUPS == 4 ? 0 : (t & 1) * 8);
    const uint32_t v_at0 = 32 * ROW + km_place<GROUPS>(2 * t, GROUPS == 4 ? g >> 1 : g >> 2) + (GROUPS == 4 ? (g & 1) * 8 : (g & 3) * 4);
    const uint32_t v_at1 = 32 * ROW + km_place<GROUPS>(2 * t + 1, GROUPS == 4 ? g >> 1 : g >> 2) + (GROUPS == 4 ? (g & 1) * 8 : (g & 3) * 4);
    for (int step = step0; step < step1; ++step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(KM_STAGES - 2) : "memory");
      __syncwarp();                                    // this step's bytes are there, and the stage before it has been read by all
      const int i8 = (step - step0) & 7;
      if (i8 == 0) ok_use = ok;
      const uint32_t here = ok_use >> (4 * i8) & 15u;
      ask();
      const int key0 = R.from + step * KM_KEYS;
      uint32_t kw[4][KW], ks[4];                       // keys 8 o + g and their scales
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        km_read<KW>(kw[o], stage + k_at + o * 8 * ROW);
        if constexpr (GROUPS == 4) km_read<1>(&ks[o], stage + CODES + (8 * o + g) * 4); else ks[o] = km_read16(stage + CODES + (8 * o + g) * 2);
      }
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
              float d[4];
              km_mma0(d, w0 & 0x00FF00FFu, w1 & 0x00FF00FFu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qb[x][j][0], qb[x][j][1]);
              km_mma(d, u0, u1, u0 & 0x00F000F0u, u1 & 0x00F000F0u, qb[x][j][2], qb[x][j][3]);
              const float d0 = d[0] + (d[1] + init[x][j]), d1 = d[2] + (d[3] + init[x][j]);
              sc[x][2 * i] = j == 0 ? (jx ? s0.y : s0.x) * d0 : fmaf(jx ? s0.y : s0.x, d0, sc[x][2 * i]);
              sc[x][2 * i + 1] = j == 0 ? (jx ? s1.y : s1.x) * d1 : fmaf(jx ? s1.y : s1.x, d1, sc[x][2 * i + 1]);
            }
          }
        }
      }
      // ---- the softmax
      const bool masked = here != 15u || key0 < clear_from || key0 + 31 > clear_to;
      if constexpr (CAP) {                              // tanh y = 1 - 2 / (1 + e^2y), off by some 2^-22 of the bound; the factor is in it then
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
      }
      if constexpr (WEIGH) {
        float sum[4];
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          sum[o] = 0.f;
#pragma unroll
          for (int x = 0; x < NT; ++x) sum[o] += sc[x][o] == -INFINITY ? 0.f : km_exp2(CAP ? sc[x][o] - lse2[x] : fmaf(sc[x][o], factor[x], -lse2[x]));
        }
        // over the four lanes with a key's rows, so that lane t has key 8 t + g
        const float y0 = (t & 1 ? sum[1] : sum[0]) + __shfl_xor_sync(0xffffffffu, t & 1 ? sum[0] : sum[1], 1);
        const float y1 = (t & 1 ? sum[3] : sum[2]) + __shfl_xor_sync(0xffffffffu, t & 1 ? sum[2] : sum[3], 1);
        const float y = (t & 2 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, t & 2 ? y0 : y1, 2);
        if (at_a != nullptr) *at_a = old_a + y;
        at_a = at_b; old_a = old_b;
        at_b = at_c; old_b = old_c;
        stage = stage == ring + (KM_STAGES - 1) * STAGE ? ring : stage + STAGE;
        continue;
      }
      uint32_t vs[2][2];                               // scales of the values 8 o + 2 t, + 1 for o = 2 u + (g & 1)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t from = stage + CODES + 32 * GROUPS + (8 * (2 * u + (g & 1)) + 2 * t) * GROUPS;
        if constexpr (GROUPS == 4) km_read<2>(vs[u], from);
        else { uint32_t both; km_read<1>(&both, from); vs[u][0] = both & 0xffffu; vs[u][1] = both >> 16; }
      }
      if (masked) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int o = 2 * u + (g & 1), key = key0 + 8 * o + 2 * t + b;
            if (!(here >> o & 1u) || key > last_place || key < low) vs[u][b] = GROUPS == 4 ? 0x78787878u : 0x7878u;      // 1, whatever lies there: its weight is 0
          }
      }
      float alpha[NT], ref[NT], times[NT];
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
        times[x] = factor[x];
      }
      // scales that call for another power of two (a byte of 48 is 2^-9, one of 128 is 2), or no numbers
      constexpr uint32_t FIRST = GROUPS == 4 ? 0x80808080u : 0x8080u, UP = GROUPS == 4 ? 0x50505050u : 0x5050u;
      const uint32_t some = vs[0][0] | vs[0][1] | vs[1][0] | vs[1][1], all = (vs[0][0] + UP) & (vs[0][1] + UP) & (vs[1][0] + UP) & (vs[1][1] + UP);
      bool far = false;                                // a maximum beyond 2^20: the bits that rounding it takes are no small part of a weight's 15 powers of two
#pragma unroll
      for (int x = 0; x < NT; ++x) far |= fabsf(m[x]) > 1048576.f;
      const bool rare = __any_sync(0xffffffffu, ((some | ~all) & FIRST) != 0 || held != 0 || far);
      uint32_t bands = 2;
      bool odd_scales = false, several = false;        // no numbers; more than one band, or such
      if (rare) {
        // four bytes at a time, what is found in a byte's first bit: which bands there are (0 is in none), and whether a byte is 248 or more
        uint32_t in0 = 0, in1 = 0, in2 = 0, in3 = 0, none = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t v = vs[w >> 1][w & 1], low = v & 0x7f7f7f7fu, above = low + 0x50505050u, some = (low + 0x7f7f7f7fu) & ~v, no = v & ((v & 0x78787878u) + 0x08080808u);
          in0 |= some & ~above;
          in1 |= above & ~v;
          in2 |= v & ~(v << 1);
          in3 |= v & (v << 1) & ~no;
          none |= no;
        }
        const uint32_t mine = (in0 & FIRST ? 1u : 0u) | (in1 & FIRST ? 2u : 0u) | (in2 & FIRST ? 4u : 0u) | (in3 & FIRST ? 8u : 0u) | (none & FIRST ? 16u : 0u);
        bands = __reduce_or_sync(0xffffffffu, mine);
        odd_scales = bands & 16u;
        several = (bands & (bands - 1)) != 0;
        bands &= 15u;
        if (bands == 0) bands = 2;
        if (__any_sync(0xffffffffu, far)) {            // scores as far below the maximum as they are, from products rounded as it was; then as if it were 0
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            if (fabsf(m[x]) <= 1048576.f || m[x] == -INFINITY) continue;
#pragma unroll
            for (int o = 0; o < 4; ++o) sc[x][o] = (CAP ? sc[x][o] : __fmul_rn(sc[x][o], factor[x])) - m[x];
            ref[x] = -15.f;
            times[x] = 1.f;
          }
        }
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          l[x] *= alpha[x];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
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
          p[o] = km_exp2(CAP ? sc[x][o] - ref[x] : fmaf(sc[x][o], times[x], -ref[x]));
          l[x] += p[o];
        }
        p2[x][0] = km_half2(p[0], p[1]);
        p2[x][1] = km_half2(p[2], p[3]);
      }
      // ---- the values.  Column g of the second operand has the weights of row 4 x + g / 2 for the 8 keys 2 u + (g & 1), and nothing for the 8 beside them.
      // Scales from 2^-9 to 2 meet the weights as they are; others, a band of 2^8 at a time, by the power of two that brings them there, and the sums with them: a weight times a scale
      // keeps its bits whatever lies beside it.  As a rule there is one band.
#pragma unroll 1
      do {
        uint32_t from = 0, size = 0, lift2 = 0;        // the band's scales as 16-bit floats, the power of two
        if (rare) {
          const int band = __ffs(bands) - 1, lift = 8 * (1 - band);
          from = band == 0 ? 1u : band == 1 ? 48u << 7 : band == 2 ? 128u << 7 : 192u << 7;
          size = (band == 0 ? 48u << 7 : band == 1 ? 128u << 7 : band == 2 ? 192u << 7 : 248u << 7) - from;
          lift2 = km_half2(km_power(lift), km_power(lift));
          if (lift != held) {
            const float f = km_power(lift - held);
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int j = 0; j < GROUPS; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) { acc[x][j][0][i] *= f; acc[x][j][1][i] *= f; }
            held = lift;
          }
        }
        bands &= bands - 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t pe[NT], po[NT];
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            const uint32_t y = km_turn(p2[x][u]);
            pe[x] = g & 1 ? 0u : y;
            po[x] = g & 1 ? y : 0u;
          }
          uint32_t vw[2][2][VW];                         // values 8 (2 u + o) + 2 t, + 1
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            km_read<VW>(vw[o][0], stage + v_at0 + (2 * u + o) * 8 * ROW);
            km_read<VW>(vw[o][1], stage + v_at1 + (2 * u + o) * 8 * ROW);
          }
          // the scales of its keys 2 t and 2 t + 1; the bytes between are a scale's first bit, 0 below 2
          uint32_t s2[GROUPS];
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) s2[j] = km_bytes(vs[u][0], vs[u][1], j == 0 ? 0x4C08 : j == 1 ? 0x5D19 : j == 2 ? 0x6E2A : 0x7F3B) >> 1;
          if (rare) {
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
              s2[j] &= 0x7F807F80u;
              if (odd_scales) {                          // no number goes into the products, where it would meet rows that do not see it: who does is noted
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  if ((s2[j] >> (16 * h) & 0x7fffu) >= 0x7c00u) {
                    s2[j] &= h ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                      const int r = 4 * x + (g >> 1), key = key0 + 16 * u + 8 * (g & 1) + 2 * t + h, at_place = base + (row0 + r) / G;
                      if (r < rows && key <= at_place && (a.window <= 0 || key > at_place - a.window)) bad[x] |= 1u << j;
                    }
                  }
              }
              if (several) s2[j] &= ((s2[j] & 0xffffu) - from < size ? 0x0000ffffu : 0u) | ((s2[j] >> 16) - from < size ? 0xffff0000u : 0u);
              s2[j] = km_mul2(s2[j], lift2);
            }
          }
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            // of two keys each: numbers 0 and 1 of this lane's four, then 2 and 3, as 1024 + c0 + 16 c1 and 1024 + 16 c1; less what makes them c - 8
            const uint32_t r0 = __byte_perm(vw[0][0][j / 2], vw[0][1][j / 2], j & 1 ? 0x7632 : 0x5410);
            const uint32_t r1 = __byte_perm(vw[1][0][j / 2], vw[1][1][j / 2], j & 1 ? 0x7632 : 0x5410);
            const uint32_t t0 = __byte_perm(r0, c_64, 0x4341), t1 = __byte_perm(r1, c_64, 0x4341);
            const uint32_t e0 = km_add2((r0 & 0x00FF00FFu) | c_1024, c_both), h0 = km_add2((r0 & 0x00F000F0u) | c_1024, c_high);
            const uint32_t e1 = km_add2((r1 & 0x00FF00FFu) | c_1024, c_both), h1 = km_add2((r1 & 0x00F000F0u) | c_1024, c_high);
            const uint32_t e2 = km_add2(t0, c_both), h2 = km_add2((t0 & 0x00F000F0u) | c_1024, c_high);
            const uint32_t e3 = km_add2(t1, c_both), h3 = km_add2((t1 & 0x00F000F0u) | c_1024, c_high);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              const uint32_t b0 = km_mul2(pe[x], s2[j]), b1 = km_mul2(po[x], s2[j]);
              km_mma(acc[x][j][0], e0, h0, e1, h1, b0, b1);
              km_mma(acc[x][j][1], e2, h2, e3, h3, b0, b1);
            }
          }
        }
      } while (bands != 0);
      stage = stage == ring + (KM_STAGES - 1) * STAGE ? ring : stage + STAGE;
    }
    // ---- the results: the unit's, or a part of them
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    if constexpr (WEIGH) {
      pos += step1 - step0;
      continue;
    }
    const bool whole = step0 == 0 && step1 == R.steps;
    const long part = 2L * me + (pos == begin ? 0 : 1);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
      bad[x] = __reduce_or_sync(0xffffffffu, bad[x] << (8 * (g >> 1))) >> (8 * t);
      const int r = 4 * x + t, row = row0 + r, h = head * G + row % G;
      const long token = R.first + row / G;
      const bool there = r < rows;
      float mul = 1.f;
      if (whole) {
        float top = m[x], total_l = l[x];
        if (a.sinks != nullptr && there) {
          const float sink = a.sinks[h] * 1.4426950408889634f;
          top = fmaxf(top, sink);
          mul = m[x] == -INFINITY ? 1.f : exp2f(m[x] - top);
          if (sink != -INFINITY) total_l = total_l * mul + exp2f(sink - top + 15.f);
        }
        if (g == 0 && there && a.lse != nullptr) a.lse[token * a.n_q + h] = total_l == 0.f ? -INFINITY : (top - 15.f + log2f(total_l)) * 0.6931471805599453f;
        mul = total_l == 0.f ? 0.f : mul / total_l;
      } else if (g == 0) {
        float* ml = a.scratch + 2L * N * RT * D + (part * RT + r) * 2;
        ml[0] = m[x];
        ml[1] = l[x];
      }
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) {
        const float f = (bad[x] >> j & 1u ? NAN : km_power(-held)) * mul;
        float y[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float* c = acc[x][j][i];
          const float c1 = c[2] + c[3], c0 = c[0] + c[1] - c1;
          y[2 * i] = c0 * f;
          y[2 * i + 1] = c1 * (0.0625f * f);
        }
        if (!whole) {
          *(float4*)&a.scratch[(part * RT + r) * D + 32 * j + 4 * g] = make_float4(y[0], y[1], y[2], y[3]);
        } else if (there) {
          bf16* to = a.out + token * a.out_stride + (long)h * D + 32 * j + 4 * g;
          const __nv_bfloat162 lo = __floats2bfloat162_rn(y[0], y[1]), hi = __floats2bfloat162_rn(y[2], y[3]);
          if (a.out_vec) *(uint2*)to = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
          else { to[0] = lo.x; to[1] = lo.y; to[2] = hi.x; to[3] = hi.y; }
        }
      }
    }
    pos += step1 - step0;
  }
}

// Units that lie in several warps: a block has one.  A thread has four numbers of a row in every `pars`-th part, in ascending order; then the threads' sums are joined.
template <int GROUPS, int NT>
__global__ void __launch_bounds__(1024, 1)
kv4_mma_join_kernel(const Kv4MmaArgs a, int N) {
  constexpr int D = GROUPS * 32, RT = 4 * NT, ITEMS = RT * D / 4;
  extern __shared__ __align__(16) float join_s[];     // [pars][ITEMS] of {4 sums}, then {maximum, sum of weights}
  pdl_wait();
  const int s = blockIdx.z, head = blockIdx.y, tile = blockIdx.x, tid = threadIdx.x, pars = blockDim.x / ITEMS, item = tid % ITEMS, par = tid / ITEMS;
  const int before = a.before[s], after = a.before[s + 1], total = a.before[a.S];
  const KmRequest R = km_request<RT, false>(a, s);
  if (after == before || tile >= R.row_tiles || (uint32_t)total == KM_MOST) return;
  const int from = before + (head * R.row_tiles + tile) * R.steps, to = from + R.steps;
  const KmRuns runs(total, N);
  const int w0 = runs.warp_of(from), w1 = runs.warp_of(to - 1);
  if (w0 == w1) return;
  const int r = item / (D / 4), d4 = item - r * (D / 4), row0 = tile * RT, row = row0 + r, G = a.n_q / a.n_kv, h = head * G + row % G;
  const bool there = row < R.rows;
  const float* part_ml = a.scratch + 2L * N * RT * D;
  float m = -INFINITY, l = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float pm, float pl, float4 o) {
    if (pl == 0.f) return;                            // a part of which the row sees nothing
    const float top = fmaxf(m, pm);
    const float f = m == -INFINITY ? 1.f : exp2f(m - top), k = pm == -INFINITY ? 1.f : exp2f(pm - top);      // no maximum and yet a sum: it is no number
    l = l * f + pl * k;
    sum.x = sum.x * f + o.x * k; sum.y = sum.y * f + o.y * k; sum.z = sum.z * f + o.z * k; sum.w = sum.w * f + o.w * k;
    m = top;
  };
  for (int w = w0 + par; w <= w1; w += 8 * pars) {   // eight parts under way
    float2 ml[8];
    float4 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = w + i * pars;
      ml[i] = make_float2(-INFINITY, 0.f);
      if (at <= w1) {
        const long part = (2L * at + (runs.begin(at) >= from ? 0 : 1)) * RT + r;
        ml[i] = *(const float2*)&part_ml[part * 2];
        o[i] = *(const float4*)&a.scratch[part * D + 4 * d4];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) add(ml[i].x, ml[i].y, o[i]);
  }
  float2* ml_s = (float2*)(join_s + 4 * pars * ITEMS);
  ((float4*)join_s)[tid] = sum;
  ml_s[tid] = make_float2(m, l);
  __syncthreads();
  if (par > 0 || !there) return;
  for (int p = 1; p < pars; ++p) add(ml_s[p * ITEMS + item].x, ml_s[p * ITEMS + item].y, ((float4*)join_s)[p * ITEMS + item]);
  float mul = 1.f;
  if (a.sinks != nullptr) {
    const float sink = a.sinks[h] * 1.4426950408889634f, top = fmaxf(m, sink);
    mul = m == -INFINITY ? 1.f : exp2f(m - top);
    if (sink != -INFINITY) l = l * mul + exp2f(sink - top + 15.f);
    m = top;
  }
  const long token = R.first + row / G;
  if (d4 == 0 && a.lse != nullptr) a.lse[token * a.n_q + h] = l == 0.f ? -INFINITY : (m - 15.f + log2f(l)) * 0.6931471805599453f;
  mul = l == 0.f ? 0.f : mul / l;
  bf16* out = a.out + token * a.out_stride + (long)h * D + 4 * d4;
  const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x * mul, sum.y * mul), hi = __floats2bfloat162_rn(sum.z * mul, sum.w * mul);
  if (a.out_vec) *(uint2*)out = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
  else { out[0] = lo.x; out[1] = lo.y; out[2] = hi.x; out[3] = hi.y; }
}

template <int GROUPS, int NT, bool CAP>
static int km_launch(const Kv4MmaArgs& a, int blocks, int max_rows, cudaStream_t stream) {
  constexpr int RT = 4 * NT;
  constexpr size_t stages = 4 * KM_STAGES * (64 * GROUPS * 16 + 64 * GROUPS);
  static bool ready[64] = {};
  const int limit = smem_limit((const void*)kv4_mma_kernel<GROUPS, NT, CAP, false>, (int)(stages + (KM_MAX_SEQS + 1) * sizeof(int)), true, ready);
  if (limit != 0) return limit;
  const int status = launch_pdl(kv4_mma_kernel<GROUPS, NT, CAP, false>, dim3(blocks), dim3(KM_THREADS), stages + (a.S + 1) * sizeof(int), stream, a);
  if (status != 0) return status;
  // threads by the parts that a unit has, about
  const int tiles = (max_rows + RT - 1) / RT;
  const long parts = 4L * blocks / ((long)a.S * a.n_kv * tiles);
  const int threads = parts > 24 ? 1024 : 256;
  return launch_pdl(kv4_mma_join_kernel<GROUPS, NT>, dim3(tiles, a.n_kv, a.S), dim3(threads), threads * 6 * sizeof(float), stream, a, 4 * blocks);
}

// parts: blocks; scratch: 8 * parts * RT * (d + 2) + S + 1 words, RT = 4 for up to 4 rows, else 8.
PHOTON_API int photon_kv4_attention_mma(const photon_kv4_attention_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d) || (c->d != 64 && c->d != 128) || c->page_size % 8 || c->num_pages <= 0) return PHOTON_ERR_UNSUPPORTED;
  if (c->S > KM_MAX_SEQS || c->n_kv > 65535 || c->scale <= 0.f || ((uintptr_t)c->k_cache | (uintptr_t)c->v_cache) % 16) return PHOTON_ERR_UNSUPPORTED;
  if (kv4_page_bytes(c->page_size, c->d) / 16 * c->num_pages * c->n_kv > 0xffffffffL) return PHOTON_ERR_UNSUPPORTED;      // a key's place in 16 bytes: 32 bits
  if (c->parts < 1 || c->scratch == nullptr) return PHOTON_ERR_ARGUMENT;
  const int rows = c->max_tokens_per_seq * (c->n_q / c->n_kv), most = rows < c->max_rows ? rows : c->max_rows;
  int shift = -1;
  for (int i = 0; i < 28; ++i) if (c->page_size == 8 << i) shift = i;
  const long words = 8L * c->parts * (most <= 4 ? 4 : 8) * (c->d + 2);
  const Kv4MmaArgs a = {(const bf16*)c->q, (bf16*)c->out, (const uint8_t*)c->k_cache, (const uint8_t*)c->v_cache, c->block_table, c->cu_tokens, c->context_lens, c->sinks, c->lse,
                        c->scratch, (int*)c->scratch + words, c->err, c->q_stride, c->out_stride, c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, c->scale, c->softcap, shift, nullptr, nullptr,
                        c->max_rows, (uintptr_t)c->q % 16 == 0 && c->q_stride % 8 == 0,
                        (uintptr_t)c->out % 8 == 0 && c->out_stride % 4 == 0};
#define ATTEND(GROUPS, NT) (c->softcap > 0.f ? km_launch<GROUPS, NT, true>(a, c->parts, most, stream) : km_launch<GROUPS, NT, false>(a, c->parts, most, stream))
  if (c->d == 64) return most <= 4 ? ATTEND(2, 1) : ATTEND(2, 2);
  return most <= 4 ? ATTEND(4, 1) : ATTEND(4, 2);
#undef ATTEND
}

template <int GROUPS, int NT, bool CAP>
static int km_weigh(const Kv4MmaArgs& a, int blocks, cudaStream_t stream) {
  constexpr size_t stages = 4 * KM_STAGES * (32 * GROUPS * 17);
  static bool ready[64] = {};
  const int limit = smem_limit((const void*)kv4_mma_kernel<GROUPS, NT, CAP, true>, (int)(stages + (KM_MAX_SEQS + 1) * sizeof(int)), true, ready);
  if (limit != 0) return limit;
  return launch_pdl(kv4_mma_kernel<GROUPS, NT, CAP, true>, dim3(blocks), dim3(KM_THREADS), stages + (a.S + 1) * sizeof(int), stream, a);
}

PHOTON_API int photon_kv4_key_weights(const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_keys <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || !c->packed || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0 || c->lse == nullptr || c->parts < 1) return PHOTON_ERR_ARGUMENT;
  if (!kv4_sizes_ok(c->page_size, c->d) || (c->d != 64 && c->d != 128) || c->page_size % 8 || c->num_pages <= 0) return PHOTON_ERR_UNSUPPORTED;
  if (c->S > KM_MAX_SEQS || c->n_kv > 65535 || c->scale <= 0.f || (uintptr_t)c->k_cache % 16) return PHOTON_ERR_UNSUPPORTED;
  if (kv4_page_bytes(c->page_size, c->d) / 16 * c->num_pages * c->n_kv > 0xffffffffL) return PHOTON_ERR_UNSUPPORTED;
  const int rows = c->max_tokens_per_seq * (c->n_q / c->n_kv);
  if (rows > 8) return PHOTON_ERR_UNSUPPORTED;        // a key's rows are one warp's
  int shift = -1;
  for (int i = 0; i < 28; ++i) if (c->page_size == 8 << i) shift = i;
  const Kv4MmaArgs a = {(const bf16*)c->q, nullptr, (const uint8_t*)c->k_cache, nullptr, c->block_table, c->cu_tokens, c->context_lens, nullptr, (float*)c->lse, nullptr, nullptr, c->err,
                        c->q_stride, 0, c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, c->scale, c->softcap, shift, c->weights, c->held, rows,
                        (uintptr_t)c->q % 16 == 0 && c->q_stride % 8 == 0, 0};
#define WEIGH(GROUPS, NT) (c->softcap > 0.f ? km_weigh<GROUPS, NT, true>(a, c->parts, stream) : km_weigh<GROUPS, NT, false>(a, c->parts, stream))
  if (c->d == 64) return rows <= 4 ? WEIGH(2, 1) : WEIGH(2, 2);
  return rows <= 4 ? WEIGH(4, 1) : WEIGH(4, 2);
#undef WEIGH
}
