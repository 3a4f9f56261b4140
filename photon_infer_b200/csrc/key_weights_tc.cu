// What each cached key got of the softmax of a request's query rows (key_weights.cu), for many rows, on tcgen05: bfloat16 queries, heads of 64 or 128, a plain bfloat16 cache or one
// in 4 bits (kv4.cuh), whose numbers bfloat16 holds exactly.
//
// A block walks a run of a request's keys, 128 at a time, for one head, beside 128 rows (tokens x query heads of the key/value head), of which the second pass takes all in turn.
// First the rows are the first operand: two threads have a row, and its maximum and its sum over the keys stay in registers.  Then, with the rows' logarithms, the keys
// are: two threads have a key and add up what the rows give it.  No score leaves tensor memory but into the registers of the thread that needs it, and a sum has one order.
//
// What bounds it: the exponentials, two for a score at 16 a cycle on an SM, take 1.1 us of the 2 to 2.5 us that a pass needs for two blocks' tiles; the rest is waiting inside a
// tile, with 16 warps on an SM, which tensor memory (2 x 128 columns a block) and shared memory allow no more of.  Two requests of 32 tokens beside 8,009 keys, 32 query heads on 8,
// heads of 128: 37 us, where key_weights_mma.cu takes 60; 8 of 64 beside 4,000: 118 and 197; up to 32 rows key_weights_mma.cu is the faster by 1 to 3 us.
#include "key_weights.cuh"
#include "tcgen05.cuh"
#include <type_traits>

#define KT_THREADS 256         // two threads for a lane of tensor memory: half of the columns each

// Waits for what was asked of tensor memory; names the registers, so that nothing reads them before.
__device__ __forceinline__ void kt_arrived(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// FINAL: the weights; else the maxima and sums of the run.
template <int D, bool PACKED, bool FINAL>
__global__ void __launch_bounds__(KT_THREADS, 2)
key_weights_tc_kernel(const KeyWeightsMmaArgs a) {
  constexpr int GROUPS = D / 32, TILE = 128 * D * 2, PIECES = PACKED ? D / 32 : D / 8, COLUMNS = 256;
  extern __shared__ uint8_t kt_smem[];
  uint8_t* k_s = (uint8_t*)(((uintptr_t)kt_smem + 1023) & ~(uintptr_t)1023);      // twice 128 keys: panels of 64 numbers, rows of 128 bytes, 128-byte swizzle
  uint8_t* q_s = k_s + 2 * TILE;
  __shared__ __align__(16) float lse_s[128];
  __shared__ float half_s[2][128];                    // what the second thread of a lane found
  __shared__ int place_s[128];
  __shared__ uint32_t there_s[4][4];                  // keys that are there, of four tiles
  __shared__ long row_s[4][KX_KEYS];                  // (page, head, slot) of a key, counted through
  __shared__ int slot_s[4][KX_KEYS];
  __shared__ __align__(8) uint64_t done;
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, own = tid & 127, half = tid >> 7;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(&tmem_s)), "n"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    tc_mbar_init(&done, 1);
    abort_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y % a.n_kv, block_r0 = FINAL ? 0 : (int)(blockIdx.y / a.n_kv) * 128;
  const int first = a.cu_tokens[seq], n = a.cu_tokens[seq + 1] - first, ctx = a.context_lens[seq], G = a.n_q / a.n_kv, rows = n * G, base = ctx - n, last_place = ctx - 1;
  const int known = a.held != nullptr ? a.held[seq] : base;
  // keys that no row sees and that have a sum already are left out
  int low = a.window > 0 ? max(0, base - a.window + 1) : 0;
  if (FINAL) low = max(0, min(low, known));
  const int tile0 = max((int)blockIdx.x * a.each, low / KX_KEYS);
  int tile1 = min(((int)blockIdx.x + 1) * a.each, (ctx + KX_KEYS - 1) / KX_KEYS);
  if (block_r0 >= rows) tile1 = tile0;
  bool fine = true;
  float m = -INFINITY, l = 0.f;                       // of row block_r0 + own, in this thread's columns; m in unscaled scores where nothing bounds them
  if (tile0 < tile1) {
    // ---- places: thread `tid` < 128 has key `tid` of a tile; the block table's entries come a tile ahead, and a tile's page and place follow from those of the one in front
    const int first_key = tile0 * KX_KEYS + own, step_pages = KX_KEYS / a.page_size, step_slots = KX_KEYS - step_pages * a.page_size;
    int next_page = 0, next_slot = 0, next_key = 0;
    struct Place { int entry, slot; };                 // entry -2: not asked for
    auto look = [&]() {                                // the tiles one behind the other; what is not there reads some entry of the table, too
      const int entry = a.table[(long)seq * a.max_pages + min(next_page, a.max_pages - 1)];
      const Place p = {half != 0 || next_key < low || next_key >= min(ctx, tile1 * KX_KEYS) ? -2 : next_page < a.max_pages ? entry : -1, next_slot};
      next_key += KX_KEYS;
      next_page += step_pages;
      next_slot += step_slots;
      if (next_slot >= a.page_size) {
        next_slot -= a.page_size;
        ++next_page;
      }
      return p;
    };
    auto settle = [&](int tile, Place p) {             // the tile's places
      if (half != 0 || tile >= tile1) return;
      const bool good = p.entry >= 0 && p.entry < a.num_pages;
      if (FINAL && !good && p.entry != -2) report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, tile * KX_KEYS + tid, p.entry);
      const uint32_t votes = __ballot_sync(0xffffffffu, good);
      if (lane == 0) there_s[tile & 3][warp] = votes;
      row_s[tile & 3][tid] = ((long)(good ? p.entry : 0) * a.n_kv + head) * a.page_size + (good ? p.slot : 0);      // else some row of the pool: what is read is not used
      if (PACKED) slot_s[tile & 3][tid] = good ? p.slot : 0;
    };
    auto piece_at = [&](uint8_t* tile, int row, int piece) { return tile + (piece >> 3) * (128 * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4); };
    constexpr int ROUNDS = KX_KEYS * PIECES / KT_THREADS;                  // of a thread, 16 bytes each
    uint4 codes[PACKED ? ROUNDS : 1];
    uint32_t scales[PACKED ? ROUNDS : 1];
    auto ask = [&](int tile) {                         // codes come into registers, numbers into shared memory
      if (tile >= tile1) return;
      const long* row = row_s[tile & 3];
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const int x = i * KT_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
        if constexpr (PACKED) {
          const int slot = slot_s[tile & 3][key];
          const uint8_t* at = (const uint8_t*)a.k + (row[key] - slot) * (GROUPS * 17);
          const uint8_t* sc = at + (long)a.page_size * (D / 2) + slot * GROUPS;
          codes[i] = *(const uint4*)(at + (long)slot * (D / 2) + 16 * piece);
          scales[i] = GROUPS == 4 ? *(const uint32_t*)sc : *(const uint16_t*)sc;
        } else {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc_smem(piece_at(k_s + (tile & 1) * TILE, key, piece))), "l"((const bf16*)a.k + row[key] * D + 8 * piece)
                       : "memory");
        }
      }
    };
    auto put = [&](int tile) {                         // codes that came, as numbers
      if (tile >= tile1) return;
#pragma unroll
      for (int i = 0; i < (PACKED ? ROUNDS : 0); ++i) {      // words t GROUPS + j
        const int x = i * KT_THREADS + tid, key = x / PIECES, piece = x - key * PIECES;
        const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int word = 4 * piece + c, tt = word / GROUPS, j = word - tt * GROUPS;
          const __nv_bfloat162 s = __float2bfloat162_rn(kv4_scale(scales[i] >> (8 * j) & 255u));
          // numbers 0 and 4, 1 and 5, 2 and 6, 3 and 7
          const uint32_t y0 = kx_scaled(w[c], 0, s), y1 = kx_scaled(w[c], 4, s), y2 = kx_scaled(w[c], 8, s), y3 = kx_scaled(w[c], 12, s);
          *(uint4*)piece_at(k_s + (tile & 1) * TILE, key, 4 * j + tt) =
              make_uint4(__byte_perm(y0, y1, 0x5410), __byte_perm(y2, y3, 0x5410), __byte_perm(y0, y1, 0x7632), __byte_perm(y2, y3, 0x7632));
        }
      }
    };
    auto stage_rows = [&](int r0) {
      constexpr int EACH = 128 * (D / 8) / KT_THREADS;
      uint4 v[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {                 // all are asked for before the first is put
        const int x = i * KT_THREADS + tid, r = x / (D / 8), piece = x - r * (D / 8), row = r0 + r, token = row / G;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows) v[i] = *(const uint4*)(a.q + (first + token) * a.q_stride + (long)(head * G + row - token * G) * D + 8 * piece);
      }
      const int row = r0 + own, token = min(row, rows - 1) / G;
      const float lse = FINAL && row < rows ? a.lse[(long)(first + token) * a.n_q + head * G + row - token * G] * 1.4426950408889634f : INFINITY;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int x = i * KT_THREADS + tid, r = x / (D / 8), piece = x - r * (D / 8);
        *(uint4*)piece_at(q_s, r, piece) = kx_queries(v[i]);
      }
      if (half != 0) return;
      place_s[tid] = row < rows ? base + token : -1;
      lse_s[tid] = lse;
    };
    const float scale2 = a.scale * 1.4426950408889634f, cap_in = 2.f * 1.4426950408889634f * a.scale / a.softcap, cap_out = a.softcap * 1.4426950408889634f;
    auto bounded = [&](float x) { return cap_out * (1.f - __fdividef(2.f, 1.f + kx_exp2(x * cap_in))); };
    // The products of a tile run while the scores of the one in front of it are worked on, and the keys behind it are on their way.
    const uint64_t k_desc = tc_desc(tc_smem(k_s)), q_desc = tc_desc(tc_smem(q_s));
    auto multiply = [&](int tile, int width) {
      if (warp == 0 && tile < tile1 && tc_elect()) {
        tc_fence_after();
        const uint32_t to = tmem + 128 * (tile & 1), idesc = FINAL ? tc_idesc(128, width) : tc_idesc(128, 128);
        const uint64_t kt = k_desc + (tile & 1) * (TILE >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {          // in 16 bytes: 16 numbers of a row, a panel
          const int at = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
          tc_mma(to, FINAL ? kt + at : q_desc + at, FINAL ? q_desc + at : kt + at, idesc, kk > 0 ? 1u : 0u);
        }
        tc_commit(&done);
      }
      __syncwarp();
    };
    auto arrived = [] {                                // this thread's part of what was asked for, for the tensor core to read
      asm volatile("cp.async.wait_all;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
    };
    uint32_t parity = 0;
    for (int r0 = block_r0; r0 < (FINAL ? rows : block_r0 + 1) && fine; r0 += 128) {
      const int width = min(128, (rows - r0 + 15) / 16 * 16);             // columns of rows
      next_page = first_key / a.page_size;
      next_slot = first_key - next_page * a.page_size;
      next_key = first_key;
      const Place place0 = look(), place1 = look();
      Place ahead = look();
      stage_rows(r0);
      settle(tile0, place0);
      settle(tile0 + 1, place1);
      __syncthreads();
      ask(tile0);
      put(tile0);
      arrived();
      __syncthreads();
      multiply(tile0, width);
      ask(tile0 + 1);
      put(tile0 + 1);
      float sum = 0.f;                                 // of key tid, half of the rows
      auto finish = [&](int tile) {
        if (FINAL && half == 0 && (there_s[tile & 3][warp & 3] >> lane & 1u)) a.weights[row_s[tile & 3][tid]] = sum + half_s[tile & 1][own];
      };
      for (int tile = tile0; tile < tile1; ++tile) {
        const int key0 = tile * KX_KEYS;
        float had = 0.f;
        if (FINAL && half == 0 && (there_s[tile & 3][warp & 3] >> lane & 1u) && (r0 > 0 || key0 + tid < known)) had = a.weights[row_s[tile & 3][tid]];
        settle(tile + 2, ahead);
        ahead = look();
        arrived();
        const bool ok = tc_wait_warp(&done, parity, &abort_s);
        parity ^= 1;
        fine = __syncthreads_and(ok);
        if (!fine) break;
        multiply(tile + 1, width);
        ask(tile + 2);
        if (tile > tile0) finish(tile - 1);
        sum = had;
        tc_fence_after();
        const uint32_t* there = there_s[tile & 3];
        const uint32_t at = tmem + 128 * (tile & 1) + ((uint32_t)(warp & 3) << 21);      // this warp's 32 lanes
        const bool clear = key0 + KX_KEYS - 1 <= base && (a.window <= 0 || key0 > last_place - a.window);      // all rows see all keys
        if constexpr (FINAL) {
          const int key = key0 + own;
          float part[4] = {};
          auto add = [&](int c0, const uint32_t* x, auto capped, auto masked) {
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              const float4 lse = *(const float4*)&lse_s[c0 + c];
              const float ref[4] = {lse.x, lse.y, lse.z, lse.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float y = __uint_as_float(x[c + i]);
                float e = decltype(capped)::value ? kx_exp2(bounded(y) - ref[i]) : kx_exp2(fmaf(y, scale2, -ref[i]));
                if constexpr (decltype(masked)::value) {
                  const int p = place_s[c0 + c + i];
                  if (!(key <= p && (a.window <= 0 || key > p - a.window))) e = 0.f;
                }
                part[i] += e;
              }
            }
          };
          auto columns = [&](auto capped) {            // 16 at a time, the next ones on their way
            uint32_t x[16], next[16];
            if (16 * half < width) {
              tc_ld8_issue(at + 16 * half, next);
              tc_ld8_issue(at + 16 * half + 8, next + 8);
            }
            for (int c0 = 16 * half; c0 < width; c0 += 32) {
              kt_arrived(next);
#pragma unroll
              for (int c = 0; c < 16; ++c) x[c] = next[c];
              if (c0 + 32 < width) {
                tc_ld8_issue(at + c0 + 32, next);
                tc_ld8_issue(at + c0 + 40, next + 8);
              }
              if (clear && r0 + c0 + 16 <= rows) add(c0, x, capped, std::false_type());
              else add(c0, x, capped, std::true_type());
            }
          };
          if (a.softcap > 0.f) columns(std::true_type());
          else columns(std::false_type());
          sum += (part[0] + part[1]) + (part[2] + part[3]);
        } else {
          const bool sure = clear && (there[0] & there[1] & there[2] & there[3]) == 0xffffffffu;
          const int p = place_s[own];
          auto columns = [&](auto capped) {
            constexpr bool CAPPED = decltype(capped)::value;
#pragma unroll
            for (int c0 = 0; c0 < KX_KEYS / 2; c0 += 32) {
              uint32_t x[32];
              tc_ld32(at + KX_KEYS / 2 * half + c0, x);
              float y[32];
#pragma unroll
              for (int c = 0; c < 32; ++c) y[c] = CAPPED ? bounded(__uint_as_float(x[c])) : __uint_as_float(x[c]);
              if (!sure) {
                const uint32_t is = there[2 * half + (c0 >> 5)];
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                  const int key = key0 + KX_KEYS / 2 * half + c0 + c;
                  if (!((is >> c & 1u) && key <= p && (a.window <= 0 || key > p - a.window))) y[c] = -INFINITY;
                }
              }
              float top[4] = {m, y[0], y[1], y[2]};
#pragma unroll
              for (int c = 3; c < 32; ++c) top[c & 3] = fmaxf(top[c & 3], y[c]);
              const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
              const float zero = now == -INFINITY ? 0.f : CAPPED ? now : now * scale2;
              float part[4] = {m == -INFINITY ? l : l * kx_exp2(CAPPED ? m - zero : fmaf(m, scale2, -zero)), 0.f, 0.f, 0.f};
#pragma unroll
              for (int c = 0; c < 32; ++c) part[c & 3] += kx_exp2(CAPPED ? y[c] - zero : fmaf(y[c], scale2, -zero));
              l = (part[0] + part[1]) + (part[2] + part[3]);
              m = now;
            }
          };
          if (a.softcap > 0.f) columns(std::true_type());
          else columns(std::false_type());
        }
        if (FINAL && half != 0) half_s[tile & 1][own] = sum;
        put(tile + 2);
        tc_fence_before();
      }
      __syncthreads();                                 // the rows, the keys and the scores are done with
      if (fine) finish(tile1 - 1);
    }
    if (!FINAL && a.softcap <= 0.f) m *= scale2;
  }
  if constexpr (!FINAL) {
    if (half != 0) {
      half_s[0][own] = m;
      half_s[1][own] = l;
    }
    __syncthreads();
    if (half == 0 && block_r0 + own < rows) {
      const int row = block_r0 + own;
      const float m2 = half_s[0][own], l2 = half_s[1][own], top = fmaxf(m, m2), zero = top == -INFINITY ? 0.f : top;
      float* to = a.scratch + ((long)(first + row / G) * a.n_q + head * G + row % G) * a.parts * 2 + 2 * blockIdx.x;
      to[0] = top;
      to[1] = (l == 0.f ? 0.f : l * kx_exp2(m - zero)) + (l2 == 0.f ? 0.f : l2 * kx_exp2(m2 - zero));
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLUMNS) : "memory");
  if (!fine && tid == 0) report_error(a.err, PHOTON_DEV_WAIT_TIMEOUT, seq, head, blockIdx.x);
}

template <int D, bool PACKED, bool FINAL>
static int kt_launch(const KeyWeightsMmaArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr size_t smem = 3 * 128 * D * 2 + 1024;
  static bool ready[64] = {};
  const int limit = smem_limit((const void*)key_weights_tc_kernel<D, PACKED, FINAL>, (int)smem, true, ready);
  if (limit != 0) return limit;
  return launch_pdl(key_weights_tc_kernel<D, PACKED, FINAL>, grid, dim3(KT_THREADS), smem, stream, a);
}

PHOTON_API int photon_key_weights_tc(const photon_key_weights_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->max_keys <= 0 || c->max_tokens_per_seq <= 0) return 0;
  if (c->dtype != PHOTON_BF16 || c->n_kv <= 0 || c->n_q <= 0 || c->n_q % c->n_kv || c->max_pages <= 0 || c->keep_scores) return PHOTON_ERR_ARGUMENT;
  if ((c->d != 64 && c->d != 128) || c->num_pages <= 0 || c->page_size <= 0 || (c->packed && !kv4_sizes_ok(c->page_size, c->d))) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)c->q | (uintptr_t)c->k_cache) % 16 || c->q_stride % 8) return PHOTON_ERR_UNSUPPORTED;
  const long rows = (long)c->max_tokens_per_seq * (c->n_q / c->n_kv), levels = (rows + 127) / 128;
  if (c->S > 65535 || c->n_kv * levels > 65535 || c->scale <= 0.f) return PHOTON_ERR_UNSUPPORTED;
  if (c->parts < 1 || (c->lse == nullptr && c->scratch == nullptr)) return PHOTON_ERR_ARGUMENT;
  const int tiles = (c->max_keys + KX_KEYS - 1) / KX_KEYS, each = (tiles + c->parts - 1) / c->parts;
  KeyWeightsMmaArgs a = {(const bf16*)c->q, c->weights, c->k_cache, c->block_table, c->cu_tokens, c->context_lens, c->held, c->sinks, c->lse, c->scratch, c->err, c->q_stride,
                         nullptr, 0, c->max_pages, c->S, c->n_q, c->n_kv, c->page_size, c->num_pages, c->window, c->parts, each, 0, c->scale, c->softcap};
#define WEIGH(FINAL, grid) (c->d == 64 ? c->packed ? kt_launch<64, true, FINAL>(a, grid, stream) : kt_launch<64, false, FINAL>(a, grid, stream) \
                                       : c->packed ? kt_launch<128, true, FINAL>(a, grid, stream) : kt_launch<128, false, FINAL>(a, grid, stream))
  if (c->lse == nullptr) {
    float* lse = c->scratch + c->scratch_rows * c->n_q * c->parts * 2;
    int status = WEIGH(false, dim3(c->parts, (unsigned)(c->n_kv * levels), c->S));
    if (status != 0) return status;
    const long blocks = ((long)c->max_tokens_per_seq * c->n_q + 3) / 4;
    if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
    status = launch_pdl(key_weights_lse_kernel, dim3((unsigned)blocks, c->S), dim3(128), 0, stream, a, lse);
    if (status != 0) return status;
    a.lse = lse;
  }
  return WEIGH(true, dim3(c->parts, c->n_kv, c->S));
#undef WEIGH
}
