// Attention for trees of drafted tokens on the fifth-generation tensor cores: bfloat16, heads of 64 or 128 numbers.
//
// The rows of a unit are the (node, query head) pairs of one request that share a key/value head, up to two tiles of 128 (whole nodes).  A unit's keys are walked in
// tiles of 128.  All units' tiles, one behind the other, are cut into equal ranges, one for each block of a grid that fills the
// chip once, so that requests of any lengths keep every SM busy to the end; a block walks the pieces of units in its range ("segments"), and units that ranges
// cut through are joined by a second kernel in a fixed order.
//
// A (key tile, row tile) pair is a job.  Two groups of four warps ("lanes") take jobs in turn: with two row tiles a lane has a row tile each, with one they take
// alternate key tiles of the same rows and add up at the segment's end.  While one lane's softmax runs, the tensor cores work for the other:
//   * warp 8 brings Q and key tiles, warp 10 value tiles, by TMA along the block table, into rings of shared memory (128-byte swizzle);
//   * one thread of warp 9 issues S = Q K^T (M 128, N 128) into the lane's score columns of tensor memory and O += P V, in halves of 64 keys, each as soon as its P is
//     there: S(0), S(1), P(0), S(2), P(1), ...  The tensor cores run them in that order, so scores that are there say that the lane's O before is too;
//   * a lane's thread owns a row: scores from tensor memory, running maximum and sum in 32 bits, P = 2^(..) as bfloat16 (eight bits of a weight are as many as the
//     values have) over the scores it came from.  O is rescaled only when a maximum grew by more than 2^8.
// Warps whose 32 rows do not exist pass their jobs on at once.
//
// Which keys a row sees: tree_attention.cuh.  Scores are chosen by the masks' bits, so that no key a row does not see touches it; values meet weights of 0, and 0 times what
// is not finite is not 0.  So in tiles where some row's mask cuts, what is not finite is set to zero in shared memory before the product, and rows that do
// see it get it back at the end from the cache (a path that no ordinary input takes).
//
// Every wait on an mbarrier is bounded: when one runs out the block raises a flag that all roles poll, records PHOTON_DEV_WAIT_TIMEOUT, waits (bounded) for
// its copies in flight, frees its tensor memory and returns.
#include "attention_tc.cuh"
#include "tree_attention.cuh"
#include <math.h>

#define TT_KT 128                                  // keys per tile
#define TT_THREADS 384
#define TT_LOG2E 1.4426950408889634f
#define TT_RESCALE_STEP 8.0f                       // log2 units that a maximum in use may lag behind

template <int D> struct Tt {
  static constexpr int DH = D / 64;                // 64-wide halves of a head
  static constexpr int TILE = 128 * 128 * DH;      // bytes of a Q, K or V tile
  static constexpr int HALF = 128 * 128;
  static constexpr int KS = D == 128 ? 3 : 6, VS = D == 128 ? 2 : 6;     // stages; keys are wanted two jobs before their values
  static constexpr int SMEM = (2 + KS + VS) * TILE + 3072;
  static constexpr int O_COL = 256;                // tensor memory: scores 2 x 128 columns, O 2 x D
};

struct TtParams {
  TreeParams t;
  int tile_rows, tile_nodes, box_rows, total_rows, page_shift;
  float scale_log2, cap_in;
  float* part_o; float* part_ml; int part_rows;    // partial results: [2 * blocks][D / 4][part_rows] of four, [2 * blocks][part_rows] of (maximum, sum)
};

// What a request asks for: its units and the tiles of each.
struct TtLoad { TreeRequest r; int tile_lo, tiles, blocks, units; };     // blocks: groups of two row tiles
__device__ __forceinline__ TtLoad tt_load(const TtParams& P, int s) {
  TtLoad q;
  q.r = tree_request(P.t, s);
  const int lo = P.t.window > 0 ? max(0, q.r.base - P.t.window + 1) : 0;
  q.tile_lo = lo / TT_KT;
  q.tiles = (q.r.base + q.r.n + TT_KT - 1) / TT_KT - q.tile_lo;
  q.blocks = (q.r.n + 2 * P.tile_nodes - 1) / (2 * P.tile_nodes);
  q.units = q.blocks * P.t.n_kv;
  return q;
}
// Warp-wide: the tiles of all units together, or (at >= 0) the request that holds tile `at` of them and the tiles before it.
__device__ __forceinline__ long long tt_scan(const TtParams& P, long long at, int& seq) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int s0 = 0; s0 < P.t.S; s0 += 32) {
    int n = 0;
    if (s0 + lane < P.t.S) { const TtLoad q = tt_load(P, s0 + lane); n = q.units * q.tiles; }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (at >= 0) {
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        seq = s0 + l;
        return before + __shfl_sync(0xffffffffu, upto - n, l);
      }
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return before;
}
// Blocks that have a range: every one of them has a tile at least.  The first tile of a block's range, and the block that has a tile.
__device__ __forceinline__ int tt_blocks(long long total, int blocks) { return (int)min((long long)blocks, total); }
__device__ __forceinline__ long long tt_first(long long total, int block, int blocks) { return total * block / blocks; }
__device__ __forceinline__ int tt_owner(long long total, long long tile, int blocks) { return (int)(((tile + 1) * blocks - 1) / total); }

// The segments of a block, in order.
struct TtSegments {
  int seq, unit, tile, left, serial;               // where the next one begins; tiles left in the block's range
  TtLoad q;
  // the segment
  int g, row0, rows, nq, tile0, ntiles, njobs, bit;
  bool whole;
  __device__ __forceinline__ void start(const TtParams& P) {
    int dummy = 0;
    const long long total = tt_scan(P, -1, dummy);
    const int blocks = tt_blocks(total, gridDim.x);
    left = 0; serial = 0; seq = 0; unit = 0; tile = 0;
    if ((int)blockIdx.x >= blocks) return;
    const long long a = tt_first(total, blockIdx.x, blocks), b = tt_first(total, blockIdx.x + 1, blocks);
    left = (int)(b - a);
    if (left > 0) {
      const int off = (int)(a - tt_scan(P, a, seq));
      q = tt_load(P, seq);
      unit = off / q.tiles; tile = off - unit * q.tiles;
    }
  }
  __device__ __forceinline__ bool next(const TtParams& P) {
    if (left <= 0) return false;
    while (unit >= q.units) {
      if (++seq >= P.t.S) return false;
      q = tt_load(P, seq); unit = 0; tile = 0;
    }
    const int rb = unit % q.blocks;
    g = unit / q.blocks;                           // row blocks of a head side by side: they read the same keys
    const int node0 = rb * 2 * P.tile_nodes;
    row0 = node0 * P.t.group;
    rows = (q.r.n - node0) * P.t.group;            // from row0 on
    nq = rows > P.tile_rows ? 2 : 1;
    ntiles = min(left, q.tiles - tile);
    tile0 = q.tile_lo + tile;
    njobs = ntiles * nq;
    whole = ntiles == q.tiles;
    bit = tile == 0 ? 1 : 0;
    left -= ntiles; tile += ntiles; ++serial;
    if (tile == q.tiles) { tile = 0; ++unit; }
    return true;
  }
};

// Jobs one behind the other, for the thread that issues the products.
struct TtJobs {
  TtSegments s;
  int i, n, tiles, qs;                             // job of the segment; jobs, key tiles and Q tiles so far (this one's included)
  __device__ __forceinline__ void start(const TtParams& P) { s.start(P); s.njobs = 0; s.nq = 0; i = 0; n = -1; tiles = 0; qs = 0; }
  __device__ __forceinline__ bool next(const TtParams& P) {
    if (++i >= s.njobs) {
      if (!s.next(P)) return false;
      i = 0; qs += s.nq;
    }
    ++n;
    if (first_use()) ++tiles;
    return true;
  }
  __device__ __forceinline__ int rt() const { return s.nq == 2 ? (i & 1) : 0; }
  __device__ __forceinline__ bool first_use() const { return s.nq == 1 || (i & 1) == 0; }
  __device__ __forceinline__ bool last_use() const { return s.nq == 1 || (i & 1) == 1; }
  __device__ __forceinline__ int q_index() const { return qs - s.nq + rt(); }
};

// The cache row of the lane's part of a key tile (P.total_rows, outside the map: zeros), for lanes below 128 / box_rows.
__device__ __forceinline__ int tt_part_row(const TtParams& P, const int* table, int g, int key, int key_lo, int key_end, int tok0, bool report) {
  if (key >= key_end || key + P.box_rows <= key_lo) return P.total_rows;
  const int pidx = P.page_shift >= 0 ? key >> P.page_shift : key / P.t.page_size;
  const int page = pidx < P.t.max_pages ? table[pidx] : -1;
  if (page < 0 || page >= P.t.num_pages) {
    if (report) report_error(P.t.err, PHOTON_DEV_BAD_PAGE, tok0, key, page);
    return -1;
  }
  return (page * P.t.n_kv + g) * P.t.page_size + (key - pidx * P.t.page_size);
}

template <int D>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const TtParams P) {
  using C = Tt<D>;
  extern __shared__ __align__(1024) unsigned char tt_dyn[];
  unsigned char* q_s = tt_dyn;                      // 2 tiles
  unsigned char* k_s = q_s + 2 * C::TILE;
  unsigned char* v_s = k_s + C::KS * C::TILE;
  float2* xch = reinterpret_cast<float2*>(v_s + C::VS * C::TILE);          // [2 lanes][128]: maximum and sum of a row
  uint64_t* q_full = reinterpret_cast<uint64_t*>(xch + 256);               // [2]
  uint64_t* q_empty = q_full + 2;                   // [2]
  uint64_t* k_full = q_empty + 2;                   // [KS] TMA -> MMA
  uint64_t* k_empty = k_full + C::KS;               // [KS] MMA -> TMA
  uint64_t* v_full = k_empty + C::KS;               // [VS]
  uint64_t* v_empty = v_full + C::VS;               // [VS]
  uint64_t* s_full = v_empty + C::VS;               // [lane] MMA -> softmax: the scores, and the O before
  uint64_t* p_full = s_full + 2;                    // [lane][half] softmax -> MMA (one arrival per warp)
  uint64_t* o_full = p_full + 4;                    // [lane] MMA -> softmax: all of a segment's O
  uint64_t* x_full = o_full + 2;                    // both lanes' maxima and sums are there (one arrival per warp)
  uint64_t* x_done = x_full + 1;                    // both lanes have read each other's O
  int* poison = reinterpret_cast<int*>(x_done + 1); // [2]: the segment (by its number's parity) whose values were not all finite
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(poison + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) { tc_mbar_init(&q_full[b], 1); tc_mbar_init(&q_empty[b], 1); tc_mbar_init(&s_full[b], 1); tc_mbar_init(&o_full[b], 1); }
    for (int s = 0; s < C::KS; ++s) { tc_mbar_init(&k_full[s], 1); tc_mbar_init(&k_empty[s], 1); }
    for (int s = 0; s < C::VS; ++s) { tc_mbar_init(&v_full[s], 1); tc_mbar_init(&v_empty[s], 1); }
    for (int b = 0; b < 4; ++b) tc_mbar_init(&p_full[b], 4);
    tc_mbar_init(x_full, 8);
    tc_mbar_init(x_done, 8);
    poison[0] = poison[1] = 0;
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();                                       // q, the cache and the step's tables come from kernels before
  // the tiles' swizzle counts from 1024-byte boundaries
  const bool aligned = (tc_smem(tt_dyn) & 1023) == 0;
  if (!aligned && threadIdx.x == 0) *abort_flag = 1;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (aligned && (warp == 8 || warp == 10)) {
      // ---------------- producers: warp 8 queries and keys, warp 10 values
      const bool elected = tc_elect(), keys = warp == 8;
      TtSegments s;
      s.start(P);
      const int boxes = TT_KT / P.box_rows;         // parts of a tile that may lie in different pages
      uint64_t* full = keys ? k_full : v_full;
      uint64_t* empty = keys ? k_empty : v_empty;
      const CUtensorMap* map = keys ? &map_k : &map_v;
      unsigned char* ring = keys ? k_s : v_s;
      const int stages = keys ? C::KS : C::VS;
      int qn = 0, n = 0, st = 0, ph = 1;            // Q tiles, tiles, the next stage and the parity its release has
      bool ok = true;
      while (ok && s.next(P)) {
        if (keys) {
          for (int j = 0; j < s.nq && ok; ++j, ++qn) {
            const int b = qn & 1;
            ok = tc_wait_warp(&q_empty[b], ((qn >> 1) & 1) ^ 1, abort_flag);
            if (ok && elected) {
              tc_mbar_expect_tx(&q_full[b], P.tile_rows * 128 * C::DH);      // rows beyond tile_rows stay as they are: nobody uses them
#pragma unroll
              for (int h = 0; h < C::DH; ++h)
                tc_tma_load3(q_s + b * C::TILE + h * C::HALF, &map_q, h * 64, s.g * P.t.group, s.q.r.tok0 + s.row0 / P.t.group + j * P.tile_nodes, &q_full[b]);
            }
          }
        }
        const int* table = P.t.block_table + (size_t)s.seq * P.t.max_pages;
        const int key_end = s.q.r.base + s.q.r.n, key_lo = P.t.window > 0 ? max(0, s.q.r.base - P.t.window + 1) : 0;
        for (int i = 0; i < s.ntiles && ok; ++i) {
          int rowc = P.total_rows;
          if (lane < boxes) rowc = tt_part_row(P, table, s.g, (s.tile0 + i) * TT_KT + lane * P.box_rows, key_lo, key_end, s.q.r.tok0, keys);
          if (rowc < 0) rowc = P.total_rows;
          ok = tc_wait_warp(&empty[st], ph, abort_flag);
          if (!ok) break;
          if (elected) tc_mbar_expect_tx(&full[st], C::TILE);
          unsigned char* dst = ring + st * C::TILE;
          for (int part = 0; part < boxes; ++part, dst += P.box_rows * 128) {
            const int row = __shfl_sync(0xffffffffu, rowc, part);
            if (elected)
#pragma unroll
              for (int h = 0; h < C::DH; ++h) tc_tma_load(dst + h * C::HALF, map, h * 64, row, &full[st]);
          }
          ++n;
          if (++st == stages) { st = 0; ph ^= 1; }
        }
      }
      if (elected && *abort_flag) {
        // copies already issued still write into this block's shared memory: wait for them, bounded
        for (int j = (qn > 2 ? qn - 2 : 0); j < qn; ++j)
          for (uint32_t w = 0; w < TC_WAIT_LIMIT && !tc_mbar_try(&q_full[j & 1], (j >> 1) & 1); ++w) {}
        for (int j = (n > stages ? n - stages : 0); j < n; ++j)
          for (uint32_t w = 0; w < TC_WAIT_LIMIT && !tc_mbar_try(&full[j % stages], (j / stages) & 1); ++w) {}
      }
    } else if (aligned && warp == 9) {
      // ---------------- MMA issuer: the warp waits, one of its lanes issues
      const bool elected = tc_elect();
      const uint32_t idesc_s = tc_idesc(128, TT_KT), idesc_o = tc_idesc(128, D) | TC_IDESC_B_MN;
      auto scores = [&](const TtJobs& J) -> bool {
        const int k = J.tiles - 1, st = k % C::KS, qi = J.q_index(), ln = J.n & 1;
        if (J.first_use() && !tc_wait(&k_full[st], (k / C::KS) & 1, abort_flag)) return false;
        if (J.i < J.s.nq && !tc_wait(&q_full[qi & 1], (qi >> 1) & 1, abort_flag)) return false;
        tc_fence_after();
        if (elected) {
          const uint32_t q_addr = tc_smem(q_s + (qi & 1) * C::TILE), k_addr = tc_smem(k_s + st * C::TILE);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            tc_mma(tmem + ln * 128, tc_desc(q_addr + (kk >> 2) * C::HALF + (kk & 3) * 32), tc_desc(k_addr + (kk >> 2) * C::HALF + (kk & 3) * 32), idesc_s,
                   kk > 0 ? 1u : 0u);
          tc_commit(&s_full[ln]);
          if (J.last_use()) tc_commit(&k_empty[st]);
          if (J.i >= J.s.njobs - J.s.nq) tc_commit(&q_empty[qi & 1]);
        }
        return true;
      };
      auto products = [&](const TtJobs& J) -> bool {
        const int v = J.tiles - 1, st = v % C::VS, ln = J.n & 1;
        if (J.first_use() && !tc_wait(&v_full[st], (v / C::VS) & 1, abort_flag)) return false;
        const uint32_t o = tmem + C::O_COL + ln * D, p = tmem + ln * 128, v_addr = tc_smem(v_s + st * C::TILE);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (!tc_wait(&p_full[2 * ln + half], (J.n >> 1) & 1, abort_flag)) return false;
          tc_fence_after();
          if (elected)
#pragma unroll
            for (int kk = half * 4; kk < half * 4 + 4; ++kk)       // 16 keys: two groups of 8 rows of V; P: 8 columns of packed pairs
              at_mma_ts(o, p + kk * 8, tc_desc_mn(v_addr + kk * 2048, C::HALF, 1024), idesc_o, (J.i >= 2 || kk > 0) ? 1u : 0u);
        }
        if (elected) {
          if (J.last_use()) tc_commit(&v_empty[st]);
          if (J.i + 2 >= J.s.njobs) tc_commit(&o_full[ln]);
        }
        return true;
      };
      TtJobs js, jp;
      js.start(P);
      jp = js;
      bool more = js.next(P), ok = true;
      if (more) ok = scores(js);
      if (more && ok) { more = js.next(P); if (more) ok = scores(js); }
      while (ok && jp.next(P)) {
        ok = products(jp);
        if (ok && more) { more = js.next(P); if (more) ok = scores(js); }
      }
      pdl_launch_dependents();                      // all products of this block are issued
    }
  } else {
    // ---------------- softmax: thread = row of a lane's jobs
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int ln = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + ln * 128, o_addr = lane_addr + C::O_COL + ln * D;
    const float c = P.scale_log2, cap = P.t.softcap, cap_in = P.cap_in * 2.8853900817779268f;     // tanh(x) = 1 - 2 / (2^(2 x log2 e) + 1)
    TtSegments s;
    if (aligned) s.start(P); else s.left = 0;
    const int boxes = TT_KT / P.box_rows;
    int n0 = 0, tiles = 0, ends = 0, exchanges = 0; // jobs and tiles before the segment; segments in which this lane had jobs; exchanges so far
    bool ok = true;
    for (; ok && s.next(P); n0 += s.njobs, tiles += s.ntiles) {
      const int first = (n0 & 1) == ln ? 0 : 1;     // this lane's first job of the segment
      const int rt = s.nq == 2 ? first : 0;
      const int row = rt * P.tile_rows + r;         // from row0 on
      const bool valid = r < P.tile_rows && row < s.rows;
      const bool busy = __any_sync(0xffffffffu, valid);
      const int t = valid ? s.q.r.tok0 + (s.row0 + row) / P.t.group : s.q.r.tok0;
      const int lo = valid && P.t.window > 0 ? max(0, P.t.positions[t] - P.t.window + 1) : 0;
      const int base = s.q.r.base, key_end = base + s.q.r.n;
      const int key_lo = P.t.window > 0 ? max(0, base - P.t.window + 1) : 0;
      const int cut_lo = P.t.window > 0 ? key_end - P.t.window : -1;       // no row's window begins behind this key
      const int* table = P.t.block_table + (size_t)s.seq * P.t.max_pages;
      // parts of a tile whose page is missing, one bit a part
      auto missing = [&](int key_base) -> uint32_t {
        const bool gone = lane < boxes && tt_part_row(P, table, s.g, key_base + lane * P.box_rows, key_lo, key_end, 0, false) < 0;
        return __ballot_sync(0xffffffffu, gone);
      };
      float m_used = -INFINITY, l = 0.f;
      for (int i = first; i < s.njobs; i += 2) {
        const int ti = s.nq == 2 ? i >> 1 : i, key_base = (s.tile0 + ti) * TT_KT, cnt = (n0 + i) >> 1;
        const uint32_t gone = missing(key_base);
        const bool edge = key_base + TT_KT > base || key_base <= cut_lo || gone != 0;
        if (edge && (s.nq == 1 || rt == 0)) {
          // values that are not finite: zeros, before this job's P says that they may be read
          const int v = tiles + ti, st = v % C::VS;
          if (!tc_wait_warp(&v_full[st], (v / C::VS) & 1, abort_flag)) { ok = false; break; }
          unsigned char* vst = v_s + st * C::TILE;
          bool found = false;
#pragma unroll 4
          for (int e = r; e < C::TILE / 16; e += 128) {
            uint4 x = *reinterpret_cast<uint4*>(vst + e * 16);
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool bad = false;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              if ((w[u] & 0x7f80u) == 0x7f80u) { w[u] &= 0xffff0000u; bad = true; }
              if ((w[u] & 0x7f800000u) == 0x7f800000u) { w[u] &= 0xffffu; bad = true; }
            }
            if (bad) {
              *reinterpret_cast<uint4*>(vst + e * 16) = make_uint4(w[0], w[1], w[2], w[3]);
              found |= key_base + ((e >> 3) & 127) < key_end;
            }
          }
          if (found) *(volatile int*)&poison[s.serial & 1] = s.serial;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // generic writes -> the tensor core's reads
        }
        if (!tc_wait_warp(&s_full[ln], cnt & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        if (!busy) {
          __syncwarp();
          if (lane == 0) { tc_mbar_arrive(&p_full[2 * ln]); tc_mbar_arrive(&p_full[2 * ln + 1]); }
          continue;
        }
        uint32_t sv[TT_KT];
#pragma unroll
        for (int u = 0; u < TT_KT; u += 32) tc_ld32_issue(s_addr + u, sv + u);
        tc_ld_wait();
        if (cap > 0.f) {
#pragma unroll
          for (int u = 0; u < TT_KT; ++u) {
            const float e = at_exp2(__uint_as_float(sv[u]) * cap_in);
            sv[u] = __float_as_uint(cap - __fdividef(2.0f * cap, e + 1.0f));
          }
        }
        if (edge) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t bits = valid ? tree_visible32(P.t, s.q.r, t, key_base + 32 * w, lo) : 0u;
            if (gone != 0) {
              for (int u = 0; u < 32; u += min(P.box_rows, 32))
                if ((gone >> ((32 * w + u) / P.box_rows)) & 1u) bits &= ~((P.box_rows >= 32 ? 0xffffffffu : (1u << P.box_rows) - 1u) << u);
            }
#pragma unroll
            for (int u = 0; u < 32; ++u) sv[32 * w + u] = (bits >> u) & 1u ? sv[32 * w + u] : 0xff800000u;       // -inf
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < TT_KT; u += 8) {
#pragma unroll
          for (int w = 0; w < 4; ++w) mx4[w] = at_max3(mx4[w], __uint_as_float(sv[u + 2 * w]), __uint_as_float(sv[u + 2 * w + 1]));
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        const float cand = fmaxf(m_used, mx * c);
        float factor = 1.f;
        const bool grow = cand > m_used + TT_RESCALE_STEP;                   // also the first finite maximum
        if (grow) { factor = at_exp2(m_used - cand); m_used = cand; l *= factor; }
        const float nsub = (m_used == -INFINITY) ? 0.f : -m_used;
        if (i >= 2 && __any_sync(0xffffffffu, grow)) {
          // rescale O: the products of the lane's job before have landed, because they were issued before these scores
#pragma unroll 1
          for (int cc = 0; cc < D; cc += 32) {
            uint32_t ov[32];
            tc_ld32(o_addr + cc, ov);
#pragma unroll
            for (int u = 0; u < 32; ++u) ov[u] = __float_as_uint(__uint_as_float(ov[u]) * factor);
            tc_st32(o_addr + cc, ov);
          }
          tc_st_wait();
        }
        // P = 2^(score c - maximum in use), packed pairs over the scores they came from (32 columns per 64 keys)
        float sum8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int u = 0; u < 64; u += 2) {
            float x0, x1;
            at_fma2(x0, x1, __uint_as_float(sv[half * 64 + u]), __uint_as_float(sv[half * 64 + u + 1]), c, nsub);
            const float p0 = at_exp2(x0), p1 = at_exp2(x1);
            at_add2(sum8[u & 6], sum8[(u & 6) + 1], p0, p1);
            pk[u >> 1] = at_pack(p0, p1);
          }
          tc_st32(s_addr + half * 32, pk);
          tc_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) tc_mbar_arrive(&p_full[2 * ln + half]);
        }
        l += ((sum8[0] + sum8[1]) + (sum8[2] + sum8[3])) + ((sum8[4] + sum8[5]) + (sum8[6] + sum8[7]));
      }
      if (!ok) break;

      // ---- the segment's end
      const bool had = first < s.njobs;             // with one key tile one of the lanes has no job
      if (had) { if (!tc_wait_warp(&o_full[ln], ends & 1, abort_flag)) break; ++ends; tc_fence_after(); }
      float f0 = 1.f, f1 = 0.f;                     // what this lane's and the other's O count for
      int col0 = 0, col1 = D;
      if (s.nq == 1) {
        // both lanes have the same rows: each takes half of the columns of both O
        xch[ln * 128 + r] = make_float2(m_used, l);
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(x_full);
        if (!tc_wait_warp(x_full, exchanges & 1, abort_flag)) break;
        tc_fence_after();                           // the other lane waited for its O before it arrived
        const float2 o = xch[(ln ^ 1) * 128 + r];
        const float top = fmaxf(m_used, o.x), sub = top == -INFINITY ? 0.f : top;
        f0 = at_exp2(m_used - sub); f1 = at_exp2(o.x - sub);
        l = l * f0 + o.y * f1;
        m_used = top;
        col0 = ln * (D / 2); col1 = col0 + D / 2;
      }
      const bool both = s.nq == 1 && s.njobs > 1;
      const bool fix = *(volatile int*)&poison[s.serial & 1] == s.serial;
      const int head = s.g * P.t.group + (valid ? (s.row0 + row) % P.t.group : 0);
      float inv = 1.f;
      if (s.whole) {
        float total = l;
        if (P.t.sinks && l != 0.f) total += exp2f(fmaf(P.t.sinks[head], TT_LOG2E, -m_used));       // the sink's weight, relative to the maximum in use
        inv = total != 0.f ? 1.f / total : 0.f;
      }
      if (busy) {
        const size_t slot = (size_t)blockIdx.x * 2 + s.bit;
        if (!s.whole && valid && col0 == 0) *reinterpret_cast<float2*>(P.part_ml + (slot * P.part_rows + row) * 2) = make_float2(m_used, l);
#pragma unroll 1
        for (int cc = col0; cc < col1; cc += 32) {
          uint32_t ov[32], ow[32];
          // a lane without jobs has nothing in its O: the other's alone counts
          tc_ld32_issue(had ? o_addr + cc : lane_addr + C::O_COL + (ln ^ 1) * D + cc, ov);
          if (both) tc_ld32_issue(lane_addr + C::O_COL + (ln ^ 1) * D + cc, ow);
          tc_ld_wait();
          float x[32];
          const float a = had ? f0 : f1;
#pragma unroll
          for (int u = 0; u < 32; ++u) x[u] = __uint_as_float(ov[u]) * a + (both ? __uint_as_float(ow[u]) * f1 : 0.f);
          if (fix && valid) {
            // what was not finite, for the rows that see it
            const bf16* vc = (const bf16*)P.t.v_cache;
            for (int ti = 0; ti < s.ntiles; ++ti) {
              const int key_base = (s.tile0 + ti) * TT_KT;
              for (int w = 0; w < 4; ++w) {
                for (uint32_t bits = tree_visible32(P.t, s.q.r, t, key_base + 32 * w, lo); bits != 0; bits &= bits - 1) {
                  const int key = key_base + 32 * w + __ffs(bits) - 1;
                  const int page = key / P.t.page_size < P.t.max_pages ? table[key / P.t.page_size] : -1;
                  if (page < 0 || page >= P.t.num_pages) continue;
                  const bf16* vr = vc + (((size_t)page * P.t.n_kv + s.g) * P.t.page_size + key % P.t.page_size) * D + cc;
#pragma unroll 1
                  for (int u = 0; u < 32; ++u) {
                    const float y = to_f32(vr[u]);
                    if (!isfinite(y)) {
#pragma unroll
                      for (int z = 0; z < 32; ++z) if (z == u) x[z] += y;
                    }
                  }
                }
              }
            }
          }
          if (valid) {
            if (s.whole) {
              bf16* dst = (bf16*)P.t.out + (size_t)t * P.t.out_stride + (size_t)head * D + cc;
#pragma unroll
              for (int u = 0; u < 32; u += 8) {
                uint4 v4;
                v4.x = at_pack(x[u] * inv, x[u + 1] * inv); v4.y = at_pack(x[u + 2] * inv, x[u + 3] * inv);
                v4.z = at_pack(x[u + 4] * inv, x[u + 5] * inv); v4.w = at_pack(x[u + 6] * inv, x[u + 7] * inv);
                *reinterpret_cast<uint4*>(dst + u) = v4;
              }
            } else {
              float4* dst = reinterpret_cast<float4*>(P.part_o) + (slot * (D / 4) + cc / 4) * P.part_rows + row;
#pragma unroll
              for (int u = 0; u < 8; ++u) dst[(size_t)u * P.part_rows] = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
            }
          }
        }
      }
      tc_fence_before();
      if (s.nq == 1) {
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(x_done);
        if (!tc_wait_warp(x_done, exchanges & 1, abort_flag)) break;
        ++exchanges;
      }
    }
  }
  // ---------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) report_error(P.t.err, PHOTON_DEV_WAIT_TIMEOUT, blockIdx.x, 0, 0);
}

// Joins the pieces of units that more than one block worked on, in the blocks' order.  A block takes 32 rows of a unit.
template <int D>
__global__ void __launch_bounds__(256)
tree_join_tc_kernel(const TtParams P, int blocks, int chunks) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b = blockIdx.x;
  const int chunk = b % chunks; b /= chunks;
  const int g = b % P.t.n_kv, seq = b / P.t.n_kv;
  const TtLoad q = tt_load(P, seq);
  const int per_block = (2 * P.tile_rows + 31) / 32;                          // chunks of a row block
  const int rb = chunk / per_block, r0 = (chunk % per_block) * 32;
  if (rb >= q.blocks || q.tiles <= 0) return;
  const int row0 = rb * 2 * P.tile_rows, rows = min(2 * P.tile_rows, q.r.n * P.t.group - row0);
  if (r0 >= rows) return;
  // the tiles before this request, and all tiles
  long long total = 0, before = 0;
  for (int s0 = 0; s0 < P.t.S; s0 += 32) {
    long long n = 0;
    if (s0 + lane < P.t.S) { const TtLoad x = tt_load(P, s0 + lane); n = (long long)x.units * x.tiles; }
    long long mine = s0 + lane < seq ? n : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { n += __shfl_xor_sync(0xffffffffu, n, o); mine += __shfl_xor_sync(0xffffffffu, mine, o); }
    total += n; before += mine;
  }
  const long long u0 = before + (long long)(g * q.blocks + rb) * q.tiles, u1 = u0 + q.tiles - 1;
  const int used = tt_blocks(total, blocks), c0 = tt_owner(total, u0, used), c1 = tt_owner(total, u1, used);
  if (c0 == c1) return;                             // one block had it all
  const int row = r0 + lane;
  const bool valid = row < rows;
  const int rr = valid ? row : rows - 1;
  const int t = q.r.tok0 + (row0 + rr) / P.t.group, head = g * P.t.group + (row0 + rr) % P.t.group;
  const float sink = P.t.sinks ? P.t.sinks[head] * TT_LOG2E : -INFINITY;
  auto slot = [&](int c) { return (size_t)2 * c + (c == c0 ? 1 : 0); };
  float top = -INFINITY;
  for (int c = c0; c <= c1; ++c) top = fmaxf(top, P.part_ml[(slot(c) * P.part_rows + rr) * 2]);
  top = fmaxf(top, sink);
  const float sub = top == -INFINITY ? 0.f : top;
  float keys = 0.f;
  for (int c = c0; c <= c1; ++c) {
    const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + (slot(c) * P.part_rows + rr) * 2);
    keys += ml.y * at_exp2(ml.x - sub);
  }
  const float sum = keys + (P.t.sinks ? at_exp2(sink - sub) : 0.f);
  const float inv = sum != 0.f && keys != 0.f ? 1.f / sum : 0.f;
  for (int cc = warp; cc < D / 4; cc += 8) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0; c <= c1; ++c) {
      const float w = at_exp2(P.part_ml[(slot(c) * P.part_rows + rr) * 2] - sub);
      const float4 x = *(reinterpret_cast<const float4*>(P.part_o) + (slot(c) * (D / 4) + cc) * P.part_rows + rr);
      if (w != 0.f) { a.x = fmaf(w, x.x, a.x); a.y = fmaf(w, x.y, a.y); a.z = fmaf(w, x.z, a.z); a.w = fmaf(w, x.w, a.w); }
    }
    if (valid) {
      uint2 v2;
      v2.x = at_pack(a.x * inv, a.y * inv); v2.y = at_pack(a.z * inv, a.w * inv);
      *reinterpret_cast<uint2*>((bf16*)P.t.out + (size_t)t * P.t.out_stride + (size_t)head * D + cc * 4) = v2;
    }
  }
}

template <int D>
static int tt_launch(TtParams& P, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, int chunks, cudaStream_t stream) {
  static bool ready[64] = {};                      // the limit is set once a device
  int st = tree_smem_limit((const void*)tree_attention_tc_kernel<D>, Tt<D>::SMEM, ready);
  if (st != 0) return st;
  st = launch_pdl(tree_attention_tc_kernel<D>, dim3(blocks), dim3(TT_THREADS), (size_t)Tt<D>::SMEM, stream, mq, mk, mv, P);
  if (st != 0) return st;
  return launch_pdl(tree_join_tc_kernel<D>, dim3((unsigned)((long)P.t.S * P.t.n_kv * chunks)), dim3(256), 0, stream, P, blocks, chunks);
}

// Rows of a unit that a partial result has room for.
static int tt_part_rows(int max_tokens, int group) {
  const int tile_nodes = 128 / group, rows = max_tokens * group, most = 2 * tile_nodes * group;
  return ((rows < most ? rows : most) + 31) / 32 * 32;
}
PHOTON_API long photon_tree_attention_tc_scratch(int max_tokens_per_seq, int n_q, int n_kv, int d, int blocks) {
  if (n_kv <= 0 || n_q < n_kv || n_q / n_kv > 128 || max_tokens_per_seq <= 0 || blocks <= 0) return 0;
  return 2L * blocks * tt_part_rows(max_tokens_per_seq, n_q / n_kv) * (d + 2);
}

PHOTON_API int photon_tree_attention_tc(const photon_tree_call* call, cudaStream_t stream) {
  if (call->S <= 0 || call->T <= 0 || call->max_tokens_per_seq <= 0) return 0;
  TtParams P;
  TreeParams& t = P.t;
  int st = tree_params(call, t);
  if (st != 0) return st;
  const int G = t.group, d = t.d, page_size = t.page_size;
  if (call->dtype != PHOTON_BF16 || (d != 64 && d != 128) || G > 128) return PHOTON_ERR_UNSUPPORTED;
  if (page_size < 8 || (page_size & 7) || !((64 % page_size) == 0 || (page_size % 64) == 0)) return PHOTON_ERR_UNSUPPORTED;
  if (((uintptr_t)t.q & 15) || (t.q_stride & 7) || ((uintptr_t)t.k_cache & 15) || ((uintptr_t)t.v_cache & 15) || ((uintptr_t)t.out & 15) || (t.out_stride & 7))
    return PHOTON_ERR_UNSUPPORTED;
  const long total_rows = (long)t.num_pages * t.n_kv * page_size;
  if (total_rows > 0x7fffff00L) return PHOTON_ERR_UNSUPPORTED;
  if (call->scratch == nullptr || call->scratch_floats < photon_tree_attention_tc_scratch(t.max_tokens, t.n_q, t.n_kv, d, call->parts)) return PHOTON_ERR_ARGUMENT;
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return PHOTON_ERR_UNSUPPORTED;
  P.tile_nodes = 128 / G; P.tile_rows = P.tile_nodes * G;
  P.box_rows = page_size < 64 ? page_size : (page_size % 128 == 0 ? 128 : 64);
  P.total_rows = (int)total_rows;
  CUtensorMap map_q, map_k, map_v;
  {
    cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)t.n_q, (cuuint64_t)t.T};
    cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)t.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)P.tile_nodes};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(&map_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(t.q), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return PHOTON_ERR_ARGUMENT;
  }
  st = make_map(&map_k, t.k_cache, total_rows, d, d, P.box_rows);
  if (st != 0) return st;
  st = make_map(&map_v, t.v_cache, total_rows, d, d, P.box_rows);
  if (st != 0) return st;
  P.page_shift = -1;
  for (int sh = 0; sh < 20; ++sh) if ((1 << sh) == page_size) P.page_shift = sh;
  P.scale_log2 = t.scale * TT_LOG2E; P.cap_in = 0.f;
  if (t.softcap > 0.f) { P.cap_in = t.scale / t.softcap; P.scale_log2 = TT_LOG2E; }
  P.part_rows = tt_part_rows(t.max_tokens, G);
  P.part_o = call->scratch;
  P.part_ml = call->scratch + 2L * call->parts * P.part_rows * d;
  // 32 rows a block of the second kernel
  const long most = (long)t.max_tokens * G, span = 2L * P.tile_rows;
  const long chunks = most / span * ((span + 31) / 32) + (most % span + 31) / 32;
  if ((long)t.S * t.n_kv * chunks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  return d == 64 ? tt_launch<64>(P, map_q, map_k, map_v, call->parts, (int)chunks, stream)
                 : tt_launch<128>(P, map_q, map_k, map_v, call->parts, (int)chunks, stream);
}
