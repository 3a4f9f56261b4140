// Attention for trees of drafted tokens on the fifth-generation tensor cores: bfloat16, heads of 64 or 128 numbers.
//
// The rows of a unit are (node, query head) pairs of one request that share a key/value head, up to 128 (whole nodes).  A unit's keys are walked in tiles of 64.  All units'
// tiles, one behind the other, are cut into equal ranges, one for each block of a grid that fills the chip once, so that requests of any
// lengths keep every SM busy to the end; a block walks the pieces of units in its range ("segments").  Units that ranges cut through are joined by a second
// kernel, in the blocks' order.  Where whole units keep the chip as busy they are dealt out whole, the longest first, and there is nothing to join.  Where there are
// few units, each is a cluster's: its blocks have equal runs of its tiles and join their results in each other's shared memory, once their rings are empty.
//
// Two blocks share an SM, so that one's loads and products run while the other begins or ends a segment.  In a block
//   * warp 4 brings Q, key and value tiles by TMA along the block table into shared memory (128-byte swizzle); keys and values share one ring;
//   * one thread of warp 5 issues S = Q K^T (M 128, N 64) into one of NB score buffers of tensor memory, and O += P V: S(0) .. S(NB - 1), P(0), S(NB), P(1), ..;
//   * warps 0-3 own one row per thread: scores from tensor memory, running maximum and sum in 32 bits, P = 2^(..) as bfloat16 (eight bits of a weight are as many
//     as the values have) over the scores it came from.  O is rescaled only when a maximum grew by more than 2^8.
// Warps whose 32 rows do not exist pass their tiles on at once.
//
// Which keys a row sees: tree_attention.cuh.  Scores are chosen by the masks' bits, so that no key a row does not see touches it; values meet weights of 0, and 0 times what
// is not finite is not 0.  So where some row's mask cuts, what is not finite is set to zero in shared memory before the product, and rows that do see it get
// it back at the end from the cache (a path that no ordinary input takes).
//
// What bounds it.  Full batches: memory.  64 requests of 32 nodes behind up to 6,000 keys (24/8 heads of 128): 170 us, 0.85 of the copy rate.  Many rows: the softmax between two products;
// 2 requests of 64 nodes behind 32,768 keys (32/8 heads of 128): 90 us, 770 TFLOP/s, tensor pipe and exponentials each below half.  Few units: begin, end and join.  8 of 27
// behind up to 2,500 (32/8 heads of 64): 20 us for 32 MB.  Measured slower there: tiles of 128 keys, a segment's end behind the next one's first scores, two threads a row,
// copies of a row with a part of a tile's keys each, weights by the old maximum before the tile's own is known.
//
// Every wait on an mbarrier is bounded: when one runs out the block raises a flag that all roles poll, records PHOTON_DEV_WAIT_TIMEOUT, waits (bounded) for
// its copies in flight, frees its tensor memory and returns.
#include "attention_tc.cuh"
#include "tree_attention.cuh"
#include <math.h>
#include <type_traits>

#define TT_KT 64                                   // keys per tile
#define TT_THREADS 192
#define TT_MAX_BLOCKS 320                          // of the first kernel's grid
#define TT_CLUSTER 8                               // blocks that may share a unit
#define TT_LOG2E 1.4426950408889634f
#define TT_RESCALE_STEP 8.0f                       // log2 units that a maximum in use may lag behind

template <int D> struct Tt {
  static constexpr int DH = D / 64;                // 64-wide halves of a head
  static constexpr int QTILE = 128 * 128 * DH;     // bytes of a Q tile
  static constexpr int TILE = TT_KT * 128 * DH;    // bytes of a K or V tile
  static constexpr int HALF = TT_KT * 128;         // of one 64-wide half of it
  static constexpr int NS = D == 128 ? 5 : 10;     // stages of the ring
  static constexpr int QS = D == 128 ? 1 : 2;      // Q tiles.  Heads of 128: with at most 64 rows one tile's room holds two
  static constexpr int SMEM = QS * QTILE + NS * TILE + 1024;      // two blocks an SM
  static constexpr int NB = D == 128 ? 2 : 3;      // score buffers: 64 columns of tensor memory each, O behind them
  static constexpr int O_COL = NB * 64;
  static constexpr int COLS = 256;
};

struct TtParams {
  TreeParams t;
  int whole, sorted, blocks_sm, cluster, levels;                   // whole units in any case: one kernel; the longest of them first; blocks that the chip holds; blocks that share a unit; most row tiles of a request
  int tile_rows, tile_nodes, box_rows, total_rows, page_shift;
  int q_slots, q_slot_bytes, q_half_bytes, q_nodes;          // Q tiles in shared memory, bytes between them and between a tile's halves, nodes of a copy
  float scale_log2, cap_in;
  int4* meta;                                      // [blocks][2]: the unit that a block begins and leaves to the next ones: (blocks behind it, first row, rows, head), (first node, ..)
  float* part_o; float* part_ml; int part_rows;    // partial results: [2 * blocks][D / 4][part_rows] of four, [2 * blocks][part_rows] of (maximum, sum)
};

// Keys and values share one ring, in the order in which they are wanted: K0 K1 V0 K2 V1 K3 V2 ..  The place in it of a block's key tile k and of its values; stage and
// parity follow from the place.  (Behind the last keys one place stays free.)
__device__ __forceinline__ int tt_place_k(int k) { return k == 0 ? 0 : 2 * k - 1; }
__device__ __forceinline__ int tt_place_v(int k) { return 2 * k + 2; }

// What a request asks for: its units and the tiles of each.
struct TtLoad { TreeRequest r; int tile_lo, tiles, blocks, units; };     // blocks: row tiles
__device__ __forceinline__ TtLoad tt_load(const TtParams& P, int s) {
  TtLoad q;
  q.r = tree_request(P.t, s);
  const int lo = P.t.window > 0 ? max(0, q.r.base - P.t.window + 1) : 0;
  q.tile_lo = lo / TT_KT;
  q.tiles = (q.r.base + q.r.n + TT_KT - 1) / TT_KT - q.tile_lo;
  q.blocks = (q.r.n + P.tile_nodes - 1) / P.tile_nodes;
  q.units = q.blocks * P.t.n_kv;
  return q;
}
// Ranges are cut from the tiles of all requests' first row tiles, then those of the second ones, and so on: a request's row tiles read the same keys, and where
// all have as many of them, as many ranges apart, at the same time.  (2 requests of 2 row tiles behind 32,768 keys read them once instead of twice: 107 -> 90 us.)
//
// Warp-wide: the tiles of all units together and in `seq` those of the longest unit.
__device__ __forceinline__ long long tt_total(const TtParams& P, int& longest) {
  const int lane = threadIdx.x & 31;
  long long total = 0;
  longest = 0;
  for (int s = lane; s < P.t.S; s += 32) {
    const TtLoad q = tt_load(P, s);
    total += (long long)q.units * q.tiles;
    if (q.units > 0) longest = max(longest, q.tiles);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  longest = __reduce_max_sync(0xffffffffu, longest);
  return total;
}
// Warp-wide: the request and its row tile that hold tile `at` of them, and the tiles before those.
__device__ __forceinline__ long long tt_find(const TtParams& P, long long at, int& seq, int& level) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (level = 0; level < P.levels; ++level) {
    for (int s0 = 0; s0 < P.t.S; s0 += 32) {
      int n = 0;
      if (s0 + lane < P.t.S) { const TtLoad q = tt_load(P, s0 + lane); n = q.blocks > level ? P.t.n_kv * q.tiles : 0; }
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > at);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        seq = s0 + l;
        return before + __shfl_sync(0xffffffffu, upto - n, l);
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  seq = P.t.S;
  return before;
}
// Whole units are dealt out with the longest first: the units before each request, for up to TT_SORTED of them; more come as they are.
#define TT_SORTED 64
struct TtOrder { int tiles[TT_SORTED]; unsigned short front[TT_SORTED], units[TT_SORTED]; };
// By the whole block, with a barrier inside.
__device__ __forceinline__ void tt_sort(const TtParams& P, TtOrder& o) {
  const int t = threadIdx.x;
  int tiles = 0, units = 0, front = 0;
  if (t < P.t.S) {
    const TtLoad q = tt_load(P, t);
    tiles = q.tiles; units = q.units;
    o.tiles[t] = tiles; o.units[t] = (unsigned short)units;
  }
  __syncthreads();
  if (t < P.t.S) {
    for (int x = 0; x < P.t.S; ++x) if (o.tiles[x] > tiles || (o.tiles[x] == tiles && x < t)) front += o.units[x];
    o.front[t] = (unsigned short)front;
  }
  __syncthreads();
}
// Warp-wide: the request that holds unit `at` of the whole units, and the units before it; false: there is no such unit.
__device__ __forceinline__ bool tt_unit(const TtParams& P, const TtOrder& o, int at, int& seq, int& before) {
  const int lane = threadIdx.x & 31;
  if (P.sorted) {
#pragma unroll
    for (int s0 = 0; s0 < TT_SORTED; s0 += 32) {
      const int s = s0 + lane;
      const bool mine = s < P.t.S && at >= o.front[s] && at < o.front[s] + o.units[s];
      const unsigned hit = __ballot_sync(0xffffffffu, mine);
      if (hit != 0) {
        seq = s0 + __ffs(hit) - 1;
        before = o.front[seq];
        return true;
      }
    }
    return false;
  }
  int total = 0;
  for (int s0 = 0; s0 < P.t.S; s0 += 32) {
    int n = 0;
    if (s0 + lane < P.t.S) n = tt_load(P, s0 + lane).units;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, total + upto > at);
    if (hit != 0) {
      const int l = __ffs(hit) - 1;
      seq = s0 + l;
      before = total + __shfl_sync(0xffffffffu, upto - n, l);
      return true;
    }
    total += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}
// Blocks that have a range: every one of them has a tile at least.  The first tile of a block's range, and the block that has a tile.
__device__ __forceinline__ int tt_blocks(long long total, int blocks) { return (int)min((long long)blocks, total); }
__device__ __forceinline__ long long tt_first(long long total, int block, int blocks) { return total * block / blocks; }
__device__ __forceinline__ int tt_owner(long long total, long long tile, int blocks) { return (int)(((tile + 1) * blocks - 1) / total); }

// The segments of a block, in order: the pieces of units in its range, or whole units.
struct TtSegments {
  int seq, unit, tile, level, left, serial, round; // where the next one begins (ranges: head and row tile); tiles left in the block's range; whole units so far
  const TtOrder* order;
  bool units_whole;
  TtLoad q;
  // the segment
  int g, row0, rows, tile0, ntiles, bit;
  bool whole;
  __device__ __forceinline__ void start(const TtParams& P, const TtOrder* o, bool w, long long total) {
    order = o; units_whole = w;
    left = 0; serial = 0; seq = 0; unit = 0; tile = 0; level = 0; round = 0; rows = 0;
    const int blocks = tt_blocks(total, gridDim.x);
    if (w || (int)blockIdx.x >= blocks) return;
    const long long first = tt_first(total, blockIdx.x, blocks);
    left = (int)(tt_first(total, blockIdx.x + 1, blocks) - first);
    const int off = (int)(first - tt_find(P, first, seq, level));
    if (seq >= P.t.S) { left = 0; return; }
    q = tt_load(P, seq);
    unit = off / q.tiles; tile = off - unit * q.tiles;
  }
  __device__ __forceinline__ void place(const TtParams& P, int rb, int h) {        // the unit's head and rows
    // Requests begin with different heads: blocks that are as far in different requests
    // otherwise read the same part of every page at a time, and some of the memory's channels wait for others (148 requests of 12,288 keys: 6 %).
    h += seq % P.t.n_kv;
    g = h < P.t.n_kv ? h : h - P.t.n_kv;
    row0 = rb * P.tile_rows;
    rows = min(q.r.n * P.t.group - row0, P.tile_rows);
  }
  __device__ __forceinline__ bool next(const TtParams& P) {       // by whole warps
    if (P.cluster > 1) {
      // one unit for the cluster, and this block's part of its tiles; a short unit leaves some blocks without
      if (round++ > 0) return false;
      rows = 0;
      const int u = blockIdx.x / P.cluster, rank = blockIdx.x - u * P.cluster, per = P.t.n_kv * P.levels;
      seq = u / per;
      if (seq >= P.t.S) return false;
      q = tt_load(P, seq);
      const int h = (u - seq * per) / P.levels, rb = u - seq * per - h * P.levels;       // row tiles of a head side by side
      if (rb >= q.blocks) return false;
      place(P, rb, h);
      // the last block, whose tiles masks cut, has a run that is no longer than the others'
      const int first = (q.tiles * rank + P.cluster - 1) / P.cluster;
      ntiles = (q.tiles * (rank + 1) + P.cluster - 1) / P.cluster - first;
      tile0 = q.tile_lo + first; whole = false; bit = 0; serial = 1;
      return ntiles > 0;
    }
    if (units_whole) {
      // the longest units first, to and fro over the blocks
      const int u = (round & 1) ? (round + 1) * (int)gridDim.x - 1 - (int)blockIdx.x : round * (int)gridDim.x + (int)blockIdx.x;
      ++round;
      int front;
      if (!tt_unit(P, *order, u, seq, front)) return false;
      q = tt_load(P, seq); unit = u - front; tile = 0; left = q.tiles;
    }
    if (left <= 0) return false;
    if (units_whole) {
      place(P, unit % q.blocks, unit / q.blocks);
    } else {
      while (unit >= P.t.n_kv || q.blocks <= level) {
        if (++seq >= P.t.S) {
          if (++level >= P.levels) return false;
          seq = 0;
        }
        q = tt_load(P, seq); unit = 0; tile = 0;
      }
      place(P, level, unit);
    }
    ntiles = min(left, q.tiles - tile);
    tile0 = q.tile_lo + tile;
    whole = ntiles == q.tiles;
    bit = tile == 0 ? 1 : 0;
    left -= ntiles; tile += ntiles; ++serial;
    if (tile == q.tiles) { tile = 0; ++unit; }
    return true;
  }
};

// softcap tanh(x / softcap) = scale x' q(y^2) of two raw scores x' at a time, y = cap_in x': tree_tanh_half's series on pairs (sm_100 has one instruction for both).
__device__ __forceinline__ uint64_t tt_both(float c) { return (uint64_t)__float_as_uint(c) << 32 | __float_as_uint(c); }
__device__ __forceinline__ void tt_cap_pair(uint32_t& a, uint32_t& b, float cap_in, float scale) {
  asm("{\n.reg .b64 x, y, z, p;\nmov.b64 x, {%0, %1};\nmul.rn.f32x2 y, x, %2;\nmul.rn.f32x2 z, y, y;\nfma.rn.f32x2 p, z, %4, %5;\nfma.rn.f32x2 p, p, z, %6;\n"
      "fma.rn.f32x2 p, p, z, %7;\nfma.rn.f32x2 p, p, z, %8;\nfma.rn.f32x2 p, p, z, %9;\nmul.rn.f32x2 x, x, %3;\nmul.rn.f32x2 x, x, p;\nmov.b64 {%0, %1}, x;\n}"
      : "+r"(a), "+r"(b)
      : "l"(tt_both(cap_in)), "l"(tt_both(scale)), "l"(tt_both(-1382.f / 155925.f)), "l"(tt_both(62.f / 2835.f)), "l"(tt_both(-17.f / 315.f)), "l"(tt_both(2.f / 15.f)),
        "l"(tt_both(-1.f / 3.f)), "l"(tt_both(1.f)));
}

template <int D>
__global__ void __launch_bounds__(TT_THREADS, 2)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const TtParams P) {
  using C = Tt<D>;
  extern __shared__ __align__(1024) unsigned char tt_dyn[];
  unsigned char* q_s = tt_dyn;
  unsigned char* kv_s = q_s + C::QS * C::QTILE;     // NS tiles
  uint64_t* q_full = reinterpret_cast<uint64_t*>(kv_s + C::NS * C::TILE);  // [2]
  uint64_t* q_empty = q_full + 2;                   // [2]
  uint64_t* full = q_empty + 2;                     // [NS] TMA -> MMA
  uint64_t* empty = full + C::NS;                   // [NS] MMA -> TMA
  uint64_t* s_full = empty + C::NS;                 // [buffer] MMA -> softmax
  uint64_t* p_full = s_full + C::NB;                // [buffer] softmax -> MMA (one arrival per warp)
  // [buffer] MMA -> softmax: the products of a tile have landed.  A barrier for each buffer: while a tile's softmax runs, all that is sure is that the products NB
  // tiles before have landed, and one barrier's parity could not tell the tiles between apart.
  uint64_t* o_full = p_full + C::NB;
  uint32_t* gone_s = reinterpret_cast<uint32_t*>(o_full + C::NB);             // [16]: parts of a key tile (by its number) whose page is missing, one bit a part
  // The last segments of odd and of even number whose values were not all finite.  A warp may be in the segment behind the one whose word another warp still has to read;
  // it is never two behind, since a segment's products want all four warps' weights.
  int* poison = reinterpret_cast<int*>(gone_s + 16);                          // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(poison + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  TtOrder* order = reinterpret_cast<TtOrder*>(tmem_slot + 2);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) { tc_mbar_init(&q_full[b], 1); tc_mbar_init(&q_empty[b], 1); }
    for (int s = 0; s < C::NS; ++s) { tc_mbar_init(&full[s], 1); tc_mbar_init(&empty[s], 1); }
    for (int b = 0; b < C::NB; ++b) { tc_mbar_init(&s_full[b], 1); tc_mbar_init(&p_full[b], 4); tc_mbar_init(&o_full[b], 1); }
    poison[0] = poison[1] = 0;
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_slot)), "n"(C::COLS) : "memory");
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
  // Ranges or whole units?  In times of a tile on an SM with two blocks (0.5 to 0.65 us): whole units take as long as the longest takes its block, or their share of the chip;
  // ranges a quarter more than their share, for what they put down and join, and the second kernel.  Measured with 32/8 heads of 128 and 128 rows a unit, ranges and whole units,
  // us: 16 requests of 2,500 keys 58 and 45, of 5,000 83 and 79; 64 of up to 2,500 106 and 69; 4 of 2,500 31 and 43; 1 of 2,500 18 and 43.
  int longest = 0;
  long long total = 0;
  bool whole = P.whole;
  if (!whole) {
    total = tt_total(P, longest);
    const float part = (float)total / (P.blocks_sm * 0.5f);
    whole = fmaxf(1.45f * longest, 1.05f * part) <= 1.25f * part + 15.f;
  }
  if (whole && P.sorted) tt_sort(P, *order);
  TtSegments s;
  s.start(P, order, whole, total);
  float row_m = -INFINITY, row_l = 0.f;             // of a row whose unit a cluster shares

  if (!aligned) {
    if (threadIdx.x == 0 && !P.whole) P.meta[2 * blockIdx.x] = make_int4(0, 0, 0, 0);       // nothing can be run
  } else if (warp == 4) {
    // ---------------- producer
    const bool elected = tc_elect();
    const int boxes = TT_KT / P.box_rows;           // parts of a tile that may lie in different pages
    int kn = 0, vn = 0, qn = 0;                     // key, value and Q tiles so far
    bool ok = true;
    // The ring's next stage for keys and for values (tt_place_k, tt_place_v step by step), and the parity that says it is free.
    int kst = 0, kph = 1, vst = 2, vph = 1;
    auto step = [&](int& st, int& ph, int by) {
      st += by;
      if (st >= C::NS) { st -= C::NS; ph ^= 1; }
    };
    // A tile whose parts' rows lie in lanes `from` .. of `rows`, in B parts.
    auto issue = [&](auto parts, const CUtensorMap* map, int st, int rows, int from) {
      constexpr int B = decltype(parts)::value;
      int row[B];
#pragma unroll
      for (int part = 0; part < B; ++part) row[part] = __shfl_sync(0xffffffffu, rows, from + part);
      if (elected) {
        unsigned char* dst = kv_s + st * C::TILE;
        tc_mbar_expect_tx(&full[st], C::TILE);
#pragma unroll
        for (int part = 0; part < B; ++part)
#pragma unroll
          for (int h = 0; h < C::DH; ++h) tc_tma_load(dst + part * (C::HALF / B) + h * C::HALF, map, h * 64, row[part], &full[st]);
      }
    };
    while (ok && s.next(P)) {
      const int* table = P.t.block_table + (size_t)s.seq * P.t.max_pages;
      const int key_end = s.q.r.base + s.q.r.n, key_lo = P.t.window > 0 ? max(0, s.q.r.base - P.t.window + 1) : 0;
      const int batch = 32 / boxes;                 // tiles whose table entries the warp asks for together, a batch ahead
      // this lane's entry of the batch that begins with tile i; -2: no row of the part is wanted
      auto entry = [&](int i) -> int {
        const int key = (s.tile0 + i) * TT_KT + lane * P.box_rows;
        if (i >= s.ntiles || key >= key_end || key + P.box_rows <= key_lo) return -2;
        const int pidx = P.page_shift >= 0 ? key >> P.page_shift : key / P.t.page_size;
        return pidx < P.t.max_pages ? table[pidx] : -1;
      };
      int page = entry(0);
      const int b = qn & (P.q_slots - 1);
      ok = tc_wait_warp(&q_empty[b], ((qn >> (P.q_slots - 1)) & 1) ^ 1, abort_flag);
      if (ok && elected) {
        tc_mbar_expect_tx(&q_full[b], P.q_nodes * P.t.group * 128 * C::DH);  // rows behind the copy stay as they are: nobody uses them
#pragma unroll
        for (int h = 0; h < C::DH; ++h)
          tc_tma_load3(q_s + b * P.q_slot_bytes + h * P.q_half_bytes, &map_q, h * 64, s.g * P.t.group, s.q.r.tok0 + s.row0 / P.t.group, &q_full[b]);
      }
      qn += ok;
      int rowc = P.total_rows, rowv = 0, fromv = 0;  // rowc: outside the map, where a part is filled with zeros
      unsigned gone = 0;
      // tile i's keys, and behind them the values of the tile before; those of the segment's last tile before the next segment's Q, which may have to wait for
      // this one's last scores
      for (int i = 0; i <= s.ntiles && ok; ++i) {
        const int j = i & (batch - 1);
        if (j == 0 && i < s.ntiles) {
          const int key = (s.tile0 + i) * TT_KT + lane * P.box_rows;
          const bool bad = page != -2 && (page < 0 || page >= P.t.num_pages);
          gone = __ballot_sync(0xffffffffu, bad);
          if (bad) report_error(P.t.err, PHOTON_DEV_BAD_PAGE, s.q.r.tok0, key, page);
          rowc = page < 0 || bad ? P.total_rows : (page * P.t.n_kv + s.g) * P.t.page_size + (P.page_shift >= 0 ? key & (P.t.page_size - 1) : key % P.t.page_size);
          page = entry(i + batch);
        }
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          const bool keys = which == 0;
          if (keys ? i == s.ntiles : vn + (i < s.ntiles) >= kn) continue;
          const int st = keys ? kst : vst;
          ok = tc_wait_warp(&empty[st], keys ? kph : vph, abort_flag);
          if (!ok) break;
          if (elected && keys) gone_s[kn & 15] = gone >> (j * boxes) & ((1u << boxes) - 1u);       // nobody reads the entry any more: this stage came free long behind the tile sixteen before
          const CUtensorMap* map = keys ? &map_k : &map_v;
          const int rows = keys ? rowc : rowv, from = keys ? j * boxes : fromv;
          switch (boxes) {
            case 1: issue(std::integral_constant<int, 1>(), map, st, rows, from); break;
            case 2: issue(std::integral_constant<int, 2>(), map, st, rows, from); break;
            case 4: issue(std::integral_constant<int, 4>(), map, st, rows, from); break;
            default: issue(std::integral_constant<int, 8>(), map, st, rows, from); break;
          }
          if (keys) { step(kst, kph, kn == 0 ? 1 : 2); ++kn; }
          else { step(vst, vph, 2); ++vn; }
        }
        rowv = rowc; fromv = j * boxes;             // values lie as keys do
      }
    }
    if (elected && *abort_flag) {
      // copies already issued still write into this block's shared memory: wait for them, bounded
      for (int j = (qn > P.q_slots ? qn - P.q_slots : 0); j < qn; ++j)
        for (uint32_t w = 0; w < TC_WAIT_LIMIT && !tc_mbar_try(&q_full[j & (P.q_slots - 1)], (j >> (P.q_slots - 1)) & 1); ++w) {}
      for (int j = (kn > C::NS ? kn - C::NS : 0); j < kn + 1; ++j) {
        const int a = tt_place_k(j), b = tt_place_v(j);
        for (uint32_t w = 0; j < kn && w < TC_WAIT_LIMIT && !tc_mbar_try(&full[a % C::NS], (a / C::NS) & 1); ++w) {}
        for (uint32_t w = 0; j < vn && w < TC_WAIT_LIMIT && !tc_mbar_try(&full[b % C::NS], (b / C::NS) & 1); ++w) {}
      }
    }
  } else if (warp == 5) {
    // ---------------- MMA issuer: the warp waits, one of its lanes issues
    const bool elected = tc_elect();
    const uint32_t idesc_s = tc_idesc(128, TT_KT), idesc_o = tc_idesc(128, D) | TC_IDESC_B_MN;
    const uint64_t q_desc = tc_desc(tc_smem(q_s)), k_desc = tc_desc(tc_smem(kv_s)), v_desc = tc_desc_mn(tc_smem(kv_s), C::HALF, 1024);
    // The next tile's scores; what its products need to know is packed into `f`: bit 0 its P's parity, 1 O has something in it, 2 and up the buffer.
    // 1: issued, 0: there is none, -1: given up.
    int i = 0, n = 0, sb = 0, sph = 0, qn = -1;     // tile of the segment, tiles so far, the next score buffer and its parity, the segment's Q tile
    s.ntiles = 0;
    auto scores = [&](uint32_t& f) -> int {
      if (i >= s.ntiles) {
        if (!s.next(P)) return 0;
        i = 0; ++qn;
        if (!tc_wait(&q_full[(qn & (P.q_slots - 1))], (qn >> (P.q_slots - 1)) & 1, abort_flag)) return -1;
      }
      const int place = tt_place_k(n), ks = place % C::NS;
      if (!tc_wait(&full[ks], (place / C::NS) & 1, abort_flag)) return -1;
      tc_fence_after();
      if (elected) {
        const uint64_t a = q_desc + (uint32_t)(((qn & (P.q_slots - 1))) * (P.q_slot_bytes >> 4)), b = k_desc + (uint32_t)(ks * (C::TILE >> 4));
        const uint32_t half = P.q_half_bytes >> 4;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma(tmem + sb * 64, a + (kk >> 2) * half + (kk & 3) * 2, b + (((kk >> 2) * C::HALF + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
        tc_commit(&s_full[sb]);
        tc_commit(&empty[ks]);
        if (i + 1 == s.ntiles) tc_commit(&q_empty[(qn & (P.q_slots - 1))]);
      }
      f = sph | (i > 0 ? 2u : 0u) | sb << 2;
      ++i; ++n;
      if (++sb == C::NB) { sb = 0; sph ^= 1; }
      return 1;
    };
    int vn = 0;
    auto products = [&](uint32_t f) -> bool {
      const int pb = f >> 2, place = tt_place_v(vn++), vs = place % C::NS;
      if (!tc_wait(&full[vs], (place / C::NS) & 1, abort_flag)) return false;
      if (!tc_wait(&p_full[pb], f & 1, abort_flag)) return false;
      tc_fence_after();
      if (elected) {
        const uint64_t v = v_desc + (uint32_t)(vs * (C::TILE >> 4));
#pragma unroll
        for (int kk = 0; kk < TT_KT / 16; ++kk)     // 16 keys: two groups of 8 rows of V; P: 8 columns of packed pairs
          at_mma_ts(tmem + C::O_COL, tmem + pb * 64 + kk * 8, v + ((kk * 2048) >> 4), idesc_o, kk > 0 ? 1u : (f >> 1) & 1u);
        tc_commit(&empty[vs]);
        tc_commit(&o_full[pb]);
      }
      return true;
    };
    uint32_t f[C::NB];
    int ahead = 0, more = 1;                        // tiles whose scores are issued and whose products are not; whether there may be another
#pragma unroll
    for (int j = 0; j < C::NB; ++j)
      if (more > 0) { more = scores(f[j]); ahead += more > 0; }
    while (ahead > 0 && more >= 0) {
      if (!products(f[0])) break;
      --ahead;
#pragma unroll
      for (int j = 0; j + 1 < C::NB; ++j) f[j] = f[j + 1];
      if (more > 0) { more = scores(f[C::NB - 1]); ahead += more > 0; }
    }
    pdl_launch_dependents();                        // all products of this block are issued
  } else {
    // ---------------- softmax: thread = row
    const int r = threadIdx.x;
    const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
    const float c = P.scale_log2, cap = P.t.softcap, cap_in = P.cap_in * 2.8853900817779268f;     // tanh(x) = 1 - 2 / (2^(2 x log2 e) + 1)
    int n = 0;                                      // tiles so far
    bool ok = true;
    auto landed = [&](int k) { return tc_wait_warp(&o_full[k % C::NB], (k / C::NB) & 1, abort_flag); };      // the products of tile k
    bool said = false;                        // what the second kernel is to do for this block
    while (ok && s.next(P)) {
      const bool valid = r < s.rows, busy = __any_sync(0xffffffffu, valid);
      const int t = s.q.r.tok0 + (valid ? (s.row0 + r) / P.t.group : 0);
      const int lo = valid && P.t.window > 0 ? max(0, P.t.positions[t] - P.t.window + 1) : 0;
      const int base = s.q.r.base, key_end = base + s.q.r.n;
      const int cut_lo = P.t.window > 0 ? key_end - P.t.window : -1;         // no row's window begins behind this key
      float m_used = -INFINITY, l = 0.f;
      for (int i = 0; i < s.ntiles; ++i, ++n) {
        const int sb = n % C::NB, ph = (n / C::NB) & 1, key_base = (s.tile0 + i) * TT_KT;
        const uint32_t s_addr = lane_addr + sb * 64;
        if (!tc_wait_warp(&s_full[sb], ph, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t gone = *(volatile uint32_t*)&gone_s[n & 15];
        const bool edge = key_base + TT_KT > base || key_base <= cut_lo || gone != 0;
        if (edge) {
          // values that are not finite, of nodes and before a row's window: zeros, before this tile's P says that they may be read
          const int place = tt_place_v(n), st = place % C::NS;
          if (!tc_wait_warp(&full[st], (place / C::NS) & 1, abort_flag)) { ok = false; break; }
          unsigned char* vst = kv_s + st * C::TILE;
          const int upto = min(max(cut_lo - key_base + 1, 0), TT_KT), from = max(min(max(base - key_base, 0), TT_KT), upto);
          bool found = false;
          auto clean = [&](int a, int b) {          // rows a .. b - 1 of the tile
#pragma unroll 2
            for (int x = a * 8 * C::DH + r; x < b * 8 * C::DH; x += 128) {
              const int key = x / (8 * C::DH), y = x % (8 * C::DH);
              uint4* at = reinterpret_cast<uint4*>(vst + (y >> 3) * C::HALF + key * 128 + (y & 7) * 16);
              const uint4 z = *at;
              uint32_t w[4] = {z.x, z.y, z.z, z.w};
              bool bad = false;
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                if ((w[u] & 0x7f80u) == 0x7f80u) { w[u] &= 0xffff0000u; bad = true; }
                if ((w[u] & 0x7f800000u) == 0x7f800000u) { w[u] &= 0xffffu; bad = true; }
              }
              if (bad) { *at = make_uint4(w[0], w[1], w[2], w[3]); found |= key_base + key < key_end; }
            }
          };
          clean(0, upto);
          clean(from, TT_KT);
          if (found) *(volatile int*)&poison[s.serial & 1] = s.serial;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // generic writes -> the tensor core's reads
        }
        if (busy) {
          uint32_t sv[TT_KT];
          tc_ld32_issue(s_addr, sv);
          tc_ld32_issue(s_addr + 32, sv + 32);
          tc_ld_wait();
          if (cap > 0.f) {
            float most = 0.f;
#pragma unroll
            for (int u = 0; u < TT_KT; u += 2) most = at_max3(most, fabsf(__uint_as_float(sv[u])), fabsf(__uint_as_float(sv[u + 1])));
            if (__all_sync(0xffffffffu, most * P.cap_in <= 0.5f)) {                                // a NaN stays one either way
#pragma unroll
              for (int u = 0; u < TT_KT; u += 2) tt_cap_pair(sv[u], sv[u + 1], P.cap_in, P.t.scale);
            } else {
#pragma unroll
              for (int u = 0; u < TT_KT; ++u) {
                const float x = at_exp2(__uint_as_float(sv[u]) * cap_in);
                sv[u] = __float_as_uint(cap - __fdividef(2.0f * cap, x + 1.0f));
              }
            }
          }
          if (edge) {
#pragma unroll
            for (int w = 0; w < TT_KT / 32; ++w) {
              uint32_t bits = valid ? tree_visible32(P.t, s.q.r, t, key_base + 32 * w, lo) : 0u;
              if (gone != 0) {
                for (int u = 0; u < 32; u += min(P.box_rows, 32))
                  if ((gone >> ((32 * w + u) / P.box_rows)) & 1u) bits &= ~((P.box_rows >= 32 ? 0xffffffffu : (1u << P.box_rows) - 1u) << u);
              }
#pragma unroll
              for (int u = 0; u < 32; ++u) sv[32 * w + u] = (bits >> u) & 1u ? sv[32 * w + u] : 0xff800000u;     // -inf
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
          const bool grow = cand > m_used + TT_RESCALE_STEP;                 // also the first finite maximum
          if (grow) { factor = at_exp2(m_used - cand); m_used = cand; l *= factor; }
          const float nsub = (m_used == -INFINITY) ? 0.f : -m_used;
          if (i > 0 && __any_sync(0xffffffffu, grow)) {
            // rescale O once the products of the tile before have landed
            if (!landed(n - 1)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < D; cc += 32) {
              uint32_t ov[32];
              tc_ld32(lane_addr + C::O_COL + cc, ov);
#pragma unroll
              for (int u = 0; u < 32; ++u) ov[u] = __float_as_uint(__uint_as_float(ov[u]) * factor);
              tc_st32(lane_addr + C::O_COL + cc, ov);
            }
            tc_st_wait();
          }
          // P = 2^(score c - maximum in use), packed pairs over the scores they came from
          float sum8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          uint32_t pk[32];
#pragma unroll
          for (int u = 0; u < 64; u += 2) {
            float x0, x1;
            at_fma2(x0, x1, __uint_as_float(sv[u]), __uint_as_float(sv[u + 1]), c, nsub);
            const float p0 = at_exp2(x0), p1 = at_exp2(x1);
            at_add2(sum8[u & 6], sum8[(u & 6) + 1], p0, p1);
            pk[u >> 1] = at_pack(p0, p1);
          }
          tc_st32(s_addr, pk);
          l += ((sum8[0] + sum8[1]) + (sum8[2] + sum8[3])) + ((sum8[4] + sum8[5]) + (sum8[6] + sum8[7]));
          tc_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(&p_full[sb]);
      }
      if (!ok) break;

      // ---- the segment's end
      if (!landed(n - 1)) break;
      tc_fence_after();
      const bool fix = *(volatile int*)&poison[s.serial & 1] == s.serial;
      const int head = s.g * P.t.group + (valid ? (s.row0 + r) % P.t.group : 0);
      const size_t slot = (size_t)blockIdx.x * 2 + s.bit;
      float inv = 1.f;
      if (s.whole) {
        float sum = l;
        if (P.t.sinks && l != 0.f) sum += exp2f(fmaf(P.t.sinks[head], TT_LOG2E, -m_used));         // the sink's weight, relative to the maximum in use
        inv = sum != 0.f ? 1.f / sum : 0.f;
      } else if (P.cluster > 1) {
        row_m = m_used; row_l = l;
      } else {
        if (valid) *reinterpret_cast<float2*>(P.part_ml + (slot * P.part_rows + r) * 2) = make_float2(m_used, l);
        if (r == 0 && s.bit) {
          // the block that begins a unit says who joins it: it ends with the unit's last tile
          const int used = tt_blocks(total, gridDim.x);
          const long long end = tt_first(total, blockIdx.x + 1, used) - 1 + (s.q.tiles - s.ntiles);
          P.meta[2 * blockIdx.x] = make_int4(tt_owner(total, end, used) - (int)blockIdx.x + 1, s.row0, s.rows, s.g);
          P.meta[2 * blockIdx.x + 1] = make_int4(s.q.r.tok0, 0, 0, 0);
        }
        if (s.bit) said = true;
      }
      if (busy) {
#pragma unroll 1
        for (int cc = 0; cc < D; cc += 32) {
          uint32_t ov[32];
          tc_ld32(lane_addr + C::O_COL + cc, ov);
          float x[32];
#pragma unroll
          for (int u = 0; u < 32; ++u) x[u] = __uint_as_float(ov[u]);
          if (fix && valid) {
            // what was not finite, for the rows that see it
            const int* table = P.t.block_table + (size_t)s.seq * P.t.max_pages;
            const bf16* vc = (const bf16*)P.t.v_cache;
#pragma unroll 1
            for (int w = 0; w < s.ntiles * (TT_KT / 32); ++w) {
              const int key0 = s.tile0 * TT_KT + 32 * w;
              for (uint32_t bits = tree_visible32(P.t, s.q.r, t, key0, lo); bits != 0; bits &= bits - 1) {
                const int key = key0 + __ffs(bits) - 1;
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
          if (P.cluster > 1) {
            // the ring has served: nothing comes behind a cluster's one unit
            float4* dst = reinterpret_cast<float4*>(kv_s) + cc / 4 * 128 + r;
#pragma unroll
            for (int u = 0; u < 8; ++u) dst[u * 128] = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
          } else if (valid) {
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
              float4* dst = reinterpret_cast<float4*>(P.part_o) + (slot * (D / 4) + cc / 4) * P.part_rows + r;
#pragma unroll
              for (int u = 0; u < 8; ++u) dst[(size_t)u * P.part_rows] = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
            }
          }
        }
      }
      tc_fence_before();                            // O is read: the next segment's P may be handed over
    }
    if (r == 0 && !said && !P.whole) P.meta[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (P.cluster > 1) {
    // ---------------- the blocks of a cluster join their unit in their order, each for its share of the columns
    float2* ml = reinterpret_cast<float2*>(kv_s + D / 4 * 128 * 16);        // [128]
    if (warp < 4) ml[threadIdx.x] = make_float2(row_m, row_l);
    tree_cluster_sync();
    const int r = threadIdx.x;
    if (warp < 4 && r < s.rows && !*abort_flag) {
      const int rank = blockIdx.x % P.cluster, t = s.q.r.tok0 + (s.row0 + r) / P.t.group, head = s.g * P.t.group + (s.row0 + r) % P.t.group;
      const float sink = P.t.sinks ? P.t.sinks[head] * TT_LOG2E : -INFINITY;
      bf16* dst = (bf16*)P.t.out + (size_t)t * P.t.out_stride + (size_t)head * D;
      // K: room for the blocks of the cluster; U: pieces of four columns at a time, so that eight loads are on their way
      auto join = [&](auto blocks, auto pieces) {
        constexpr int K = decltype(blocks)::value, U = decltype(pieces)::value;
        float w[K], l[K], sum = 0.f, top = sink;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          w[k] = k < P.cluster ? tree_peer(&ml[r].x, k) : -INFINITY;
          l[k] = k < P.cluster ? tree_peer(&ml[r].y, k) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) top = fmaxf(top, w[k]);
        const float sub = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const bool none = tree_nothing(w[k], l[k]);
          w[k] = at_exp2(w[k] - sub);               // 0 for what is not there
          sum += l[k] * w[k];
          if (none) w[k] = TREE_NOTHING;
        }
        sum += at_exp2(sink - sub);
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        const int end = D / 8 * (rank + 1) / P.cluster * 2;
#pragma unroll 1
        for (int c4 = D / 8 * rank / P.cluster * 2; c4 < end; c4 += U) {
          float4 y[K][U];
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (k < P.cluster) y[k][u] = tree_peer4(reinterpret_cast<const float*>(kv_s) + (min(c4 + u, D / 4 - 1) * 128 + r) * 4, k);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < K; ++k)
              if (k < P.cluster && !(w[k] < 0.f)) {
                a.x = fmaf(w[k], y[k][u].x, a.x); a.y = fmaf(w[k], y[k][u].y, a.y); a.z = fmaf(w[k], y[k][u].z, a.z); a.w = fmaf(w[k], y[k][u].w, a.w);
              }
            if (c4 + u < end) {
              uint2 v;
              v.x = at_pack(a.x * inv, a.y * inv); v.y = at_pack(a.z * inv, a.w * inv);
              *reinterpret_cast<uint2*>(dst + (c4 + u) * 4) = v;
            }
          }
        }
      };
      if (P.cluster == 2) join(std::integral_constant<int, 2>(), std::integral_constant<int, 4>());
      else if (P.cluster <= 4) join(std::integral_constant<int, 4>(), std::integral_constant<int, 2>());
      else join(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    }
    tree_cluster_sync();                            // the others have read this block's results
  }
  // ---------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::COLS) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) report_error(P.t.err, PHOTON_DEV_WAIT_TIMEOUT, blockIdx.x, 0, 0);
}

// Joins the pieces of the units that blocks of the first kernel shared, in their order.  A unit's record stands at the block that began it; each block here finds
// the records and takes its share of the work, 32 rows and 32 columns at a time.
template <int D>
__global__ void __launch_bounds__(256)
tree_join_tc_kernel(const TtParams P, int blocks, int chunks) {
  __shared__ short first_s[TT_MAX_BLOCKS];         // the blocks that began a shared unit
  __shared__ int count_s[TT_MAX_BLOCKS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  unsigned mine[(TT_MAX_BLOCKS + 255) / 256];      // this warp's 32 blocks at a time: those that began one
#pragma unroll
  for (int k = 0; k < (TT_MAX_BLOCKS + 255) / 256; ++k) {
    const int c = k * 256 + threadIdx.x, parts = c < blocks ? P.meta[2 * c].x : 0;
    mine[k] = __ballot_sync(0xffffffffu, parts >= 2 && parts <= TT_MAX_BLOCKS);
    if (lane == 0 && c < TT_MAX_BLOCKS) count_s[c >> 5] = __popc(mine[k]);
  }
  __syncthreads();
  int units = 0;
#pragma unroll
  for (int w = 0; w < TT_MAX_BLOCKS / 32; ++w) {
    if (w % 8 == warp && (mine[w / 8] >> lane & 1u)) first_s[units + __popc(mine[w / 8] & ((1u << lane) - 1u))] = (short)(w * 32 + lane);
    units += count_s[w];
  }
  __syncthreads();
  for (int item = blockIdx.x; item < units * chunks * (D / 32); item += gridDim.x) {
    const int c0 = first_s[item / (chunks * (D / 32))], r0 = item / (D / 32) % chunks * 32, cc = item % (D / 32) * 8 + warp;
    const int4 a0 = P.meta[2 * c0];
    const int parts = a0.x, rows = a0.z;
    if (r0 >= rows) continue;
    const int tok0 = P.meta[2 * c0 + 1].x;
    const bool valid = r0 + lane < rows;
    const int rr = valid ? r0 + lane : rows - 1;
    const int t = tok0 + (a0.y + rr) / P.t.group, head = a0.w * P.t.group + (a0.y + rr) % P.t.group;
    auto slot = [&](int i) { return (size_t)2 * (c0 + i) + (i == 0 ? 1 : 0); };
    // the maximum and sum so far, the sink first; eight pieces are on their way at a time
    float top = P.t.sinks ? P.t.sinks[head] * TT_LOG2E : -INFINITY, sum = P.t.sinks ? 1.f : 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (top == -INFINITY) sum = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 8) {
      float2 ml[8];
      float4 y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = min(i0 + k, parts - 1);
        ml[k] = *reinterpret_cast<const float2*>(P.part_ml + (slot(i) * P.part_rows + rr) * 2);
        y[k] = *(reinterpret_cast<const float4*>(P.part_o) + (slot(i) * (D / 4) + cc) * P.part_rows + rr);
      }
      float most = top;
#pragma unroll
      for (int k = 0; k < 8; ++k) most = fmaxf(most, ml[k].x);
      const float sub = most == -INFINITY ? 0.f : most, old = at_exp2(top - sub);
      sum *= old; a.x *= old; a.y *= old; a.z *= old; a.w *= old;
      top = most;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (i0 + k >= parts) continue;
        const float w = at_exp2(ml[k].x - sub);
        sum += ml[k].y * w;
        if (!tree_nothing(ml[k].x, ml[k].y)) { a.x = fmaf(w, y[k].x, a.x); a.y = fmaf(w, y[k].y, a.y); a.z = fmaf(w, y[k].z, a.z); a.w = fmaf(w, y[k].w, a.w); }
      }
    }
    if (valid) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      uint2 v2;
      v2.x = at_pack(a.x * inv, a.y * inv); v2.y = at_pack(a.z * inv, a.w * inv);
      *reinterpret_cast<uint2*>((bf16*)P.t.out + (size_t)t * P.t.out_stride + (size_t)head * D + cc * 4) = v2;
    }
  }
}

template <int D>
static int tt_launch(TtParams& P, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, int blocks, cudaStream_t stream) {
  static bool ready[64] = {};                      // the limit is set once a device
  int st = tree_smem_limit((const void*)tree_attention_tc_kernel<D>, Tt<D>::SMEM, ready);
  if (st != 0) return st;
  if (P.cluster > 1)
    return tree_launch_clusters(tree_attention_tc_kernel<D>, (long)blocks, P.cluster, TT_THREADS, (size_t)Tt<D>::SMEM, stream, mq, mk, mv, P);
  st = launch_pdl(tree_attention_tc_kernel<D>, dim3(blocks), dim3(TT_THREADS), (size_t)Tt<D>::SMEM, stream, mq, mk, mv, P);
  if (st != 0 || P.whole) return st;
  const int chunks = (P.part_rows + 31) / 32;
  const int items = blocks * chunks * (D / 32), grid = 2 * P.blocks_sm;     // four blocks an SM
  return launch_pdl(tree_join_tc_kernel<D>, dim3((unsigned)(items < grid ? items : grid)), dim3(256), 0, stream, P, blocks, chunks);
}

// Rows of a unit that a partial result has room for.
static int tt_part_rows(int max_tokens, int group) {
  const long most = 128 / group * group, rows = (long)max_tokens * group;
  return (int)((rows < most ? rows : most) + 31) / 32 * 32;
}
PHOTON_API long photon_tree_attention_tc_scratch(int max_tokens_per_seq, int n_q, int n_kv, int d, int blocks) {
  if (n_kv <= 0 || n_q < n_kv || n_q / n_kv > 128 || max_tokens_per_seq <= 0 || blocks <= 0) return 0;
  return 8L * blocks + 2L * blocks * tt_part_rows(max_tokens_per_seq, n_q / n_kv) * (d + 2);
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
  if (((uintptr_t)t.q & 15) || (t.q_stride & 7) || ((uintptr_t)t.k_cache & 15) || ((uintptr_t)t.v_cache & 15) || ((uintptr_t)t.out & 15) || (t.out_stride & 7) ||
      t.q_stride < (long)t.n_q * d)                // a tensor map's stride holds the dimensions before it
    return PHOTON_ERR_UNSUPPORTED;
  const long total_rows = (long)t.num_pages * t.n_kv * page_size;
  if (total_rows > 0x7fffff00L) return PHOTON_ERR_UNSUPPORTED;
  P.whole = call->scratch == nullptr;
  P.blocks_sm = 2 * photon_sm_count();
  P.cluster = call->cluster;
  if (P.cluster < 1 || P.cluster > TT_CLUSTER || (P.cluster > 1 && (!P.whole || call->parts % P.cluster))) return PHOTON_ERR_ARGUMENT;
  P.sorted = P.cluster == 1 && t.S <= TT_SORTED && (long)t.S * t.n_kv * ((t.max_tokens + 128 / G - 1) / (128 / G)) <= 65535;
  if (!P.whole && call->parts > TT_MAX_BLOCKS) return PHOTON_ERR_ARGUMENT;
  if (!P.whole && call->scratch_floats < photon_tree_attention_tc_scratch(t.max_tokens, t.n_q, t.n_kv, d, call->parts)) return PHOTON_ERR_ARGUMENT;
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return PHOTON_ERR_UNSUPPORTED;
  P.tile_nodes = 128 / G; P.tile_rows = P.tile_nodes * G;
  P.levels = (t.max_tokens + P.tile_nodes - 1) / P.tile_nodes;
  P.box_rows = page_size < TT_KT ? page_size : TT_KT;
  P.total_rows = (int)total_rows;
  // Q tiles: with at most 64 rows (in whole groups of 8, which the swizzle needs) two have room where one of 128 has
  const bool small = d == 128 && (long)t.max_tokens * G <= 64;
  P.q_slots = d == 64 || small ? 2 : 1;
  P.q_nodes = small ? 64 / G : P.tile_nodes;
  P.q_half_bytes = small ? 64 * 128 : 128 * 128;
  P.q_slot_bytes = P.q_half_bytes * (d / 64);
  CUtensorMap map_q, map_k, map_v;
  {
    cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)t.n_q, (cuuint64_t)t.T};
    cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)t.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)P.q_nodes};
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
  P.meta = reinterpret_cast<int4*>(call->scratch);
  P.part_o = call->scratch + 8L * call->parts;
  P.part_ml = P.part_o + 2L * call->parts * P.part_rows * d;
  return d == 64 ? tt_launch<64>(P, map_q, map_k, map_v, call->parts, stream) : tt_launch<128>(P, map_q, map_k, map_v, call->parts, stream);
}
