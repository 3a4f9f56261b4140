// Tokens leave a paged cache: of every layer and key/value head the keys with the largest sums stay and move to the front of the request's pages, in their order.
//
// evict_select: a block has one (entry, request, head).  The first and the last keys stay; of the others the `want` largest sums: three passes over the sums find the
// smallest one that stays, 11, 11 and 10 bits at a time (a sum's bits in an order that whole numbers have; -0 is 0, a NaN is above all), and a last pass, every thread with a run of
// neighbours, writes the keys that stay in ascending order, as many of the smallest as are wanted from the lowest places on.
// evict_move: a block moves a slice of the rows of one (entry, request, head, plane) as they are.  Row j comes from place kept[j] >= j, so a run of rows
// is read as a whole before it is written, and what a later run reads lies behind all that an earlier one wrote.
//
// What bounds it: memory, where there is much to move: 8 requests of up to 6,001 keys that keep 2,048, 28 layers, 8 heads of 128 in 16 bits, 520 us on caches that hold their keys as they came, 0.83 of
// the copy rate by the rows that may move.  Rows that lie where they belong are not moved: calls in a row on the same caches take 370 to 440.  With little to move two chains of latencies: one
// request, 1,152 to 1,024, 16 layers, 8 heads of 64 in 4 bits, 17.5 us.  Sums that stay in shared memory and places found once for a batch of rows: 684 to 445 us in a row.
#include "common.cuh"
#include "limits.cuh"

#define EV_THREADS 512
#define EV_MOVERS 256
#define EV_BATCH 512            // rows whose places a block knows at a time
#define EV_DEPTH 8               // rows that a thread has under way
#define EV_SHARED 49152          // bytes of sums that stay in shared memory, at most: two blocks an SM and more

struct EvictArgs {
  uint8_t* kv; float* weights; const int* table; const int* context_lens; int* new_lens; int* kept; int* err;
  int entries, planes, num_pages, n_kv, page_size, page_shift, max_pages, S, keep, first, last;
  int room;                      // words of sums in shared memory
  long page_bytes;               // of one head
  int row_bytes, scale_bytes;    // of one key; the scales of a cache in 4 bits lie behind a page's rows
};

__device__ __forceinline__ uint32_t evict_order(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The exclusive sum of a block's numbers, and their total.  `warp_s`: one word a warp.
__device__ __forceinline__ int evict_scan(int x, int* warp_s, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  __syncthreads();
  if (lane == 31) warp_s[warp] = upto;
  __syncthreads();
  int before = upto - x, all = 0;
  for (int i = 0; i < EV_THREADS / 32; ++i) {
    const int y = warp_s[i];
    if (i < warp) before += y;
    all += y;
  }
  *total = all;
  return before;
}

// Where they fit, the sums' bits stay in shared memory, every thread's run an odd number of words from the next one's; else they are read again in every pass.
__global__ void __launch_bounds__(EV_THREADS)
evict_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t order_s[];
  __shared__ int bins[2048];
  __shared__ int digit_s, above_s, warp_s[EV_THREADS / 32];
  pdl_wait();
  const int head = blockIdx.x % a.n_kv, seq = blockIdx.x / a.n_kv % a.S, entry = blockIdx.x / a.n_kv / a.S, tid = threadIdx.x;
  const int len = a.context_lens[seq];
  if (head == 0 && entry == 0 && tid == 0) a.new_lens[seq] = min(len, a.keep);
  if (len <= a.keep) return;
  const int first = min(a.first, a.keep), last = min(a.last, a.keep - first), lo = first, hi = len - last, count = hi - lo;
  int want = a.keep - first - last;
  int* kept = a.kept + (long)blockIdx.x * a.keep;
  for (int j = tid; j < first; j += EV_THREADS) kept[j] = j;
  for (int j = tid; j < last; j += EV_THREADS) kept[a.keep - last + j] = hi + j;
  if (want <= 0) return;
  const int* table = a.table + (long)seq * a.max_pages;
  const float* sums = a.weights + ((long)entry * a.num_pages * a.n_kv + head) * a.page_size;
  auto order = [&](int at) -> uint32_t {             // of key lo + at
    const int key = lo + at, pidx = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size, page = pidx < a.max_pages ? table[pidx] : -1;
    if (page < 0 || page >= a.num_pages) return 0;
    return evict_order(sums[(long)page * a.n_kv * a.page_size + key - pidx * a.page_size]);
  };
  // a thread has a run of neighbouring keys in the end
  const int run = (count + EV_THREADS - 1) / EV_THREADS, pitch = run | 1;
  const bool in_shared = pitch * EV_THREADS <= a.room;
  auto place = [&](int at) { return at / run * pitch + at % run; };
  if (in_shared)
    for (int at = tid; at < count; at += EV_THREADS) order_s[place(at)] = order(at);
  uint32_t prefix = 0, mask = 0;                     // the bits found so far of the smallest sum that stays
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, size = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < size; i += EV_THREADS) bins[i] = 0;
    __syncthreads();
    if (in_shared) {
      for (int i = 0; i < run && tid * run + i < count; ++i) {
        const uint32_t u = order_s[tid * pitch + i];
        if ((u & mask) == prefix) atomicAdd(&bins[u >> shift & (size - 1)], 1);
      }
    } else {
      for (int at = tid; at < count; at += EV_THREADS) {
        const uint32_t u = order(at);
        if ((u & mask) == prefix) atomicAdd(&bins[u >> shift & (size - 1)], 1);
      }
    }
    __syncthreads();
    // the bin, from the top, in which the wanted number is reached: a thread has size / 512 neighbouring bins
    const int mine = size / EV_THREADS, top = size - 1 - tid * mine;
    int n = 0, total;
    for (int i = 0; i < mine; ++i) n += bins[top - i];
    int before = evict_scan(n, warp_s, &total);
    if (before < want && before + n >= want) {
      for (int i = 0; i < mine; ++i) {
        if (before + bins[top - i] >= want) { digit_s = top - i; above_s = before; break; }
        before += bins[top - i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)digit_s << shift;
    mask |= (uint32_t)(size - 1) << shift;
    want -= above_s;
    __syncthreads();
  }
  // in ascending order: what is above the border, and the first `want` of what lies on it
  const int from = min(tid * run, count), to = min(from + run, count);
  int ties = 0, above = 0, total;
  for (int at = from; at < to; ++at) {
    const uint32_t u = in_shared ? order_s[tid * pitch + at - from] : order(at);
    ties += u == prefix;
    above += u > prefix;
  }
  const int ties_before = evict_scan(ties, warp_s, &total), take = max(0, min(ties, want - ties_before));
  int put = first + evict_scan(above + take, warp_s, &total), left = take;
  for (int at = from; at < to; ++at) {
    const uint32_t u = in_shared ? order_s[tid * pitch + at - from] : order(at);
    if (u > prefix || (u == prefix && left-- > 0)) kept[put++] = lo + at;
  }
}

// Rows of `bytes` bytes, one behind the other from `base` on in every page: `pieces` pieces of V of the rows that move, from `piece0` on.  A batch's places are found once for all pieces.
template <typename V>
__device__ __forceinline__ void evict_rows(uint8_t* base, long page_step, int bytes, const int* __restrict__ kept, const int* __restrict__ table, const EvictArgs& a, int piece0,
                                           int pieces, long* from_s, long* to_s, int report = -1) {      // report: the request whose pages that are not there are recorded
  const int per = EV_MOVERS / pieces, sub = threadIdx.x / pieces, piece = piece0 + threadIdx.x - sub * pieces;
  auto place = [&](int key) -> long {
    const int pidx = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size, page = pidx < a.max_pages ? table[pidx] : -1;
    if (page < 0 || page >= a.num_pages) return -1;
    return page * page_step + (long)(key - pidx * a.page_size) * bytes;
  };
  for (int j0 = 0; j0 < a.keep; j0 += EV_BATCH) {
    const int here = min(EV_BATCH, a.keep - j0);
    __syncthreads();                                  // the batch in front of it is done with
    int key[EV_BATCH / EV_MOVERS];
#pragma unroll
    for (int i = 0; i < EV_BATCH / EV_MOVERS; ++i) {
      const int r = i * EV_MOVERS + threadIdx.x;
      key[i] = r < here ? kept[j0 + r] : -1;
    }
#pragma unroll
    for (int i = 0; i < EV_BATCH / EV_MOVERS; ++i) {
      const int r = i * EV_MOVERS + threadIdx.x;
      if (r >= here) continue;
      long from = key[i] == j0 + r && report < 0 ? -1 : place(key[i]);
      if (from < 0 && report >= 0) report_error(a.err, PHOTON_DEV_BAD_PAGE, report, key[i], key[i] / a.page_size < a.max_pages ? table[key[i] / a.page_size] : -1);
      if (key[i] == j0 + r) from = -1;
      from_s[r] = from;
      to_s[r] = from < 0 ? -1 : place(j0 + r);
    }
    __syncthreads();
    for (int r0 = 0; r0 < here; r0 += per * EV_DEPTH) {
      V x[EV_DEPTH];
      long at[EV_DEPTH];
#pragma unroll
      for (int i = 0; i < EV_DEPTH; ++i) {
        const int r = r0 + i * per + sub;
        at[i] = -1;
        if (sub < per && r < here) {
          at[i] = to_s[r];
          if (at[i] >= 0) x[i] = *((const V*)(base + from_s[r]) + piece);
        }
      }
      __syncthreads();                                // all are read before the first is written
#pragma unroll
      for (int i = 0; i < EV_DEPTH; ++i) if (at[i] >= 0) *((V*)(base + at[i]) + piece) = x[i];
    }
  }
}

__global__ void __launch_bounds__(EV_MOVERS)
evict_move_kernel(const EvictArgs a, int slices, int slice_pieces, int kinds) {      // kinds: rows of every plane, scales of every plane where there are some, sums
  __shared__ long from_s[EV_BATCH], to_s[EV_BATCH];
  pdl_wait();
  const int slice = blockIdx.x % slices, what = blockIdx.x / slices % kinds, unit = blockIdx.x / slices / kinds;
  const int head = unit % a.n_kv, seq = unit / a.n_kv % a.S, entry = unit / a.n_kv / a.S;
  if (a.context_lens[seq] <= a.keep || a.keep <= 0) return;
  const int* kept = a.kept + (long)unit * a.keep;
  const int* table = a.table + (long)seq * a.max_pages;
  if (what == kinds - 1) {                           // the sums, and pages that are not there
    if (slice > 0) return;
    evict_rows<float>((uint8_t*)(a.weights + ((long)entry * a.num_pages * a.n_kv + head) * a.page_size), (long)a.n_kv * a.page_size * 4, 4, kept, table, a, 0, 1, from_s, to_s, seq);
    return;
  }
  const bool of_scales = what >= a.planes;
  uint8_t* base = a.kv + (((long)entry * a.planes + what % a.planes) * a.num_pages * a.n_kv + head) * a.page_bytes;
  const int pieces = a.row_bytes / 16, piece0 = slice * slice_pieces;
  if (!of_scales) {
    if (piece0 < pieces) evict_rows<uint4>(base, a.n_kv * a.page_bytes, a.row_bytes, kept, table, a, piece0, min(slice_pieces, pieces - piece0), from_s, to_s);
  } else if (slice == 0) {
    uint8_t* scales = base + (long)a.page_size * a.row_bytes;
    if (a.scale_bytes % 4 == 0) evict_rows<uint32_t>(scales, a.n_kv * a.page_bytes, a.scale_bytes, kept, table, a, 0, a.scale_bytes / 4, from_s, to_s);
    else if (a.scale_bytes % 2 == 0) evict_rows<uint16_t>(scales, a.n_kv * a.page_bytes, a.scale_bytes, kept, table, a, 0, a.scale_bytes / 2, from_s, to_s);
    else evict_rows<uint8_t>(scales, a.n_kv * a.page_bytes, a.scale_bytes, kept, table, a, 0, a.scale_bytes, from_s, to_s);
  }
}

PHOTON_API int photon_cache_evict(const photon_evict_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->entries <= 0) return 0;
  if (c->planes <= 0 || c->num_pages <= 0 || c->n_kv <= 0 || c->page_size <= 0 || c->max_pages <= 0 || c->keep < 0 || c->first < 0 || c->last < 0 || c->max_keys < 0) return PHOTON_ERR_ARGUMENT;
  if (c->row_bytes <= 0 || c->row_bytes % 16 || (uintptr_t)c->kv % 16 || c->row_bytes / 16 > EV_MOVERS) return PHOTON_ERR_UNSUPPORTED;
  // a run of every thread and a word
  const long words = (((long)c->max_keys + EV_THREADS - 1) / EV_THREADS | 1) * EV_THREADS;
  const int room = words * 4 <= EV_SHARED ? (int)words : 0;
  int shift = -1;
  for (int i = 0; i < 31; ++i) if (c->page_size == 1 << i) shift = i;
  const EvictArgs a = {(uint8_t*)c->kv, c->weights, c->block_table, c->context_lens, c->new_lens, c->kept, c->err, c->entries, c->planes, c->num_pages, c->n_kv, c->page_size, shift,
                 c->max_pages, c->S, c->keep, c->first, c->last, room, (long)c->page_size * (c->row_bytes + c->scale_bytes), c->row_bytes, c->scale_bytes};
  const long units = (long)c->entries * c->S * c->n_kv;
  // Whole rows where there are enough of them to fill the chip, else parts of 32 bytes or more for several blocks.
  const int pieces = c->row_bytes / 16;
  long want = (8L * photon_sm_count() + units * c->planes - 1) / (units * c->planes);
  if (want > (pieces + 1) / 2) want = (pieces + 1) / 2;
  const int slice_pieces = (int)((pieces + want - 1) / want), slices = (pieces + slice_pieces - 1) / slice_pieces;
  const int kinds = c->planes * (c->scale_bytes > 0 ? 2 : 1) + 1;
  const long blocks = units * kinds * slices;
  if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  static bool ready[64] = {};
  const int limit = smem_limit((const void*)evict_select_kernel, EV_SHARED, false, ready);
  if (limit != 0) return limit;
  const int status = launch_pdl(evict_select_kernel, dim3((unsigned)units), dim3(EV_THREADS), (size_t)room * 4, stream, a);
  if (status != 0 || c->keep == 0) return status;
  return launch_pdl(evict_move_kernel, dim3((unsigned)blocks), dim3(EV_MOVERS), 0, stream, a, slices, slice_pieces, kinds);
}
