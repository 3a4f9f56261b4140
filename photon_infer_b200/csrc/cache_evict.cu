// Tokens leave a paged cache: of every layer and key/value head the keys with the largest sums stay and move to the front of the request's pages, in their order.
//
// evict_select: a block has one (entry, request, head).  The first and the last keys stay; of the others the `want` largest sums: three passes over the sums find the
// smallest one that stays, 11, 11 and 10 bits at a time (a sum's bits in an order that whole numbers have; -0 is 0, a NaN is above all), and a last pass writes the keys
// that stay in ascending order, as many of the smallest as are wanted from the lowest places on.
// evict_move: a block moves a slice of the rows of one (entry, request, head, plane) as they are.  Row j comes from place kept[j] >= j, so a run of rows
// is read as a whole before it is written, and what a later run reads lies behind all that an earlier one wrote.
#include "common.cuh"

#define EV_THREADS 512
#define EV_MOVERS 256
#define EV_DEPTH 4               // rows that a thread has under way

struct EvictArgs {
  uint8_t* kv; float* weights; const int* table; const int* context_lens; int* new_lens; int* kept; int* err;
  int entries, planes, num_pages, n_kv, page_size, max_pages, S, keep, first, last;
  long page_bytes;               // of one head
  int row_bytes, scale_bytes;    // of one key; the scales of a cache in 4 bits lie behind a page's rows
};

__device__ __forceinline__ uint32_t evict_order(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(EV_THREADS)
evict_select_kernel(const EvictArgs a) {
  __shared__ int bins[2048];
  __shared__ int digit_s, above_s, warp_s[EV_THREADS / 32], warp_t[EV_THREADS / 32];
  pdl_wait();
  const int head = blockIdx.x % a.n_kv, seq = blockIdx.x / a.n_kv % a.S, entry = blockIdx.x / a.n_kv / a.S, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = a.context_lens[seq];
  if (head == 0 && entry == 0 && tid == 0) a.new_lens[seq] = min(len, a.keep);
  if (len <= a.keep) return;
  const int first = min(a.first, a.keep), last = min(a.last, a.keep - first), lo = first, hi = len - last;
  int want = a.keep - first - last;
  int* kept = a.kept + (long)blockIdx.x * a.keep;
  const int* table = a.table + (long)seq * a.max_pages;
  const float* sums = a.weights + ((long)entry * a.num_pages * a.n_kv + head) * a.page_size;
  auto order = [&](int key) -> uint32_t {
    const int pidx = key / a.page_size, page = pidx < a.max_pages ? table[pidx] : -1;
    if (page < 0 || page >= a.num_pages) return 0;
    return evict_order(sums[(long)page * a.n_kv * a.page_size + key - pidx * a.page_size]);
  };
  uint32_t prefix = 0, mask = 0;                     // the bits found so far of the smallest sum that stays
  for (int pass = 0; pass < 3 && want > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, size = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < size; i += EV_THREADS) bins[i] = 0;
    __syncthreads();
    for (int key = lo + tid; key < hi; key += EV_THREADS) {
      const uint32_t u = order(key);
      if ((u & mask) == prefix) atomicAdd(&bins[u >> shift & (size - 1)], 1);
    }
    __syncthreads();
    // the bin, from the top, in which the wanted number is reached: a thread has size / 512 neighbouring bins
    const int mine = size / EV_THREADS, top = size - 1 - tid * mine;
    int count = 0;
    for (int i = 0; i < mine; ++i) count += bins[top - i];
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) warp_s[warp] = upto;
    __syncthreads();
    int before = upto - count;
    for (int i = 0; i < warp; ++i) before += warp_s[i];
    if (before < want && before + count >= want) {
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
  for (int j = tid; j < first; j += EV_THREADS) kept[j] = j;
  for (int j = tid; j < last; j += EV_THREADS) kept[a.keep - last + j] = hi + j;
  if (a.keep - first - last <= 0) return;
  int written = first, ties = 0;
  for (int k0 = lo; k0 < hi; k0 += EV_THREADS) {
    const int key = k0 + tid;
    const uint32_t u = key < hi ? order(key) : 0;
    const bool above = key < hi && u > prefix, tie = key < hi && u == prefix;
    const unsigned votes = __ballot_sync(0xffffffffu, tie);
    __syncthreads();
    if (lane == 0) warp_t[warp] = __popc(votes);
    __syncthreads();
    int tied = ties + __popc(votes & ((1u << lane) - 1)), all_ties = ties;
    for (int i = 0; i < EV_THREADS / 32; ++i) {
      if (i < warp) tied += warp_t[i];
      all_ties += warp_t[i];
    }
    const bool stays = above || (tie && tied < want);
    const unsigned stay = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) warp_s[warp] = __popc(stay);
    __syncthreads();
    int at = written + __popc(stay & ((1u << lane) - 1)), all = written;
    for (int i = 0; i < EV_THREADS / 32; ++i) {
      if (i < warp) at += warp_s[i];
      all += warp_s[i];
    }
    if (stays) kept[at] = key;
    written = all;
    ties = all_ties;
  }
}

// Rows of `bytes` bytes, one behind the other from `base` on in every page: the pieces [slice] of V of the rows that move.
template <typename V>
__device__ __forceinline__ void evict_rows(uint8_t* base, long page_step, int bytes, const int* __restrict__ kept, const int* __restrict__ table, const EvictArgs& a, int piece0,
                                           int pieces) {
  const int per = EV_MOVERS / pieces, sub = threadIdx.x / pieces, piece = piece0 + threadIdx.x - sub * pieces;
  auto place = [&](int key) -> V* {
    const int pidx = key / a.page_size, page = pidx < a.max_pages ? table[pidx] : -1;
    if (page < 0 || page >= a.num_pages) return nullptr;
    return (V*)(base + page * page_step + (long)(key - pidx * a.page_size) * bytes) + piece;
  };
  for (int j0 = 0; j0 < a.keep; j0 += per * EV_DEPTH) {
    V x[EV_DEPTH];
    V* to[EV_DEPTH];
#pragma unroll
    for (int i = 0; i < EV_DEPTH; ++i) {
      const int j = j0 + i * per + sub;
      to[i] = nullptr;
      if (sub < per && j < a.keep && kept[j] != j) {
        const V* from = place(kept[j]);
        if (from != nullptr) { to[i] = place(j); x[i] = *from; }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EV_DEPTH; ++i) if (to[i] != nullptr) *to[i] = x[i];
  }
}

__global__ void __launch_bounds__(EV_MOVERS)
evict_move_kernel(const EvictArgs a, int slices, int slice_pieces) {
  pdl_wait();
  const int slice = blockIdx.x % slices, what = blockIdx.x / slices % (a.planes + 1);
  const long unit = blockIdx.x / slices / (a.planes + 1);
  const int head = (int)(unit % a.n_kv), seq = (int)(unit / a.n_kv % a.S), entry = (int)(unit / a.n_kv / a.S);
  if (a.context_lens[seq] <= a.keep || a.keep <= 0) return;
  const int* kept = a.kept + unit * a.keep;
  const int* table = a.table + (long)seq * a.max_pages;
  if (what == a.planes) {                            // the sums, and pages that are not there
    if (slice > 0) return;
    for (int j = threadIdx.x; j < a.keep; j += EV_MOVERS) {
      const int pidx = kept[j] / a.page_size, page = pidx < a.max_pages ? table[pidx] : -1;
      if (page < 0 || page >= a.num_pages) report_error(a.err, PHOTON_DEV_BAD_PAGE, seq, kept[j], page);
    }
    evict_rows<float>((uint8_t*)(a.weights + ((long)entry * a.num_pages * a.n_kv + head) * a.page_size), (long)a.n_kv * a.page_size * 4, 4, kept, table, a, 0, 1);
    return;
  }
  uint8_t* base = a.kv + (((long)entry * a.planes + what) * a.num_pages * a.n_kv + head) * a.page_bytes;
  const int pieces = a.row_bytes / 16, piece0 = slice * slice_pieces;
  if (piece0 < pieces) evict_rows<uint4>(base, a.n_kv * a.page_bytes, a.row_bytes, kept, table, a, piece0, min(slice_pieces, pieces - piece0));
  if (slice == slices - 1 && a.scale_bytes > 0) {
    __syncthreads();
    uint8_t* scales = base + (long)a.page_size * a.row_bytes;
    if (a.scale_bytes % 4 == 0) evict_rows<uint32_t>(scales, a.n_kv * a.page_bytes, a.scale_bytes, kept, table, a, 0, a.scale_bytes / 4);
    else if (a.scale_bytes % 2 == 0) evict_rows<uint16_t>(scales, a.n_kv * a.page_bytes, a.scale_bytes, kept, table, a, 0, a.scale_bytes / 2);
    else evict_rows<uint8_t>(scales, a.n_kv * a.page_bytes, a.scale_bytes, kept, table, a, 0, a.scale_bytes);
  }
}

PHOTON_API int photon_cache_evict(const photon_evict_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->entries <= 0) return 0;
  if (c->planes <= 0 || c->num_pages <= 0 || c->n_kv <= 0 || c->page_size <= 0 || c->max_pages <= 0 || c->keep < 0 || c->first < 0 || c->last < 0) return PHOTON_ERR_ARGUMENT;
  if (c->row_bytes <= 0 || c->row_bytes % 16 || (uintptr_t)c->kv % 16 || c->row_bytes / 16 > EV_MOVERS) return PHOTON_ERR_UNSUPPORTED;
  EvictArgs a = {(uint8_t*)c->kv, c->weights, c->block_table, c->context_lens, c->new_lens, c->kept, c->err, c->entries, c->planes, c->num_pages, c->n_kv, c->page_size,
                 c->max_pages, c->S, c->keep, c->first, c->last, (long)c->page_size * (c->row_bytes + c->scale_bytes), c->row_bytes, c->scale_bytes};
  const long units = (long)c->entries * c->S * c->n_kv;
  const int pieces = c->row_bytes / 16, slice_pieces = pieces < 2 ? pieces : 2, slices = (pieces + slice_pieces - 1) / slice_pieces;
  const long blocks = units * (c->planes + 1) * slices;
  if (blocks > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  const int status = launch_pdl(evict_select_kernel, dim3((unsigned)units), dim3(EV_THREADS), 0, stream, a);
  if (status != 0 || c->keep == 0) return status;
  return launch_pdl(evict_move_kernel, dim3((unsigned)blocks), dim3(EV_MOVERS), 0, stream, a, slices, slice_pieces);
}
