// Rows and pages of a paged cache moved inside it, in all layers at once.
//
// The pools of a cache group lie in one tensor [entries][planes][pages][n_kv][page_size][d]; what is moved is moved as it is, in pieces of up to 16 bytes.
//
// cache_keep: the rows of a tree's accepted nodes go to the places behind the request's cached tokens.  Node i of request s lies at key base + i;
// path[s][j], j < counts[s], goes to key base + j.  A path ascends from its root, so path[j] >= j: a row is never needed after a later one has been written.  A
// thread owns one piece of the rows of one head and moves eight rows at a time: all eight are read before the first is written, and what a later eight read lies
// behind all that an earlier eight wrote.  A block's threads share the list of moves, up to 256 at a time behind a barrier, and nothing of the rows.
// Bound by the latency of one round (path, table, rows, rows back) for few rows: 8 requests, 16 layers of 8 heads of 64: 2.9 us (3.2 with the path read behind the count);
// 48 requests, 28 layers of 8 heads of 128, 44 MB read and written: 12.3 us (3.6 TB/s, rows of 256 bytes in no order; 13.0 with a block for every 256 pieces, two rounds
// of blocks); 20 requests of as many layers in 32 bits 7.2 (8.7).
//
// cache_copy_pages: page pairs[i][0] onto page pairs[i][1]; a block copies a part of one page in one plane, 64 bytes a thread in flight.
// 512 pages of 28 layers, 1.88 GB: 285 us, the copy rate; 8 pages of 16 layers 2.0 us.
#include "common.cuh"

#define CR_THREADS 256
#define CR_ROWS 8                                  // rows of a path that a thread moves at a time
#define CR_BLOCKS 4                                // an SM, of a kernel that moves rows: a second round of blocks would go the way to the rows again
#define CR_PIECES 4                                // pieces of a page that a thread copies at a time

template <typename V>
__global__ void __launch_bounds__(CR_THREADS)
cache_keep_kernel(V* __restrict__ kv, long units, int num_pages, int n_kv, int page_size, int pieces, const int* __restrict__ block_table,
                  int max_pages, const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, const int* __restrict__ path,
                  const int* __restrict__ counts, int D, int* err) {
  __shared__ long long src_s[CR_THREADS], dst_s[CR_THREADS];      // rows (page, slot) of the moves that there are, a block's worth at a time
  pdl_wait();
  const int seq = blockIdx.y;
  const int node = 1 + (int)threadIdx.x < D ? path[(size_t)seq * D + 1 + threadIdx.x] : 0;      // beside the count, not behind it
  const int first = cu_tokens[seq], n = cu_tokens[seq + 1] - first, base = context_lens[seq] - n;
  const int count = min(counts[seq], D);
  if (count < 2) return;
  const int* table = block_table + (size_t)seq * max_pages;
  const long page_step = (long)n_kv * page_size * pieces;                     // from a page's row to the same row of the next page
  auto place = [&](int key) -> long long {         // page and slot of a key, packed; -1: no page
    const int pidx = key / page_size;
    const int page = key >= 0 && pidx < max_pages ? table[pidx] : -1;
    if (page < 0 || page >= num_pages) {
      if (blockIdx.x == 0) report_error(err, PHOTON_DEV_BAD_PAGE, seq, key, page);
      return -1;
    }
    return (long long)page << 32 | (key - pidx * page_size);
  };
  for (int j0 = 1; j0 < count; j0 += CR_THREADS) {
    const int here = min(CR_THREADS, count - j0), j = j0 + (int)threadIdx.x;
    __syncthreads();
    if (j < count) {
      const int from = j0 == 1 ? node : path[(size_t)seq * D + j];
      long long src = -1, dst = -1;
      if (from < j || from >= n) {
        if (blockIdx.x == 0) report_error(err, PHOTON_DEV_BAD_TOKEN, seq, from, n);
      } else if (from > j) {                       // a row that is already there stays
        src = place(base + from);
        dst = place(base + j);
      }
      src_s[threadIdx.x] = dst < 0 ? -1 : src;
      dst_s[threadIdx.x] = dst;
    }
    __syncthreads();
    for (long unit = (long)blockIdx.x * CR_THREADS + threadIdx.x; unit < units; unit += (long)gridDim.x * CR_THREADS) {      // (entry and plane, head, piece)
      const long head = unit / pieces, plane = head / n_kv;
      V* rows = kv + (plane * num_pages * n_kv + (head - plane * n_kv)) * (long)page_size * pieces + (unit - head * pieces);
      auto at = [&](long long p) { return rows + (p >> 32) * page_step + (long)(uint32_t)p * pieces; };
      for (int k = 0; k < here; k += CR_ROWS) {
        V x[CR_ROWS];
#pragma unroll
        for (int i = 0; i < CR_ROWS; ++i) if (k + i < here && src_s[k + i] >= 0) x[i] = *at(src_s[k + i]);
#pragma unroll
        for (int i = 0; i < CR_ROWS; ++i) if (k + i < here && src_s[k + i] >= 0) *at(dst_s[k + i]) = x[i];
      }
    }
  }
}

template <typename V>
__global__ void __launch_bounds__(CR_THREADS)
cache_copy_pages_kernel(V* __restrict__ kv, int planes, int num_pages, long pieces, int parts, const int* __restrict__ pairs, int count, int* err) {
  pdl_wait();
  const int part = blockIdx.x % parts;
  const long long plane = blockIdx.x / parts % planes;
  const int pair = blockIdx.x / parts / planes;
  const int from = pairs[2 * pair], to = pairs[2 * pair + 1];
  if (from < 0 || from >= num_pages || to < 0 || to >= num_pages) {
    if (threadIdx.x == 0 && part == 0 && plane == 0) report_error(err, PHOTON_DEV_BAD_PAGE, pair, from, to);
    return;
  }
  if (from == to) return;
  const V* src = kv + (plane * num_pages + from) * pieces;
  V* dst = kv + (plane * num_pages + to) * pieces;
  const long first = (long)part * CR_THREADS * CR_PIECES + threadIdx.x;
  V x[CR_PIECES];
#pragma unroll
  for (int i = 0; i < CR_PIECES; ++i) if (first + i * CR_THREADS < pieces) x[i] = src[first + i * CR_THREADS];
#pragma unroll
  for (int i = 0; i < CR_PIECES; ++i) if (first + i * CR_THREADS < pieces) dst[first + i * CR_THREADS] = x[i];
}

// The widest piece that an address and a row allow.
static int piece_bytes(const void* p, long row_bytes) {
  for (int b = 16; b > 2; b >>= 1) if ((uintptr_t)p % b == 0 && row_bytes % b == 0) return b;
  return 2;
}

PHOTON_API int photon_cache_keep(const photon_keep_call* c, cudaStream_t stream) {
  if (c->S <= 0 || c->D <= 0 || c->planes <= 0) return 0;
  if (c->dtype != PHOTON_F32 && c->dtype != PHOTON_BF16) return PHOTON_ERR_ARGUMENT;
  if (c->num_pages <= 0 || c->n_kv <= 0 || c->page_size <= 0 || c->d <= 0 || c->max_pages <= 0) return PHOTON_ERR_ARGUMENT;
  if (c->S > 65535) return PHOTON_ERR_UNSUPPORTED;
  const long row = (long)c->d * (c->dtype == PHOTON_F32 ? 4 : 2);
  const int b = piece_bytes(c->kv, row), pieces = (int)(row / b);
  const long units = (long)c->planes * c->n_kv * pieces;
  const long blocks = (units + CR_THREADS - 1) / CR_THREADS, most = (CR_BLOCKS * photon_sm_count() + c->S - 1) / c->S;
  const dim3 grid((unsigned)(blocks < most ? blocks : most), (unsigned)c->S);
#define KEEP(V) launch_pdl(cache_keep_kernel<V>, grid, dim3(CR_THREADS), 0, stream, (V*)c->kv, units, c->num_pages, c->n_kv, c->page_size, pieces, c->block_table, \
                           c->max_pages, c->cu_tokens, c->context_lens, c->path, c->counts, c->D, c->err)
  return b == 16 ? KEEP(uint4) : b == 8 ? KEEP(uint2) : b == 4 ? KEEP(uint32_t) : KEEP(uint16_t);
#undef KEEP
}

PHOTON_API int photon_cache_copy_pages(void* kv, int dtype, int planes, int num_pages, long page_elems, const int* pairs, int count, int* err,
                                       cudaStream_t stream) {
  if (count <= 0 || planes <= 0) return 0;
  if (dtype != PHOTON_F32 && dtype != PHOTON_BF16) return PHOTON_ERR_ARGUMENT;
  if (num_pages <= 0 || page_elems <= 0) return PHOTON_ERR_ARGUMENT;
  const long bytes = page_elems * (dtype == PHOTON_F32 ? 4 : 2);
  const int b = piece_bytes(kv, bytes);
  const long pieces = bytes / b, parts = (pieces + CR_THREADS * CR_PIECES - 1) / (CR_THREADS * CR_PIECES);
  if (parts * planes * count > 0x7fffffffL) return PHOTON_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(parts * planes * count));
#define COPY(V) launch_pdl(cache_copy_pages_kernel<V>, grid, dim3(CR_THREADS), 0, stream, (V*)kv, planes, num_pages, pieces, (int)parts, pairs, count, err)
  return b == 16 ? COPY(uint4) : b == 8 ? COPY(uint2) : b == 4 ? COPY(uint32_t) : COPY(uint16_t);
#undef COPY
}
