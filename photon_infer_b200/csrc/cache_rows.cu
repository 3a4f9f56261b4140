// Rows and pages of a paged cache moved inside it, in all layers at once.
//
// The pools of a cache group lie in one tensor [entries][planes][pages][n_kv][page_size][d]; what is moved is moved as it is, in pieces of
// up to 16 bytes.
//
// cache_keep: the rows of a tree's accepted nodes go to the places behind the request's cached tokens.  Node i of request s lies at key base + i;
// path[s][j], j < counts[s], goes to key base + j.  A path ascends from its root, so path[j] >= j: a row is never needed after a later one has
// been written, and a warp that has all pieces of a head's rows reads a few rows before it writes them.
//
// cache_copy_pages: page pairs[i][0] onto page pairs[i][1].
#include "common.cuh"

#define CR_THREADS 256

template <typename V>
__global__ void __launch_bounds__(CR_THREADS)
cache_keep_kernel(V* __restrict__ kv, int planes, int num_pages, int n_kv, int page_size, int pieces, const int* __restrict__ block_table,
                  int max_pages, const int* __restrict__ cu_tokens, const int* __restrict__ context_lens, const int* __restrict__ path,
                  const int* __restrict__ counts, int D, int* err) {
  pdl_wait();
  const int seq = blockIdx.y, lane = threadIdx.x & 31;
  const int unit = blockIdx.x * (CR_THREADS / 32) + (threadIdx.x >> 5);       // (entry and plane, head)
  if (unit >= planes * n_kv) return;
  const int plane = unit / n_kv, g = unit - plane * n_kv;
  const int n = cu_tokens[seq + 1] - cu_tokens[seq], base = context_lens[seq] - n;
  const int count = min(counts[seq], D);
  const int* table = block_table + (size_t)seq * max_pages;
  auto row_of = [&](int key) -> long long {
    const int pidx = key / page_size;
    const int page = key >= 0 && pidx < max_pages ? table[pidx] : -1;
    if (page < 0 || page >= num_pages) {
      if (unit == 0 && lane == 0) report_error(err, PHOTON_DEV_BAD_PAGE, seq, key, page);
      return -1;
    }
    return ((((long long)plane * num_pages + page) * n_kv + g) * page_size + (key - pidx * page_size)) * pieces;
  };
  for (int j = 1; j < count; ++j) {
    const int from = path[(size_t)seq * D + j];
    if (from == j) continue;                       // already there
    if (from < j || from >= n) {
      if (unit == 0 && lane == 0) report_error(err, PHOTON_DEV_BAD_TOKEN, seq, from, n);
      continue;
    }
    const long long src = row_of(base + from), dst = row_of(base + j);
    if (src < 0 || dst < 0) continue;
    for (int e = lane; e < pieces; e += 32) kv[dst + e] = kv[src + e];
    __syncwarp();
  }
}

template <typename V>
__global__ void __launch_bounds__(CR_THREADS)
cache_copy_pages_kernel(V* __restrict__ kv, int num_pages, long pieces, const int* __restrict__ pairs, int* err) {
  pdl_wait();
  const int from = pairs[2 * blockIdx.y], to = pairs[2 * blockIdx.y + 1];
  if (from < 0 || from >= num_pages || to < 0 || to >= num_pages) {
    if (threadIdx.x == 0) report_error(err, PHOTON_DEV_BAD_PAGE, blockIdx.y, from, to);
    return;
  }
  if (from == to) return;
  const long long plane = blockIdx.x;
  const V* src = kv + (plane * num_pages + from) * pieces;
  V* dst = kv + (plane * num_pages + to) * pieces;
  for (long e = threadIdx.x; e < pieces; e += CR_THREADS) dst[e] = src[e];
}

// The widest piece that an address and a row allow.
static int piece_bytes(const void* p, long row_bytes) {
  for (int b = 16; b > 2; b >>= 1) if ((uintptr_t)p % b == 0 && row_bytes % b == 0) return b;
  return 2;
}

PHOTON_API int photon_cache_keep(void* kv, int dtype, int planes, int num_pages, int n_kv, int page_size, int d, const int* block_table,
                                 int max_pages, const int* cu_tokens, const int* context_lens, const int* path, const int* counts, int S,
                                 int D, int* err, cudaStream_t stream) {
  if (S <= 0 || D <= 0 || planes <= 0) return 0;
  if (dtype != PHOTON_F32 && dtype != PHOTON_BF16) return PHOTON_ERR_ARGUMENT;
  if (num_pages <= 0 || n_kv <= 0 || page_size <= 0 || d <= 0 || max_pages <= 0) return PHOTON_ERR_ARGUMENT;
  if (S > 65535) return PHOTON_ERR_UNSUPPORTED;
  const long row = (long)d * (dtype == PHOTON_F32 ? 4 : 2);
  const int b = piece_bytes(kv, row);
  const dim3 grid((unsigned)(((long)planes * n_kv + CR_THREADS / 32 - 1) / (CR_THREADS / 32)), (unsigned)S);
  const int pieces = (int)(row / b);
#define KEEP(V) launch_pdl(cache_keep_kernel<V>, grid, dim3(CR_THREADS), 0, stream, (V*)kv, planes, num_pages, n_kv, page_size, pieces, block_table, \
                           max_pages, cu_tokens, context_lens, path, counts, D, err)
  return b == 16 ? KEEP(uint4) : b == 8 ? KEEP(uint2) : b == 4 ? KEEP(uint32_t) : KEEP(uint16_t);
#undef KEEP
}

PHOTON_API int photon_cache_copy_pages(void* kv, int dtype, int planes, int num_pages, long page_elems, const int* pairs, int count, int* err,
                                       cudaStream_t stream) {
  if (count <= 0 || planes <= 0) return 0;
  if (dtype != PHOTON_F32 && dtype != PHOTON_BF16) return PHOTON_ERR_ARGUMENT;
  if (num_pages <= 0 || page_elems <= 0) return PHOTON_ERR_ARGUMENT;
  if (count > 65535) return PHOTON_ERR_UNSUPPORTED;
  const long bytes = page_elems * (dtype == PHOTON_F32 ? 4 : 2);
  const int b = piece_bytes(kv, bytes);
  const dim3 grid((unsigned)planes, (unsigned)count);
#define COPY(V) launch_pdl(cache_copy_pages_kernel<V>, grid, dim3(CR_THREADS), 0, stream, (V*)kv, num_pages, bytes / b, pairs, err)
  return b == 16 ? COPY(uint4) : b == 8 ? COPY(uint2) : b == 4 ? COPY(uint32_t) : COPY(uint16_t);
#undef COPY
}
