// Rows and pages of the paged cache moved on the device, over all cache slots of a group at once (any element type: bytes).
//
// A group's pool is (slots, pages, parts, page_size, width): parts = 2 x kv heads for separate keys and values, kv heads where a
// token's key and value lie side by side, 1 for a latent. A token's row is `width` values in each of slots x parts places.
#include "common.cuh"

namespace {
constexpr int KEEP_THREADS = 256;
constexpr int KEEP_NODES = 1024;      // kept rows of a request at most

template <typename V>
struct Pool {
  V* data;
  long long slot_stride, page_stride, part_stride;      // in units of V
  int slots, parts, width, page_size, num_pages;
};

// The kept nodes of a request's tree: place start + path[k] -> start + k. path rises, so path[k] >= k and a place is read
// before or at the time it is written if the kept nodes go in order: a thread owns PER vectors of every row (each of one slot and part)
// and takes a few rows at a time, loads first, so eight loads are in flight. Grid (slots x parts x vectors of a row, requests). Bound by the
// chain count -> path -> page -> row in every block, so blocks are few where there is enough to do: PER = 4 (64 requests of up to
// 16 nodes, 32 layers of 8 heads of 128: 12 us with 4,096 blocks, 11 with 512 and all of them on the chip at once).
template <typename V, int PER>
__global__ void __launch_bounds__(KEEP_THREADS)
keep_rows_kernel(const Pool<V> P, const int* __restrict__ table, int S, int mb, const int* __restrict__ seg,
                 const int* __restrict__ path, const int* __restrict__ count, int N, int* err) {
  __shared__ long long s_from[KEEP_NODES], s_to[KEEP_NODES];
  __shared__ int s_bad;
  fz_grid_launch_dependents();
  fz_grid_wait();
  const int s = blockIdx.y, row0 = seg[4 * s], nodes = seg[4 * s + 1], start = seg[4 * s + 2];
  const int kept = count[s];
  if (nodes <= 0 || kept <= 0) return;
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  const bool fits = row0 >= 0 && nodes <= N - row0 && kept <= nodes && kept <= KEEP_NODES && start >= 0 && start <= (long long)mb * P.page_size;
  for (int k = threadIdx.x; fits && k < kept; k += KEEP_THREADS) {
    const int from = path[row0 + k];
    int bad = from < k || from >= nodes || (k > 0 && from <= path[row0 + k - 1]) ? FZ_ERR_ROW_RANGE : 0;
    long long at[2] = {-1, -1};
    if (!bad) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const long long place = (long long)start + (w ? k : from), pi = place / P.page_size;
        const int page = pi < mb ? table[(size_t)s * mb + pi] : -1;
        if (page < 0 || page >= P.num_pages) bad = FZ_ERR_NO_PAGE;
        at[w] = (long long)page * P.page_stride + (place - pi * P.page_size) * P.width;
      }
    }
    if (bad) atomicOr(&s_bad, bad);
    s_from[k] = at[0];
    s_to[k] = at[1];
  }
  __syncthreads();
  const int bad = fits ? s_bad : FZ_ERR_ROW_RANGE;
  if (bad) {      // (a request with a path that is none is left as it is)
    if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(err, bad);
    return;
  }
  const int per_slot = P.parts * P.width;
  V* base[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const long long e = ((long long)blockIdx.x * PER + i) * KEEP_THREADS + threadIdx.x;
    const int slot = (int)(e / per_slot), in_slot = (int)(e - (long long)slot * per_slot);
    const int part = in_slot / P.width, v = in_slot - part * P.width;
    base[i] = slot < P.slots ? P.data + slot * P.slot_stride + part * P.part_stride + v : nullptr;
  }
  int k = 0;
  while (k < kept && s_from[k] == s_to[k]) ++k;      // (the root, and a chain that stands: already there)
  constexpr int ROWS = 8 / PER;
  for (; k < kept; k += ROWS) {
    V x[ROWS][PER];
#pragma unroll
    for (int u = 0; u < ROWS; ++u)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (k + u < kept && base[i]) x[u][i] = base[i][s_from[k + u]];
#pragma unroll
    for (int u = 0; u < ROWS; ++u)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (k + u < kept && base[i]) base[i][s_to[k + u]] = x[u][i];
  }
}

// Page src[i] -> dst[i] in every slot. A page of a slot is one run of page_units vectors; grid (parts of a run, slots, pages).
constexpr int COPY_THREADS = 256, COPY_UNROLL = 4;
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS)
copy_pages_kernel(V* __restrict__ pool, long long slot_stride, int page_units, int num_pages, const int* __restrict__ src,
                  const int* __restrict__ dst, int* err) {
  fz_grid_launch_dependents();
  fz_grid_wait();
  const int from = src[blockIdx.z], to = dst[blockIdx.z];
  if (from < 0 || to < 0 || from >= num_pages || to >= num_pages) {
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(err, FZ_ERR_NO_PAGE);
    return;
  }
  const V* a = pool + blockIdx.y * slot_stride + (long long)from * page_units;
  V* b = pool + blockIdx.y * slot_stride + (long long)to * page_units;
  const int at = blockIdx.x * (COPY_THREADS * COPY_UNROLL) + threadIdx.x;
  V x[COPY_UNROLL];
#pragma unroll
  for (int u = 0; u < COPY_UNROLL; ++u)
    if (at + u * COPY_THREADS < page_units) x[u] = a[at + u * COPY_THREADS];
#pragma unroll
  for (int u = 0; u < COPY_UNROLL; ++u)
    if (at + u * COPY_THREADS < page_units) b[at + u * COPY_THREADS] = x[u];
}

template <typename V>
int keep(void* pool, int slots, int num_pages, int parts, int page_size, int row_bytes, const int* table, int S, int mb, const int* seg,
         const int* path, const int* count, int N, int* err, cudaStream_t stream) {
  Pool<V> P;
  P.data = (V*)pool;
  P.width = row_bytes / (int)sizeof(V);
  P.part_stride = (long long)page_size * P.width;
  P.page_stride = parts * P.part_stride;
  P.slot_stride = num_pages * P.page_stride;
  P.slots = slots, P.parts = parts, P.page_size = page_size, P.num_pages = num_pages;
  const long long vectors = (long long)slots * parts * P.width;
  const int per = vectors * S >= 4LL * KEEP_THREADS * 148 ? 4 : 1;
  const long long blocks = (vectors + per * KEEP_THREADS - 1) / (per * KEEP_THREADS);
  if (blocks > 2147483647LL || (long long)parts * P.width > 2147483647LL) return FZ_TOO_LARGE;
  const dim3 grid((unsigned)blocks, (unsigned)S);
  const cudaError_t e = per == 4 ? fz_launch(keep_rows_kernel<V, 4>, grid, dim3(KEEP_THREADS), 0, stream, P, table, S, mb, seg, path, count, N, err)
                                 : fz_launch(keep_rows_kernel<V, 1>, grid, dim3(KEEP_THREADS), 0, stream, P, table, S, mb, seg, path, count, N, err);
  return e == cudaSuccess ? FZ_OK : (int)e;
}

template <typename V>
int copy(void* pool, int slots, int num_pages, long long page_bytes, const int* src, const int* dst, int M, int* err, cudaStream_t stream) {
  const long long units = page_bytes / (long long)sizeof(V), blocks = (units + COPY_THREADS * COPY_UNROLL - 1) / (COPY_THREADS * COPY_UNROLL);
  if (units > 2147483647LL) return FZ_TOO_LARGE;
  const cudaError_t e = fz_launch(copy_pages_kernel<V>, dim3((unsigned)blocks, (unsigned)slots, (unsigned)M), dim3(COPY_THREADS), 0, stream, (V*)pool,
                                  units * num_pages, (int)units, num_pages, src, dst, err);
  return e == cudaSuccess ? FZ_OK : (int)e;
}

// The widest vector that divides a row (or a page) and its address.
#define FZ_BY_WIDTH(bytes, f, ...)                                                        \
  do {                                                                                    \
    const uintptr_t w__ = (uintptr_t)(bytes) | (uintptr_t)pool;                           \
    if (w__ % 16 == 0) return f<uint4>(__VA_ARGS__);                                      \
    if (w__ % 8 == 0) return f<uint2>(__VA_ARGS__);                                       \
    if (w__ % 4 == 0) return f<unsigned int>(__VA_ARGS__);                                \
    return f<unsigned short>(__VA_ARGS__);                                                \
  } while (0)
}  // namespace

// pool: (slots, num_pages, parts, page_size, row_bytes), contiguous; table (S, mb); seg (S, 4) = (first row, rows, first place of
// the tree, anything); path (N,): path[first row + k] = node of the k-th kept row, rising; count (S,).
FZ_API int fz_keep_rows(void* pool, int slots, int num_pages, int parts, int page_size, int row_bytes, const int* table, int S, int mb,
                        const int* seg, const int* path, const int* count, int N, int* err, cudaStream_t stream) {
  if (S <= 0 || slots <= 0) return FZ_OK;
  if (num_pages <= 0 || parts <= 0 || page_size <= 0 || row_bytes <= 0 || row_bytes % 2 || mb <= 0 || N < 0) return FZ_BAD_SHAPE;
  if (S > 65535) return FZ_TOO_LARGE;
  if ((uintptr_t)pool & 1) return FZ_BAD_ALIGNMENT;
  FZ_BY_WIDTH(row_bytes, keep, pool, slots, num_pages, parts, page_size, row_bytes, table, S, mb, seg, path, count, N, err, stream);
}

// src, dst (M,): page ids. No page may be a destination twice, or a source and a destination.
FZ_API int fz_copy_pages(void* pool, int slots, int num_pages, long long page_bytes, const int* src, const int* dst, int M, int* err,
                         cudaStream_t stream) {
  if (M <= 0 || slots <= 0) return FZ_OK;
  if (num_pages <= 0 || page_bytes <= 0 || page_bytes % 2) return FZ_BAD_SHAPE;
  if (M > 65535 || slots > 65535) return FZ_TOO_LARGE;
  if ((uintptr_t)pool & 1) return FZ_BAD_ALIGNMENT;
  FZ_BY_WIDTH(page_bytes, copy, pool, slots, num_pages, page_bytes, src, dst, M, err, stream);
}

#ifdef FZ_TIMELINE
FZ_TIMELINE_READER(cache_rows)
#endif
