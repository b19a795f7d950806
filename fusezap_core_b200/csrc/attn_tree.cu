// Attention of drafted tokens that form a tree, over the paged cache (both dtypes): rows of a step whose keys are the cached
// places before the request's tree and, of the tree's own places, those whose bit is set for the row.
//
// The two kinds of key go separate ways. All rows of a request see the same cached places (but for a window's edge), so these
// are a dense problem: the query heads of a kv head times a few nodes are the rows of a tile, keys and values are read once
// for all of them, and the key axis is cut into pieces that leave unnormalised rows and (maximum, sum) in float32 scratch.
// A row sees few nodes of its tree (its ancestors), scattered and different for every row: the kernel that merges the pieces
// walks the row's set bits, a warp per row and head, so nothing of a node that a row does not see enters its sums, whatever the
// node's place holds.
//
// `attn_tree_context_kernel` here is the general kernel of the first kind, plain float32 FMA from tiles in shared memory: the
// float32 path, and head and page sizes that the tensor-core kernel (attn_tree_tc.cu) refuses.
// Keys are cut at places that depend on the request's own length only, and a tile's rows do not mix: what this kernel leaves of a row
// does not depend on the other requests of the step, and in float32 the row's result does not either. (In bfloat16 the kernel that joins adds a
// row's terms up in another order where a step has many rows, see `launch_merge`.)
#include "attn_tree.cuh"

namespace {
using namespace fztree;

constexpr int THREADS = 256;

// The context of one request as the kernels cut it: places [first, end), in pieces of `piece` from `first` on. first: the
// first place that any row sees, rounded down to a multiple of 64. Up to 32 pieces of at least 64 places (a key tile): the pieces' results
// are written and read once more, (hd + 2) floats a row against 2 hd values a key, but a step of short contexts has few blocks otherwise (4
// requests of 13 nodes behind 500 places, 14 heads of 64 over 2: 46 us with pieces of 256 and tiles of 64 rows, 19 with pieces of 64 and
// tiles of 16).
__host__ __device__ __forceinline__ int piece_length(int places) {
  const int p = ((places + 31) / 32 + 63) / 64 * 64;
  return p < 64 ? 64 : p;
}

struct Args {
  const int *pos, *seg, *table;
  int S, mb;
  long long page_stride;
  int page_size, num_pages, N, Hq, Hkv, hd, window, pieces;
  float scale_log2;
  float *part_o, *part_ml;
  int* err;
};

__device__ __forceinline__ float4 four(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 four(const __nv_bfloat16* p) {
  const uint2 u = *(const uint2*)p;
  const float2 a = __bfloat1622float2(*(const __nv_bfloat162*)&u.x), b = __bfloat1622float2(*(const __nv_bfloat162*)&u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

// Grid (row tiles, kv heads x parts of a kv head's query heads, pieces). 16 x 16 threads; thread (tx, ty) has rows ty + 16 i
// of the tile, keys tx + 16 j of a key tile and dimensions 4 tx + 64 j of the result. RM: rows of a tile, KT: keys of a key
// tile, DPT: dimensions per thread (16 DPT >= hd, the rest zeros).
template <typename T, int DPT, int RM, int KT>
__global__ void __launch_bounds__(THREADS)
attn_tree_context_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool, const Args A) {
  constexpr int HD = 16 * DPT, RPT = RM / 16, KPT = KT / 16, KS = HD + 16 / sizeof(T);
  extern __shared__ __align__(16) unsigned char tree_smem[];
  T* Ks = (T*)tree_smem;                          // [2][KT][KS]
  T* Vs = Ks + 2 * KT * KS;                       // [2][KT][HD]
  float* Qs = (float*)(Vs + 2 * KT * HD);         // [RM][HD]
  float* Ps = Qs + RM * HD;                       // [RM][KT + 4]
  fz_grid_launch_dependents();
  const int G = A.Hq / A.Hkv, GH = G < RM ? G : RM, NB = RM / GH, parts = (G + GH - 1) / GH;
  const int kvh = blockIdx.y / parts, part = blockIdx.y - kvh * parts;
  const int heads = min(GH, G - part * GH), head0 = kvh * G + part * GH;
  fz_grid_wait();
  int s, node0;
  const bool there = find_tile(blockIdx.x, A.seg, A.S, NB, A.N, (long long)A.mb * A.page_size, s, node0);
  int row0 = 0, nodes = 0, start = 0, first = 0, begin = 0, end = 0;
  if (there) {
    row0 = A.seg[4 * s] + node0;
    nodes = min(NB, A.seg[4 * s + 1] - node0);
    start = A.seg[4 * s + 2];
    first = context_first(start, A.window);
    const int piece = piece_length(start - first);
    begin = first + blockIdx.z * piece;
    end = min(start, begin + piece);
    if (blockIdx.z == 0 && first + (long long)A.pieces * piece < start && threadIdx.x == 0) atomicOr(A.err, FZ_ERR_POS_RANGE);      // longer than announced
  }
  if (!there || begin >= end) return;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, rows = nodes * heads;
  const int* trow = A.table + (size_t)s * A.mb;
  const long long head_off = (long long)kvh * A.page_size * A.hd;
  const int seen_from = A.window > 0 ? max(0, start - A.window + 1) : 0;      // (pages before it may have been given back)

  auto fetch = [&](int key0, int buf) {
    T* K = Ks + buf * KT * KS;
    T* V = Vs + buf * KT * HD;
    constexpr int PER = 16 / sizeof(T), CH = HD / PER;      // 16-byte chunks of a key
    for (int e = tid; e < 2 * KT * CH; e += THREADS) {
      const int which = e / (KT * CH), f = e - which * KT * CH, j = f / CH, d = (f - j * CH) * PER, key = key0 + j;
      const T* src = nullptr;
      if (key >= seen_from && key < end && d < A.hd) {
        const int pi = key / A.page_size;
        const int page = pi < A.mb ? trow[pi] : -1;
        if (page >= 0 && page < A.num_pages) src = (which ? v_pool : k_pool) + (long long)page * A.page_stride + head_off + (long long)(key - pi * A.page_size) * A.hd + d;
        else atomicOr(A.err, FZ_ERR_NO_PAGE);
      }
      T* dst = which ? V + j * HD + d : K + j * KS + d;
      fz_copy16(dst, src ? src : k_pool, src != nullptr);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  fetch(begin, 0);
  for (int e = tid; e < RM * HD; e += THREADS) {
    const int r = e / HD, d = e - r * HD;
    Qs[e] = r < rows && d < A.hd ? Cvt<T>::to_f(q[((size_t)(row0 + r / heads) * A.Hq + head0 + r % heads) * A.hd + d]) : 0.f;
  }
  int lo[RPT];
  int lo_max = 0;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = ty + 16 * i;
    lo[i] = r < rows && A.window > 0 ? max(0, A.pos[row0 + r / heads] - A.window + 1) : 0;
    if (A.window > 0) lo_max = max(lo_max, lo[i]);
  }
  lo_max = A.window > 0 ? __syncthreads_or(lo_max > begin) : 0;      // a row of the tile may not see all of the piece
  float m[RPT], l[RPT], o[RPT][DPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < DPT; ++j) o[i][j] = 0.f;
  }
  int buf = 0;
  for (int key0 = begin; key0 < end; key0 += KT, buf ^= 1) {
    if (key0 + KT < end) {
      fetch(key0 + KT, buf ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const T* K = Ks + buf * KT * KS;
    const T* V = Vs + buf * KT * HD;
    float sc[RPT][KPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < KPT; ++j) sc[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      float4 kk[KPT];
#pragma unroll
      for (int j = 0; j < KPT; ++j) kk[j] = four(K + (tx + 16 * j) * KS + d);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float4 qq = four(Qs + (ty + 16 * i) * HD + d);
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          sc[i][j] = fmaf(qq.x, kk[j].x, sc[i][j]);
          sc[i][j] = fmaf(qq.y, kk[j].y, sc[i][j]);
          sc[i][j] = fmaf(qq.z, kk[j].z, sc[i][j]);
          sc[i][j] = fmaf(qq.w, kk[j].w, sc[i][j]);
        }
      }
    }
    // online softmax in the exp2 domain; a row's 16 threads share its maximum and sum
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const int key = key0 + tx + 16 * j;
        sc[i][j] = key < end && key >= lo[i] ? sc[i][j] * A.scale_log2 : -INFINITY;
        mx = fmaxf(mx, sc[i][j]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[i], mx), mu = mn == -INFINITY ? 0.f : mn, corr = exp2f(m[i] - mu);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const float e = exp2f(sc[i][j] - mu);
        sum += e;
        Ps[(ty + 16 * i) * (KT + 4) + tx + 16 * j] = e;
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[i] = fmaf(l[i], corr, sum);
#pragma unroll
      for (int j = 0; j < DPT; ++j) o[i][j] *= corr;
    }
    __syncwarp();      // (a row's weights are written and read by the same half warp)
    const bool edge = lo_max != 0;
    for (int j = 0; j < KT; j += 4) {
      float4 p[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) p[i] = four(Ps + (ty + 16 * i) * (KT + 4) + j);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int c = 0; c < DPT; c += 4) {
          const float4 v = four(V + (j + u) * HD + 4 * tx + 16 * c);
#pragma unroll
          for (int i = 0; i < RPT; ++i) {
            const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
            // (a key before the row's window takes no part, whatever its value: 0 * inf)
            if (!edge || key0 + j + u >= lo[i]) {
              o[i][c] = fmaf(w, v.x, o[i][c]);
              o[i][c + 1] = fmaf(w, v.y, o[i][c + 1]);
              o[i][c + 2] = fmaf(w, v.z, o[i][c + 2]);
              o[i][c + 3] = fmaf(w, v.w, o[i][c + 3]);
            }
          }
        }
      }
    }
    __syncthreads();      // the tile is consumed
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = ty + 16 * i;
    if (r >= rows) continue;
    const size_t at = ((size_t)(row0 + r / heads) * A.Hq + head0 + r % heads) * A.pieces + blockIdx.z;
    if (tx == 0) *(float2*)(A.part_ml + 2 * at) = make_float2(m[i], l[i]);
#pragma unroll
    for (int c = 0; c < DPT; c += 4) {
      const int d = 4 * tx + 16 * c;
      if (d < A.hd) *(float4*)(A.part_o + at * A.hd + d) = make_float4(o[i][c], o[i][c + 1], o[i][c + 2], o[i][c + 3]);
    }
  }
}

// Where a row's pieces lie in the general kernel's scratch.
struct Pieces {
  const float *part_o, *part_ml;
  int pieces, Hq, window;
  __device__ __forceinline__ int2 early(int, int) const { return make_int2(0, 0); }
  __device__ __forceinline__ Range range(int2, int n, int h, int, int, int, int, int start, int) const {
    const int places = start - context_first(start, window), piece = piece_length(places);
    return {min(pieces, (places + piece - 1) / piece), ((size_t)n * Hq + h) * pieces, 1, 0, 0};
  }
};

template <typename T, int DPT, int RM, int KT>
int launch_context(const void* q, const void* k, const void* v, const Args& A, int tiles, cudaStream_t stream) {
  constexpr int HD = 16 * DPT;
  const size_t smem = sizeof(T) * 2 * KT * (2 * HD + 16 / sizeof(T)) + sizeof(float) * (RM * HD + RM * (KT + 4));
  auto kern = attn_tree_context_kernel<T, DPT, RM, KT>;
  static_assert(sizeof(T) * 2 * KT * (2 * HD + 16 / sizeof(T)) + sizeof(float) * (RM * HD + RM * (KT + 4)) <= FZ_MOST_SMEM);
  FZ_RAISE_SMEM(kern);
  const int G = A.Hq / A.Hkv, GH = G < RM ? G : RM;
  const dim3 grid((unsigned)tiles, (unsigned)(A.Hkv * ((G + GH - 1) / GH)), (unsigned)A.pieces);
  const cudaError_t e = fz_launch(kern, grid, dim3(THREADS), smem, stream, (const T*)q, (const T*)k, (const T*)v, A);
  return e == cudaSuccess ? FZ_OK : (int)e;
}

template <typename T>
int context(const void* q, const void* k, const void* v, const Args& A, cudaStream_t stream) {
  const int G = A.Hq / A.Hkv;
  // tiles of 16 rows where a request's rows fill no more than one of those on average, or where larger ones would be too few blocks
  const bool few = (long long)A.N * G <= 16LL * A.S || ((long long)A.N * G / 64 + A.S) * A.Hkv * A.pieces < 2 * 148;
  auto tiles = [&](int RM) {
    const int NB = RM / (G < RM ? G : RM);
    const long long t = (long long)A.N / NB + A.S;
    return (int)(t < A.N ? t : A.N);
  };
  if (A.hd <= 64) return few ? launch_context<T, 4, 16, 64>(q, k, v, A, tiles(16), stream) : launch_context<T, 4, 64, 64>(q, k, v, A, tiles(64), stream);
  if (A.hd <= 128) return few ? launch_context<T, 8, 16, 64>(q, k, v, A, tiles(16), stream) : launch_context<T, 8, 64, 64>(q, k, v, A, tiles(64), stream);
  if (A.hd <= 256) return launch_context<T, 16, 16, 32>(q, k, v, A, tiles(16), stream);
  return launch_context<T, 32, 16, 16>(q, k, v, A, tiles(16), stream);
}
}  // namespace

FZ_API int fz_attn_tree_check(int Hq, int Hkv, int hd) {
  return Hq <= 0 || Hkv <= 0 || Hq % Hkv || hd <= 0 || hd % 16 || hd > 512 ? FZ_BAD_SHAPE : FZ_OK;
}

// The pieces that the general kernel cuts a context of at most `max_context` places into (the scratch: N * Hq * pieces *
// (hd + 2) floats).
FZ_API int fz_attn_tree_pieces(int max_context, int window) {
  int places = max_context > 0 ? max_context : 1;
  if (window > 0 && places > window + 64) places = window + 64;
  // (a shorter context may be cut into as many pieces: 32 of its own length)
  const int most = (places + 63) / 64;
  return most < 32 ? most : 32;
}

// q, out: (N, Hq hd); seg (S, 4) = (first row, rows, first place of the tree, anything); ancestors (N, words): bit j of a row's
// words: place `first place + j` is seen. part: N * Hq * pieces * (hd + 2) floats, 16-byte aligned.
FZ_API int fz_attn_tree(const void* q, const void* k_pool, const void* v_pool, const int* pos, const int* seq_row, const int* seg, int S,
                        const int* ancestors, int words, const int* table, int mb, long long page_stride, int page_size, int num_pages,
                        void* out, int dtype, int N, int Hq, int Hkv, int hd, float scale, int window, int pieces, float* part, int* err,
                        cudaStream_t stream) {
  if (N <= 0) return FZ_OK;
  if (fz_attn_tree_check(Hq, Hkv, hd) != FZ_OK || S <= 0 || words <= 0 || mb <= 0 || page_size <= 0 || num_pages <= 0 || pieces <= 0 || pieces > 32) return FZ_BAD_SHAPE;
  if (Hq > 65535) return FZ_TOO_LARGE;
  if (dtype != FZ_F32 && dtype != FZ_BF16) return FZ_BAD_DTYPE;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)part) & 15 || page_stride % (dtype == FZ_F32 ? 4 : 8)) return FZ_BAD_ALIGNMENT;
  const Args A = {pos, seg, table, S, mb, page_stride, page_size, num_pages, N, Hq, Hkv, hd, window, pieces, scale * 1.4426950408889634f,
            part, part + (size_t)N * Hq * pieces * hd, err};
  const int st = dtype == FZ_F32 ? context<float>(q, k_pool, v_pool, A, stream) : context<__nv_bfloat16>(q, k_pool, v_pool, A, stream);
  if (st != FZ_OK) return st;
  const Pieces P = {A.part_o, A.part_ml, pieces, Hq, window};
  const TreeArgs R = {pos, seq_row, seg, ancestors, table, S, words, mb, page_stride, page_size, num_pages, N, Hq, Hkv, hd, A.scale_log2, window, err};
  return dtype == FZ_F32 ? launch_merge<float>((const float*)q, (const float*)k_pool, (const float*)v_pool, (float*)out, P, R, stream)
                         : launch_merge<__nv_bfloat16>((const __nv_bfloat16*)q, (const __nv_bfloat16*)k_pool, (const __nv_bfloat16*)v_pool,
                                                       (__nv_bfloat16*)out, P, R, stream);
}

#ifdef FZ_TIMELINE
FZ_TIMELINE_READER(attn_tree)
#endif
