// Shared by the kernels that attend over a tree of drafted tokens: which rows a tile has, where a request's cached context
// begins, and the kernel that joins the context's pieces with the row's own ancestors.
#pragma once
#include "common.cuh"
#include <math.h>

namespace fztree {

// The first place of the context that any row of a request sees, rounded down to a multiple of 64 (the rows' own windows, which
// begin there or later, are the kernels' business). start: the first place of the tree, the smallest position of its rows.
__host__ __device__ __forceinline__ int context_first(int start, int window) {
  if (window <= 0 || start < window) return 0;
  return (start - window + 1) & ~63;
}

// Tile number `tile` of a step whose requests' rows are cut into tiles of NB nodes: its request and its first node within it. The
// whole warp takes part.
__device__ __forceinline__ bool find_tile(int tile, const int* __restrict__ seg, int S, int NB, int& s, int& node0) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int s0 = 0; s0 < S; s0 += 32) {
    const int n = s0 + lane < S ? max(seg[4 * (s0 + lane) + 1], 0) : 0;
    const int t = (n + NB - 1) / NB;
    int upto = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + upto > tile);
    if (hit) {
      const int who = __ffs(hit) - 1;
      s = s0 + who;
      node0 = (tile - base - (__shfl_sync(0xffffffffu, upto - t, who))) * NB;
      return true;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

struct TreeArgs {
  const int *pos, *seq_row, *seg, *ancestors, *table;
  int S, words, mb;
  long long page_stride;
  int page_size, num_pages, N, Hq, Hkv, hd;
  float scale_log2;
  int window;
  int* err;
};

// Where a row's pieces of the context lie in the scratch (place `first + i * step` of its rows), and the context places [extra_from,
// extra_to) that the row sees beside them.
struct Range {
  int pieces;
  size_t first;
  int step, extra_from, extra_to;
};

__device__ __forceinline__ float4 load4(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 u = *(const uint2*)p;
  const float2 a = __bfloat1622float2(*(const __nv_bfloat162*)&u.x), b = __bfloat1622float2(*(const __nv_bfloat162*)&u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void save4(float* p, float4 v) { *(float4*)p = v; }
__device__ __forceinline__ void save4(__nv_bfloat16* p, float4 v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *(uint2*)p = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
}

constexpr int MERGE_WARPS = 8;

// A warp per row and head; a lane has the dimensions 4 lane + 128 c. The context's pieces in rising order of their keys, then
// the row's set bits in rising order, four keys at a time so that their loads and their sums over the lanes overlap. m, l, o:
// maximum (exp2 domain), sum of weights and weighted values so far, float32.
template <typename T, typename Where, int CH>
__global__ void __launch_bounds__(32 * MERGE_WARPS)
attn_tree_merge_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool, T* __restrict__ out,
                       const Where where, const TreeArgs A) {
  fz_grid_launch_dependents();
  fz_grid_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = blockIdx.x, h = blockIdx.y * MERGE_WARPS + warp;
  if (h >= A.Hq) return;
  T* dst = out + ((size_t)n * A.Hq + h) * A.hd;
  const int s = A.seq_row[n];
  const bool there = s >= 0 && s < A.S && n >= A.seg[4 * s] && n - A.seg[4 * s] < A.seg[4 * s + 1];
  if (!there) {      // a padding row
    if (s >= 0 && lane == 0) atomicOr(A.err, FZ_ERR_ROW_RANGE);
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (4 * lane + 128 * c < A.hd) save4(dst + 4 * lane + 128 * c, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int row0 = A.seg[4 * s], nodes = A.seg[4 * s + 1], start = A.seg[4 * s + 2], kvh = h / (A.Hq / A.Hkv);
  float m = -INFINITY, l = 0.f;
  float4 o[CH], qv[CH];
  const T* from = q + ((size_t)n * A.Hq + h) * A.hd;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const bool in = 4 * lane + 128 * c < A.hd;
    o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    qv[c] = in ? load4(from + 4 * lane + 128 * c) : o[c];
  }
  const int group = A.Hq / A.Hkv;
  const Range range = where.range(n, h, s, n - row0, kvh, h - kvh * group, nodes, start, A.pos[n]);
  const int pieces = range.pieces;
  for (int f0 = 0; f0 < pieces; f0 += 32) {
    const int here = min(32, pieces - f0);
    const float2 ml = lane < here ? *(const float2*)(where.part_ml + 2 * (range.first + (size_t)(f0 + lane) * range.step)) : make_float2(-INFINITY, 0.f);
    float top = ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float mn = fmaxf(m, top);
    if (mn == -INFINITY) continue;      // (no row of these pieces saw a key)
    const float corr = exp2f(m - mn), e = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mn);
    m = mn;
    l *= corr;
#pragma unroll
    for (int c = 0; c < CH; ++c) { o[c].x *= corr; o[c].y *= corr; o[c].z *= corr; o[c].w *= corr; }
#pragma unroll 4
    for (int f = 0; f < here; ++f) {
      const float w = __shfl_sync(0xffffffffu, e, f), add = __shfl_sync(0xffffffffu, ml.y, f);
      if (w == 0.f) continue;      // (a piece of which the row sees nothing may hold anything)
      l = fmaf(add, w, l);
      const float* src = where.part_o + (range.first + (size_t)(f0 + f) * range.step) * A.hd;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (4 * lane + 128 * c < A.hd) {
          const float4 v = *(const float4*)(src + 4 * lane + 128 * c);
          o[c].x = fmaf(v.x, w, o[c].x); o[c].y = fmaf(v.y, w, o[c].y); o[c].z = fmaf(v.z, w, o[c].z); o[c].w = fmaf(v.w, w, o[c].w);
        }
      }
    }
  }
  const int* trow = A.table + (size_t)s * A.mb;
  // up to four places (-1: none)
  auto attend = [&](const int (&places)[4]) {
    float4 kv[4][CH], vv[4][CH];
    float sc[4];
    bool ok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      ok[u] = places[u] >= 0;
      long long off = 0;
      if (ok[u]) {
        const int pi = places[u] / A.page_size;
        const int page = pi < A.mb ? trow[pi] : -1;
        ok[u] = page >= 0 && page < A.num_pages;
        if (ok[u]) off = (long long)page * A.page_stride + ((long long)kvh * A.page_size + (places[u] - pi * A.page_size)) * A.hd;
        else if (lane == 0) atomicOr(A.err, FZ_ERR_NO_PAGE);
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const bool in = ok[u] && 4 * lane + 128 * c < A.hd;
        kv[u][c] = in ? load4(k_pool + off + 4 * lane + 128 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        vv[u][c] = in ? load4(v_pool + off + 4 * lane + 128 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      sc[u] = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        sc[u] = fmaf(qv[c].x, kv[u][c].x, sc[u]); sc[u] = fmaf(qv[c].y, kv[u][c].y, sc[u]);
        sc[u] = fmaf(qv[c].z, kv[u][c].z, sc[u]); sc[u] = fmaf(qv[c].w, kv[u][c].w, sc[u]);
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1)
#pragma unroll
      for (int u = 0; u < 4; ++u) sc[u] += __shfl_xor_sync(0xffffffffu, sc[u], x);
    float mn = m;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      sc[u] = ok[u] ? sc[u] * A.scale_log2 : -INFINITY;
      mn = fmaxf(mn, sc[u]);
    }
    const float mu = mn == -INFINITY ? 0.f : mn, corr = exp2f(m - mu);
    m = mn;
    l *= corr;
#pragma unroll
    for (int c = 0; c < CH; ++c) { o[c].x *= corr; o[c].y *= corr; o[c].z *= corr; o[c].w *= corr; }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (!ok[u]) continue;
      const float e = exp2f(sc[u] - mu);
      l += e;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        o[c].x = fmaf(vv[u][c].x, e, o[c].x); o[c].y = fmaf(vv[u][c].y, e, o[c].y);
        o[c].z = fmaf(vv[u][c].z, e, o[c].z); o[c].w = fmaf(vv[u][c].w, e, o[c].w);
      }
    }
  };
  for (int x = range.extra_from; x < range.extra_to; x += 4) {
    const int places[4] = {x, x + 1 < range.extra_to ? x + 1 : -1, x + 2 < range.extra_to ? x + 2 : -1, x + 3 < range.extra_to ? x + 3 : -1};
    attend(places);
  }
  for (int w0 = 0; w0 < A.words && 32 * w0 < nodes; ++w0) {
    unsigned bits = (unsigned)A.ancestors[(size_t)n * A.words + w0];
    if (nodes - 32 * w0 < 32) bits &= (1u << (nodes - 32 * w0)) - 1u;
    while (bits) {
      int places[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        places[u] = bits ? start + 32 * w0 + __ffs(bits) - 1 : -1;
        bits &= bits - 1;
      }
      attend(places);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;      // (a row that sees no key gives zeros)
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (4 * lane + 128 * c < A.hd)
      save4(dst + 4 * lane + 128 * c, make_float4(o[c].x * inv, o[c].y * inv, o[c].z * inv, o[c].w * inv));
}

template <typename T, typename Where>
int launch_merge(const T* q, const T* k, const T* v, T* out, const Where& where, const TreeArgs& A, cudaStream_t stream) {
  const dim3 grid((unsigned)A.N, (unsigned)((A.Hq + MERGE_WARPS - 1) / MERGE_WARPS));
  cudaError_t e;
  if (A.hd <= 128) e = fz_launch(attn_tree_merge_kernel<T, Where, 1>, grid, dim3(32 * MERGE_WARPS), 0, stream, q, k, v, out, where, A);
  else if (A.hd <= 256) e = fz_launch(attn_tree_merge_kernel<T, Where, 2>, grid, dim3(32 * MERGE_WARPS), 0, stream, q, k, v, out, where, A);
  else e = fz_launch(attn_tree_merge_kernel<T, Where, 4>, grid, dim3(32 * MERGE_WARPS), 0, stream, q, k, v, out, where, A);
  return e == cudaSuccess ? FZ_OK : (int)e;
}

}  // namespace fztree
