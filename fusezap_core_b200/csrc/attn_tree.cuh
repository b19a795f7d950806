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

// Nodes of a request whose rows lie in the step and whose tree begins within its block table (`places` long); else none of it is touched, and
// its rows are reported.
__device__ __forceinline__ int sound_nodes(int row0, int nodes, int start, int N, long long places) {
  return row0 >= 0 && nodes > 0 && nodes <= N - row0 && start >= 0 && start <= places ? nodes : 0;
}

// Tile number `tile` of a step whose requests' rows are cut into tiles of NB nodes: its request and its first node within it. The
// whole warp takes part.
__device__ __forceinline__ bool find_tile(int tile, const int* __restrict__ seg, int S, int NB, int N, long long places, int& s, int& node0) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int s0 = 0; s0 < S; s0 += 32) {
    const int* e = seg + 4 * (s0 + lane);
    const int n = s0 + lane < S ? sound_nodes(e[0], e[1], e[2], N, places) : 0;
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

// 16 bytes of T as float32.
__device__ __forceinline__ void as_floats(const uint4& r, float (&v)[4]) {
  v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void as_floats(const uint4& r, float (&v)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(*(const __nv_bfloat162*)&w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 as_raw(const float (&v)[4]) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
__device__ __forceinline__ uint4 as_raw(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *(const uint32_t*)&p;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int MERGE_WARPS = 8;

// A warp is cut into groups of LANES lanes: a group's lane has the dimensions VEC (lane + LANES c) + 0 .. VEC - 1, c < D / VEC, of one
// head's row. Two ways to use the groups:
//   SHARE false   a warp per row and head: pieces of the context and places go round the groups in rising order, every group keeps its own
//                 maximum, sum and values, and the groups' are joined at the end. Few rows: the chain of loads is short.
//   SHARE true    a warp per row and as many query heads of one kv head as there are groups, which all see the same places: keys and
//                 values are asked for once for all of them, and a quarter of the warps do. Many rows: one round of warps instead of several.
// m, l, o: maximum (exp2 domain), sum of weights and weighted values so far, float32; the context's pieces first, then the tree's places in
// rising order, then those that the row sees beside them. Bound by the chain of loads (row -> request -> pieces, pages -> values) and by
// fetching its instructions, hence short loops instead of unrolled ones, and no spills: local memory is as far away as the rest (a
// warp with four dimensions a lane and eight places at a time took 15 us from start to end, this one 4).
template <typename T, typename Where, int LANES, int D, bool SHARE>
__global__ void __launch_bounds__(32 * MERGE_WARPS, D == 8 ? 4 : SHARE ? 3 : 2)
attn_tree_merge_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool, T* __restrict__ out,
                       const Where where, const TreeArgs A) {
  constexpr int VEC = 16 / sizeof(T), NC = D / VEC, GROUPS = 32 / LANES, STEP = SHARE ? 1 : GROUPS;
  fz_grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane / LANES, gl = lane % LANES;
  const int n = blockIdx.x, group = A.Hq / A.Hkv, job = blockIdx.y * MERGE_WARPS + warp;
  const int parts = SHARE ? (group + GROUPS - 1) / GROUPS : group;      // warps of a kv head
  const int kvh = job / parts, in_group = SHARE ? (job - kvh * parts) * GROUPS + g : job - kvh * parts, h = kvh * group + in_group;
  fz_grid_wait();
  if (kvh >= A.Hkv) return;
  const bool mine = in_group < group;      // (the last warp of a kv head may have groups without a head)
  const size_t at = ((size_t)n * A.Hq + (mine ? h : 0)) * A.hd;
  const int s = A.seq_row[n];
  unsigned bits = (unsigned)A.ancestors[(size_t)n * A.words];
  const int2 record = where.early(n, kvh);
  const int pos = A.window > 0 ? A.pos[n] : 0;
  uint4 qr[NC];
  float o[D];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = VEC * (gl + LANES * c);
    qr[c] = d < A.hd ? *(const uint4*)(q + at + d) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < D; ++i) o[i] = 0.f;
  const bool named = s >= 0 && s < A.S;
  const int row0 = named ? A.seg[4 * s] : 0, start = named ? A.seg[4 * s + 2] : 0;
  const int nodes = named ? sound_nodes(row0, A.seg[4 * s + 1], start, A.N, (long long)A.mb * A.page_size) : 0;
  if (!named || n < row0 || n - row0 >= nodes) {      // a padding row
    if (s >= 0 && lane == 0) atomicOr(A.err, FZ_ERR_ROW_RANGE);
    if (mine)
      for (int d = VEC * (SHARE ? gl : lane); d < A.hd; d += (SHARE ? LANES : 32) * VEC) *(uint4*)(out + at + d) = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const Range range = where.range(record, n, mine ? h : 0, n - row0, mine ? in_group : 0, group, nodes, start, pos);
  // the pages of the tree's first places, a lane each
  const int* trow = A.table + (size_t)s * A.mb;
  const int page0 = start / A.page_size;
  const int pages = page0 + lane < A.mb && (long long)(page0 + lane) * A.page_size < (long long)start + nodes ? trow[page0 + lane] : -1;
  float m = -INFINITY, l = 0.f;
  // the context's pieces
#pragma unroll 2
  for (int f = SHARE ? 0 : g; f < range.pieces; f += STEP) {
    const size_t slot = range.first + (size_t)f * range.step;
    const float2 ml = *(const float2*)(where.part_ml + 2 * slot);
    const float* src = where.part_o + slot * A.hd;
    float4 v[D / 4];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const int d = VEC * (gl + LANES * c) + i;
        v[(c * VEC + i) / 4] = d < A.hd ? *(const float4*)(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    if (ml.x == -INFINITY) continue;      // (a piece of which the row sees nothing may hold anything)
    const float mn = fmaxf(m, ml.x), corr = exp2f(m - mn), w = exp2f(ml.x - mn);
    m = mn;
    l = l * corr + ml.y * w;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      o[4 * i] = o[4 * i] * corr + v[i].x * w, o[4 * i + 1] = o[4 * i + 1] * corr + v[i].y * w;
      o[4 * i + 2] = o[4 * i + 2] * corr + v[i].z * w, o[4 * i + 3] = o[4 * i + 3] * corr + v[i].w * w;
    }
  }
  // places, STEP x AT at a time: the tree's whose bit is set, then the others
  constexpr int AT = SHARE ? 2 : 1;
  int w0 = 0, extra = range.extra_from;
  if (nodes < 32) bits &= (1u << nodes) - 1u;
#pragma unroll 1
  for (;;) {
    while (!bits && ++w0 < A.words && 32 * w0 < nodes) {
      bits = (unsigned)A.ancestors[(size_t)n * A.words + w0];
      if (nodes - 32 * w0 < 32) bits &= (1u << (nodes - 32 * w0)) - 1u;
    }
    int place[AT];
    if (bits) {
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        place[u] = -1;
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          if ((SHARE || i == g) && bits) place[u] = start + 32 * w0 + __ffs(bits) - 1;
          bits &= bits - 1;
        }
      }
    } else if (extra < range.extra_to) {
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        place[u] = extra + (SHARE ? 0 : g) < range.extra_to ? extra + (SHARE ? 0 : g) : -1;
        extra += STEP;
      }
    } else {
      break;
    }
    uint4 kr[AT][NC], vr[AT][NC];
    bool seen[AT];
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      const int pi = place[u] / A.page_size, near = __shfl_sync(0xffffffffu, pages, (pi - page0) & 31);
      const int page = place[u] < 0 ? -1 : pi >= page0 && pi < page0 + 32 ? near : pi < A.mb ? trow[pi] : -1;
      seen[u] = page >= 0 && page < A.num_pages;
      if (place[u] >= 0 && !seen[u] && gl == 0) atomicOr(A.err, FZ_ERR_NO_PAGE);
      const long long off = seen[u] ? (long long)page * A.page_stride + ((long long)kvh * A.page_size + (place[u] - pi * A.page_size)) * A.hd : 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = VEC * (gl + LANES * c);
        const bool in = seen[u] && d < A.hd;
        kr[u][c] = in ? *(const uint4*)(k_pool + off + d) : make_uint4(0u, 0u, 0u, 0u);
        vr[u][c] = in ? *(const uint4*)(v_pool + off + d) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    float sc[AT];
    float mn = m;
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      sc[u] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float x[VEC], y[VEC];
        as_floats(kr[u][c], x);
        as_floats(qr[c], y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sc[u] = fmaf(y[i], x[i], sc[u]);
      }
#pragma unroll
      for (int x = LANES / 2; x > 0; x >>= 1) sc[u] += __shfl_xor_sync(0xffffffffu, sc[u], x);
      sc[u] = seen[u] ? sc[u] * A.scale_log2 : -INFINITY;
      mn = fmaxf(mn, sc[u]);
    }
    const float mu = mn == -INFINITY ? 0.f : mn, corr = exp2f(m - mu);
    m = mn;
    l *= corr;
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] *= corr;
#pragma unroll
    for (int u = 0; u < AT; ++u) {
      if (!seen[u]) continue;
      const float e = exp2f(sc[u] - mu);
      l += e;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float x[VEC];
        as_floats(vr[u][c], x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[c * VEC + i] = fmaf(x[i], e, o[c * VEC + i]);
      }
    }
  }
  // the groups' results
  if (!SHARE) {
    float top = m;
#pragma unroll
    for (int x = LANES; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float w = m == -INFINITY ? 0.f : exp2f(m - top);
    l *= w;
#pragma unroll
    for (int x = LANES; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
    for (int i = 0; i < D; ++i) {
      o[i] = w == 0.f ? 0.f : o[i] * w;
#pragma unroll
      for (int x = LANES; x < 32; x <<= 1) o[i] += __shfl_xor_sync(0xffffffffu, o[i], x);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;      // (a row that sees no key gives zeros)
  if (SHARE ? mine : g == 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = VEC * (gl + LANES * c);
      float x[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = l == 0.f ? 0.f : o[c * VEC + i] * inv;
      if (d < A.hd) *(uint4*)(out + at + d) = as_raw(x);
    }
  }
}

template <typename T, int LANES, int D, bool SHARE, typename Where>
int launch_merge_as(const T* q, const T* k, const T* v, T* out, const Where& where, const TreeArgs& A, cudaStream_t stream) {
  const int group = A.Hq / A.Hkv, jobs = SHARE ? A.Hkv * ((group + 32 / LANES - 1) / (32 / LANES)) : A.Hq;
  const dim3 grid((unsigned)A.N, (unsigned)((jobs + MERGE_WARPS - 1) / MERGE_WARPS));
  const cudaError_t e = fz_launch(attn_tree_merge_kernel<T, Where, LANES, D, SHARE>, grid, dim3(32 * MERGE_WARPS), 0, stream, q, k, v, out, where, A);
  return e == cudaSuccess ? FZ_OK : (int)e;
}

template <typename T, typename Where>
int launch_merge(const T* q, const T* k, const T* v, T* out, const Where& where, const TreeArgs& A, cudaStream_t stream) {
  // bfloat16: warps share their loads between heads where there are several heads of a kv head and more rows x heads than two blocks per
  // SM hold. float32: never, since the two ways add a row's terms up in another order, and a row's sums are not to depend on the step.
  if constexpr (sizeof(T) == 2) {
    if (A.Hq > A.Hkv && (long long)A.N * A.Hq > 148LL * 2 * MERGE_WARPS) {
      if (A.hd <= 64) return launch_merge_as<T, 8, 8, true>(q, k, v, out, where, A, stream);
      if (A.hd <= 128) return launch_merge_as<T, 8, 16, true>(q, k, v, out, where, A, stream);
    }
  }
  if (A.hd <= 64) return launch_merge_as<T, 8, 8, false>(q, k, v, out, where, A, stream);
  if (A.hd <= 128) return launch_merge_as<T, 8, 16, false>(q, k, v, out, where, A, stream);
  if (A.hd <= 256) return launch_merge_as<T, 16, 16, false>(q, k, v, out, where, A, stream);
  return launch_merge_as<T, 32, 16, false>(q, k, v, out, where, A, stream);
}

}  // namespace fztree
