// The verdict on a tree of drafted tokens against the target's logits, from given random numbers (float64 throughout).
//
// A request's walk starts at its root, the token already chosen. At a node, p = softmax(logits / T) is the target's distribution
// of the next token, q that of the drafter, from which the node's children were drawn one after the other without replacement
// (without a drafter's logits: q puts all on the child). A child x with uniform number u stands if u q(x) < p(x), and the walk goes
// on from it; else p becomes max(p - q, 0) over its sum, q loses x and is scaled to sum 1, and the next child is tried. Where no
// child stands, the next token is drawn from what p is then, so the tokens are distributed as the target's own (recursive
// rejection sampling). T <= 0: the child that is the argmax stands, else the argmax is the next token.
//
// The tokens of a row are shared by the BLOCKS blocks of a cluster, one cluster per request: a walk is a chain of passes over one
// row pair each (statistics of a node: maximum and sum; after a rejection: the sums of the new p and q), each ended by one exchange
// through distributed shared memory after which all blocks know the sums and take the same decisions. Only the rows of nodes
// that the walk visits are read. A pass keeps its sums per warp, whose tokens are one run each, so the last pass before the draw
// already says in whose run the drawn token lies: one warp walks that run again, in index order.
// exp in float64 by a table of 2^(j/64) and a Taylor polynomial (the table-driven method of P. T. P. Tang, 1989): ten float64
// operations a token, so that a pass is not bound by them (a draw's place among 100,000 running sums needs more than 32 bits).
#include "common.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

namespace {
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MAX_NODES = 1024;      // nodes of a tree

struct Ref {      // a row's scale: token x weighs exp((x - top) / T)
  double scale, top;      // 64 log2(e) / T, and the row's maximum
};

// The token's weight, tab[j] = 2^(j / 64); 1 for x = top exactly. -inf gives 0, NaN and +inf NaN. Here and where p and q are
// made from weights the roundings are written out: every place that needs a token's p gets the same bits.
__device__ __forceinline__ double weight(float x, const Ref& r, const double* tab) {
  const double t = __dmul_rn(__dadd_rn((double)x, -r.top), r.scale);      // 64 log2 of the weight
  if (!(t > -65000.0)) return t == t ? 0.0 : t;          // (below 2^-1015: nothing beside a maximum of 1)
  const double big = 6755399441055744.0;                 // 1.5 * 2^52: the low bits of the sum are the nearest whole number
  const double shifted = __dadd_rn(t, big), f = __dadd_rn(t, -__dadd_rn(shifted, -big));
  const int k = __double2loint(shifted);
  constexpr double c1 = 0.010830424696249145, c2 = 5.86490495505617e-05, c3 = 2.1173137155464776e-07,
                   c4 = 5.732851688640402e-10;      // (ln 2 / 64)^i / i!
  const double e = __dmul_rn(tab[k & 63], fma(f, fma(f, fma(f, fma(f, c4, c3), c2), c1), 1.0));
  return __hiloint2double(__double2hiint(e) + ((k >> 6) << 20), __double2loint(e));
}

__device__ __forceinline__ bool better(float v, int i, float bv, int bi) {      // numpy.argmax: a NaN is the maximum, then the lower index
  if (bi < 0) return i >= 0;
  if (i < 0) return false;
  const bool vn = isnan(v), bn = isnan(bv);
  if (vn != bn) return vn;
  if (!vn && v != bv) return v > bv;
  return i < bi;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Stat { float top; double sum; };
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, double scale, const double* tab) {
  if (a.top == b.top) return {a.top, a.sum + b.sum};      // (two without tokens: -inf, 0)
  const Stat &hi = a.top > b.top ? a : b, &lo = a.top > b.top ? b : a;
  if (lo.sum == 0.0) return {hi.top, hi.sum + lo.sum};
  return {hi.top, fma(lo.sum, weight(lo.top, Ref{scale, (double)hi.top}, tab), hi.sum)};
}

struct Slot {      // what a block tells the others after a pass
  float top_p, top_q;
  double sum_p, sum_q;
  int arg;
};

struct Shared {
  double tab[64];
  Slot slot[2];
  float top_p[WARPS], top_q[WARPS];
  double sum_p[WARPS], sum_q[WARPS], run[WARPS];
  int arg[WARPS];
  // the rejected siblings at the node: token, 1 / sum of p after it, 1 / sum of q before it
  double scale_p[MAX_NODES], scale_q[MAX_NODES];
  int token[MAX_NODES];
};

template <int BLOCKS>
__global__ void __launch_bounds__(THREADS, 1)
verify_kernel(const float* __restrict__ logits, const float* __restrict__ draft, const float* __restrict__ temperature,
              const double* __restrict__ uniform, const int* __restrict__ tokens, const int* __restrict__ parents,
              const int* __restrict__ seg, int N, int V, int* __restrict__ path, int* __restrict__ count, int* __restrict__ next_ids, int* err) {
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  fz_grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int s = blockIdx.x / BLOCKS, rank = blockIdx.x % BLOCKS;
  if (tid < 64) sh.tab[tid] = exp2((double)tid / 64.0);
  fz_grid_wait();
  const int row0 = seg[4 * s], n = seg[4 * s + 1];
  const bool first = rank == 0 && tid == 0;
  if (n <= 0 || row0 < 0 || row0 + n > N || n > MAX_NODES) {      // (the whole cluster)
    if (first) {
      if (n > 0) atomicOr(err, FZ_ERR_ROW_RANGE);
      count[s] = 0;
      next_ids[s] = -1;
    }
    return;
  }
  __syncthreads();
  const float T = temperature[s];
  const bool greedy = !(T > 0.f);
  const double scale = 92.33248261689366 / (double)T;      // 64 log2(e) / T
  // this warp's run of tokens: [lo, hi), within the block's part of the vocabulary; multiples of four
  const int per_warp = ((V + BLOCKS * WARPS - 1) / (BLOCKS * WARPS) + 3) & ~3;
  const int lo = min(V, (rank * WARPS + warp) * per_warp), hi = min(V, lo + per_warp);
  const bool vec = (V & 3) == 0 && (((uintptr_t)logits | (uintptr_t)draft) & 15) == 0;
  int turn = 0;
  // Every block leaves its slot; after the barrier all read all of them (the next exchange writes the other slot).
  auto exchange = [&](Slot mine, Slot& got, bool with_max) {
    if (tid == 0) sh.slot[turn] = mine;
    if (BLOCKS == 1) __syncthreads();
    else cluster.sync();
    Slot r = lane < BLOCKS ? (BLOCKS == 1 ? sh.slot[turn] : *cluster.map_shared_rank(&sh.slot[turn], lane)) : Slot{-INFINITY, -INFINITY, 0.0, 0.0, -1};
    turn ^= 1;
#pragma unroll
    for (int o = 1; o < BLOCKS; o <<= 1) {
      Slot b;
      b.top_p = __shfl_xor_sync(0xffffffffu, r.top_p, o);
      b.top_q = __shfl_xor_sync(0xffffffffu, r.top_q, o);
      b.sum_p = __shfl_xor_sync(0xffffffffu, r.sum_p, o);
      b.sum_q = __shfl_xor_sync(0xffffffffu, r.sum_q, o);
      b.arg = __shfl_xor_sync(0xffffffffu, r.arg, o);
      if (greedy) {
        if (better(b.top_p, b.arg, r.top_p, r.arg)) { r.top_p = b.top_p; r.arg = b.arg; }
      } else if (with_max) {
        const Stat p = join({r.top_p, r.sum_p}, {b.top_p, b.sum_p}, scale, sh.tab), q = join({r.top_q, r.sum_q}, {b.top_q, b.sum_q}, scale, sh.tab);
        r.top_p = p.top, r.sum_p = p.sum, r.top_q = q.top, r.sum_q = q.sum;
      } else {
        r.sum_p += b.sum_p;
        r.sum_q += b.sum_q;
      }
    }
    got.top_p = __shfl_sync(0xffffffffu, r.top_p, 0);
    got.top_q = __shfl_sync(0xffffffffu, r.top_q, 0);
    got.sum_p = __shfl_sync(0xffffffffu, r.sum_p, 0);
    got.sum_q = __shfl_sync(0xffffffffu, r.sum_q, 0);
    got.arg = __shfl_sync(0xffffffffu, r.arg, 0);
  };
  auto each = [&](const float* row, auto f) {      // f(index, x) over the warp's run
    if (vec) {
      for (int i = lo + 4 * lane; i < hi; i += 128) {
        const float4 x = *(const float4*)(row + i);
        f(i, x.x); f(i + 1, x.y); f(i + 2, x.z); f(i + 3, x.w);
      }
    } else {
      for (int i = lo + lane; i < hi; i += 32) f(i, row[i]);
    }
  };
  auto row_stat = [&](const float* row) {      // maximum and sum of the warp's run, in one pass: a lane's sum goes by its own maximum
    float top = -INFINITY;
    double sum = 0.0;
    each(row, [&](int, float x) {
      if (x > top) {
        if (sum != 0.0) sum *= weight(top, Ref{scale, (double)x}, sh.tab);
        top = x;
      }
      if (x != -INFINITY) sum += weight(x, Ref{scale, (double)top}, sh.tab);      // (a token left out has none, also ahead of a first one)
    });
    Stat st = {top, sum};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) st = join(st, {__shfl_xor_sync(0xffffffffu, st.top, o), __shfl_xor_sync(0xffffffffu, st.sum, o)}, scale, sh.tab);
    return st;
  };
  auto next_child = [&](int node, int after) {      // the node's next child behind `after`, or -1
    for (int j0 = after + 1; j0 < n; j0 += 32) {
      const unsigned hit = __ballot_sync(0xffffffffu, j0 + lane < n && parents[row0 + j0 + lane] == node);
      if (hit) return j0 + __ffs(hit) - 1;
    }
    return -1;
  };

  int node = 0, kept = 1, result = V - 1;
  if (first) path[row0] = 0;
  for (;;) {
    const float* lrow = logits + (size_t)(row0 + node) * V;
    const float* drow = draft ? draft + (size_t)(row0 + node) * V : nullptr;
    int child = next_child(node, node);
    Slot mine = {-INFINITY, -INFINITY, 0.0, 0.0, -1}, all;
    if (greedy) {
      float bv = -INFINITY;
      int bi = -1;
      each(lrow, [&](int i, float x) { if (better(x, i, bv, bi)) { bv = x; bi = i; } });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        if (better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
      }
      if (lane == 0) { sh.top_p[warp] = bv; sh.arg[warp] = bi; }
      __syncthreads();
      if (tid == 0)
        for (int w = 0; w < WARPS; ++w)
          if (better(sh.top_p[w], sh.arg[w], mine.top_p, mine.arg)) { mine.top_p = sh.top_p[w]; mine.arg = sh.arg[w]; }
      exchange(mine, all, false);
      while (child >= 0 && tokens[row0 + child] != all.arg) child = next_child(node, child);
      if (child < 0) {
        result = all.arg;
        break;
      }
      node = child;
      if (first) path[row0 + kept] = node;
      ++kept;
      continue;
    }
    // statistics of the node's rows (the drafter's only where there is a child to try)
    const bool with_q = drow && child >= 0;
    {
      const Stat p = row_stat(lrow), q = with_q ? row_stat(drow) : Stat{-INFINITY, 0.0};
      if (lane == 0) { sh.top_p[warp] = p.top; sh.sum_p[warp] = p.sum; sh.top_q[warp] = q.top; sh.sum_q[warp] = q.sum; }
      __syncthreads();
      if (warp == 0) {
        Stat a = lane < WARPS ? Stat{sh.top_p[lane], sh.sum_p[lane]} : Stat{-INFINITY, 0.0}, b = lane < WARPS ? Stat{sh.top_q[lane], sh.sum_q[lane]} : Stat{-INFINITY, 0.0};
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) {
          a = join(a, {__shfl_xor_sync(0xffffffffu, a.top, o), __shfl_xor_sync(0xffffffffu, a.sum, o)}, scale, sh.tab);
          b = join(b, {__shfl_xor_sync(0xffffffffu, b.top, o), __shfl_xor_sync(0xffffffffu, b.sum, o)}, scale, sh.tab);
        }
        mine = {a.top, b.top, a.sum, b.sum, 0};
      }
    }
    exchange(mine, all, true);
    const Ref rp = {scale, (double)all.top_p}, rq = {scale, (double)all.top_q};
    const double inv_p = 1.0 / all.sum_p;
    double inv_q = with_q ? 1.0 / all.sum_q : 0.0, total = all.sum_p;      // total: the sum over all tokens of what `run` sums over a warp's
    double run = sh.sum_p[warp] == 0.0 ? 0.0 : sh.sum_p[warp] * weight(sh.top_p[warp], rp, sh.tab);
    bool plain = true;                  // the draw goes by p itself (weights not divided by their sum), nothing has been rejected
    int rejected = 0;
    // p and q of a token after `r` rejections
    auto p_after = [&](int i, float x, float d, int r, double& qv) {
      double pv = __dmul_rn(weight(x, rp, sh.tab), inv_p);
      double base = with_q ? weight(d, rq, sh.tab) : 0.0;
      for (int k = 0; k < r; ++k) {
        const bool it = i == sh.token[k];
        const double qk = with_q ? __dmul_rn(base, sh.scale_q[k]) : it ? 1.0 : 0.0;
        pv = __dmul_rn(fmax(__dadd_rn(pv, -qk), 0.0), sh.scale_p[k]);
        if (it) base = 0.0;
      }
      qv = base;      // (not yet divided by its sum)
      return pv;
    };
    bool stands = false;
    while (child >= 0) {
      const int x = tokens[row0 + child];
      const bool ok = x >= 0 && x < V;
      if (!ok && first) atomicOr(err, FZ_ERR_TOKEN_RANGE);
      double qx = 1.0, px = 0.0;
      if (ok) {
        double base;
        px = p_after(x, lrow[x], with_q ? drow[x] : 0.f, rejected, base);
        if (with_q) qx = __dmul_rn(base, inv_q);
      }
      if (uniform[row0 + child] * qx < px) { stands = true; break; }
      // rejected: the sums of what p and q are now
      __syncthreads();      // (nobody still reads the list's last entry)
      if (tid == 0) { sh.token[rejected] = ok ? x : -1; sh.scale_p[rejected] = 1.0; sh.scale_q[rejected] = inv_q; }
      __syncthreads();
      double sp = 0.0, sq = 0.0;
      if (with_q && vec) {
        for (int i = lo + 4 * lane; i < hi; i += 128) {
          const float4 a = *(const float4*)(lrow + i), b = *(const float4*)(drow + i);
          double q0, q1, q2, q3;
          sp += p_after(i, a.x, b.x, rejected + 1, q0); sp += p_after(i + 1, a.y, b.y, rejected + 1, q1);
          sp += p_after(i + 2, a.z, b.z, rejected + 1, q2); sp += p_after(i + 3, a.w, b.w, rejected + 1, q3);
          sq += (q0 + q1) + (q2 + q3);
        }
      } else if (with_q) {
        for (int i = lo + lane; i < hi; i += 32) {
          double qv;
          sp += p_after(i, lrow[i], drow[i], rejected + 1, qv);
          sq += qv;
        }
      } else {
        each(lrow, [&](int i, float v) { double qv; sp += p_after(i, v, 0.f, rejected + 1, qv); });
      }
      sp = warp_sum_d(sp);
      sq = warp_sum_d(sq);
      if (lane == 0) { sh.sum_p[warp] = sp; sh.sum_q[warp] = sq; }
      __syncthreads();
      Slot m2 = {0.f, 0.f, 0.0, 0.0, 0};
      if (tid == 0)
        for (int w = 0; w < WARPS; ++w) { m2.sum_p += sh.sum_p[w]; m2.sum_q += sh.sum_q[w]; }
      exchange(m2, all, false);
      if (all.sum_p > 0.0) {
        total = 1.0;
        plain = false;
        run = sp / all.sum_p;
        if (tid == 0) sh.scale_p[rejected] = 1.0 / all.sum_p;
      } else if (tid == 0) {      // nothing is left: p stays what it was (the rejection had no probability)
        sh.scale_q[rejected] = 0.0;
        if (!with_q) sh.token[rejected] = -1;
      }
      __syncthreads();
      if (with_q) inv_q = all.sum_q > 0.0 ? 1.0 / all.sum_q : 0.0;
      ++rejected;
      child = next_child(node, child);
    }
    if (stands) {
      node = child;
      if (first) path[row0 + kept] = node;
      ++kept;
      continue;
    }
    // the draw: the first token whose running sum, in index order, exceeds u * total. Blocks' runs before this one's first.
    const double target = uniform[row0] * total;
    if (lane == 0) sh.run[warp] = run;
    __syncthreads();
    mine = {0.f, 0.f, 0.0, 0.0, 0};
    if (tid == 0)
      for (int w = 0; w < WARPS; ++w) mine.sum_p += sh.run[w];
    if (tid == 0) sh.slot[turn] = mine;
    if (BLOCKS == 1) __syncthreads();
    else cluster.sync();
    // where the warp's run begins and ends among the running sums: the blocks before, then the warps before, added up the same way by
    // all, so that every end is the next one's beginning
    double blocks = 0.0, part = 0.0, behind = 0.0;
    for (int b = 0; b < BLOCKS; ++b) {
      const double sum = BLOCKS == 1 ? 0.0 : cluster.map_shared_rank(&sh.slot[turn], b)->sum_p;
      if (b < rank) blocks += sum;
      else if (b > rank) behind += sum;
    }
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) part += sh.run[w];
      else if (w > warp) behind += sh.run[w];
    }
    const double before = blocks + part;
    turn ^= 1;
    result = -1;
    // (behind = 0: u so near 1 that the sums' roundings end below the target: the last token that has any probability)
    if (run > 0.0 && before <= target && (blocks + (part + run) > target || behind == 0.0)) {
      double at = before;
      int found = -1, last = -1;
      for (int i0 = lo; i0 < hi && found < 0; i0 += 32) {
        const int i = i0 + lane;
        double w = 0.0, unused;
        if (i < hi) w = plain ? weight(lrow[i], rp, sh.tab) : p_after(i, lrow[i], with_q ? drow[i] : 0.f, rejected, unused);
        double upto = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && at + upto > target), some = __ballot_sync(0xffffffffu, w > 0.0);
        if (hit) found = i0 + __ffs(hit) - 1;
        if (some) last = i0 + 31 - __clz(some);
        at += __shfl_sync(0xffffffffu, upto, 31);
      }
      result = found >= 0 ? found : last;      // (the run's sum, taken in another order, was a little larger)
    }
    break;
  }
  // the block and warp that hold the token, or (a row without a distribution) nobody: V - 1
  if (greedy) {
    if (first) next_ids[s] = result;
  } else {
    const bool mine = __any_sync(0xffffffffu, result >= 0);
    if (lane == 0) sh.arg[warp] = mine ? result : -1;
    __syncthreads();
    Slot out = {0.f, 0.f, 0.0, 0.0, -1};
    if (tid == 0)
      for (int w = 0; w < WARPS; ++w) out.arg = max(out.arg, sh.arg[w]);
    if (tid == 0) sh.slot[turn] = out;
    if (BLOCKS == 1) __syncthreads();
    else cluster.sync();
    if (first) {
      int id = -1;
      for (int b = 0; b < BLOCKS; ++b) id = max(id, BLOCKS == 1 ? sh.slot[turn].arg : cluster.map_shared_rank(&sh.slot[turn], b)->arg);
      next_ids[s] = id >= 0 ? id : V - 1;
    }
  }
  if (first) count[s] = kept;
  if (rank == 0)
    for (int k = kept + tid; k < n; k += THREADS) path[row0 + k] = -1;
  if (BLOCKS > 1) cluster.sync();      // nobody leaves while its slots may still be read
}

template <int BLOCKS>
int launch(const float* logits, const float* draft, const float* temperature, const double* uniform, const int* tokens, const int* parents,
           const int* seg, int S, int N, int V, int* path, int* count, int* next_ids, int* err, cudaStream_t stream) {
  auto kern = verify_kernel<BLOCKS>;
  if (BLOCKS > 8) {
    static const cudaError_t wide = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (wide != cudaSuccess) return (int)wide;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)S * BLOCKS);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (BLOCKS > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = BLOCKS;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (fz_pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, logits, draft, temperature, uniform, tokens, parents, seg, N, V, path, count, next_ids, err);
  return e == cudaSuccess ? FZ_OK : (int)e;
}
}  // namespace

// Blocks per request: as many as the chip holds at once beside the other requests' (14 clusters of eight, 32 of four, 74 of two),
// each with 2,048 tokens and more.
FZ_API int fz_verify_blocks(int S, int V) {
  int b = S <= 14 ? 8 : S <= 32 ? 4 : S <= 74 ? 2 : 1;
  while (b > 1 && V < 2048 * b) b >>= 1;
  return b;
}

// logits, draft (or null): (N, V) float32; temperature (S,); uniform (N,) in [0, 1): a child's own, the root's for the draw;
// tokens, parents (N,): a node's parent within its request's rows (the root, node 0: -1); seg (S, 4) = (first row, rows, ..);
// path (N,): the kept nodes of every request from its first row on, then -1; count (S,); next_ids (S,).
FZ_API int fz_verify_tree(const float* logits, const float* draft, const float* temperature, const double* uniform, const int* tokens,
                          const int* parents, const int* seg, int S, int N, int V, int* path, int* count, int* next_ids, int* err,
                          cudaStream_t stream) {
  if (S <= 0) return FZ_OK;
  if (V <= 0 || N < 0) return FZ_BAD_SHAPE;
  if ((long long)S * 16 > 2147483647LL) return FZ_TOO_LARGE;
#define FZ_V(B_) return launch<B_>(logits, draft, temperature, uniform, tokens, parents, seg, S, N, V, path, count, next_ids, err, stream)
  switch (fz_verify_blocks(S, V)) {
    case 16: FZ_V(16);
    case 8: FZ_V(8);
    case 4: FZ_V(4);
    case 2: FZ_V(2);
    default: FZ_V(1);
  }
#undef FZ_V
}

#ifdef FZ_TIMELINE
FZ_TIMELINE_READER(verify)
#endif
