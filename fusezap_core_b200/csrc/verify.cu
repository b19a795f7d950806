// The verdict on a tree of drafted tokens against the target's logits, from given random numbers: float64's, taken in float32 where that
// cannot differ.
//
// A request's walk starts at its root, the token already chosen. At a node, p = softmax(logits / T) is the target's distribution
// of the next token, q that of the drafter, from which the node's children were drawn one after the other without replacement
// (without a drafter's logits: q puts all on the child). A child x with uniform number u stands if u q(x) < p(x), and the walk goes
// on from it; else p becomes max(p - q, 0) over its sum, q loses x and is scaled to sum 1, and the next child is tried. Where no
// child stands, the next token is drawn from what p is then, so the tokens are distributed as the target's own (recursive
// rejection sampling). T <= 0: the child that is the argmax stands, else the argmax is the next token.
//
// The tokens of a row are shared by the BLOCKS blocks of a cluster, one cluster per request. A walk is a chain of passes over one
// row pair each, ended by one exchange through distributed shared memory, after which all blocks know the sums and take the same
// decisions. Only the rows of nodes that the walk visits are read. The kinds of pass:
//   quick   maximum and sum of p's and q's row, exponentials in float32, once per visited node. Whether a child stands is decided from
//           these sums unless u q(x) lies within MARGIN of p(x); the sums are off by 5e-6 (short rows) to 4e-4 at most (see `quick_chunk`);
//   first   float64, where a child falls, or is too near to call, or the draw is due: the exact sums, and with them at once the sum of
//           max(p - q, 0). That one takes p's and q's exact sums beforehand, which are not known yet: with the quick sums' ratio a0 for
//           a, S(a) = sum max(a p - q, 0) is S(a0) + (a - a0) times the p for which a0 p > q, but for tokens that change sides between a0
//           and a. Those within 2^-19 of their border are therefore left out, and added with the exact a by a second exchange where there
//           are any; where a0 turns out to be off by more than half of that, or a lane has met several, a `next` pass does it. (Taken
//           for good, what changes sides is |a - a0| times its p, with nothing to compare it to: a token that has nearly all of p and q makes the
//           sum wrong by a thousandth, and it scales all that follows.)
//   next    float64, for every further sibling that falls: the sums of the new p and q.
// Sums are kept per warp, whose tokens are one run each, so the last pass before the draw already says in whose run the drawn token
// lies: its block's threads walk that run again, a few neighbouring tokens each. A draw's place among 100,000 running sums needs more
// than 32 bits.
#include "common.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;

namespace {
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int MAX_NODES = 1024;      // nodes of a tree
constexpr float MARGIN = 1e-3f;      // of p(x): a decision nearer than that is taken in float64

constexpr int MOST_TOKENS = 8 << 20;      // of a vocabulary (see `quick_chunk`)

// (Above 1e30: 1e30, where logits of everyday size weigh the same already; times 1 / inf, -inf would be a NaN.)
__device__ __forceinline__ float temperature_of(const float* temperature, int s) {
  const float t = temperature[s];
  return t > 1e30f ? 1e30f : t;
}

// Whether a request has rows, all of them in the step, and no more than a tree may have; else it has no verdict, and no row is its own.
__device__ __forceinline__ bool sound(int row0, int n, int N) { return n > 0 && row0 >= 0 && n <= N - row0 && n <= MAX_NODES; }

struct Ref {      // a row's scale: token x weighs exp((x - top) / T)
  double scale, top;      // 128 log2(e) / T, and the row's maximum
  unsigned far;           // the high word of the difference at which a token would weigh 2^-1015: below it tokens weigh exactly 0
};
constexpr double NOTHING = 1e-290;      // weights and probabilities up to this count as 0

// The token's weight; 1 for x = top exactly. t = 128 log2 of it, k = t rounded, f = t - k, 2^(t / 128) = 2^(k / 128 div 128) *
// table[k mod 128] * 2^(f / 128) (the table-driven method of P. T. P. Tang, 1989), the last by its Taylor polynomial up to f^5 with that term
// economized (C. Lanczos: f^5 / 512 of Chebyshev's fifth polynomial of 2 f left out, which makes the rest of degree four), 8e-17 off. In all
// off by 6e-16 of itself (table, polynomial, their product) and, as any float64 exponential of a quotient, by |ln| of it times 2^-52. The
// degree is what sums of p - q need, where p and q are nearly the same and what is left of them carries their errors whole: one of three
// is 2e-12 off.
// tab: this lane's copy of the table, of which shared memory holds sixteen side by side: the lanes of half a warp, whose k are
// anything, then never meet in a bank (with one copy the reads took as long as all the rest of a pass). A
// row that holds a NaN or +inf is not asked for. Here and where p and q are made from weights the roundings are written out: every place that
// needs a token's p gets the same bits.
// LIFT: tokens too far below for a weight get 2^-1015 or so instead of 0, in fewer instructions (the first pass over 64 x 6 rows of 151,936
// tokens, the whole call: 130 us with exact zeros, 129 like this): for sums that are divided by no less than 1e-6 after it, where that is NOTHING.
constexpr int TABLE = 128, COPIES = 16;
template <bool LIFT = false>
__device__ __forceinline__ double weight(float x, const Ref& r, const double* tab) {
  double d = __dadd_rn((double)x, -r.top);                // 0 or negative, -inf for x = -inf: the larger high word is the lower number
  const bool none = (unsigned)__double2hiint(d) > r.far;
  if (LIFT) d = __hiloint2double((int)min((unsigned)__double2hiint(d), r.far), __double2loint(d));
  const double big = 6755399441055744.0;                  // 1.5 * 2^52: the low bits of the sum are the nearest whole number
  const double shifted = __fma_rn(d, r.scale, big);
  const double f = __fma_rn(d, r.scale, -__dadd_rn(shifted, -big));
  const int k = __double2loint(shifted);
  constexpr double c1 = 0.0054152123481238145, c2 = 1.4662262387640425e-05, c3 = 2.646643357113146e-08, c4 = 3.583032305400251e-11;
  const double e = __dmul_rn(tab[(k & (TABLE - 1)) * COPIES], __fma_rn(f, __fma_rn(f, __fma_rn(f, __fma_rn(f, c4, c3), c2), c1), 1.0));
  const double w = __hiloint2double(__double2hiint(e) + (k & ~(TABLE - 1)) * (1048576 / TABLE), __double2loint(e));
  return !LIFT && none ? 0.0 : w;
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

struct alignas(16) Slot {      // what a block tells the others after a pass
  double sum_p, sum_q, over, under;
  int near;
};
struct alignas(8) Found {     // a node's rows, quick; or the argmax (p.top, arg)
  float top_p, sum_p, top_q, sum_q;
  int arg, bad;      // bad: 1 p's row has no distribution, 2 q's
};

constexpr int CHUNK = 16;      // tokens of a row that a lane has in registers at a time

// A lane's CHUNK tokens of a warp's 32 * CHUNK from i0 on, -inf from hi on: token j is i0 + 4 lane + step(j).
__device__ __forceinline__ constexpr int step(int j) { return 128 * (j >> 2) + (j & 3); }
__device__ __forceinline__ void load_chunk(const float* __restrict__ row, int i0, int hi, bool vec, int lane, float (&x)[CHUNK]) {
  const int at = i0 + 4 * lane;
  if (vec) {
#pragma unroll
    for (int j = 0; j < CHUNK; j += 4) {
      const float4 v = at + step(j) < hi ? *(const float4*)(row + at + step(j)) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      x[j] = v.x, x[j + 1] = v.y, x[j + 2] = v.z, x[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < CHUNK; ++j) x[j] = at + step(j) < hi ? row[at + step(j)] : -INFINITY;
  }
}

__device__ __forceinline__ float quick_exp2(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}

// A row's maximum and sum of weights, quick: float32.
struct Quick { float top, sum; };

// A chunk joins a lane's statistics; its sum goes by its own maximum so far. How far off a sum may be, of itself: a weight 2^-22.5
// (ex2.approx) and four roundings of the exponent t, 4 |t| 2^-24 ln 2, where |t| is log2(V) on average over p (the entropy of p is that
// average plus log2 of the sum, and at most log2(V)): 4e-6; a chunk's addition, and its rescaling where the maximum grew, 4e-7 at most,
// 1,024 chunks (vocabularies of eight million): 4e-4. MARGIN covers both sums. A NaN makes the sum one, +inf the maximum or the sum.
__device__ __forceinline__ void quick_chunk(const float (&x)[CHUNK], Quick& r, float scale2) {
  float m = r.top;
#pragma unroll
  for (int j = 0; j < CHUNK; ++j) m = fmaxf(m, x[j]);
  if (m > r.top) {
    r.sum = r.sum == 0.f ? 0.f : r.sum * quick_exp2((r.top - m) * scale2);
    r.top = m;
  }
  const float from = r.top == -INFINITY ? 0.f : r.top;
  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < CHUNK; ++j) part[j & 3] += quick_exp2((x[j] - from) * scale2);
  r.sum += (part[0] + part[1]) + (part[2] + part[3]);
}

// The statistics of a warp's run of one or two rows.
__device__ __forceinline__ void quick_rows(const float* __restrict__ lrow, const float* __restrict__ drow, int lo, int hi, bool vec, int lane, float scale2,
                                           Quick& p, Quick& q) {
  for (int i0 = lo; i0 < hi; i0 += 32 * CHUNK) {
    float a[CHUNK], b[CHUNK];
    load_chunk(lrow, i0, hi, vec, lane, a);
    if (drow) load_chunk(drow, i0, hi, vec, lane, b);
    quick_chunk(a, p, scale2);
    if (drow) quick_chunk(b, q, scale2);
  }
}

__device__ __forceinline__ bool is_bad(const Quick& r) { return !(r.top < INFINITY) || !(r.sum < INFINITY); }

// The lanes' (the first `width` of them; a power of two) statistics as one, in every one of these lanes.
__device__ __forceinline__ void join_lanes(Quick& r, int width, float scale2) {
  float m = r.top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < width) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float v = r.sum == 0.f ? 0.f : r.sum * quick_exp2((r.top - m) * scale2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < width) v += __shfl_xor_sync(0xffffffffu, v, o);
  r = {m, v};
}

// The quick statistics of all rows ahead of the walks, which then start a node with its rows' sums in hand: a row's slices are evenly
// spread over the SMs, where walks are as long as they are (see `fz_verify_ahead`). stats: (N, slices). A row is p's and, where its node has
// children, q's; of a greedy request the argmax of p's alone.
// One (row, lane < width) each: the joined statistics in every lane.
__device__ __forceinline__ Found join_found(const Found& mine, bool greedy, int width, float scale2) {
  Found r = mine;
  if (greedy) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o >= width) continue;
      const float v = __shfl_xor_sync(0xffffffffu, r.top_p, o);
      const int i = __shfl_xor_sync(0xffffffffu, r.arg, o);
      if (better(v, i, r.top_p, r.arg)) { r.top_p = v; r.arg = i; }
    }
  } else {
    Quick p = {r.top_p, r.sum_p}, q = {r.top_q, r.sum_q};
    r.bad = (int)__reduce_or_sync(0xffffffffu, (unsigned)r.bad);
    join_lanes(p, width, scale2);
    join_lanes(q, width, scale2);
    r.top_p = p.top, r.sum_p = p.sum, r.top_q = q.top, r.sum_q = q.sum;
  }
  return r;
}
__device__ __forceinline__ Found nobody() { return {-INFINITY, 0.f, -INFINITY, 0.f, -1, 0}; }

// A warp's run of a node's rows (drow null: p's alone), joined.
__device__ __forceinline__ Found find_warp(const float* __restrict__ lrow, const float* __restrict__ drow, int lo, int hi, bool vec, int lane, bool greedy,
                                           float scale2) {
  Found r = nobody();
  if (greedy) {
    for (int i0 = lo; i0 < hi; i0 += 32 * CHUNK) {
      float x[CHUNK];
      load_chunk(lrow, i0, hi, vec, lane, x);
#pragma unroll
      for (int j = 0; j < CHUNK; ++j) {
        const int i = i0 + 4 * lane + step(j);
        if (i < hi && better(x[j], i, r.top_p, r.arg)) { r.top_p = x[j]; r.arg = i; }
      }
    }
  } else {
    Quick p = {-INFINITY, 0.f}, q = {-INFINITY, 0.f};
    quick_rows(lrow, drow, lo, hi, vec, lane, scale2, p, q);
    r = {p.top, p.sum, q.top, q.sum, 0, (is_bad(p) ? 1 : 0) | (is_bad(q) ? 2 : 0)};
  }
  return join_found(r, greedy, 32, scale2);
}

// A warp's part of the first exact pass: of p's weights (without token `gone`'s where there is no drafter), q's without it, max(a0 p - q,
// 0), and the p for which that is not 0, these two without the tokens whose a0 p is within 2^-NEAR of q: on which side of a p they lie is
// for the exact a to say. A lane keeps one such token (`at`: the lane's own, -1 for none); near: how many lanes have one, MANY for each that
// has met several.
constexpr int NEAR = 19, MANY = 1 << 16;
struct Part {
  double sum_p, sum_q, over, under;
  int near, at;
};
__device__ __noinline__ Part first_sums(const float* __restrict__ lrow, const float* __restrict__ drow, int lo, int hi, bool vec, int lane, const Ref& rp_,
                                        const Ref& rq_, const double* tab, double a0, int gone) {
  const Ref rp = rp_, rq = rq_;
  double sp = 0.0, sq = 0.0, so = 0.0, su = 0.0;
  int near = 0, at = -1;
  for (int i0 = lo; i0 < hi; i0 += 32 * CHUNK) {
    float a[CHUNK], b[CHUNK];
    load_chunk(lrow, i0, hi, vec, lane, a);
    const int it = gone - i0 - 4 * lane;
    if (drow) {
      load_chunk(drow, i0, hi, vec, lane, b);
      unsigned close = 0;
#pragma unroll
      for (int j = 0; j < CHUNK; ++j) {      // (tokens from hi on weigh nothing)
        const double wp = weight<true>(a[j], rp, tab), wq = weight<true>(b[j], rq, tab), over = fma(a0, wp, -wq);
        sp += wp;
        if (it != step(j)) sq += wq;
        // (high words compare as the numbers do, and 2^-NEAR is a subtraction there; weights below 2^-1004 are never near)
        const bool here = (__double2hiint(over) & 0x7fffffff) <= __double2hiint(wq) - (NEAR << 20);
        if (here) close |= 1u << j;
        if (!here && __double2hiint(over) >= 0) {      // (the sign bit)
          so += over;
          su += wp;
        }
      }
      if (close) {
        at = i0 + 4 * lane + step(__ffs(close) - 1);
        near = near || (close & (close - 1)) ? MANY : 1;
      }
    } else {
#pragma unroll
      for (int j = 0; j < CHUNK; ++j) {
        const double wp = weight<true>(a[j], rp, tab);
        if (it != step(j)) sp += wp;
      }
    }
  }
  return {warp_sum_d(sp), warp_sum_d(sq), warp_sum_d(so), warp_sum_d(su), __reduce_add_sync(0xffffffffu, near), at};
}

// A child that has fallen: its token, 1 / the sum of p after it, 1 / the sum of q before it.
struct Fallen { double scale_p, scale_q; int token; };

// A warp's part of a further pass: p and q after `rejected` children, `p_after` below for four tokens side by side.
__device__ __noinline__ Part next_sums(const float* __restrict__ lrow, const float* __restrict__ drow, int lo, int hi, bool vec, int lane, const Ref& rp_,
                                       const Ref& rq_, const double* tab, double inv_p, const Fallen* fallen, int rejected) {
  const Ref rp = rp_, rq = rq_;
  double sp = 0.0, sq = 0.0;
  for (int i0 = lo; i0 < hi; i0 += 32 * CHUNK) {
    float a[CHUNK], b[CHUNK];
    load_chunk(lrow, i0, hi, vec, lane, a);
    if (drow) load_chunk(drow, i0, hi, vec, lane, b);
#pragma unroll
    for (int j0 = 0; j0 < CHUNK; j0 += 4) {
      double pv[4], qv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        pv[j] = __dmul_rn(weight(a[j0 + j], rp, tab), inv_p);
        qv[j] = drow ? weight(b[j0 + j], rq, tab) : 0.0;
      }
      for (int k = 0; k < rejected; ++k) {
        const int it = fallen[k].token - i0 - 4 * lane;
        const double kp = fallen[k].scale_p, kq = fallen[k].scale_q;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool here = it == step(j0 + j);
          const double qk = drow ? __dmul_rn(qv[j], kq) : here ? 1.0 : 0.0;
          pv[j] = __dmul_rn(fmax(__dadd_rn(pv[j], -qk), 0.0), kp);
          if (here) qv[j] = 0.0;
        }
      }
      sp += (pv[0] + pv[1]) + (pv[2] + pv[3]);
      sq += (qv[0] + qv[1]) + (qv[2] + qv[3]);
    }
  }
  return {warp_sum_d(sp), warp_sum_d(sq), 0.0, 0.0, 0, -1};
}

struct Shared {
  double tab[TABLE * COPIES];
  Slot slot[2], block[16], sums;
  Found found[2], warp_found[WARPS], node_found;
  int who;
  Part part[WARPS];
  double run[WARPS], warp_begin[WARPS + 1], block_begin[17];
  // the request's tree
  double uniform[MAX_NODES];
  int token[MAX_NODES], parent[MAX_NODES];
  Fallen fallen[MAX_NODES];      // the node's children that have fallen
};

constexpr int AHEAD_THREADS = 256, AHEAD_WARPS = AHEAD_THREADS / 32, MAX_SLICES = 32;
__global__ void __launch_bounds__(AHEAD_THREADS)
verify_stats_kernel(const float* __restrict__ logits, const float* __restrict__ draft, const float* __restrict__ temperature,
                    const int* __restrict__ parents, const int* __restrict__ seg, int S, int N, int V, Found* __restrict__ stats) {
  __shared__ Found s_found[AHEAD_WARPS];
  fz_grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  fz_grid_wait();
  const int row = blockIdx.x, slices = gridDim.y;
  int s = -1, row0 = 0, n = 0;
  for (int s0 = 0; s0 < S && s < 0; s0 += 32) {
    const int2 sg = s0 + lane < S ? make_int2(seg[4 * (s0 + lane)], seg[4 * (s0 + lane) + 1]) : make_int2(0, 0);
    const unsigned hit = __ballot_sync(0xffffffffu, sound(sg.x, sg.y, N) && row >= sg.x && row - sg.x < sg.y);
    if (hit) {
      const int who = __ffs(hit) - 1;
      s = s0 + who;
      row0 = __shfl_sync(0xffffffffu, sg.x, who);
      n = __shfl_sync(0xffffffffu, sg.y, who);
    }
  }
  if (s < 0) return;
  const float T = temperature_of(temperature, s);
  const bool greedy = !(T > 0.f);
  bool with_q = false;
  if (draft && !greedy)
    for (int j0 = row - row0 + 1; j0 < n && !with_q; j0 += 32) with_q = __any_sync(0xffffffffu, j0 + lane < n && parents[row0 + j0 + lane] == row - row0);
  const float scale2 = (float)fmin(1.4426950408889634 / (double)T, 3.4e38);
  const int per_warp = ((V + slices * AHEAD_WARPS - 1) / (slices * AHEAD_WARPS) + 3) & ~3;
  const int lo = min(V, ((int)blockIdx.y * AHEAD_WARPS + warp) * per_warp), hi = min(V, lo + per_warp);
  const bool vec = (V & 3) == 0 && (((uintptr_t)logits | (uintptr_t)draft) & 15) == 0;
  const Found mine = find_warp(logits + (size_t)row * V, with_q ? draft + (size_t)row * V : nullptr, lo, hi, vec, lane, greedy, scale2);
  if (lane == 0) s_found[warp] = mine;
  __syncthreads();
  if (warp == 0) {
    const Found all = join_found(lane < AHEAD_WARPS ? s_found[lane] : nobody(), greedy, AHEAD_WARPS, scale2);
    if (lane == 0) stats[(size_t)row * slices + blockIdx.y] = all;
  }
}

template <int BLOCKS>
__global__ void __launch_bounds__(THREADS, 1)
verify_kernel(const float* __restrict__ logits, const float* __restrict__ draft, const float* __restrict__ temperature,
              const double* __restrict__ uniform, const int* __restrict__ tokens, const int* __restrict__ parents,
              const int* __restrict__ seg, int N, int V, int* __restrict__ path, int* __restrict__ count, int* __restrict__ next_ids,
              const Found* __restrict__ stats, int slices, int* err) {
  extern __shared__ __align__(16) unsigned char verify_smem[];
  Shared& sh = *(Shared*)verify_smem;
  cg::cluster_group cluster = cg::this_cluster();
  fz_grid_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int s = blockIdx.x / BLOCKS, rank = blockIdx.x % BLOCKS;
  if (tid < TABLE) {
    const double v = exp2((double)tid / TABLE);
    for (int c = 0; c < COPIES; ++c) sh.tab[tid * COPIES + c] = v;
  }
  const double* tab = sh.tab + lane % COPIES;
  fz_grid_wait();
  const int row0 = seg[4 * s], n = seg[4 * s + 1];
  const float T = temperature_of(temperature, s);
  const bool first = rank == 0 && tid == 0;
  if (!sound(row0, n, N)) {      // (the whole cluster)
    if (first) {
      if (n > 0) atomicOr(err, FZ_ERR_ROW_RANGE);
      count[s] = 0;
      next_ids[s] = -1;
    }
    return;
  }
  for (int i = tid; i < n; i += THREADS) {
    sh.uniform[i] = uniform[row0 + i];
    sh.token[i] = tokens[row0 + i];
    sh.parent[i] = parents[row0 + i];
  }
  __syncthreads();
  const bool greedy = !(T > 0.f);
  const double scale = 184.6649652337873 / (double)T;      // 128 log2(e) / T
  const unsigned far = (unsigned)__double2hiint(-(1015.0 * 0.6931471805599453) * (double)T);
  const float scale2 = (float)fmin(1.4426950408889634 / (double)T, 3.4e38);
  // this warp's run of tokens: [lo, hi), within the block's part of the vocabulary; multiples of four
  const int per_warp = ((V + BLOCKS * WARPS - 1) / (BLOCKS * WARPS) + 3) & ~3;
  const int lo = min(V, (rank * WARPS + warp) * per_warp), hi = min(V, lo + per_warp);
  const bool vec = (V & 3) == 0 && (((uintptr_t)logits | (uintptr_t)draft) & 15) == 0;
  int turn = 0;
  // Every block leaves what it found in a slot of its own; after the barrier the first warp of every block reads all of them (loads from
  // other blocks by all warps would queue: 28 against 16 us for a walk of one request), joins them in the same order everywhere and
  // tells its block. The next exchange writes the other slot.
  auto exchange_sums = [&](const Slot& mine) -> Slot {      // mine: the first warp's
    if (tid == 0) sh.slot[turn] = mine;
    if (BLOCKS > 1) {
      cluster.sync();
      if (warp == 0) {
        Slot r = {0.0, 0.0, 0.0, 0.0, 0};
        if (lane < BLOCKS) sh.block[lane] = r = *cluster.map_shared_rank(&sh.slot[turn], lane);
#pragma unroll
        for (int o = BLOCKS >> 1; o > 0; o >>= 1) {
          r.sum_p += __shfl_xor_sync(0xffffffffu, r.sum_p, o);
          r.sum_q += __shfl_xor_sync(0xffffffffu, r.sum_q, o);
          r.over += __shfl_xor_sync(0xffffffffu, r.over, o);
          r.under += __shfl_xor_sync(0xffffffffu, r.under, o);
          r.near += __shfl_xor_sync(0xffffffffu, r.near, o);
        }
        if (lane == 0) sh.sums = r;
      }
    } else if (tid == 0) {
      sh.block[0] = sh.sums = mine;
    }
    turn ^= 1;
    __syncthreads();
    return sh.sums;
  };
  auto next_child = [&](int node, int after) {      // the node's next child behind `after`, or -1
    for (int j0 = after + 1; j0 < n; j0 += 32) {
      const unsigned hit = __ballot_sync(0xffffffffu, j0 + lane < n && sh.parent[j0 + lane] == node);
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
    // the drafter's row only where there is a child to try; the first child's own values on their way meanwhile
    const bool with_q = drow && child >= 0 && !greedy;
    int x = child >= 0 ? sh.token[child] : 0;
    bool ok = x >= 0 && x < V;
    float lx = ok ? lrow[x] : 0.f, dx = ok && with_q ? drow[x] : 0.f;
    Found all = nobody();
    if (stats) {
      if (lane < slices) all = stats[(size_t)(row0 + node) * slices + lane];
      all = join_found(all, greedy, 32, scale2);
    } else {
      // few requests: the rows of the node that comes next if the first child stands are brought into L2 meanwhile (where requests are
      // many their own loads keep the memory busy)
      if (BLOCKS >= 8 && child >= 0) {
        const bool inner = draft && !greedy && next_child(child, child) >= 0;
        for (int i = lo + 32 * lane; i < hi; i += 32 * 32) {
          asm volatile("prefetch.global.L2 [%0];" ::"l"(logits + (size_t)(row0 + child) * V + i));
          if (inner) asm volatile("prefetch.global.L2 [%0];" ::"l"(draft + (size_t)(row0 + child) * V + i));
        }
      }
      const Found mine = find_warp(lrow, with_q ? drow : nullptr, lo, hi, vec, lane, greedy, scale2);
      if (lane == 0) sh.warp_found[warp] = mine;
      __syncthreads();
      if (warp == 0) {
        Found r = join_found(lane < WARPS ? sh.warp_found[lane] : nobody(), greedy, WARPS, scale2);
        if (lane == 0) (BLOCKS > 1 ? sh.found[turn] : sh.node_found) = r;
      }
      if (BLOCKS > 1) {
        cluster.sync();
        if (warp == 0) {
          Found r = nobody();
          if (lane < BLOCKS) r = *cluster.map_shared_rank(&sh.found[turn], lane);
          r = join_found(r, greedy, BLOCKS, scale2);
          if (lane == 0) sh.node_found = r;
        }
        turn ^= 1;
      }
      __syncthreads();
      all = sh.node_found;
    }
    if (greedy) {
      while (child >= 0 && sh.token[child] != all.arg) child = next_child(node, child);
      if (child < 0) {
        result = all.arg;
        break;
      }
      node = child;
      if (first) path[row0 + kept] = node;
      ++kept;
      continue;
    }
    if ((all.bad & 1) || !(all.sum_p > 0.f)) break;      // a row without a distribution: V - 1
    const bool dead_q = with_q && ((all.bad & 2) || !(all.sum_q > 0.f));      // a drafter's row without one: no child stands, p stays
    const Ref rp = {scale, (double)all.top_p, far}, rq = {scale, (double)all.top_q, far};
    const float near_p = 1.f / all.sum_p, near_q = with_q && !dead_q ? 1.f / all.sum_q : 0.f;      // quick
    double inv_p = 0.0, inv_q = 0.0;      // exact
    // what the draw goes by: a warp's or block's part is (sum_p or over + shift * under) * unit of its sums, the whole 1 or all of p
    double total = 0.0, shift = 0.0, unit = 1.0;
    double own_p = 0.0, own_over = 0.0, own_under = 0.0;
    bool exact = false, stale = false;  // stale: the last pass's sums are not the draw's
    bool by_over = false, plain = true;   // plain: the draw goes by p itself (weights not divided by their sum)
    int rejected = 0;
    // p of a token after `r` rejections, and its q before it is divided by its sum
    auto p_after = [&](int i, float l, float d, int r, double& qv) {
      double pv = __dmul_rn(weight(l, rp, tab), inv_p);
      double base = with_q ? weight(d, rq, tab) : 0.0;
      for (int k = 0; k < r; ++k) {
        const bool it = i == sh.fallen[k].token;
        const double qk = with_q ? __dmul_rn(base, sh.fallen[k].scale_q) : it ? 1.0 : 0.0;
        pv = __dmul_rn(fmax(__dadd_rn(pv, -qk), 0.0), sh.fallen[k].scale_p);
        if (it) base = 0.0;
      }
      qv = base;
      return pv;
    };
    // one exchange of the warps' parts
    auto add_up = [&](const Part& part) {
      if (lane == 0) sh.part[warp] = part;
      __syncthreads();
      Slot mine = {0.0, 0.0, 0.0, 0.0, 0};
      if (warp == 0) {
        const Part z = lane < WARPS ? sh.part[lane] : Part{0.0, 0.0, 0.0, 0.0, 0, -1};
        mine = {warp_sum_d(z.sum_p), warp_sum_d(z.sum_q), warp_sum_d(z.over), warp_sum_d(z.under), __reduce_add_sync(0xffffffffu, z.near)};
      }
      return exchange_sums(mine);
    };
    // The first pass in float64: exact sums, and if a child x has fallen (x = -1: none) the sums of p and q after it. Returns false where
    // the sum of max(p - q, 0) is not to be had this way: too small (p and q nearly the same), more than one token of a lane near its border,
    // or a0 further off than the border's width covers.
    auto first_pass = [&](int gone, float lg, float dg, bool fell) -> bool {
      const double a0 = with_q ? (double)near_p / (double)near_q : 0.0;
      Part mine = first_sums(lrow, with_q ? drow : nullptr, lo, hi, vec, lane, rp, rq, tab, a0, gone);
      Slot sum = add_up(mine);
      const double wg = gone >= 0 ? weight(lg, rp, tab) : 0.0, dgw = gone >= 0 && with_q ? weight(dg, rq, tab) : 0.0;
      const double all_p = with_q ? sum.sum_p : sum.sum_p + wg, all_q = sum.sum_q + dgw;
      inv_p = 1.0 / all_p;
      if (with_q) inv_q = 1.0 / all_q;
      exact = true;
      own_p = mine.sum_p, own_over = mine.over, own_under = mine.under, shift = 0.0, unit = 1.0, total = sum.sum_p, plain = true, by_over = false;
      if (!fell) return true;
      // the list's entry for x; the draw's sums
      double left = 0.0;
      bool good = true;
      if (with_q) {
        double da = all_q / all_p - a0;
        good = fabs(da) <= a0 * (0.5 / (1 << NEAR)) && sum.near < MANY;
        if (good && sum.near > 0) {      // the tokens near the border, now that it is known
          double over = 0.0;
          if (mine.at >= 0) {
            const double wp = weight<true>(lrow[mine.at], rp, tab), wq = weight<true>(drow[mine.at], rq, tab);
            over = fmax(fma(da, wp, fma(a0, wp, -wq)), 0.0);
          }
          mine.over = fma(da, mine.under, mine.over) + warp_sum_d(over);
          mine.under = da = 0.0;
          sum = add_up(mine);
          own_over = mine.over, own_under = 0.0;
        }
        left = (sum.over + da * sum.under) / all_q;
        good = good && left > 1e-6;
        if (good) shift = da, unit = 1.0 / (all_q * left), total = 1.0, plain = false, by_over = true;
      } else if (sum.sum_p > NOTHING) {
        left = sum.sum_p / all_p;
        unit = 1.0 / sum.sum_p, total = 1.0, plain = false;
      } else {
        stale = true;      // (p, all of it on the fallen child, stays what it was)
      }
      if (!good) return false;
      if (tid == 0) {
        sh.fallen[0] = {left > 0.0 ? 1.0 / left : 1.0, inv_q, !with_q && left <= 0.0 ? -1 : gone};
      }
      __syncthreads();
      if (with_q) inv_q = sum.sum_q > NOTHING ? 1.0 / sum.sum_q : 0.0;
      rejected = 1;
      return true;
    };
    // a further pass: child `gone` falls from p and q as `rejected` children have left them
    auto next_pass = [&](int gone, bool fell) {      // (not fell: the sums as they are)
      __syncthreads();      // (nobody still reads the list's last entry)
      if (tid == 0 && fell) sh.fallen[rejected] = {1.0, inv_q, gone};
      __syncthreads();
      if (fell) ++rejected;
      const Part mine = next_sums(lrow, with_q ? drow : nullptr, lo, hi, vec, lane, rp, rq, tab, inv_p, sh.fallen, rejected);
      const Slot left = add_up(mine);
      own_p = mine.sum_p, shift = 0.0, total = 1.0, plain = by_over = false;
      if (!fell) {
        unit = 1.0, total = left.sum_p, stale = false;
        return;
      }
      const int k = rejected - 1;
      stale = !(left.sum_p > NOTHING);      // nothing is left: p stays what it was (the rejection had no probability)
      if (!stale) unit = 1.0 / left.sum_p;
      if (tid == 0) {
        if (!stale) sh.fallen[k].scale_p = unit;
        else sh.fallen[k].scale_q = 0.0;
        if (stale && !with_q) sh.fallen[k].token = -1;
      }
      __syncthreads();
      if (with_q) inv_q = left.sum_q > NOTHING ? 1.0 / left.sum_q : 0.0;
    };
    bool stands = false;
    for (;;) {
      enum { EXACT, FALL_FIRST, FALL_NEXT, RECOUNT } todo = EXACT;
      int gone = -1;
      float lg = 0.f, dg = 0.f;
      if (child < 0 || dead_q) {
        if (exact && !stale) break;      // (the draw's sums are there)
        if (exact) todo = RECOUNT;
      } else {
        if (!ok && first) atomicOr(err, FZ_ERR_TOKEN_RANGE);
        bool sure = true, yes;
        if (!exact && ok) {      // from the quick sums
          const float px = quick_exp2((lx - all.top_p) * scale2) * near_p, qx = with_q ? quick_exp2((dx - all.top_q) * scale2) * near_q : 1.f;
          const float ux = (float)sh.uniform[child] * qx;
          sure = lx == -INFINITY || (px > 1e-30f && fabsf(ux - px) > MARGIN * px);
          yes = ux < px;
        } else {
          double qx = 1.0, px = 0.0, base;
          if (ok) {
            px = p_after(x, lx, dx, rejected, base);
            if (with_q) qx = __dmul_rn(base, inv_q);
          }
          yes = sh.uniform[child] * qx < (px > NOTHING ? px : 0.0);
        }
        if (sure) {
          if (yes) { stands = true; break; }
          todo = exact ? FALL_NEXT : FALL_FIRST;
          if (ok) gone = x, lg = lx, dg = dx;
          child = next_child(node, child);      // (the next child's own values on their way meanwhile)
          x = child >= 0 ? sh.token[child] : 0;
          ok = x >= 0 && x < V;
          lx = ok ? lrow[x] : 0.f, dx = ok && with_q ? drow[x] : 0.f;
        }
      }
      if (todo < FALL_NEXT && !first_pass(gone, lg, dg, todo == FALL_FIRST)) todo = FALL_NEXT;
      if (todo >= FALL_NEXT) next_pass(gone, todo == FALL_NEXT);
    }
    if (stands) {
      node = child;
      if (first) path[row0 + kept] = node;
      ++kept;
      continue;
    }
    // The draw: the first token whose running sum, in index order, exceeds u * total. Where the blocks' runs begin among the running
    // sums, then this block's warps': each end is the next one's beginning, the same number in every block.
    const double target = fmax(sh.uniform[0], 0.0) * total;      // (a NaN: 0)
    if (lane == 0) sh.run[warp] = (by_over ? fmax(fma(shift, own_under, own_over), 0.0) : own_p) * unit;
    __syncthreads();
    if (warp == 0) {
      const Slot b = lane < BLOCKS ? sh.block[lane] : Slot{0.0, 0.0, 0.0, 0.0, 0};
      double run = (by_over ? fmax(fma(shift, b.under, b.over), 0.0) : b.sum_p) * unit;
#pragma unroll
      for (int o = 1; o < BLOCKS; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
      }
      if (lane < BLOCKS) sh.block_begin[lane + 1] = run;
      const double start = __shfl_sync(0xffffffffu, run, (rank + 31) & 31);      // (the block before's end)
      double w = lane < WARPS ? sh.run[lane] : 0.0;
#pragma unroll
      for (int o = 1; o < WARPS; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += v;
      }
      if (lane == 0) sh.block_begin[0] = 0.0, sh.who = -1;
      if (lane < WARPS) sh.warp_begin[lane + 1] = (rank > 0 ? start : 0.0) + w;
      if (lane == 0) sh.warp_begin[0] = rank > 0 ? start : 0.0;
    }
    __syncthreads();
    // the last block that has any probability and begins at or before the target holds the token (u may be so near 1 that the sums'
    // roundings end below the target)
    int holder = 0;
    for (int b = 1; b < BLOCKS; ++b)
      if (sh.block_begin[b] <= target && sh.block_begin[b + 1] - sh.block_begin[b] > NOTHING) holder = b;
    if (holder == rank) {
      // its last such warp; then all threads share that warp's run, a few neighbouring tokens each
      int who = 0;
      for (int w = 1; w < WARPS; ++w)
        if (sh.run[w] > NOTHING && sh.warp_begin[w] <= target) who = w;
      const double begin = sh.warp_begin[who];
      const int from = min(V, (rank * WARPS + who) * per_warp), to = min(V, from + per_warp);
      const int each = (to - from + THREADS - 1) / THREADS, i0 = min(to, from + tid * each), i1 = min(to, i0 + each);
      auto value = [&](int i) {
        double unused;
        const double v = plain ? weight(lrow[i], rp, tab) : p_after(i, lrow[i], with_q ? drow[i] : 0.f, rejected, unused);
        return v > NOTHING ? v : 0.0;
      };
      double mass = 0.0;
      int i = i0;
      for (; i + 4 <= i1; i += 4) {
        const double v0 = value(i), v1 = value(i + 1), v2 = value(i + 2), v3 = value(i + 3);
        mass += (v0 + v1) + (v2 + v3);
      }
      for (; i < i1; ++i) mass += value(i);
      double upto = mass;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      __syncthreads();      // (the runs have been read)
      if (lane == 31) sh.run[warp] = upto;
      __syncthreads();
      if (warp == 0) {
        double w = lane < WARPS ? sh.run[lane] : 0.0;
#pragma unroll
        for (int o = 1; o < WARPS; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, w, o);
          if (lane >= o) w += v;
        }
        if (lane < WARPS) sh.warp_begin[lane + 1] = begin + w;
        if (lane == 0) sh.warp_begin[0] = begin;
      }
      __syncthreads();
      // the last thread that has any and begins at or before the target; its warp walks that thread's tokens together
      const double at = sh.warp_begin[warp] + (upto - mass);
      if (mass > 0.0 && at <= target) atomicMax(&sh.who, tid);
      __syncthreads();
      if (sh.who < 0 && tid == 0) next_ids[s] = V - 1;      // (a run whose sum is the roundings of sums that cancel)
      if (sh.who >= 0 && sh.who >> 5 == warp) {
        const int src = sh.who & 31, t0 = __shfl_sync(0xffffffffu, i0, src), t1 = __shfl_sync(0xffffffffu, i1, src);
        double run = __shfl_sync(0xffffffffu, at, src);
        int found = -1, last = -1;
        for (int t = t0; t < t1 && found < 0; t += 32) {
          const double v = t + lane < t1 ? value(t + lane) : 0.0;
          double w = v;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
          }
          const unsigned hit = __ballot_sync(0xffffffffu, v > 0.0 && run + w > target), some = __ballot_sync(0xffffffffu, v > 0.0);
          if (hit) found = t + __ffs(hit) - 1;
          if (some) last = t + 31 - __clz(some);
          run += __shfl_sync(0xffffffffu, w, 31);
        }
        if (lane == 0) next_ids[s] = found >= 0 ? found : last;
      }
    }
    result = -1;      // (written)
    break;
  }
  if (first) {
    if (result >= 0) next_ids[s] = result;
    count[s] = kept;
  }
  if (rank == 0)
    for (int k = kept + tid; k < n; k += THREADS) path[row0 + k] = -1;
  if (BLOCKS > 1) cluster.sync();      // nobody leaves while its slots may still be read
}

template <int BLOCKS>
int launch(const float* logits, const float* draft, const float* temperature, const double* uniform, const int* tokens, const int* parents,
           const int* seg, int S, int N, int V, int* path, int* count, int* next_ids, const Found* stats, int slices, int* err, cudaStream_t stream) {
  auto kern = verify_kernel<BLOCKS>;
  FZ_RAISE_SMEM(kern);
  if (BLOCKS > 8) {
    static const cudaError_t wide = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (wide != cudaSuccess) return (int)wide;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)S * BLOCKS);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = sizeof(Shared);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, logits, draft, temperature, uniform, tokens, parents, seg, N, V, path, count, next_ids, stats, slices, err);
  return e == cudaSuccess ? FZ_OK : (int)e;
}
}  // namespace

// Blocks per request: as many as the chip holds at once beside the other requests' (8 clusters of sixteen, 14 of eight, 32 of four, 74 of
// two), each with 2,048 tokens and more. us at 128,256 tokens with 2, 4, 8 and 16 blocks: one request with 5 nodes 28, 21, 18, 17; 8 with 16
// 131, 76, 54, 44; 64 with 6 at 151,936 tokens 129, 145, 182, 265.
FZ_API int fz_verify_blocks(int S, int V) {
  int b = S <= 8 ? 16 : S <= 14 ? 8 : S <= 32 ? 4 : S <= 74 ? 2 : 1;
  while (b > 1 && V < 2048 * b) b >>= 1;
  return b;
}

// Slices of a row whose quick statistics a kernel of its own takes ahead of the walks (0: none; the scratch: N * slices * 24 bytes).
// It reads rows that no walk visits, but all SMs share it evenly, while walks differ in length: it pays where trees are small, two to six
// nodes on average (us without and with it, a drafter's logits throughout: 64 chains of up to 6 nodes over 151,936 tokens 141 and 129, 16 of
// 8 over 128,256 83 and 59; 30 trees of 10 73 and 107, 8 of 16 43 and 64; single nodes, 64 of them 32 and 37).
FZ_API int fz_verify_ahead(int S, int N, int V) {
  if (N < 2 * S || N > 6 * S) return 0;
  int slices = (8 * 148 + N - 1) / N;
  if (slices > MAX_SLICES) slices = MAX_SLICES;
  while (slices > 1 && V < 4096 * slices) --slices;
  return slices;
}

// logits, draft (or null): (N, V) float32; temperature (S,); uniform (N,) in [0, 1): a child's own, the root's for the draw;
// tokens, parents (N,): a node's parent within its request's rows (the root, node 0: -1); seg (S, 4) = (first row, rows, ..);
// path (N,): the kept nodes of every request from its first row on, then -1; count (S,); next_ids (S,). scratch: as `fz_verify_ahead`
// says, 8-byte aligned.
FZ_API int fz_verify_tree(const float* logits, const float* draft, const float* temperature, const double* uniform, const int* tokens,
                          const int* parents, const int* seg, int S, int N, int V, int* path, int* count, int* next_ids, void* scratch, int slices,
                          int* err, cudaStream_t stream) {
  static_assert(sizeof(Found) == 24, "what callers size the scratch by");
  if (S <= 0) return FZ_OK;
  if (V <= 0 || N < 0 || slices < 0 || slices > MAX_SLICES || (slices > 0 && !scratch)) return FZ_BAD_SHAPE;
  if ((uintptr_t)scratch & 7) return FZ_BAD_ALIGNMENT;
  if ((long long)S * 16 > 2147483647LL || V > MOST_TOKENS) return FZ_TOO_LARGE;
  Found* stats = slices > 0 ? (Found*)scratch : nullptr;
  if (stats && N > 0) {
    const cudaError_t e = fz_launch(verify_stats_kernel, dim3((unsigned)N, (unsigned)slices), dim3(AHEAD_THREADS), 0, stream, logits, draft, temperature,
                                    parents, seg, S, N, V, stats);
    if (e != cudaSuccess) return (int)e;
  }
#define FZ_V(B_) return launch<B_>(logits, draft, temperature, uniform, tokens, parents, seg, S, N, V, path, count, next_ids, stats, slices, err, stream)
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
