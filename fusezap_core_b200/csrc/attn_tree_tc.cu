// The cached context of drafted trees (see attn_tree.cu) on the 5th-generation tensor cores, bf16.
//
// A tile's 128 rows are the 128 TMEM lanes: NB = 128 / G nodes of one request times the G query heads of one kv head, so keys
// and values are fetched once for all of them. Work is counted in units, a key tile of 128 places for one (request, kv head, row
// tile) item; the persistent grid has one block per SM and every block takes an equal run of the units, whatever the requests'
// lengths: a run cuts items where it must, at most one at either end. Each stretch of an item leaves unnormalised rows and
// (maximum, sum) in float32 scratch, from scratch row 128 * block + the rows of the items before (both rise along the runs, and an
// item has 128 rows at most, so no two stretches overlap); the merge kernel finds a row's stretches by a record. Nothing is planned on the host and no launch size depends on the requests'
// lengths. (The cuts follow from all requests of the step together: a row's last bits may depend on its neighbours.)
// Bound by HBM up to about 128 rows per kv head: 64 KB of keys and values per unit at head size 128, 1.5 us of an SM's share of
// the bandwidth, against 1,024 clocks of MMA and as many of exponentials. Blocks of 19 warps:
//   warps 0, 18 TMA producers: warp 0 queries and keys, warp 18 values (a page's rows of one kv head are boxes of the pool seen as a
//               2-D array of rows, 128-byte swizzle), each into a ring of its own, as far ahead as the ring allows;
//   warp 1      one lane issues tcgen05.mma. The tiles of a run alternate between two streams, each with its own scores, weights and
//               output in tensor memory and its own eight softmax warps, so that one stream's exponentials run beside the other's products:
//               S = Q K^T (128 x 128 x hd), then, once the weights P are written over the scores, O += P V and the stream's next S;
//   warps 2..17 softmax, two threads per row and stream, 64 columns each: online in the exp2 domain, float32 maximum and sum, P as
//               bf16 (half a step, 2^-8 of a weight: the tensor core's operand type); O is rescaled in tensor memory only where a row's
//               maximum has grown by more than 2^8. At a stretch's end the two streams' results are joined, four threads a row. Warps
//               whose rows are all padding only keep the barriers going.
// All rows of a request see the same places [a, b) here (with a window: those that every row sees, from first place + nodes -
// window on; the merge kernel walks the few before), so scores are masked in the first and last tile alone, and value rows
// outside [a, b) never meet the tensor core: products take whole groups of 16 places, and a group cut by an end is filled by the
// producer's lanes, zeros outside. What a page holds beside the context therefore does not matter.
// Waits are bounded; a wait that gives up sets the error bit. No multicast.
#include "attn_tree.cuh"
#include "umma.cuh"

namespace {
using namespace fztree;
using namespace fztma;
using namespace fzumma;

constexpr int BM = 128, BN = 128, THREADS = 608;
constexpr float RESCALE_STEP = 8.f;

// The warp that issues MMAs runs together, with values that are the same in all lanes, and one lane's instruction counts (`lead`): the
// operands of an MMA are then computed once for the warp. Inside a branch of one lane every operand is moved there for every
// instruction, and issuing 8 + 8 MMAs per key tile took longer than fetching the tile: a request of 27 nodes behind 30,000 places 43 us, 64
// requests of 6 behind 4,096 165, 4 of 64 behind 12,000 91, like this 37, 151 and 73.
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      ::"r"(smem_u32(bar)), "r"(lead) : "memory");
}
__device__ __forceinline__ int same(int v) { return __shfl_sync(0xffffffffu, v, 0); }      // a value that is the same in all lanes, known to be

// The context places of a request that the units cover, in key tiles, and its row tiles.
__host__ __device__ __forceinline__ void request_units(int n, int start, int window, int NB, int& a, int& tiles, int& row_tiles) {
  a = window > 0 ? max(0, start + n - window) : 0;
  tiles = n > 0 && a < start ? (start + BN - 1) / BN - a / BN : 0;
  row_tiles = n > 0 ? (n + NB - 1) / NB : 0;
}

struct Sizes {
  const int* seg;
  int S, NB, Hkv, window, N;
  long long places;      // of a block table
};

// A block's share of an item: `count` key tiles of the places [a, b) from place `key0` on, for `rows` (node, head) rows from row `row` on.
// before: (node, head) rows of the items before it; stretches: how many the item has in all where this is its first, else 0.
struct Stretch {
  int s, kvh, row, rows, key0, count, a, b, before, stretches;
};
constexpr int RING = 8;      // stretches that the key producer may be ahead of the others' reading (the queries' one buffer keeps it within four)

// The walk of a block over its run of units, one stretch at a time, by the warp that fetches queries and keys; it leaves every stretch in
// shared memory for the other roles, ahead of its data (each role walking by itself took 2 us of the softmax warps' time between two requests,
// and their registers). Requests are looked up only where the run crosses from one to the next; within a request the next item
// follows by counting.
struct Walk {
  int G, u, u1;                                    // the next unit, the run's end
  int s, n, row0, a, b, tiles, row_tiles;          // the request
  int end, nodes_before;                           // its last unit + 1, nodes of the requests before it
  int chunk, chunk_units, chunk_nodes;             // where the look-up goes on: 32 requests from `chunk`, units and nodes before them
  int kvh, rt;                                     // the item

  // Sum of all requests' units.
  static __device__ __forceinline__ int sum(const Sizes& Z) {
    const int lane = threadIdx.x & 31;
    int total = 0;
    for (int s = lane; s < Z.S; s += 32) {
      int a, tiles, row_tiles;
      const int* e = Z.seg + 4 * s;
      const int start = e[2];
      request_units(sound_nodes(e[0], e[1], start, Z.N, Z.places), start, Z.window, Z.NB, a, tiles, row_tiles);
      total += Z.Hkv * row_tiles * tiles;
    }
    return __reduce_add_sync(0xffffffffu, total);
  }
  // The request that holds unit u, and the item and tile within it.
  __device__ __forceinline__ void find(const Sizes& Z) {
    const int lane = threadIdx.x & 31;
    int units = chunk_units, nodes = chunk_nodes;
    for (int s0 = chunk; s0 < Z.S; s0 += 32) {
      int nn = 0, bb = 0, rr = 0, aa = 0, tt = 0, rt_ = 0;
      if (s0 + lane < Z.S) {
        const int* e = Z.seg + 4 * (s0 + lane);
        rr = e[0], bb = e[2], nn = sound_nodes(rr, e[1], bb, Z.N, Z.places);
        request_units(nn, bb, Z.window, Z.NB, aa, tt, rt_);
      }
      const int mine_u = Z.Hkv * rt_ * tt;
      int iu = mine_u, in = nn;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, iu, o), y = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) { iu += x; in += y; }
      }
      const unsigned hit = __ballot_sync(0xffffffffu, units + iu > u);
      if (hit) {
        const int who = __ffs(hit) - 1;
        chunk = s0, chunk_units = units, chunk_nodes = nodes;
        s = s0 + who;
        n = __shfl_sync(0xffffffffu, nn, who), b = __shfl_sync(0xffffffffu, bb, who), row0 = __shfl_sync(0xffffffffu, rr, who);
        a = __shfl_sync(0xffffffffu, aa, who), tiles = __shfl_sync(0xffffffffu, tt, who), row_tiles = __shfl_sync(0xffffffffu, rt_, who);
        end = units + __shfl_sync(0xffffffffu, iu, who);
        const int begin = end - __shfl_sync(0xffffffffu, mine_u, who);
        nodes_before = nodes + __shfl_sync(0xffffffffu, in - nn, who);
        const int within = u - begin, k = within / tiles;
        kvh = k / row_tiles;
        rt = k - kvh * row_tiles;
        tile = within - k * tiles;
        return;
      }
      units += __shfl_sync(0xffffffffu, iu, 31);
      nodes += __shfl_sync(0xffffffffu, in, 31);
    }
  }
  int tile;      // the stretch's first within its item
  // The next stretch; false at the run's end. share: units per block.
  __device__ __forceinline__ bool next(const Sizes& Z, int share, Stretch& x) {
    if (u >= u1) return false;
    if (u >= end) {
      find(Z);
    } else {
      tile = 0;
      if (++rt == row_tiles) rt = 0, ++kvh;
    }
    const int node0 = rt * Z.NB, count = min(tiles - tile, u1 - u);
    x = {s, kvh, row0 + node0, min(Z.NB, n - node0) * G, (a / BN + tile) * BN, count, a, b,
         (nodes_before * Z.Hkv + kvh * n + node0) * G,
         tile == 0 ? (u + tiles - 1) / share - u / share + 1 : 0};
    u += count;
    return true;
  }
};

template <int HD, int BOX>
__global__ void __launch_bounds__(THREADS, 1)
attn_tree_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const __nv_bfloat16* __restrict__ v_pool,
                    const Sizes Z, const int* __restrict__ table, int mb, int page_size, int num_pages, int Hq, float scale_log2,
                    int N, float* __restrict__ part_o, float* __restrict__ part_ml, int2* __restrict__ records, int* err) {
  constexpr int HALVES = HD / 64;                     // 64-column halves of a head
  constexpr int STAGES = HD <= 64 ? 6 : 3;            // key tiles and value tiles in flight
  constexpr int HALF_BYTES = 128 * 128;               // 128 rows of 128 bytes
  constexpr int Q_BYTES = HALVES * HALF_BYTES, KV_BYTES = HALVES * HALF_BYTES;
  constexpr int TMEM_COLS = 512;                      // S0 / P0: 0.., S1 / P1: 128.., O0: 256.., O1: 256 + HD..
  constexpr int OPS = (BN / BOX) * HALVES;            // TMA boxes per key tile, for K and again for V
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t s_q = smem_u32(smem), s_k = s_q + Q_BYTES, s_v = s_k + STAGES * KV_BYTES;
  float* s_mx = (float*)(smem + Q_BYTES + 2 * STAGES * KV_BYTES);      // [stream][half][128 rows]
  uint64_t* q_full = (uint64_t*)(s_mx + 4 * BM);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;          // STAGES each
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* s_ready = v_empty + STAGES;    // one per stream
  uint64_t* p_ready = s_ready + 2;
  uint64_t* o_ready = p_ready + 2;
  uint64_t* listed = o_ready + 2;          // RING: stretch j stands in ring[j % RING]
  Stretch* ring = (Stretch*)(listed + RING);
  uint32_t* tmem_slot = (uint32_t*)(ring + RING);
  int* flag = (int*)(tmem_slot + 1);

  const int tid = threadIdx.x, warp = same(tid >> 5), lane = tid & 31;
  if (s_q & 1023u) {      // (the swizzle needs it; the declaration asks for it)
    fz_grid_wait();
    if (tid == 0) atomicOr(err, FZ_ERR_WAIT_TIMEOUT);
    return;
  }
  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_ready[i], 1);
      mbar_init(&p_ready[i], 256);
      mbar_init(&o_ready[i], 1);
    }
    for (int i = 0; i < RING; ++i) mbar_init(&listed[i], 1);
    flag[0] = 0;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(tmem_slot, TMEM_COLS);
  // (brought into L2 ahead of the wait on the kernel before; read behind it)
  if (warp == 2)
    for (int i = lane * 8; i < Z.S; i += 256) asm volatile("prefetch.global.L2 [%0];" ::"l"(Z.seg + 4 * i));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = (uint32_t)same((int)*tmem_slot);
  fz_grid_launch_dependents();
  fz_grid_wait();
  const int G = Hq / Z.Hkv;
  const int total = Walk::sum(Z), share = (total + gridDim.x - 1) / gridDim.x;
  const int u0 = min(total, (int)blockIdx.x * share), u1 = min(total, u0 + share);
  // Every role goes through the same stretches and counts the key tiles it has gone through (`g`, up to u1 - u0): ring stages, streams and
  // barrier phases follow from that count and carry over from one stretch to the next.
  bool ok = true;
  Stretch x;
  auto read = [&](int j) -> bool {      // stretch number j, once the key producer has listed it
    if (!__all_sync(0xffffffffu, mbar_wait(&listed[j % RING], (j / RING) & 1))) return false;
    x = ring[j % RING];
    return true;
  };

  if (warp == 0 || warp == 18) {
    // ---------------- producers
    const bool is_v = warp == 18;
    const int rows_per_page = 2 * Z.Hkv * page_size;
    int g = 0, n_q = 0;
    Walk walk;
    walk.G = G, walk.u = u0, walk.u1 = u1, walk.end = walk.chunk = walk.chunk_units = walk.chunk_nodes = 0;
    while (ok && g < u1 - u0) {
      if (is_v) {
        if (!(ok = read(n_q++))) break;
      } else {
        walk.next(Z, share, x);
        if (lane == 0) {
          ring[n_q % RING] = x;
          mbar_arrive(&listed[n_q % RING]);
        }
        // the one Q buffer is free once the last score product of the stretch before is done
        if (n_q > 0) ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (n_q - 1) & 1));
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(q_full, Z.NB * G * 128 * HALVES);
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf)
            asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                         ::"r"(s_q + hf * HALF_BYTES), "l"(&q_map), "r"(smem_u32(q_full)), "r"(64 * hf), "r"(x.kvh * G), "r"(x.row) : "memory");
        }
        ++n_q;
      }
      const int* trow = table + (size_t)x.s * mb;
      for (int t = 0; t < x.count && ok; ++t, ++g) {
        const int s = g % STAGES, round = g / STAGES;
        const int key0 = x.key0 + t * BN;
        // op -> (page box, column half). Keys: boxes with any place of [a, b). Values: boxes of groups of 16 places that lie in it whole.
        int op_row[(OPS + 31) / 32];
        uint32_t bytes = 0;
#pragma unroll
        for (int j = 0; j < (OPS + 31) / 32; ++j) {
          const int op = lane + 32 * j;
          op_row[j] = -1;
          if (op < OPS) {
            const int key = key0 + (op / HALVES) * BOX, group = key & ~15;
            if (is_v ? group >= x.a && group + 16 <= x.b : key + BOX > x.a && key < x.b) {
              const int pi = key / page_size;
              const int page = pi < mb ? trow[pi] : -1;
              if (page >= 0 && page < num_pages) op_row[j] = page * rows_per_page + (is_v ? Z.Hkv * page_size : 0) + x.kvh * page_size + (key - pi * page_size);
              else if (!is_v) atomicOr(err, FZ_ERR_NO_PAGE);
            }
          }
          bytes += op_row[j] >= 0 ? BOX * 128u : 0u;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) bytes += __shfl_xor_sync(0xffffffffu, bytes, o);
        uint64_t* full = is_v ? &v_full[s] : &k_full[s];
        uint64_t* empty = is_v ? &v_empty[s] : &k_empty[s];
        if (round > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty, (round - 1) & 1));
        if (!ok) break;
        const uint32_t dst = (is_v ? s_v : s_k) + s * KV_BYTES, bar = smem_u32(full);
        if (is_v) {
          // the groups that an end of [a, b) cuts: by hand, zeros for the places outside
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int end = e ? x.b : x.a, group = end & ~15;
            if ((end & 15) == 0 || group < key0 || group >= key0 + BN || (e && group < x.a)) continue;      // (both ends in one group: filled once)
            for (int c = lane; c < 16 * HD / 8; c += 32) {
              const int row = c / (HD / 8), chunk = c - row * (HD / 8), key = group + row;
              uint4 v = make_uint4(0u, 0u, 0u, 0u);
              if (key >= x.a && key < x.b) {
                const int pi = key / page_size;
                const int page = pi < mb ? trow[pi] : -1;
                if (page >= 0 && page < num_pages)
                  v = *(const uint4*)(v_pool + ((long long)page * rows_per_page + x.kvh * page_size + (key - pi * page_size)) * HD + chunk * 8);
              }
              const int r = key - key0, hf = chunk >> 3, col = chunk & 7;
              const uint32_t at = dst + hf * HALF_BYTES + r * 128 + ((col ^ (r & 7)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        if (lane == 0) mbar_expect_tx(full, bytes);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < (OPS + 31) / 32; ++j) {
          const int op = lane + 32 * j;
          if (op < OPS && op_row[j] >= 0) tma_load_2d_u32(dst + (op % HALVES) * HALF_BYTES + (op / HALVES) * BOX * 128, &kv_map, bar, 64 * (op % HALVES), op_row[j]);
        }
      }
    }
    if (!ok && lane == 0) flag[0] = 1;
  } else if (warp == 1) {
    // ---------------- MMA issuer (the warp goes through the stretches together, lane 0's instructions count)
    constexpr uint32_t idesc_s = make_idesc(BM, BN, false), idesc_pv = make_idesc(BM, HD, true);
    const uint32_t lead = lane == 0;
    // The scores run two tiles ahead of the products with the values: two walks over the same stretches.
    int st = 0, sg = 0, n_q = 0, scores = 0;   // the score walk: tile within its stretch, tiles so far, stretches so far, tiles of its stretch
    auto issue_s = [&]() -> bool {             // S(sg) = Q K(sg)^T into the scores of stream sg & 1; frees the key stage when done
      if (st == 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&listed[n_q % RING], (n_q / RING) & 1))) return false;
        scores = same(ring[n_q % RING].count);
        if (!__all_sync(0xffffffffu, mbar_wait(q_full, n_q & 1))) return false;
      }
      const int s = sg % STAGES;
      if (!__all_sync(0xffffffffu, mbar_wait(&k_full[s], (sg / STAGES) & 1))) return false;
      tc_fence_after();
      const uint32_t tmem_s = tmem_base + (uint32_t)(sg & 1) * 128u;
      const uint64_t dq = desc_k_major(s_q), dk = desc_k_major(s_k + s * KV_BYTES);
#pragma unroll
      for (int i = 0; i < 4 * HALVES; ++i) {      // 16 dimensions each: 32 bytes along a half's rows
        const uint64_t step = (uint64_t)((i >> 2) * (HALF_BYTES >> 4) + 2 * (i & 3));
        mma_ss(lead, tmem_s, dq + step, dk + step, idesc_s, i ? 1u : 0u);
      }
      mma_commit(lead, &s_ready[sg & 1]);
      mma_commit(lead, &k_empty[s]);
      if (st + 1 == scores) mma_commit(lead, q_empty);      // the stretch's last score product: Q may be overwritten when it is done
      ++sg;
      if (++st == scores) {
        st = 0;
        ++n_q;
      }
      return true;
    };
    int g = 0, n_x = 0;
    for (int i = 0; i < 2 && ok && sg < u1 - u0; ++i) ok = issue_s();
    while (ok && g < u1 - u0) {
      if (!(ok = read(n_x++))) break;
      const int xa = same(x.a), xb = same(x.b), xkey0 = same(x.key0), xcount = same(x.count);
      for (int t = 0; t < xcount && ok; ++t, ++g) {
        const int s = g % STAGES, tq = g & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[s], (g / STAGES) & 1) && mbar_wait(&p_ready[tq], (g >> 1) & 1));      // P(g) written, O rescaled if it had to be
        if (!ok) break;
        tc_fence_after();
        const uint32_t tmem_p = tmem_base + (uint32_t)tq * 128u, tmem_o = tmem_base + 256u + (uint32_t)(tq * HD);
        const int key0 = xkey0 + t * BN;
        const int k0 = max(0, (xa - key0) >> 4), k1 = min(BN / 16, (xb - key0 + 15) >> 4);      // groups with places of [a, b)
        // (P: the first 64 places over score columns 0..31, the others over 64..95; V: 16 places are 2,048 bytes, 128 in a descriptor)
        const uint64_t dv = desc_mn_major(s_v + s * KV_BYTES, HALF_BYTES);
        if (k0 == 0 && k1 == BN / 16) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            mma_ts(lead, tmem_o, tmem_p + (uint32_t)(kk < 4 ? 8 * kk : 64 + 8 * (kk - 4)), dv + (uint64_t)(128 * kk), idesc_pv, (t >= 2 || kk > 0) ? 1u : 0u);
        } else {
          for (int kk = k0; kk < k1; ++kk)
            mma_ts(lead, tmem_o, tmem_p + (uint32_t)(kk < 4 ? 8 * kk : 64 + 8 * (kk - 4)), dv + (uint64_t)(128 * kk), idesc_pv, (t >= 2 || kk > k0) ? 1u : 0u);
        }
        if (t + 2 >= xcount) mma_commit(lead, &o_ready[tq]);      // the stream's last of the stretch
        mma_commit(lead, &v_empty[s]);
        if (sg < u1 - u0) ok = issue_s();      // the stream's next scores go behind the product that reads its P
      }
    }
    if (!ok && lane == 0) flag[0] = 1;
  } else {
    // ---------------- softmax: warps 2..9 stream 0, warps 10..17 stream 1; two threads per row
    constexpr int OD = HD / 2, JD = HD / 4;      // output dimensions per thread: of its stream's rescaling, of the joined result
    const int idx = warp - 2, tq = idx >> 3, hf = (idx >> 2) & 1, quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t lane_sel = (uint32_t)(quad * 32) << 16;
    const uint32_t t_s = tmem_base + (uint32_t)(tq * 128 + hf * 64) + lane_sel;    // this thread's 64 scores; its P over the first 32 columns
    const uint32_t t_o = tmem_base + 256u + (uint32_t)(tq * HD + hf * OD) + lane_sel;
    const int pair_bar = 1 + tq * 4 + quad, quad_bar = 9 + quad;
    float* mx_mine = s_mx + (tq * 2 + hf) * BM + r;
    const float* mx_other = s_mx + (tq * 2 + (hf ^ 1)) * BM + r;
    int g0 = 0, n_x = 0, n_s = 0, n_o[2] = {0, 0};      // tiles of the block, of this stream, and stretches with tiles of either stream so far
    while (ok && g0 < u1 - u0) {
      if (!(ok = read(n_x++))) break;
      // where the item's rows will find their stretches, from the block that has its first: (scratch row of the first, stretches)
      if (x.stretches > 0 && idx == 0) {
        for (int i = lane; i < x.rows / G; i += 32)
          records[(size_t)(x.row + i) * Z.Hkv + x.kvh] = make_int2(blockIdx.x * BM + x.before, x.stretches);
      }
      const bool live = quad * 32 < x.rows;      // (the warp has rows)
      const int first = (g0 ^ tq) & 1;           // the first tile of the stretch that is this stream's
      float m_run = -INFINITY, l_part = 0.f;     // the maximum in use (exp2 domain) and this thread's half of the row's sum
      for (int t = first; t < x.count && ok; t += 2) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_ready[tq], n_s & 1));
        if (!ok) break;
        ++n_s;
        if (!live) {
          mbar_arrive(&p_ready[tq]);
          continue;
        }
        tc_fence_after();
        const int key0 = x.key0 + t * BN + hf * 64;
        const bool full = key0 >= x.a && key0 + 64 <= x.b;
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          tmem_ld32(t_s + (uint32_t)c, v);
          if (!full) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = key0 + c + j >= x.a && key0 + c + j < x.b ? v[j] : -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            mx4[0] = fmax3(mx4[0], v[j], v[j + 1]); mx4[1] = fmax3(mx4[1], v[j + 2], v[j + 3]);
            mx4[2] = fmax3(mx4[2], v[j + 4], v[j + 5]); mx4[3] = fmax3(mx4[3], v[j + 6], v[j + 7]);
          }
        }
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        *mx_mine = mx;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        mx = fmaxf(mx, *mx_other);
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");    // both have read: the slots may be written again
        // (the stream's last P V product is complete: the scores just waited for were issued behind it)
        const float m_new = fmaxf(m_run, mx * scale_log2);
        const bool grow = m_new > m_run + RESCALE_STEP;
        if (__any_sync(0xffffffffu, grow)) {
          const float corr = grow ? fast_exp2(m_run - m_new) : 1.f;
          if (t >= 2) {
            const float2 c2 = make_float2(corr, corr);
#pragma unroll
            for (int c = 0; c < OD; c += 32) {
              float ov[32];
              tmem_ld32(t_o + (uint32_t)c, ov);
              uint32_t ow[32];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float2 sc = __fmul2_rn(make_float2(ov[2 * j], ov[2 * j + 1]), c2);
                ow[2 * j] = __float_as_uint(sc.x);
                ow[2 * j + 1] = __float_as_uint(sc.y);
              }
              tmem_st32(t_o + (uint32_t)c, ow);
            }
          }
          if (grow) {
            l_part *= corr;
            m_run = m_new;
          }
        }
        const float mu = m_run == -INFINITY ? 0.f : m_run;
        const float2 sc2 = make_float2(scale_log2, scale_log2), nmu2 = make_float2(-mu, -mu);
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          float v[32];
          tmem_ld32(t_s + (uint32_t)c, v);
          uint32_t w[16];
          if (full) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 z = __ffma2_rn(make_float2(v[2 * j], v[2 * j + 1]), sc2, nmu2);
              const float2 e = ((0x52u >> (j & 7)) & 1u) ? exp2_fma2(z) : make_float2(fast_exp2(z.x), fast_exp2(z.y));      // 3 pairs in 8
              sum2[j & 1] = __fadd2_rn(sum2[j & 1], e);
              const __nv_bfloat162 pk = __floats2bfloat162_rn(e.x, e.y);
              w[j] = *(const uint32_t*)&pk;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int key = key0 + c + 2 * j;
              const float s0 = key >= x.a && key < x.b ? v[2 * j] : -INFINITY, s1 = key + 1 >= x.a && key + 1 < x.b ? v[2 * j + 1] : -INFINITY;
              const float2 z = __ffma2_rn(make_float2(s0, s1), sc2, nmu2);
              const float2 e = make_float2(fast_exp2(z.x), fast_exp2(z.y));
              sum2[j & 1] = __fadd2_rn(sum2[j & 1], e);
              const __nv_bfloat162 pk = __floats2bfloat162_rn(e.x, e.y);
              w[j] = *(const uint32_t*)&pk;
            }
          }
          tmem_st16(t_s + (uint32_t)(c >> 1), w);
        }
        l_part += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
        tc_fence_before();
        mbar_arrive(&p_ready[tq]);
      }
      if (!ok) break;
      // the stretch's end: both streams' last products, then the two results joined, a quarter of the dimensions per thread
      const bool has[2] = {x.count > ((g0 ^ 0) & 1), x.count > ((g0 ^ 1) & 1)};
      // (warps without rows do not wait here: the barriers below, which keep a row quarter's warps within one stretch of one another,
      // are not theirs, and a phase that has come round twice cannot be told from one that has not)
      for (int j = 0; j < 2 && ok; ++j) {
        if (has[j] && live) ok = __all_sync(0xffffffffu, mbar_wait(&o_ready[j], n_o[j] & 1));
        n_o[j] += has[j];
      }
      g0 += x.count;
      if (!ok) break;
      if (!live) continue;
      tc_fence_after();
      if (hf == 0) s_mx[tq * 2 * BM + r] = m_run;
      asm volatile("bar.sync %0, 128;" ::"r"(quad_bar) : "memory");
      const float m0 = s_mx[r], m1 = s_mx[2 * BM + r], m = fmaxf(m0, m1), mu = m == -INFINITY ? 0.f : m;
      asm volatile("bar.sync %0, 128;" ::"r"(quad_bar) : "memory");
      *mx_mine = l_part;
      asm volatile("bar.sync %0, 128;" ::"r"(quad_bar) : "memory");
      const float f0 = fast_exp2(m0 - mu), f1 = fast_exp2(m1 - mu);      // (a stream without tiles: maximum -inf, weight 0)
      const float l = (s_mx[r] + s_mx[BM + r]) * f0 + (s_mx[2 * BM + r] + s_mx[3 * BM + r]) * f1;
      const size_t row0 = (size_t)blockIdx.x * BM + x.before;
      const bool fits = x.before >= 0 && x.before <= N * Hq - x.rows;
      if (!fits && lane == 0) atomicOr(err, FZ_ERR_ROW_RANGE);      // (requests that share rows)
      // A lane has one row: a store instruction would touch 32 lines with 16 bytes each. So every four lanes exchange first, four vectors
      // of four dimensions each: then a lane has vector `lane % 4` of all four rows, and an instruction writes 64 bytes of eight rows.
      const int d0 = (tq * 2 + hf) * JD, base = quad * 32 + (lane & ~3);
#pragma unroll 1
      for (int c = 0; c < JD; c += 16) {
        float a[16], b[16];
        tmem_ld16(tmem_base + 256u + (uint32_t)(d0 + c) + lane_sel, a);
        tmem_ld16(tmem_base + 256u + (uint32_t)(HD + d0 + c) + lane_sel, b);
#pragma unroll
        for (int j = 0; j < 16; ++j) a[j] = (has[0] ? a[j] * f0 : 0.f) + (has[1] ? b[j] * f1 : 0.f);
#pragma unroll
        for (int k = 2; k > 0; k >>= 1) {
          const bool up = lane & k;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i & k) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float got = __shfl_xor_sync(0xffffffffu, up ? a[4 * i + j] : a[4 * (i | k) + j], k);
              if (up) a[4 * i + j] = got;
              else a[4 * (i | k) + j] = got;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)      // (a[4 j ..] is now vector lane % 4 of row `base + j`)
          if (fits && base + j < x.rows)
            *(float4*)(part_o + (row0 + base + j) * HD + d0 + c + 4 * (lane & 3)) = make_float4(a[4 * j], a[4 * j + 1], a[4 * j + 2], a[4 * j + 3]);
      }
      if (fits && r < x.rows && d0 == 0) *(float2*)(part_ml + 2 * (row0 + r)) = make_float2(m, l);
      // nobody of this row quarter starts on the next stretch's tiles (whose products overwrite O) before all four have read
      tc_fence_before();
      asm volatile("bar.sync %0, 128;" ::"r"(quad_bar) : "memory");
    }
    if (!ok) flag[0] = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
  if (tid == 0 && flag[0]) atomicOr(err, FZ_ERR_WAIT_TIMEOUT);
}

// Where a row's stretches lie: as the record says that the block with its item's first stretch has left (none for an item without units).
struct Stretches {
  const float *part_o, *part_ml;
  const int2* records;
  int NB, Hkv, window, rows;      // rows: of the scratch
  __device__ __forceinline__ int2 early(int n, int kvh) const { return records[(size_t)n * Hkv + kvh]; }
  __device__ __forceinline__ Range range(int2 record, int, int, int node, int head_in_group, int group, int nodes, int start, int pos) const {
    int a, tiles, row_tiles;
    request_units(nodes, start, window, NB, a, tiles, row_tiles);
    Range x;
    x.extra_from = x.extra_to = 0;
    if (window > 0) {      // places that this row sees and a later one does not
      x.extra_from = max(0, pos - window + 1);
      x.extra_to = min(a, start);
    }
    const bool there = tiles > 0 && record.x >= 0 && record.y > 0 && record.y <= rows / BM && record.x <= rows - BM * record.y;
    x.pieces = there ? record.y : 0;
    x.first = there ? (size_t)record.x + (node % NB) * group + head_in_group : 0;
    x.step = BM;
    return x;
  }
};

int sm_count() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) sms = 148;
  }
  return sms;
}

// Queries as (N, Hq, hd): boxes of NB nodes x the G heads of a kv head x 64 columns. The pool as rows of hd values: boxes of `box` rows x 64.
int encode(const void* p, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, CUtensorMap* out) {
  EncodeTiled enc = encode_fn();
  if (!enc) return FZ_NO_DRIVER_ENTRY;
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? FZ_OK : FZ_TMAP_ENCODE;
}
int query_map(const void* q, int N, int Hq, int hd, int G, int NB, CUtensorMap* out) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)Hq, (cuuint64_t)N}, strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)Hq * hd * 2};
  const cuuint32_t box[3] = {64u, (cuuint32_t)G, (cuuint32_t)NB};
  return encode(q, 3, dims, strides, box, out);
}
int pool_map(const void* pool, long long rows, int hd, int box_rows, CUtensorMap* out) {
  const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)hd * 2};
  const cuuint32_t box[2] = {64u, (cuuint32_t)box_rows};
  return encode(pool, 2, dims, strides, box, out);
}

template <int HD, int BOX>
int launch(const CUtensorMap& qm, const CUtensorMap& kvm, const void* v_pool, const Sizes& Z, const int* table, int mb, int page_size, int num_pages,
           int N, int Hq, float scale_log2, int blocks, float* part_o, float* part_ml, int2* records, int* err, cudaStream_t stream) {
  constexpr int HALVES = HD / 64, STAGES = HD <= 64 ? 6 : 3;
  constexpr size_t smem = (size_t)HALVES * 128 * 128 * (1 + 2 * STAGES) + 4 * BM * 4 + 8 * (8 + 4 * STAGES + RING) + RING * sizeof(Stretch) + 8;
  static_assert(smem <= FZ_MOST_SMEM);
  auto kern = attn_tree_tc_kernel<HD, BOX>;
  FZ_RAISE_SMEM(kern);
  const cudaError_t e = fz_launch(kern, dim3((unsigned)blocks), dim3(THREADS), smem, stream, qm, kvm, (const __nv_bfloat16*)v_pool, Z, table, mb, page_size,
                                  num_pages, Hq, scale_log2, N, part_o, part_ml, records, err);
  return e == cudaSuccess ? FZ_OK : (int)e;
}
}  // namespace

// Head sizes 64 and 128, up to 128 query heads per kv head, pages of 8 or a multiple of 16 places.
FZ_API int fz_attn_tree_tc_check(int Hq, int Hkv, int hd, int page_size) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > BM) return FZ_BAD_SHAPE;
  if (hd != 64 && hd != 128) return FZ_BAD_SHAPE;
  if (!(page_size == 8 || (page_size > 0 && page_size % 16 == 0))) return FZ_BAD_SHAPE;
  return FZ_OK;
}

// Rows of the scratch (each hd + 2 floats; behind them 2 * N * Hkv ints): every (node, head) once, and once more where a block's run cuts its
// item.
FZ_API long long fz_attn_tree_tc_rows(int N, int Hq) { return (long long)N * Hq + (long long)BM * sm_count(); }

// As fz_attn_tree; k_pool and v_pool are the two parts of one pool (pages, 2, Hkv, page_size, hd) of num_pages pages.
FZ_API int fz_attn_tree_tc(const void* q, const void* k_pool, const void* v_pool, const int* pos, const int* seq_row, const int* seg, int S,
                           const int* ancestors, int words, const int* table, int mb, long long page_stride, int page_size, int num_pages, void* out,
                           int N, int Hq, int Hkv, int hd, float scale, int window, float* part, int* err, cudaStream_t stream) {
  if (N <= 0) return FZ_OK;
  if (fz_attn_tree_tc_check(Hq, Hkv, hd, page_size) != FZ_OK || S <= 0 || words <= 0 || mb <= 0 || num_pages <= 0) return FZ_BAD_SHAPE;
  if (page_stride != 2LL * Hkv * page_size * hd || (const __nv_bfloat16*)v_pool != (const __nv_bfloat16*)k_pool + (long long)Hkv * page_size * hd)
    return FZ_BAD_SHAPE;
  if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out | (uintptr_t)part) & 15) return FZ_BAD_ALIGNMENT;
  const long long pool_rows = (long long)num_pages * 2 * Hkv * page_size;
  if (pool_rows > 2147483647LL) return FZ_TOO_LARGE;
  const int G = Hq / Hkv, NB = BM / G, blocks = sm_count();
  CUtensorMap qm, kvm;
  int st = query_map(q, N, Hq, hd, G, NB, &qm);
  if (st != FZ_OK) return st;
  const int box = page_size == 8 ? 8 : 16;
  if ((st = pool_map(k_pool, pool_rows, hd, box, &kvm)) != FZ_OK) return st;
  const float scale_log2 = scale * 1.4426950408889634f;
  const long long rows = fz_attn_tree_tc_rows(N, Hq);
  if (rows > 2147483647LL) return FZ_TOO_LARGE;
  float* part_ml = part + (size_t)rows * hd;
  int2* records = (int2*)(part_ml + (size_t)rows * 2);
  const Sizes Z = {seg, S, NB, Hkv, window, N, (long long)mb * page_size};
#define FZ_T(HD_, BOX_) st = launch<HD_, BOX_>(qm, kvm, v_pool, Z, table, mb, page_size, num_pages, N, Hq, scale_log2, blocks, part, part_ml, records, err, stream)
  if (hd == 64 && box == 8) FZ_T(64, 8);
  else if (hd == 64) FZ_T(64, 16);
  else if (box == 8) FZ_T(128, 8);
  else FZ_T(128, 16);
#undef FZ_T
  if (st != FZ_OK) return st;
  const Stretches P = {part, part_ml, records, NB, Hkv, window, (int)rows};
  const TreeArgs R = {pos, seq_row, seg, ancestors, table, S, words, mb, page_stride, page_size, num_pages, N, Hq, Hkv, hd, scale_log2, window, err};
  return launch_merge<__nv_bfloat16>((const __nv_bfloat16*)q, (const __nv_bfloat16*)k_pool, (const __nv_bfloat16*)v_pool, (__nv_bfloat16*)out, P, R, stream);
}

#ifdef FZ_TIMELINE
FZ_TIMELINE_READER(attn_tree_tc)
#endif
