// Softmax attention of lists that share a prefix, on the 5th-generation tensor cores (formulas in xdlb200.h).
//
// A tile is 128 rows of scores: R = 128 / share query rows of one prefix's lists, with the `share` heads that read one head of keys side by side.
// It meets the keys of its prefix, and those of its lists' own that lie between the first that its first row sees and the last that its last row
// does, 128 at a time; a row's own keys are one interval, so that lists and the order in a list are one comparison with two ends. The prefix is
// read once for all rows of a tile, whatever lists they are of.
// An item is a tile and a head of keys, a unit one block of keys of an item. The units of all items lie in one line that is cut into equal parts,
// one a CTA; a part that ends inside an item leaves its sums (fp32, with the running maximum and sum) in the workspace, and a last kernel joins
// them in order. prefix_plan_kernel lays the line out from the offsets, which only the device knows.
//
// In a CTA one warp loads (TMA), one issues the MMAs, and two groups of four warps take the blocks of keys in turn, each with scores, weights and
// sums of its own in tensor memory: while one makes weights of its scores, the tensor cores are at the other's. A thread has a row; a maximum
// that has not grown by more than 2^8 leaves the sums as they are (weights up to 256 fit both types), so that they are seldom moved.
#pragma once

#include <algorithm>

#include "xb_heads.cuh"
#include "xb_umma.cuh"

namespace xb {
namespace {

constexpr int PFX_KEYS = 128, PFX_ROWS = 128, PFX_THREADS = 320, PFX_LOADER = 8, PFX_MMA = 9;
constexpr float PFX_GROWTH = 8.f;

struct PrefixTile {
  int row0, rows;                          // query rows
  int prefix0, prefix_n;
  int own0, own_n;                         // the own keys that any of its rows sees
  int own_full;                            // the first of them that all of its rows see
  int list0, list1;                        // its first row's list, and its last row's
  int units;
};
struct PrefixParams {
  Lists lists, own;                        // rows of q; rows of k and v
  const int32_t* members;                  // [prefixes + 1], null: as many lists each
  const int32_t* prefix_offsets;           // [prefixes + 1], null: as many rows each
  int64_t prefix_rows;
  int prefixes, H, Hkv, share, R, d;
  float scale;                             // times log2(e)
  Heads y, v;
  int vec_y;
  // workspace
  PrefixTile* tiles;
  int64_t* ends;                           // [tiles + 1]: units before a tile (of one head)
  int* first_tile;                         // [groups + 1]
  float* part;                             // [2 CTAs][128][d]
  float2* part_ml;                         // [2 CTAs][128]
  int max_tiles, ctas;
};

// ---- the plan ----
// Lists of group g: those ahead of the first member (no prefix), of prefix g - 1, and those behind the last member (no prefix).
__device__ __forceinline__ int group_begin(const PrefixParams& p, int g) {
  if (g == 0) return 0;
  if (g == p.prefixes + 2 || p.prefixes == 0) return p.lists.batch;
  if (!p.members) return (g - 1) * (p.lists.batch / p.prefixes);
  const int m = p.members[g - 1];
  return m < 0 ? 0 : m > p.lists.batch ? p.lists.batch : m;
}
__device__ __forceinline__ int64_t prefix_begin(const PrefixParams& p, int i) {
  if (!p.prefix_offsets) return (int64_t)i * (p.prefix_rows / p.prefixes);
  const int64_t o = p.prefix_offsets[i];
  return o < 0 ? 0 : o > p.prefix_rows ? p.prefix_rows : o;
}
// the list of a row, from lo to hi (that of a later row): the last that begins at it or ahead of it
__device__ __forceinline__ int list_of(const Lists& l, int64_t row, int lo, int hi) {
  if (!l.offsets) return l.per > 0 ? (int)(row / l.per) : 0;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (l.begin(mid) <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// the own keys that a row sees: a list's last row sees all of them, each row before it one less
__device__ __forceinline__ void own_of(const PrefixParams& p, int64_t row, int list, int64_t& lo, int64_t& hi) {
  lo = p.own.begin(list);
  hi = p.own.begin(list + 1) - (p.lists.begin(list + 1) - 1 - row);
  if (hi < lo) hi = lo;
}
template <int WARPS>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s_sums, int64_t& total) {      // exclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t t = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += t;
  }
  __syncthreads();
  if (lane == 31) s_sums[warp] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_sums[w];
    total += s_sums[w];
  }
  return before + x - v;
}
constexpr int PLAN_THREADS = 1024;
__global__ void __launch_bounds__(PLAN_THREADS) prefix_plan_kernel(const PrefixParams p) {
  pdl_begin();
  __shared__ int64_t s_sums[PLAN_THREADS / 32];
  const int groups = p.prefixes == 0 ? 1 : p.prefixes + 2;
  int64_t total = 0, sum;
  for (int g0 = 0; g0 < groups; g0 += PLAN_THREADS) {
    const int g = g0 + (int)threadIdx.x;
    int64_t n = 0;
    if (g < groups) {
      const int64_t rows = p.lists.begin(group_begin(p, g + 1)) - p.lists.begin(group_begin(p, g));
      n = rows > 0 ? (rows + p.R - 1) / p.R : 0;
    }
    const int64_t at = total + block_scan<PLAN_THREADS / 32>(n, s_sums, sum);
    if (g < groups) p.first_tile[g] = (int)min(at, (int64_t)p.max_tiles);
    total += sum;
  }
  const int tiles = (int)min(total, (int64_t)p.max_tiles);
  if (threadIdx.x == 0) p.first_tile[groups] = tiles;
  __syncthreads();
  int64_t units = 0;
  for (int t0 = 0; t0 < tiles; t0 += PLAN_THREADS) {
    const int t = t0 + (int)threadIdx.x;
    PrefixTile x = {};
    if (t < tiles) {
      int lo = 0, hi = groups - 1;                        // the group: the last that begins at the tile or ahead of it
      while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (p.first_tile[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      const int l0 = group_begin(p, lo), l1 = group_begin(p, lo + 1);
      const int64_t begin = p.lists.begin(l0) + (int64_t)(t - p.first_tile[lo]) * p.R, end = min(begin + p.R, p.lists.begin(l1));
      x.row0 = (int)begin; x.rows = (int)max(end - begin, (int64_t)0);
      if (lo > 0 && lo <= p.prefixes) {
        const int64_t a = prefix_begin(p, lo - 1), b = prefix_begin(p, lo);
        x.prefix0 = (int)a; x.prefix_n = (int)max(b - a, (int64_t)0);
      }
      x.list0 = list_of(p.lists, begin, l0, max(l1 - 1, l0));
      x.list1 = list_of(p.lists, max(end - 1, begin), x.list0, max(l1 - 1, l0));
      if (p.own.rows > 0) {
        int64_t a, b, c, e;
        own_of(p, begin, x.list0, a, b);
        own_of(p, max(end - 1, begin), x.list1, c, e);
        x.own0 = (int)a; x.own_n = (int)max(e - a, (int64_t)0);
        x.own_full = x.list0 == x.list1 ? (int)(b - a) : 0;
      }
      x.units = max((x.prefix_n + PFX_KEYS - 1) / PFX_KEYS + (x.own_n + PFX_KEYS - 1) / PFX_KEYS, 1);
      p.tiles[t] = x;
    }
    const int64_t at = units + block_scan<PLAN_THREADS / 32>(x.units, s_sums, sum);
    if (t < tiles) p.ends[t] = at;
    units += sum;
  }
  if (threadIdx.x == 0) p.ends[tiles] = units;
}

// Where a CTA's part of the line begins: tile, head of keys, block of keys.
struct PrefixAt {
  int tile, head, unit;
};
__device__ __forceinline__ PrefixAt part_begin(const PrefixParams& p, int tiles, int64_t all, int cta, int ctas) {
  PrefixAt at = {tiles, 0, 0};
  if (cta >= ctas) return at;
  const int64_t x = all * cta / ctas;
  int lo = 0, hi = tiles - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (p.ends[mid] * p.Hkv <= x) lo = mid;
    else hi = mid - 1;
  }
  const int64_t units = p.ends[lo + 1] - p.ends[lo], in = x - p.ends[lo] * p.Hkv;
  at.tile = lo; at.head = (int)(in / units); at.unit = (int)(in % units);
  // small items stay whole: what a cut saves is less than joining costs
  if (units * ctas * 4 <= all && at.unit > 0) {
    if (2 * at.unit >= units && ++at.head == p.Hkv) {
      at.head = 0;
      ++at.tile;
    }
    at.unit = 0;
  }
  return at;
}

// ---- the kernel ----
template <int DP>
struct PrefixShape {
  static constexpr int Q = 2, K = DP == 128 ? 3 : 5, V = DP == 128 ? 2 : 5;                     // buffers
  static constexpr int TILE = 128 * DP * 2, BOX = 128 * 128;
  struct Control {                         // behind the buffers (the kernel has no other shared memory, so that its buffers begin on 1024 bytes)
    uint64_t q_full[Q], q_empty[Q], k_full[K], k_empty[K], v_full[V], v_empty[V];
    uint64_t s_full[2], p_ready[2], o_done[2], o_free, met, drained;
    float2 ml[2][PFX_ROWS];                // maximum and sum of either group's rows
    PrefixAt part[2];
    int bad[2];
    uint32_t tmem;
  };
  static constexpr int SMEM = (Q + K + V) * TILE + (int)sizeof(Control);
  static_assert(SMEM <= 227 * 1024, "");
  // columns of tensor memory: the scores of both groups, their sums; weights where there is room, else over the scores that they are made of
  static constexpr uint32_t S = 0, O = 256, P = DP == 128 ? 0 : 384, P_STEP = DP == 128 ? 128 : 64;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// halves that are infinite or NaN
template <bool BF16>
__device__ __forceinline__ bool half_is_bad(uint32_t h) {
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  return (h & E) == E;
}

// A CTA's pieces in order: an item, its blocks of keys [k0, k1), and whether these are all of them.
struct PrefixPiece {
  PrefixTile t;
  int head, k0, k1, prefix_tiles, n;       // n: blocks of keys
  bool whole, head_part;                   // head_part: the item began in a CTA before
};
template <typename F>
__device__ __forceinline__ void each_piece(const PrefixParams& p, const PrefixAt& from, const PrefixAt& to, F visit) {
  PrefixAt at = from;
  while (at.tile < to.tile || (at.tile == to.tile && (at.head < to.head || (at.head == to.head && at.unit < to.unit)))) {
    PrefixPiece x;
    x.t = p.tiles[at.tile];
    x.head = at.head;
    x.k0 = at.unit;
    const bool ends_inside = at.tile == to.tile && at.head == to.head;
    x.k1 = ends_inside ? to.unit : x.t.units;
    x.prefix_tiles = (x.t.prefix_n + PFX_KEYS - 1) / PFX_KEYS;
    x.n = x.t.prefix_n + x.t.own_n > 0 ? x.k1 - x.k0 : 0;
    x.whole = x.k0 == 0 && x.k1 == x.t.units;
    x.head_part = x.k0 > 0;
    if (!visit(x)) return;
    at.unit = 0;
    if (++at.head == p.Hkv) {
      at.head = 0;
      ++at.tile;
    }
  }
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(PFX_THREADS, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ CUtensorMap map_pk, const __grid_constant__ CUtensorMap map_pv, const __grid_constant__ PrefixParams p) {
  using namespace umma;
  using T = PrefixShape<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *smem_q = smem, *smem_k = smem_q + T::Q * T::TILE, *smem_v = smem_k + T::K * T::TILE;
  typename T::Control& ctl = *reinterpret_cast<typename T::Control*>(smem_v + T::V * T::TILE);
  auto &q_full = ctl.q_full, &q_empty = ctl.q_empty;
  auto &k_full = ctl.k_full, &k_empty = ctl.k_empty;
  auto &v_full = ctl.v_full, &v_empty = ctl.v_empty;
  auto &s_full = ctl.s_full, &p_ready = ctl.p_ready, &o_done = ctl.o_done;
  auto &o_free = ctl.o_free, &met = ctl.met, &drained = ctl.drained;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::Q; ++s) { mbar_init(smem_u32(&q_full[s]), 1); mbar_init(smem_u32(&q_empty[s]), 1); }
    for (int s = 0; s < T::K; ++s) { mbar_init(smem_u32(&k_full[s]), 1); mbar_init(smem_u32(&k_empty[s]), 1); }
    for (int s = 0; s < T::V; ++s) { mbar_init(smem_u32(&v_full[s]), 1); mbar_init(smem_u32(&v_empty[s]), 1); }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&s_full[w]), 1);
      mbar_init(smem_u32(&p_ready[w]), 128);
      mbar_init(smem_u32(&o_done[w]), 1);
    }
    mbar_init(smem_u32(&o_free), 256);
    mbar_init(smem_u32(&met), 256);
    mbar_init(smem_u32(&drained), 1);
    fence_barrier_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    prefetch_tensormap(&map_pk);
    prefetch_tensormap(&map_pv);
    ctl.bad[0] = ctl.bad[1] = 0;
  }
  if (warp == PFX_MMA) tmem_alloc(smem_u32(&ctl.tmem), 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = ctl.tmem;
  pdl_wait();
  if (threadIdx.x < 2) {
    const int tiles = p.first_tile[p.prefixes == 0 ? 1 : p.prefixes + 2];
    const int64_t all = tiles > 0 ? p.ends[tiles] * p.Hkv : 0;
    const int ctas = (int)min(all, (int64_t)gridDim.x);
    ctl.part[threadIdx.x] = part_begin(p, tiles, all, blockIdx.x + threadIdx.x, ctas);
  }
  __syncthreads();
  const PrefixAt from = ctl.part[0], to = ctl.part[1];

  if (warp == PFX_LOADER) {
    int qn = 0, kn = 0, vn = 0;            // tiles asked for so far
    bool ok = true;
    each_piece(p, from, to, [&](const PrefixPiece& x) {
      if (x.n == 0) return true;
      const int qs = qn % T::Q;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&q_empty[qs]), ((uint32_t)(qn / T::Q) & 1u) ^ 1u, 81)))) return false;
      if (lane == 0) {
        const uint32_t bar = smem_u32(&q_full[qs]), dst = smem_u32(smem_q + qs * T::TILE);
        mbar_arrive_expect_tx(bar, (uint32_t)(DP / 64 * 128 * p.share * p.R));
#pragma unroll
        for (int b = 0; b < DP / 64; ++b) tma_load_4d(dst + b * T::BOX, &map_q, bar, b * 64, 0, x.head, x.t.row0);
      }
      ++qn;
      auto load = [&](bool keys, int j) {
        const bool prefix = j < x.prefix_tiles;
        const int row = prefix ? x.t.prefix0 + j * PFX_KEYS : x.t.own0 + (j - x.prefix_tiles) * PFX_KEYS;
        int& n = keys ? kn : vn;
        const int S = keys ? T::K : T::V, s = n % S;
        const uint32_t empty = smem_u32(keys ? &k_empty[s] : &v_empty[s]), full = smem_u32(keys ? &k_full[s] : &v_full[s]);
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty, ((uint32_t)(n / S) & 1u) ^ 1u, keys ? 82 : 83)))) return false;
        if (lane == 0) {
          const uint32_t dst = smem_u32((keys ? smem_k : smem_v) + s * T::TILE);
          const CUtensorMap* map = keys ? (prefix ? &map_pk : &map_k) : (prefix ? &map_pv : &map_v);
          mbar_arrive_expect_tx(full, (uint32_t)T::TILE);
#pragma unroll
          for (int b = 0; b < DP / 64; ++b) tma_load_3d(dst + b * T::BOX, map, full, b * 64, x.head, row);
        }
        ++n;
        return true;
      };
      if (!load(true, x.k0)) return false;
      for (int j = x.k0; j < x.k1; ++j) {
        if (j + 1 < x.k1 && !load(true, j + 1)) return false;
        if (!load(false, j)) return false;
      }
      return true;
    });
    if (!ok) {                             // nothing that was asked for arrives after this CTA has ended
      for (int i = 1; i <= T::Q && i <= qn; ++i) mbar_wait(smem_u32(&q_full[(qn - i) % T::Q]), (uint32_t)((qn - i) / T::Q) & 1u, 84);
      for (int i = 1; i <= T::K && i <= kn; ++i) mbar_wait(smem_u32(&k_full[(kn - i) % T::K]), (uint32_t)((kn - i) / T::K) & 1u, 84);
      for (int i = 1; i <= T::V && i <= vn; ++i) mbar_wait(smem_u32(&v_full[(vn - i) % T::V]), (uint32_t)((vn - i) / T::V) & 1u, 84);
    }
  } else if (warp == PFX_MMA) {
    constexpr int FMT = BF16 ? 1 : 0;
    const uint32_t idesc_s = make_idesc(128, PFX_KEYS, FMT), idesc_o = make_idesc(128, DP, FMT) | IDESC_B_MN;
    const int steps = (p.d + 15) / 16;
    int qn = 0, kn = 0, vn = 0, pieces = 0;
    int sn[2] = {0, 0};                    // blocks of either group so far (scores asked for)
    int on[2] = {0, 0};                    // products with the weights asked for
    bool ok = true;
    auto wait = [&](uint64_t* bar, int phase, int site) { return ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), (uint32_t)phase & 1u, site)); };
    each_piece(p, from, to, [&](const PrefixPiece& x) {
      if (x.n == 0) return true;
      const int qs = qn % T::Q;
      if (!wait(&q_full[qs], qn / T::Q, 85)) return false;
      const uint32_t q = smem_u32(smem_q + qs * T::TILE);
      auto scores = [&](int i) {
        const int w = i & 1, s = kn % T::K;
        if (!wait(&k_full[s], kn / T::K, 86)) return false;
        // the group's weights lie over its scores (or its scores' next ones are made into them): the product that reads them has ended
        if (on[w] > 0 && !wait(&o_done[w], on[w] - 1, 87)) return false;
        tc_fence_after_sync();
        const uint32_t k = smem_u32(smem_k + s * T::TILE), to_s = tmem + T::S + w * 128;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
          if (kk < steps)
            mma_f16_ss_elect(to_s, make_desc_sw128(q + (kk / 4) * T::BOX + (kk % 4) * 32, 1024), make_desc_sw128(k + (kk / 4) * T::BOX + (kk % 4) * 32, 1024),
                             idesc_s, kk > 0 ? 1u : 0u);
        mma_commit_elect(smem_u32(&k_empty[s]));
        mma_commit_elect(smem_u32(&s_full[w]));
        ++kn;
        ++sn[w];
        if (i == x.n - 1) mma_commit_elect(smem_u32(&q_empty[qs]));
        return true;
      };
      if (!scores(0)) return false;
      if (x.n > 1 && !scores(1)) return false;
      for (int i = 0; i < x.n; ++i) {
        const int w = i & 1, s = vn % T::V;
        if (!wait(&p_ready[w], on[w], 88)) return false;
        if (!wait(&v_full[s], vn / T::V, 89)) return false;
        if (i < 2 && pieces > 0 && !wait(&o_free, pieces - 1, 90)) return false;
        tc_fence_after_sync();
        const uint32_t v = smem_u32(smem_v + s * T::TILE), to_o = tmem + T::O + w * DP, from_p = tmem + T::P + w * T::P_STEP;
#pragma unroll
        for (int kk = 0; kk < PFX_KEYS / 16; ++kk)
          mma_f16_ts_elect(to_o, from_p + kk * 8, make_desc_sw128_mn(v + kk * 2048, T::BOX), idesc_o, (i >= 2 || kk > 0) ? 1u : 0u);
        mma_commit_elect(smem_u32(&v_empty[s]));
        mma_commit_elect(smem_u32(&o_done[w]));
        ++vn;
        ++on[w];
        if (i + 2 < x.n && !scores(i + 2)) return false;
      }
      ++qn;
      ++pieces;
      return true;
    });
    if (!ok) {                             // the products in flight end before their tensor memory is given back
      mma_commit_elect(smem_u32(&drained));
      mbar_wait(smem_u32(&drained), 0, 91);
    }
  } else {
    const int w = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) * 32u << 16;
    const uint32_t my_s = tmem + T::S + w * 128 + lanes, my_p = tmem + T::P + w * T::P_STEP + lanes, my_o = tmem + T::O + w * DP + lanes;
    int sn = 0, on[2] = {0, 0}, seq = 0, pieces = 0;       // blocks of this group; products of either; blocks of the CTA; pieces with blocks
    each_piece(p, from, to, [&](const PrefixPiece& x) {
      const int g = row % p.share;
      const bool there = row < x.t.rows * p.share;
      const int64_t q_row = x.t.row0 + row / p.share;
      const int q_head = x.head * p.share + g;
      // the own keys that the row sees, counted from the tile's first
      int lo = 0, hi = 0;
      if (there && x.t.own_n > 0) {
        int64_t a, b;
        own_of(p, q_row, list_of(p.lists, q_row, x.t.list0, x.t.list1), a, b);
        lo = (int)min(max(a - x.t.own0, (int64_t)0), (int64_t)x.t.own_n);
        hi = (int)min(max(b - x.t.own0, (int64_t)0), (int64_t)x.t.own_n);
      }
      float m = -INFINITY, l = 0.f;
      for (int i = w; i < x.n; i += 2) {
        const int j = x.k0 + i;
        const bool prefix = j < x.prefix_tiles;
        const int key0 = prefix ? j * PFX_KEYS : (j - x.prefix_tiles) * PFX_KEYS;
        const int in = min(PFX_KEYS, (prefix ? x.t.prefix_n : x.t.own_n) - key0);             // keys of the block
        const bool masked = in < PFX_KEYS || (!prefix && (x.t.list0 != x.t.list1 || key0 + PFX_KEYS > x.t.own_full));
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[w]), (uint32_t)sn & 1u, 92))) return false;
        tc_fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_nowait(my_s + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld(s[c]);
        if (masked) {
          const int c0 = prefix ? 0 : max(lo - key0, 0), c1 = prefix ? in : min(hi - key0, in);
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c < c0 || c >= c1) s[c / 32][c % 32] = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; ++c) top[c % 4] = fmaxf(top[c % 4], __uint_as_float(s[c / 32][c % 32]));
        const float next = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        if (__any_sync(0xffffffffu, (next - m) * p.scale > PFX_GROWTH)) {
          // (m is -infinity: nothing has been summed; no maximum yet: nothing to move)
          const float by = m == next || m == -INFINITY ? 1.f : ex2((m - next) * p.scale);
          m = next;
          l *= by;
          if (i >= 2) {
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_done[w]), (uint32_t)(on[w] - 1) & 1u, 93))) return false;
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              uint32_t o[32];
              tmem_ld32_nowait(my_o + c, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
              tmem_st16(my_o + c, o);
              tmem_st16(my_o + c + 16, o + 16);
            }
          }
        }
        // The exponents: scale s - scale m in one FMA. A rounded scale m is the same factor to all of a row's weights, but of scores far beyond what
        // a softmax tells apart (masks of the type's lowest value) it would be a large one: those have m taken off first.
        float base = m == -INFINITY ? 0.f : m * p.scale;
        if (__any_sync(0xffffffffu, fabsf(base) > 1e6f)) {
          const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c / 32][c % 32] = __float_as_uint(__uint_as_float(s[c / 32][c % 32]) - off);
          base = 0.f;
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t weights[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float a = ex2(fmaf(__uint_as_float(s[c][e]), p.scale, -base)), b = ex2(fmaf(__uint_as_float(s[c][e + 1]), p.scale, -base));
            sum[e / 2 % 2] += a;
            sum[2 + e / 2 % 2] += b;
            weights[e / 2] = pack_weights<BF16>(a, b);
          }
          tmem_st16(my_p + c * 16, weights);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (masked) {
          // Zero weights take no part only beside finite values: rows behind the keys become zeros, and where rows see different keys, infinities and
          // NaN too (what they are to the rows that see them is made up for at the end).
          const int vs = (seq + i) % T::V;
          if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&v_full[vs]), (uint32_t)((seq + i) / T::V) & 1u, 94))) return false;
          uint8_t* v = smem_v + vs * T::TILE;
#pragma unroll 4
          for (int e = row; e < DP / 64 * 1024; e += 128) {
            const int r = e >> 3 & 127;
            uint4* at = reinterpret_cast<uint4*>(v + (e >> 10) * T::BOX + r * 128 + (e & 7) * 16);
            if (r >= in) {
              *at = make_uint4(0u, 0u, 0u, 0u);
            } else if (!prefix) {
              uint4 t = *at;
              uint32_t* h = reinterpret_cast<uint32_t*>(&t);
              bool bad = false;
#pragma unroll
              for (int z = 0; z < 4; ++z) bad |= half_is_bad<BF16>(h[z]) || half_is_bad<BF16>(h[z] >> 16);
              if (bad) {
#pragma unroll
                for (int z = 0; z < 4; ++z) h[z] &= (half_is_bad<BF16>(h[z]) ? 0u : 0xffffu) | (half_is_bad<BF16>(h[z] >> 16) ? 0u : 0xffff0000u);
                *at = t;
                ctl.bad[pieces & 1] = pieces + 1;
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&p_ready[w]));
        ++sn;
        ++on[w];
      }
      // both groups' sums together: a thread has half of its row's columns
      float f[2] = {1.f, 0.f}, top = -INFINITY, all = 0.f;
      bool bad = false;
      if (x.n > 0) {
        on[w ^ 1] += (x.n + w) / 2;                        // (this group counted its own)
        // (what stands there of the piece before has been read)
        if (pieces > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_free), (uint32_t)(pieces - 1) & 1u, 98))) return false;
        ctl.ml[w][row] = make_float2(m, l);
        mbar_arrive(smem_u32(&met));
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&met), (uint32_t)pieces & 1u, 95))) return false;
        const float2 a = ctl.ml[0][row], b = ctl.ml[1][row];
        bad = ctl.bad[pieces & 1] == pieces + 1;
        top = fmaxf(a.x, b.x);
        f[0] = a.x == -INFINITY ? 0.f : ex2((a.x - top) * p.scale);
        f[1] = b.x == -INFINITY ? 0.f : ex2((b.x - top) * p.scale);
        all = a.y * f[0] + b.y * f[1];
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_done[0]), (uint32_t)(on[0] - 1) & 1u, 96))) return false;
        if (x.n > 1 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&o_done[1]), (uint32_t)(on[1] - 1) & 1u, 97))) return false;
        tc_fence_after_sync();
      }
      const int slot = 2 * blockIdx.x + (x.head_part ? 0 : 1);
      const float by = x.whole && all > 0.f ? 1.f / all : x.whole && all == 0.f ? 0.f : x.whole ? all : 1.f;       // (NaN: as it is)
#pragma unroll 1
      for (int c0 = w * (DP / 2); c0 < (w + 1) * (DP / 2); c0 += 32) {
        float o[32];
        if (x.n > 0) {
          uint32_t a[32], b[32];
          tmem_ld32_nowait(tmem + T::O + lanes + c0, a);
          if (x.n > 1) tmem_ld32_nowait(tmem + T::O + DP + lanes + c0, b);
          tmem_wait_ld(a);
          if (x.n > 1) tmem_wait_ld(b);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = (__uint_as_float(a[e]) * f[0] + (x.n > 1 ? __uint_as_float(b[e]) * f[1] : 0.f)) * by;
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (there && bad) {                                // infinities and NaN among the own values that the row sees in these blocks
          const int k_lo = max(lo, max(x.k0 - x.prefix_tiles, 0) * PFX_KEYS), k_hi = min(hi, (x.k1 - x.prefix_tiles) * PFX_KEYS);
          for (int k = k_lo; k < k_hi; ++k) {
            const uint16_t* v = p.v.get<uint16_t>((int64_t)x.t.own0 + k, x.head);
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (c0 + e >= p.d) break;
              const uint16_t t = v[c0 + e];
              if (half_is_bad<BF16>(t)) o[e] += BF16 ? __uint_as_float((uint32_t)t << 16) : __half2float(__ushort_as_half(t));
            }
          }
        }
        if (there && x.whole) {
          uint16_t* y = const_cast<uint16_t*>(p.y.get<uint16_t>(q_row, q_head)) + c0;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (c0 + e >= p.d) break;                      // (d is whole pieces of 8)
            uint4 t;
            t.x = pack_weights<BF16>(o[e], o[e + 1]); t.y = pack_weights<BF16>(o[e + 2], o[e + 3]);
            t.z = pack_weights<BF16>(o[e + 4], o[e + 5]); t.w = pack_weights<BF16>(o[e + 6], o[e + 7]);
            if (p.vec_y) {
              *reinterpret_cast<uint4*>(y + e) = t;
            } else {
              const uint32_t h[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
              for (int z = 0; z < 8; ++z) y[e + z] = (uint16_t)(h[z / 2] >> (16 * (z & 1)));
            }
          }
        } else if (there) {
          float* part = p.part + ((int64_t)slot * PFX_ROWS + row) * p.d + c0;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            if (c0 + e >= p.d) break;
            *reinterpret_cast<float4*>(part + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        __syncwarp();                                      // the lanes meet ahead of the next loads from tensor memory
      }
      if (!x.whole && there && w == 0) p.part_ml[(int64_t)slot * PFX_ROWS + row] = make_float2(top, all);
      if (x.n > 0) {
        tc_fence_before_sync();
        mbar_arrive(smem_u32(&o_free));
        seq += x.n;
        ++pieces;
      }
      return true;
    });
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == PFX_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
  pdl_release();
}

// The parts of items that were cut, joined in the order of their CTAs. Block (c, y) has the item in which CTA c's part begins, if it began in the CTA
// before: every gridDim.y-th of its rows from y on, a warp a row.
constexpr int JOIN_THREADS = 128;
template <bool BF16>
__global__ void __launch_bounds__(JOIN_THREADS) prefix_join_kernel(const PrefixParams p) {
  pdl_begin();
  const int tiles = p.first_tile[p.prefixes == 0 ? 1 : p.prefixes + 2];
  const int64_t units = tiles > 0 ? p.ends[tiles] * p.Hkv : 0;
  const int ctas = (int)min(units, (int64_t)p.ctas), c = blockIdx.x + 1, lane = threadIdx.x & 31;
  if (c >= ctas) return;
  const PrefixAt at = part_begin(p, tiles, units, c, ctas);
  if (at.unit == 0) return;
  const PrefixAt before = part_begin(p, tiles, units, c - 1, ctas);
  if (before.tile == at.tile && before.head == at.head && before.unit > 0) return;      // cut before already
  int last = c;                                                                          // the CTA with the item's end
  while (last + 1 < ctas) {
    const PrefixAt next = part_begin(p, tiles, units, last + 1, ctas);
    if (next.tile != at.tile || next.head != at.head || next.unit == 0) break;
    ++last;
  }
  const PrefixTile t = p.tiles[at.tile];
  auto slot_of = [&](int cta) { return (int64_t)(cta == c - 1 ? 2 * cta + 1 : 2 * cta) * PFX_ROWS; };
  for (int row = blockIdx.y * (JOIN_THREADS / 32) + threadIdx.x / 32; row < t.rows * p.share; row += gridDim.y * (JOIN_THREADS / 32)) {
    float top = -INFINITY;
    for (int i = c - 1 + lane; i <= last; i += 32) top = fmaxf(top, p.part_ml[slot_of(i) + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float all = 0.f;
    const int col = lane * 4;
#pragma unroll 4
    for (int i = c - 1; i <= last; ++i) {
      const float2 ml = p.part_ml[slot_of(i) + row];
      const float f = ml.x == -INFINITY ? 0.f : ex2((ml.x - top) * p.scale);
      all += ml.y * f;
      if (col < p.d) {
        const float4 v = *reinterpret_cast<const float4*>(p.part + (slot_of(i) + row) * p.d + col);
        o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
      }
    }
    const float by = all > 0.f ? 1.f / all : all;
    if (col < p.d) {
      uint16_t* y = const_cast<uint16_t*>(p.y.get<uint16_t>(t.row0 + row / p.share, at.head * p.share + row % p.share)) + col;
      const uint32_t lo = pack_weights<BF16>(o.x * by, o.y * by), hi = pack_weights<BF16>(o.z * by, o.w * by);
      if (p.vec_y) {
        *reinterpret_cast<uint2*>(y) = make_uint2(lo, hi);
      } else {
        y[0] = (uint16_t)lo; y[1] = (uint16_t)(lo >> 16); y[2] = (uint16_t)hi; y[3] = (uint16_t)(hi >> 16);
      }
    }
  }
}

}  // namespace
}  // namespace xb
