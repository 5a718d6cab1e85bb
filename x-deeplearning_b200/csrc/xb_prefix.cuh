// Softmax attention of lists that share a prefix, on the 5th-generation tensor cores (formulas in xdlb200.h).
//
// An item is one or two tiles of 128 rows of scores (R = 128 / share query rows of one prefix's lists, with the `share` heads that read one head of
// keys side by side) and that head of keys. It meets the keys of its prefix, and those of its lists' own that lie between the first that its first
// row sees and the last that its last row does, in blocks of 128 (units). A row's own keys are one interval, so that lists and the order in a list
// are one comparison with two ends. The prefix is read once for all rows of an item, whatever lists they are of.
//
// prefix_plan_kernel puts the units of all items in a line, from the offsets that only the device knows, and cuts it into equal parts, one a CTA.
// Where the items of a prefix are longer than a part, they lie side by side in chunks of a part's length: CTAs that run at the same time then read
// the same keys, which come from memory once. (512 rows of 4 heads on 100003 keys, one item after another: 4 times the bytes.) What a CTA has of an
// item that is not whole goes to the workspace as sums in fp32 with their running maximum, and a last kernel joins those in order.
//
// In a CTA (16 warps) two groups of four warps make weights of scores, each with a warp that issues its MMAs and with scores, weights and sums of its own
// in tensor memory: one tile each of an item of two, whose keys they share, or of a single tile every other block of keys. While one makes weights,
// the tensor cores are at the other's. A thread has a row; a maximum that has not grown by more than 2^8 leaves the sums as they are (weights up to
// 256 times that of the maximum in use fit both types), so that they are seldom moved. fp16 weights are 2^7 times as large: below that one's range they are known to
// 2^-32 of the largest, not 2^-25. One more warp loads (TMA), one works the pieces out ahead of the others, and four clear what must
// not take part of the blocks of values that some row sees in part (in the groups themselves that was a sixth of the time of short lists).
//
// What bounds it is neither memory nor the tensor cores but the way from scores to weights: 128 exponentials a row and block at 16 a cycle and SM, 1024
// cycles for a block of 128 rows, with the maximum, the packing and the loads and stores of tensor memory 1500 to 2100; and some 18000 cycles an item of
// few blocks (offsets, the first keys, the results). Single calls (back to back 3 to 13 us less): 512 candidates of 4 heads of 128 on one prefix of 100003 rows: 165 us
// (its products: 62); 74 requests of 1000 candidates on 100 rows each, 4 heads of 64: 127 us (bytes 24); 256 lists of up to 300 rows that 8 prefixes of up to 4000
// serve, 32 heads on 8 of 128, one new row each: 205 us (bytes 69); 64 lists of up to 500 rows, whole, 16 prefixes of up to 1000, 8 heads of 64: 400 us (products 48).
// Instructions are not always at hand (no_instruction 0.9 to 1.5 stalls an issue): one more wait in line costs 1 to 6 % of some calls.
#pragma once

#include <algorithm>

#include "xb_heads.cuh"
#include "xb_mma_half.cuh"
#include "xb_umma.cuh"

namespace xb {
namespace {

constexpr int PFX_KEYS = 128, PFX_ROWS = 128, PFX_THREADS = 512, PFX_LOADER = 8, PFX_MMA = 9, PFX_SLOTS = 4;
constexpr int PFX_RING = 2, PFX_TAKERS = 15;               // pieces ahead; warps that take them
constexpr float PFX_GROWTH = 8.f;
constexpr int PFX_KEPT = 128;                              // blocks after which a group's sums are taken out of the tensor cores
template <bool BF16>
constexpr float PFX_UP = BF16 ? 0.f : 7.f;                 // the power of two that the weight of a row's maximum is

struct PrefixItem {
  int row0, rows;                          // query rows
  int prefix0, prefix_n;
  int own0, own_n;                         // the own keys that any of its rows sees; from here on counted from the first of them
  int end0, begin1;                        // where those of the first tile's rows end and those of the second's begin
  int full0, full1;                        // up to where all rows of a tile see them, if its rows are of one list (else 0)
  int list[4];                             // the lists of the first and the last row of either tile
};
struct PrefixGroup {                       // the lists of a prefix
  int64_t weight;                          // units of tiles ahead of it (for one head of keys)
  int first, blocks, chunks, tiles;        // its first item; blocks of its prefix's keys, and the chunks that they go by; tiles of its items
};
struct PrefixAt {                          // a place in the line: group, head of keys, chunk, item, block of keys
  int group, head, chunk, item, unit;
};
struct PrefixRecord {                      // sums in the workspace: of which item and head, from which block of keys on (item -1: none)
  int item, head, unit, pad;
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
  PrefixItem* items;
  int64_t* own_weight;                     // [items + 1]: units of tiles of own keys ahead of an item
  PrefixGroup* groups;                     // [groups + 1]
  PrefixAt* begins;                        // [CTAs + 1]
  PrefixRecord* records;                   // [CTAs][PFX_SLOTS]
  float4* part;                            // [CTAs][PFX_SLOTS][d / 4][part_rows]: the rows' pieces of four side by side
  float2* part_ml;                         // [CTAs][PFX_SLOTS][part_rows]
  float4* kept;                            // [CTAs][d / 4][2][128]: sums of either group's rows in long pieces (null: there are none)
  int max_items, ctas, n_groups, part_rows;
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
// (members that do not ascend: no list)
__device__ __forceinline__ int group_end(const PrefixParams& p, int g) { return max(group_begin(p, g + 1), group_begin(p, g)); }
__device__ __forceinline__ int64_t prefix_begin(const PrefixParams& p, int i) {
  if (!p.prefix_offsets) return (int64_t)i * (p.prefix_rows / p.prefixes);
  const int64_t o = p.prefix_offsets[i];
  return o < 0 ? 0 : o > p.prefix_rows ? p.prefix_rows : o;
}
// the list of a row, from lo to hi (that of a later row): the last that begins at it or ahead of it
__device__ __noinline__ int list_of(const Lists& l, int64_t row, int lo, int hi) {
  if (!l.offsets) return l.per > 0 ? (int)((uint32_t)row / (uint32_t)l.per) : 0;      // (rows are counted in 31 bits)
#pragma unroll 1
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (l.begin(mid) <= row) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// the own keys that a row sees: a list's last row sees all of them, each row before it one less
__device__ __noinline__ void own_of(const Lists& lists, const Lists& own, int64_t row, int list, int64_t& lo, int64_t& hi) {
  lo = own.begin(list);
  hi = own.begin(list + 1) - max(lists.begin(list + 1) - 1 - row, (int64_t)0);
  if (hi < lo) hi = lo;
}
// the same of a row in one of some lists, counted from key own0 and cut to own_n
__device__ __noinline__ int2 row_keys(const PrefixParams& p, int row, int list_a, int list_b, int own0, int own_n) {
  int64_t a, b;
  own_of(p.lists, p.own, row, list_of(p.lists, row, list_a, list_b), a, b);
  return make_int2((int)min(max(a - own0, (int64_t)0), (int64_t)own_n), (int)min(max(b - own0, (int64_t)0), (int64_t)own_n));
}
constexpr int PLAN_THREADS = 1024, PLAN_GROUPS = 1024, PLAN_ITEMS = 2048;      // (what shared memory holds of a plan; larger ones are in the workspace alone)
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s_sums, int64_t& total) {      // exclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t t = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += t;
  }
  __syncthreads();                         // (what stands there of the scan before has been read)
  if (lane == 31) s_sums[warp] = x;
  __syncthreads();
  int64_t sums = lane < (int)blockDim.x / 32 ? s_sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t t = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += t;
  }
  total = __shfl_sync(0xffffffffu, sums, 31);
  const int64_t before = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
  return (warp > 0 ? before : 0) + x - v;
}

// Chunk c of a prefix's blocks begins at c blocks / chunks. All items of a group and a head of keys, in the line: for every chunk but the last its
// blocks of item after item, then item after item the last chunk's with the own keys behind them. A block of an item of two tiles counts twice.
__device__ __noinline__ int64_t quotient64(int64_t a, int64_t b) { return a / b; }
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {      // (of numbers that are not negative; 64-bit division takes 100 instructions)
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : quotient64(a, b);
}
__device__ __forceinline__ int chunk_begin(const PrefixGroup& g, int c) { return g.chunks == 1 ? c * g.blocks : (int)quotient((int64_t)c * g.blocks, g.chunks); }
__device__ __forceinline__ int item_blocks(const PrefixItem& x, int prefix_blocks) {
  return max(prefix_blocks + (x.own_n + PFX_KEYS - 1) / PFX_KEYS, 1);        // (an item without keys is one block, for its rows' zeros)
}
__device__ __forceinline__ PrefixAt line_place(const PrefixParams& p, const PrefixGroup* groups, const int64_t* own_weight, int64_t x, int64_t all, int ctas) {
  int lo = 0, hi = p.n_groups - 1;
#pragma unroll 1
  while (lo < hi) {                        // the last group that begins at x or ahead of it
    const int mid = lo + (hi - lo + 1) / 2;
    if (groups[mid].weight * p.Hkv <= x) lo = mid;
    else hi = mid - 1;
  }
  const PrefixGroup g = groups[lo];
  const int n = groups[lo + 1].first - g.first;
  const int64_t weight = groups[lo + 1].weight - g.weight;
  PrefixAt at;
  at.group = lo;
  at.head = (int)quotient(x - g.weight * p.Hkv, weight);
  int64_t r = x - g.weight * p.Hkv - at.head * weight;
  const int last = chunk_begin(g, g.chunks - 1);
  if (r < (int64_t)g.tiles * last) {
    const int u = (int)quotient(r, g.tiles);
    int c = (int)quotient((int64_t)u * g.chunks, g.blocks);
    while (chunk_begin(g, c + 1) <= u) ++c;
    const int b = chunk_begin(g, c), len = chunk_begin(g, c + 1) - b;
    r -= (int64_t)g.tiles * b;
    const int i = (int)min(quotient(r, 2 * len), (int64_t)n - 1), w = i == n - 1 ? g.tiles - 2 * i : 2;
    at.chunk = c; at.item = g.first + i; at.unit = b + (int)(w == 2 ? (r - (int64_t)i * 2 * len) >> 1 : r - (int64_t)i * 2 * len);
    return at;
  }
  r -= (int64_t)g.tiles * last;
  const int rem = g.blocks - last;
  const int64_t own = own_weight[g.first];
  lo = 0;
  hi = n - 1;
#pragma unroll 1
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if ((int64_t)mid * 2 * rem + own_weight[g.first + mid] - own <= r) lo = mid;
    else hi = mid - 1;
  }
  r -= (int64_t)lo * 2 * rem + own_weight[g.first + lo] - own;
  const int w = lo == n - 1 ? g.tiles - 2 * lo : 2;
  at.chunk = g.chunks - 1; at.item = g.first + lo; at.unit = last + (int)(w == 2 ? r >> 1 : r);
  // small items stay whole: what a cut saves is less than joining costs
  if (g.chunks == 1 && at.unit > 0) {
    const int blocks = g.blocks + (int)((own_weight[at.item + 1] - own_weight[at.item]) >> (w - 1));
    if ((int64_t)blocks * w * ctas * 4 <= all) {
      if (2 * at.unit >= blocks) {
        if (lo + 1 < n) {
          ++at.item;
        } else {
          at.item = g.first;
          if (++at.head == p.Hkv) {
            at.head = 0;
            ++at.group;
            while (at.group < p.n_groups && groups[at.group + 1].first == groups[at.group].first) ++at.group;      // (groups without rows)
            at.chunk = 0;
            at.item = at.group < p.n_groups ? groups[at.group].first : 0;
          }
        }
      }
      at.unit = 0;
    }
  }
  return at;
}

// One block: three sums over groups and items and a search a CTA, each behind a read or two from memory. 74 requests of 1000 candidates: 11 us with the
// sums in the workspace, whose every read takes 0.4 us.
__global__ void __launch_bounds__(PLAN_THREADS) prefix_plan_kernel(const __grid_constant__ PrefixParams p) {
  pdl_begin();
  __shared__ int64_t s_sums[PLAN_THREADS / 32], s_own[PLAN_ITEMS + 1];
  __shared__ PrefixGroup s_groups[PLAN_GROUPS + 1];
  const int threads = blockDim.x, n_groups = p.n_groups, step = 2 * p.R;
  PrefixGroup* groups = n_groups <= PLAN_GROUPS ? s_groups : p.groups;
  int64_t total = 0, sum;
#pragma unroll 1
  for (int g0 = 0; g0 < n_groups; g0 += threads) {
    const int g = g0 + (int)threadIdx.x;
    PrefixGroup x = {};
    int64_t n = 0;
    if (g < n_groups) {
      const int64_t rows = p.lists.begin(group_end(p, g)) - p.lists.begin(group_begin(p, g));
      n = rows > 0 ? (rows + step - 1) / step : 0;
      x.tiles = rows > 0 ? (int)((rows + p.R - 1) / p.R) : 0;
      if (g > 0 && g <= p.prefixes) x.blocks = (int)((max(prefix_begin(p, g) - prefix_begin(p, g - 1), (int64_t)0) + PFX_KEYS - 1) / PFX_KEYS);
    }
    const int64_t at = total + block_scan(n, s_sums, sum);
    x.first = (int)min(at, (int64_t)p.max_items);
    // (members that do not ascend name lists twice: a group has the tiles of the items that there is room for)
    if (at + n > p.max_items) x.tiles = (int)min((int64_t)x.tiles, 2 * ((int64_t)p.max_items - x.first));
    if (g < n_groups) groups[g] = x;
    total += sum;
  }
  const int items = (int)min(total, (int64_t)p.max_items);
  int64_t* own_weight = items <= PLAN_ITEMS ? s_own : p.own_weight;
  if (threadIdx.x == 0) {
    const PrefixGroup x = {0, items, 0, 1, 0};
    groups[n_groups] = x;
  }
  __syncthreads();
  int64_t own_total = 0;
#pragma unroll 1
  for (int t0 = 0; t0 < items; t0 += threads) {
    const int t = t0 + (int)threadIdx.x;
    int64_t weight = 0;
    if (t < items) {
      int lo = 0, hi = n_groups - 1;                      // the group: the last that begins at the item or ahead of it
#pragma unroll 1
      while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (groups[mid].first <= t) lo = mid;
        else hi = mid - 1;
      }
      PrefixItem x = {};
      const int l0 = group_begin(p, lo), l1 = group_end(p, lo) - 1;
      const int64_t begin = p.lists.begin(l0) + (int64_t)(t - groups[lo].first) * step;
      const int64_t end = max(min(begin + step, p.lists.begin(l1 + 1)), begin + 1), mid = min(begin + p.R, end);
      x.row0 = (int)begin; x.rows = (int)(end - begin);
      if (lo > 0 && lo <= p.prefixes) {
        const int64_t a = prefix_begin(p, lo - 1), b = prefix_begin(p, lo);
        x.prefix0 = (int)a; x.prefix_n = (int)max(b - a, (int64_t)0);
      }
      x.list[0] = list_of(p.lists, begin, l0, l1);
      x.list[1] = list_of(p.lists, mid - 1, x.list[0], l1);
      x.list[2] = mid < end ? list_of(p.lists, mid, x.list[1], l1) : x.list[1];
      x.list[3] = mid < end ? list_of(p.lists, end - 1, x.list[2], l1) : x.list[1];
      if (p.own.rows > 0) {
        // first and last row of either tile: where their own keys begin and end (all reads at once)
        const int64_t row[4] = {begin, mid - 1, min(mid, end - 1), end - 1};
        int64_t from[4], to[4], last[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) { from[k] = p.own.begin(x.list[k]); to[k] = p.own.begin(x.list[k] + 1); last[k] = p.lists.begin(x.list[k] + 1) - 1; }
#pragma unroll
        for (int k = 0; k < 4; ++k) to[k] = max(to[k] - max(last[k] - row[k], (int64_t)0), from[k]);
        const int64_t b0 = from[0], e0 = to[0], e1 = to[1], b2 = from[2], e2 = to[2], e3 = to[3];
        const int64_t n = max(e3 - b0, (int64_t)0);
        auto in = [&](int64_t k) { return (int)min(max(k - b0, (int64_t)0), n); };
        x.own0 = (int)b0; x.own_n = (int)n; x.end0 = in(e1); x.begin1 = mid < end ? in(b2) : 0;
        x.full0 = x.list[0] == x.list[1] ? in(e0) : 0;
        x.full1 = x.list[2] == x.list[3] ? in(e2) : 0;
      }
      p.items[t] = x;
      const int blocks = (x.prefix_n + PFX_KEYS - 1) / PFX_KEYS;
      weight = (int64_t)(item_blocks(x, blocks) - blocks) * (mid < end ? 2 : 1);
    }
    const int64_t at = own_total + block_scan(weight, s_sums, sum);
    if (t < items) own_weight[t] = at;
    own_total += sum;
  }
  if (threadIdx.x == 0) own_weight[items] = own_total;
  __syncthreads();
  int64_t all = 0;
#pragma unroll 1
  for (int g0 = 0; g0 < n_groups; g0 += threads) {
    const int g = g0 + (int)threadIdx.x;
    int64_t weight = 0;
    if (g < n_groups) weight = (int64_t)groups[g].tiles * groups[g].blocks + own_weight[groups[g + 1].first] - own_weight[groups[g].first];
    const int64_t at = all + block_scan(weight, s_sums, sum);
    if (g < n_groups) groups[g].weight = at;
    all += sum;
  }
  if (threadIdx.x == 0) groups[n_groups].weight = all;
  all *= p.Hkv;
  const int ctas = (int)min(all, (int64_t)p.ctas);
#pragma unroll 1
  for (int g = threadIdx.x; g < n_groups; g += threads) {
    // (several items, each longer than a part: as many chunks as parts of an item)
    const int64_t chunks = groups[g].tiles > 2 && all > 0 ? quotient(2 * (int64_t)groups[g].blocks * ctas, all) : 1;
    groups[g].chunks = (int)max(min(chunks, (int64_t)groups[g].blocks), (int64_t)1);
  }
  __syncthreads();
#pragma unroll 1
  for (int c = threadIdx.x; c <= p.ctas; c += threads) {
    PrefixAt at = {n_groups, 0, 0, 0, 0};
    if (c < ctas) at = line_place(p, groups, own_weight, quotient(all * c, ctas), all, ctas);
    p.begins[c] = at;
  }
  if (groups == s_groups)
#pragma unroll 1
    for (int g = threadIdx.x; g <= n_groups; g += threads) p.groups[g] = s_groups[g];
}

// ---- the kernel ----
// A CTA's pieces in order: an item, its blocks of keys [k0, k1), and whether these are all of them.
struct PrefixPiece {
  PrefixItem t;
  int item, head, k0, k1, prefix_blocks, slot;
  int clean0, clean1, clean2;              // blocks [clean0, clean1) and from clean2 on hold values that some row does not see beside ones that it does
  bool valid;                              // (false: there are no more)
  bool whole, two;                         // two tiles
  bool empty;                              // no keys: the rows' zeros
  // The blocks of either group of warps: of a single tile every other one, else what its tile's rows see: all but [hole0, hole1), up to `end`.
  struct Walk {
    int begin, end, n;
  } walk[2];
  int step, hole0, hole1;
  // (by comparison: a place counted at run time would put the piece into memory)
  __device__ __forceinline__ Walk of(int w) const { return {w ? walk[1].begin : walk[0].begin, w ? walk[1].end : walk[0].end, w ? walk[1].n : walk[0].n}; }
  __device__ __forceinline__ bool cleaned(int j) const { return (j >= clean0 && j < clean1) || j >= clean2; }
  __device__ __forceinline__ int next(int w, int j) const {
    j += step;
    return w == 1 && j >= hole0 && j < hole1 ? hole1 : j;
  }
};
template <int DP>
struct PrefixShape {
  static constexpr int Q = DP == 128 ? 1 : 2, K = DP == 128 ? 3 : 5, V = DP == 128 ? 2 : 5;     // buffers (of queries: an item's)
  static constexpr int TILE = 128 * DP * 2, BOX = 128 * 128;
  struct Control {                         // behind the buffers (the kernel has no other shared memory, so that its buffers begin on 1024 bytes)
    uint64_t q_full[Q], q_empty[Q], k_full[K], k_empty[K], v_full[V], v_clean[V], v_empty[V];
    uint64_t s_full[2], s_read[2], p_ready[2], o_done[2], o_free[2], met, drained[2];
    uint64_t piece_full[PFX_RING], piece_empty[PFX_RING];
    PrefixPiece ring[PFX_RING];
    float2 ml[2][PFX_ROWS];                // maximum and sum of either group's rows
    // Of the two pieces that are under way the first and the last block in which bad values were found: the piece's number + 1 in the high word, the block
    // (the first one's counted down) in the low one.
    unsigned long long bad_first[2], bad_last[2];
    int lock, progress;
    uint32_t tmem;
  };
  static constexpr int SMEM = (2 * Q + K + V) * TILE + (int)sizeof(Control);
  static_assert(SMEM <= 227 * 1024 - 64, "");
  // Columns of tensor memory: the scores of both groups, their sums; weights where there is room, else over the scores that they are made of
  // (whose next ones then wait for the weights' product).
  static constexpr bool APART = DP == 64;
  static constexpr uint32_t S = 0, O = 256, P = APART ? 384 : 0, P_STEP = APART ? 64 : 128;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
// mbar_wait with a limit on its tries, each of which ends after a microsecond at the latest: it stands in the code in many places, and takes a
// quarter of the instructions of one that looks at the clock.
constexpr int PFX_TRIES = 1 << 21;
__device__ __forceinline__ bool mbar_spin(uint32_t bar, uint32_t parity, int site) {
  if (umma::mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (int i = 0; i < PFX_TRIES; ++i)
    if (umma::mbar_try_wait_for(bar, parity, 1000u)) return true;
  umma::wait_gave_up(site);
  return false;
}
// One that may last as long as a piece, whose blocks only the memory bounds (a group of warps that has nothing to do in it waits for what comes behind): the limit
// is on the time in which nothing goes on (`progress`: blocks asked for). Everywhere it would cost 4 to 8 %.
__device__ __forceinline__ bool mbar_spin_long(uint32_t bar, uint32_t parity, const int* progress, int site) {
  if (umma::mbar_try_wait(bar, parity)) return true;
  int seen = -1;
#pragma unroll 1
  for (int now = 0; now != seen;) {
    seen = now;
#pragma unroll 1
    for (int i = 0; i < PFX_TRIES; ++i)
      if (umma::mbar_try_wait_for(bar, parity, 1000u)) return true;
    now = *reinterpret_cast<const volatile int*>(progress);
  }
  umma::wait_gave_up(site);
  return false;
}
__device__ __forceinline__ void mbar_arrive_twice(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], 2;" ::"r"(bar) : "memory"); }
// A lock between two warps, held for the time of a product and the issue of the scores behind it. False: it was not to be had (with the limit of the waits).
__device__ __forceinline__ bool take(int* lock, int lane) {
  int ok = 1;
  if (lane == 0) {
    int tries = 0;
#pragma unroll 1
    while (atomicCAS(lock, 0, 1) != 0 && ++tries < PFX_TRIES) {}
    if (tries == PFX_TRIES) {
      umma::wait_gave_up(99);
      ok = 0;
    }
  }
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
__device__ __forceinline__ void let_go(int* lock, int lane) {
  __syncwarp();
  if (lane == 0) atomicExch(lock, 0);
  __syncwarp();
}
// shares of a launch's registers: every warp of four that begin at a multiple of four
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <bool BF16>
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// A value that all lanes have, told to the compiler as such: what the MMAs take then stands in uniform registers.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
// the lowest n bits, n cut to [0, 32]
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }

// A CTA's pieces are worked out by a warp of their own, ahead of the others, which take them from a ring in shared memory: the plan's reads, each
// behind the other, stand in nobody's way, and the walk is in the code once.
template <typename F>
__device__ __forceinline__ void make_pieces(const PrefixParams& p, F put) {
  PrefixAt at = p.begins[blockIdx.x];
  const PrefixAt to = p.begins[blockIdx.x + 1];
  int slot = 0;
#pragma unroll 1
  while (at.group < to.group || (at.group == to.group && at.group < p.n_groups)) {
    const bool here = at.group == to.group && at.head == to.head && at.chunk == to.chunk && at.item == to.item;
    if (here && at.unit >= to.unit) return;
    const PrefixGroup g = p.groups[at.group];
    const int behind = p.groups[at.group + 1].first;
    PrefixPiece x;
    x.t = p.items[at.item];
    x.item = at.item;
    x.head = at.head;
    x.prefix_blocks = g.blocks;
    const int blocks = item_blocks(x.t, g.blocks), end = at.chunk == g.chunks - 1 ? blocks : chunk_begin(g, at.chunk + 1);
    x.k0 = at.unit;
    x.k1 = here ? to.unit : end;
    x.whole = x.k0 == 0 && x.k1 == blocks;
    x.two = x.t.rows > p.R;
    x.empty = x.t.prefix_n + x.t.own_n == 0;
    x.valid = true;
    x.slot = min(slot, PFX_SLOTS - 1);
    // (a prefix's last block, if it is not full; own blocks but those that all rows see whole: of one list, which all of the item's rows are in)
    x.clean0 = x.t.prefix_n % PFX_KEYS ? g.blocks - 1 : g.blocks;
    x.clean1 = g.blocks;
    x.clean2 = g.blocks + (x.t.list[0] == x.t.list[3] ? min(x.t.full0, x.t.own_n) / PFX_KEYS : 0);
    x.step = x.two ? 1 : 2;
    x.hole0 = x.two ? g.blocks : 0;
    x.hole1 = x.two ? g.blocks + x.t.begin1 / PFX_KEYS : 0;
    const int end0 = x.two ? min(x.k1, g.blocks + (x.t.end0 + PFX_KEYS - 1) / PFX_KEYS) : x.k1;
    x.walk[0] = {x.k0, end0, max((end0 - x.k0 + x.step - 1) / x.step, 0)};
    const int first1 = x.two ? (x.k0 >= x.hole0 && x.k0 < x.hole1 ? x.hole1 : x.k0) : x.k0 + 1;
    const int left_out = x.two ? max(min(x.hole1, x.k1) - max(x.hole0, first1), 0) : 0;
    x.walk[1] = {first1, x.k1, max((x.k1 - first1 + x.step - 1) / x.step - left_out, 0)};
    if (!put(x) || here) return;
    if (!x.whole) ++slot;
    if (++at.item == behind) {
      at.item = g.first;
      if (++at.chunk == g.chunks) {
        at.chunk = 0;
        if (++at.head == p.Hkv) {
          at.head = 0;
          do ++at.group;
          while (at.group < p.n_groups && p.groups[at.group + 1].first == p.groups[at.group].first);
          if (at.group >= p.n_groups) return;
          at.item = p.groups[at.group].first;
        }
      }
    }
    at.unit = chunk_begin(p.groups[at.group], at.chunk);
  }
}
// false: a wait ran out. AHEAD: a warp that may be done with pieces that others are still at (the loader, the MMAs and the clearing go through all blocks).
template <bool AHEAD, typename C, typename F>
__device__ __forceinline__ bool each_piece(C& ctl, int lane, F visit) {
#pragma unroll 1
  for (int n = 0;; ++n) {
    const uint32_t full = umma::smem_u32(&ctl.piece_full[n % PFX_RING]), parity = (uint32_t)(n / PFX_RING) & 1u;
    if (!__all_sync(0xffffffffu, AHEAD ? mbar_spin_long(full, parity, &ctl.progress, 80) : mbar_spin(full, parity, 80))) return false;
    const PrefixPiece x = ctl.ring[n % PFX_RING];
    __syncwarp();
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&ctl.piece_empty[n % PFX_RING]));
    if (!x.valid) return true;
    if (!visit(x)) return false;
  }
}

// Infinities and NaN among own values, which the products were made without, added to a row's results or sums (whose own, of a prefix or of scores, they
// meet there). For columns [c0, c1) and keys [k0, k1).
template <bool BF16>
__device__ __noinline__ void spread_bad(const Heads v, int64_t row0, int head, int c0, int c1, int k0, int k1, uint16_t* y, float* part, int64_t part_step) {
#pragma unroll 1
  for (int c = c0; c < c1; c += 8) {       // (rows are on 16 bytes, columns whole pieces of 8)
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = k0; k < k1; ++k) {
      const uint4 t = *reinterpret_cast<const uint4*>(v.get<uint16_t>(row0 + k, head) + c);
      const uint32_t h[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t x = (uint16_t)(h[e / 2] >> (16 * (e & 1)));
        if (half_is_bad<BF16>(x)) sum[e] += BF16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (sum[e] == 0.f) continue;
      if (y) {
        const float all = sum[e] + (BF16 ? __uint_as_float((uint32_t)y[c + e] << 16) : __half2float(__ushort_as_half(y[c + e])));
        y[c + e] = (uint16_t)pack_weights<BF16>(all, all);
      } else {
        part[((c + e) / 4) * part_step + e % 4] += sum[e];
      }
    }
  }
}

// The tensor cores cut off what they add below 2^-23 of a running sum, 8 times a block: over 1000 blocks of equal keys that is 0.04 % of the sum, over 32 768
// 1.4 %. So sums of long pieces leave them every PFX_KEPT blocks, for fp32 ones in the workspace, which are rounded: (those so far, moved from their maximum to m)
// + the tensor cores', of a row's d columns, when `done` has come to its phase. `back`: the sum goes to tensor memory. False: a wait ran out.
__device__ __noinline__ bool keep_sums(uint32_t done, uint32_t phase, uint32_t tmem, float4* kept, int d, float* max, float m, float scale, bool more, bool back) {
  if (!__all_sync(0xffffffffu, mbar_spin(done, phase & 1u, 78))) return false;
  umma::tc_fence_after_sync();
  const float before = *max, by = before == m || before == -INFINITY ? 1.f : ex2((before - m) * scale);
  *max = m;
#pragma unroll 1
  for (int c = 0; c < d; c += 16) {
    uint32_t o[16];
    umma::tmem_ld16_nowait(tmem + c, o);
    umma::tmem_wait_ld(o);
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      if (c + e >= d) break;
      float4* at = kept + (c + e) / 4 * (2 * PFX_ROWS);
      float4 t = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
      if (more) {
        const float4 k = *at;
        t.x = fmaf(k.x, by, t.x); t.y = fmaf(k.y, by, t.y); t.z = fmaf(k.z, by, t.z); t.w = fmaf(k.w, by, t.w);
      }
      if (back) {
        o[e] = __float_as_uint(t.x); o[e + 1] = __float_as_uint(t.y); o[e + 2] = __float_as_uint(t.z); o[e + 3] = __float_as_uint(t.w);
      } else {
        *at = t;
      }
    }
    __syncwarp();                          // the lanes meet ahead of the next access to tensor memory
    if (back) umma::tmem_st16(tmem + c, o);
  }
  if (back) {
    umma::tmem_wait_st();
    umma::tc_fence_before_sync();
  }
  return true;
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(PFX_THREADS, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                        const __grid_constant__ CUtensorMap map_pk, const __grid_constant__ CUtensorMap map_pv, const __grid_constant__ PrefixParams p) {
  using namespace umma;
  using T = PrefixShape<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *smem_q = smem, *smem_k = smem_q + 2 * T::Q * T::TILE, *smem_v = smem_k + T::K * T::TILE;
  typename T::Control& ctl = *reinterpret_cast<typename T::Control*>(smem_v + T::V * T::TILE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < T::Q; ++s) { mbar_init(smem_u32(&ctl.q_full[s]), 1); mbar_init(smem_u32(&ctl.q_empty[s]), 10); }
    for (int s = 0; s < T::K; ++s) { mbar_init(smem_u32(&ctl.k_full[s]), 1); mbar_init(smem_u32(&ctl.k_empty[s]), 2); }
    for (int s = 0; s < T::V; ++s) { mbar_init(smem_u32(&ctl.v_full[s]), 1); mbar_init(smem_u32(&ctl.v_clean[s]), 128); mbar_init(smem_u32(&ctl.v_empty[s]), 3); }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&ctl.s_full[w]), 1);
      mbar_init(smem_u32(&ctl.s_read[w]), 128);
      mbar_init(smem_u32(&ctl.p_ready[w]), 128);
      mbar_init(smem_u32(&ctl.o_done[w]), 1);
      mbar_init(smem_u32(&ctl.o_free[w]), 256);
      mbar_init(smem_u32(&ctl.drained[w]), 1);
      ctl.bad_first[w] = ctl.bad_last[w] = 0;
    }
    for (int r = 0; r < PFX_RING; ++r) { mbar_init(smem_u32(&ctl.piece_full[r]), 1); mbar_init(smem_u32(&ctl.piece_empty[r]), PFX_TAKERS); }
    mbar_init(smem_u32(&ctl.met), 256);
    ctl.lock = ctl.progress = 0;
    fence_barrier_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    prefetch_tensormap(&map_pk);
    prefetch_tensormap(&map_pv);
  }
  if (warp == PFX_MMA) tmem_alloc(smem_u32(&ctl.tmem), 512);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = ctl.tmem;
  pdl_wait();

  if (warp >= 12) {
    registers_down<48>();                  // (a launch gives 512 threads 128 each: 2 x 192 + 80 + 48 is the same)
    // Zero weights take no part only beside finite values: in blocks that not all rows see whole, rows behind the keys become zeros, and of own keys
    // infinities and NaN too (what they are to the rows that see them is made up for at the end).
    const int thread = threadIdx.x & 127;
    int vn = 0, pieces = 0;
    each_piece<false>(ctl, lane, [&](const PrefixPiece& x) {
      if (x.empty) return true;
#pragma unroll 1
      for (int j = x.k0; j < x.k1; ++j, ++vn) {
        const int s = vn % T::V;
        if (!__all_sync(0xffffffffu, mbar_spin(smem_u32(&ctl.v_full[s]), (uint32_t)(vn / T::V) & 1u, 94))) return false;
        if (x.cleaned(j)) {
          const bool prefix = j < x.prefix_blocks;
          const int in = min(PFX_KEYS, prefix ? x.t.prefix_n - j * PFX_KEYS : x.t.own_n - (j - x.prefix_blocks) * PFX_KEYS);      // keys of the block
          uint8_t* v = smem_v + s * T::TILE;
#pragma unroll 1
          for (int e = in * 8 + thread; e < 1024; e += 128)
#pragma unroll
            for (int b = 0; b < DP / 64; ++b) *reinterpret_cast<uint4*>(v + b * T::BOX + e * 16) = make_uint4(0u, 0u, 0u, 0u);
          if (!prefix) {
            uint32_t sick = 0u;            // (0 * t is 0 but for those)
#pragma unroll 4
            for (int e = 0; e < DP / 64 * 8; ++e) {
              if (thread + e % 8 * 128 >= in * 8) continue;
              const uint4 t = *reinterpret_cast<const uint4*>(v + e / 8 * T::BOX + (thread + e % 8 * 128) * 16);
              sick = fma_zero<BF16>(t.x, sick);
              sick = fma_zero<BF16>(t.y, sick);
              sick = fma_zero<BF16>(t.z, sick);
              sick = fma_zero<BF16>(t.w, sick);
            }
            if (half_is_bad<BF16>(sick) || half_is_bad<BF16>(sick >> 16)) {
              const unsigned long long piece = (unsigned long long)(pieces + 1) << 32;
              atomicMax(&ctl.bad_first[pieces & 1], piece | (unsigned)(INT32_MAX - j));
              atomicMax(&ctl.bad_last[pieces & 1], piece | (unsigned)j);
#pragma unroll 1
              for (int e = thread; e < in * 8; e += 128)
#pragma unroll 1
                for (int b = 0; b < DP / 64; ++b) {
                  uint32_t* h = reinterpret_cast<uint32_t*>(v + b * T::BOX + e * 16);
#pragma unroll 1
                  for (int z = 0; z < 4; ++z) h[z] &= (half_is_bad<BF16>(h[z]) ? 0u : 0xffffu) | (half_is_bad<BF16>(h[z] >> 16) ? 0u : 0xffff0000u);
                }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        mbar_arrive(smem_u32(&ctl.v_clean[s]));
        bool fine = true;                  // (its buffer is loaded again only when all have been here)
        if (thread == 0) {
          fine = mbar_spin(smem_u32(&ctl.v_clean[s]), (uint32_t)(vn / T::V) & 1u, 94);
          mbar_arrive(smem_u32(&ctl.v_empty[s]));
        }
        if (!__all_sync(0xffffffffu, fine)) return false;
      }
      ++pieces;
      return true;
    });
  } else if (warp >= 8) {
    registers_down<80>();
    if (warp == PFX_LOADER) {
      int qn = 0, kn = 0, vn = 0;          // items and blocks asked for so far
      bool ok = true;
      each_piece<false>(ctl, lane, [&](const PrefixPiece& x) {
        if (x.empty) return true;
        const int qs = qn % T::Q;
        if (!(ok = __all_sync(0xffffffffu, mbar_spin(smem_u32(&ctl.q_empty[qs]), ((uint32_t)(qn / T::Q) & 1u) ^ 1u, 81)))) return false;
        if (lane == 0) {
          const uint32_t bar = smem_u32(&ctl.q_full[qs]), dst = smem_u32(smem_q + qs * 2 * T::TILE);
          mbar_arrive_expect_tx(bar, (uint32_t)((x.two ? 2 : 1) * DP / 64 * 128 * p.share * p.R));
          for (int t = 0; t < (x.two ? 2 : 1); ++t)
#pragma unroll
            for (int b = 0; b < DP / 64; ++b) tma_load_4d(dst + t * T::TILE + b * T::BOX, &map_q, bar, b * 64, 0, x.head, x.t.row0 + t * p.R);
        }
        ++qn;
        // keys a block ahead of values
        const int n = 2 * (x.k1 - x.k0);
#pragma unroll 1
        for (int i = 0; i < n + 1; ++i) {
          // K0, K1, V0, K2, V1, ..: odd places but the first are keys
          const bool keys = i == 0 || (i & 1) == 1;
          const int j = x.k0 + (i == 0 ? 0 : keys ? (i + 1) / 2 : i / 2 - 1);
          if (j >= x.k1) continue;
          const bool prefix = j < x.prefix_blocks;
          const int row = prefix ? x.t.prefix0 + j * PFX_KEYS : x.t.own0 + (j - x.prefix_blocks) * PFX_KEYS;
          const int s = keys ? kn % T::K : vn % T::V, turn = keys ? kn / T::K : vn / T::V;
          const uint32_t empty = smem_u32(keys ? &ctl.k_empty[s] : &ctl.v_empty[s]), full = smem_u32(keys ? &ctl.k_full[s] : &ctl.v_full[s]);
          if (!(ok = __all_sync(0xffffffffu, mbar_spin(empty, ((uint32_t)turn & 1u) ^ 1u, keys ? 82 : 83)))) return false;
          if (lane == 0) {
            const uint32_t dst = smem_u32((keys ? smem_k : smem_v) + s * T::TILE);
            const CUtensorMap* map = keys ? (prefix ? &map_pk : &map_k) : (prefix ? &map_pv : &map_v);
            mbar_arrive_expect_tx(full, (uint32_t)T::TILE);
#pragma unroll
            for (int b = 0; b < DP / 64; ++b) tma_load_3d(dst + b * T::BOX, map, full, b * 64, x.head, row);
            atomicAdd(&ctl.progress, 1);
          }
          kn += keys;
          vn += !keys;
        }
        return true;
      });
      if (!ok) {                           // nothing that was asked for arrives after this CTA has ended
        for (int i = 1; i <= T::Q && i <= qn; ++i) mbar_spin(smem_u32(&ctl.q_full[(qn - i) % T::Q]), (uint32_t)((qn - i) / T::Q) & 1u, 84);
        for (int i = 1; i <= T::K && i <= kn; ++i) mbar_spin(smem_u32(&ctl.k_full[(kn - i) % T::K]), (uint32_t)((kn - i) / T::K) & 1u, 84);
        for (int i = 1; i <= T::V && i <= vn; ++i) mbar_spin(smem_u32(&ctl.v_full[(vn - i) % T::V]), (uint32_t)((vn - i) / T::V) & 1u, 84);
      }
    } else if (warp == PFX_MMA + 2) {
      int n = 0;
      bool ok = true;
      auto put = [&](const PrefixPiece& x) {
        if (!(ok = __all_sync(0xffffffffu, mbar_spin_long(smem_u32(&ctl.piece_empty[n % PFX_RING]), ((uint32_t)(n / PFX_RING) & 1u) ^ 1u, &ctl.progress, 79)))) return false;
        if (lane == 0) {
          ctl.ring[n % PFX_RING] = x;
          mbar_arrive(smem_u32(&ctl.piece_full[n % PFX_RING]));
        }
        __syncwarp();
        ++n;
        return true;
      };
      make_pieces(p, put);
      if (ok) {
        PrefixPiece none = {};
        put(none);
      }
    } else if (warp < PFX_MMA + 2) {
      // A warp for each group. Where a group's weights lie over its scores, its product and the scores after it are made at a stretch, one group
      // at a time (the lock): the groups fall out of step, one's MMAs beside the other's weights. (Without the lock both groups wait for both: 179 us in place
      // of 173 for the rows below; with the lock let go between the two 182; one warp for both spends 400 cycles between MMAs looking for what is ready.)
      constexpr int FMT = BF16 ? 1 : 0;
      const int w = warp - PFX_MMA;
      const uint32_t idesc_s = make_idesc(128, PFX_KEYS, FMT), idesc_o = make_idesc(128, DP, FMT) | IDESC_B_MN;
      const uint32_t to_s = uniform(tmem + T::S + w * 128), to_o = uniform(tmem + T::O + w * DP), from_p = uniform(tmem + T::P + w * T::P_STEP);
      int qn = 0, kn = 0, vn = 0, pieces = 0;              // items; blocks whose keys and values are behind this warp
      int on = 0;                                          // its products so far
      bool ok = true;
      auto wait = [&](uint64_t* bar, int phase, int site) { return ok = __all_sync(0xffffffffu, mbar_spin(smem_u32(bar), (uint32_t)phase & 1u, site)); };
      each_piece<false>(ctl, lane, [&](const PrefixPiece& x) {
        if (x.empty) return true;
        const int qs = qn % T::Q, k_first = kn, v_first = vn;
        if (!wait(&ctl.q_full[qs], qn / T::Q, 85)) return false;
        const uint64_t q = make_desc_sw128(uniform(smem_u32(smem_q + (qs * 2 + (x.two ? w : 0)) * T::TILE)), 1024);
        // Blocks ahead of j that this group has no use for are given back: one after the other, keys and values, as they are loaded (keys alone
        // only where a block or two lie between: a loader that waits for buffers of values loads no keys either).
        auto give_back = [&](int j, bool values) {
          const int n = j - x.k0;
#pragma unroll 1
          while (kn - k_first < n || (values && vn - v_first < n)) {
            if (kn - k_first < n) {
              if (!wait(&ctl.k_full[kn % T::K], kn / T::K, 86)) return false;
              if (lane == 0) mbar_arrive(smem_u32(&ctl.k_empty[kn % T::K]));
              ++kn;
            }
            if (values && vn - v_first < min(kn - k_first, n)) {
              if (!wait(&ctl.v_full[vn % T::V], vn / T::V, 86)) return false;
              if (lane == 0) mbar_arrive(smem_u32(&ctl.v_empty[vn % T::V]));
              ++vn;
            }
          }
          return true;
        };
        auto keys_of = [&](int j, bool values) { return give_back(j, values) && wait(&ctl.k_full[kn % T::K], kn / T::K, 86); };
        // The blocks in order, a step behind: scores of block `ask`, then the product with the weights of the block before it. Where these lie over the
        // scores, the product comes first.
        const int end = x.of(w).end;
        int ask = x.of(w).begin, j = end;                // (j: the block whose weights come next; none yet)
        bool first = true;
        int since = 0;                                   // products since the sums have last been taken out
#pragma unroll 1
        while (ask < end || j < end) {
          // a block further on than two: the loader may wait for this block's values to be done with
          const bool near = j >= end || ask - j <= 2;
          const bool product_first = j < end && (!T::APART || !near || ask >= end);
          bool held = false;
#pragma unroll 1
          for (int turn = 0; turn < 2; ++turn) {
            if ((turn == 0) == product_first) {
              if (j >= end) continue;
              if (near && ask < end && product_first && !keys_of(ask, false)) return false;
              if (!give_back(j, true)) return false;
              const int s = vn % T::V;
              const uint64_t v = make_desc_sw128_mn(uniform(smem_u32(smem_v + s * T::TILE)), T::BOX);
              // (v_full first: a buffer is loaded again when the one before has been cleaned, and a phase of v_clean is told from the one before it only then;
              // blocks that this group gave back may not have been. One wait in the code: with two, 512 rows of 4 heads of 128 on 100003 keys take 176 us, not 165.)
#pragma unroll 1
              for (int c = 0; c < (x.cleaned(j) ? 2 : 1); ++c)
                if (!wait(c ? &ctl.v_clean[s] : &ctl.v_full[s], vn / T::V, 89)) return false;
              // (in this order: with its first weights of the piece the group has seen the phase ahead of o_free's, which is told from it only then)
              if (!wait(&ctl.p_ready[w], on, 88)) return false;
              if (first && pieces > 0 && !wait(&ctl.o_free[w], pieces - 1, 90)) return false;
              if (!T::APART && !(ok = held = take(&ctl.lock, lane))) return false;
              tc_fence_after_sync();
#pragma unroll
              for (int kk = 0; kk < PFX_KEYS / 16; ++kk) mma_f16_ts_elect(to_o, from_p + kk * 8, v + kk * 128, idesc_o, (since > 0 || kk > 0) ? 1u : 0u);
              mma_commit_elect(smem_u32(&ctl.o_done[w]));
              mma_commit_elect(smem_u32(&ctl.v_empty[s]));
              ++vn;
              ++on;
              first = false;
              if (++since == PFX_KEPT) since = 0;
              if (held && !near) {
                let_go(&ctl.lock, lane);
                held = false;
              }
            } else if (ask < end) {
              if (!held && !keys_of(ask, j >= end || !near)) return false;
              if (T::APART && j < end && !product_first && !wait(&ctl.s_read[w], on, 87)) return false;      // (the scores before these have been read)
              // Scores over weights: the product that reads these has ended (products and scores have different accumulators, and no order is promised
              // between MMAs of which one writes what another reads). 512 rows of 4 heads of 128 on 100003 keys: 169 us without this wait, 173 with it, when it came in.
              if (!T::APART && on > 0 && !wait(&ctl.o_done[w], on - 1, 77)) return false;
              const int s = kn % T::K;
              // (a descriptor's address counts 16 bytes: a step of 16 elements is 2, a box of 64 columns 1024)
              const uint64_t k = make_desc_sw128(uniform(smem_u32(smem_k + s * T::TILE)), 1024);
              tc_fence_after_sync();
#pragma unroll
              for (int kk = 0; kk < DP / 16; ++kk)
                mma_f16_ss_elect(to_s, q + (kk / 4) * (T::BOX / 16) + (kk % 4) * 2, k + (kk / 4) * (T::BOX / 16) + (kk % 4) * 2, idesc_s, kk > 0 ? 1u : 0u);
              mma_commit_elect(smem_u32(&ctl.s_full[w]));
              mma_commit_elect(smem_u32(&ctl.k_empty[s]));
              ++kn;
            }
          }
          if (held) let_go(&ctl.lock, lane);
          j = ask;
          if (ask < end) ask = x.next(w, ask);
        }
        if (!give_back(x.k1, true)) return false;
        if (first) {
          if (lane == 0) mbar_arrive(smem_u32(&ctl.q_empty[qs]));
        } else {
          mma_commit_elect(smem_u32(&ctl.q_empty[qs]));
        }
        ++qn;
        ++pieces;
        return true;
      });
      if (!ok) {                           // the products in flight end before their tensor memory is given back
        mma_commit_elect(smem_u32(&ctl.drained[w]));
        mbar_spin(smem_u32(&ctl.drained[w]), 0, 91);
      }
    }
  } else {
    registers_up<192>();
    const int w = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) * 32u << 16;
    const uint32_t my_s = tmem + T::S + w * 128 + lanes, my_p = tmem + T::P + w * T::P_STEP + lanes, my_o = tmem + T::O + w * DP + lanes;
    int sn = 0, pieces = 0, mets = 0;      // this group's blocks; pieces with keys; meetings of the groups
    int other = 0;                                         // the other group's blocks
    int slots = 0;
    auto wait = [&](uint64_t* bar, int phase, int site) { return __all_sync(0xffffffffu, mbar_spin(smem_u32(bar), (uint32_t)phase & 1u, site)); };
    auto wait_long = [&](uint64_t* bar, int phase, int site) {
      return __all_sync(0xffffffffu, mbar_spin_long(smem_u32(bar), (uint32_t)phase & 1u, &ctl.progress, site));
    };
    each_piece<true>(ctl, lane, [&](const PrefixPiece& x) {
      const int tile = x.two ? w : 0, tile_row = tile * p.R + row / p.share;
      const bool there = row < p.R * p.share && tile_row < x.t.rows;
      const int64_t q_row = (int64_t)x.t.row0 + tile_row;
      const int q_head = x.head * p.share + row % p.share;
      // The own keys that the row sees, counted from the item's first. Where its list needs no search the offsets are read now and used when the first
      // own block comes; else when the first block is out of hand.
      int lo = 0, hi = 0;
      bool known = x.t.own_n == 0;
      const int list_a = tile ? x.t.list[2] : x.t.list[0], list_b = tile ? x.t.list[3] : x.t.list[1];
      const int list = !p.lists.offsets ? (int)((uint32_t)q_row / (uint32_t)p.lists.per) : list_a == list_b ? list_a : -1;
      const bool early = there && !known && list >= 0 && list < p.lists.batch;
      int raw_own[2] = {0, 0}, raw_behind = 0;             // (as they stand in memory: nothing is made of them before they are needed)
      if (early) {
        if (p.own.offsets) { raw_own[0] = p.own.offsets[list]; raw_own[1] = p.own.offsets[list + 1]; }
        if (p.lists.offsets) raw_behind = p.lists.offsets[list + 1];
      }
      auto know = [&]() {
        known = true;
        if (early) {
          auto cut = [](const Lists& of, int raw, int i) { return of.offsets ? min(max((int64_t)raw, (int64_t)0), of.rows) : (int64_t)i * of.per; };
          const int64_t begin = cut(p.own, raw_own[0], list), last = cut(p.own, raw_own[1], list + 1) - max(cut(p.lists, raw_behind, list + 1) - 1 - q_row, (int64_t)0);
          lo = (int)min(max(begin - x.t.own0, (int64_t)0), (int64_t)x.t.own_n);
          hi = (int)min(max(max(last, begin) - x.t.own0, (int64_t)0), (int64_t)x.t.own_n);
        } else if (there) {
          const int2 keys = row_keys(p, (int)q_row, list_a, list_b, x.t.own0, x.t.own_n);
          lo = keys.x;
          hi = keys.y;
        }
        __syncwarp();
      };
      float m = -INFINITY, l = 0.f;
      int mine = 0;
      int stop = x.of(w).n > PFX_KEPT ? PFX_KEPT - 1 : -1;                                    // the block behind which sums are taken out, at the last one put back
      if (!x.empty) {
        const int end = x.of(w).end;
#pragma unroll 1
        for (int j = x.of(w).begin; j < end; j = x.next(w, j), ++mine) {
          const bool prefix = j < x.prefix_blocks;
          const int key0 = (prefix ? j : j - x.prefix_blocks) * PFX_KEYS;
          const int in = min(PFX_KEYS, (prefix ? x.t.prefix_n : x.t.own_n) - key0);           // keys of the block
          const bool masked = in < PFX_KEYS || (!prefix && (key0 < (tile ? x.t.begin1 : 0) || key0 + PFX_KEYS > (tile ? x.t.full1 : x.t.full0)));
          if (masked && !prefix && !known) know();
          if (!wait_long(&ctl.s_full[w], sn, 92)) return false;
          tc_fence_after_sync();
          // Sums so far are moved to a maximum that has grown. (m is -infinity: nothing has been summed; no maximum yet: nothing to move.)
          auto move_sums = [&](float next) {
            if (__any_sync(0xffffffffu, there && (next - m) * p.scale > PFX_GROWTH)) {       // (what stands in rows that are none has no say in the others' roundings)
              const float by = m == next || m == -INFINITY ? 1.f : ex2((m - next) * p.scale);
              m = next;
              l *= by;
              if (mine % PFX_KEPT == 0) return true;       // (the tensor cores have none)
              if (!wait(&ctl.o_done[w], sn - 1, 93)) return false;
              tc_fence_after_sync();
#pragma unroll 1
              for (int c = 0; c < DP; c += 16) {
                uint32_t o[16];
                tmem_ld16_nowait(my_o + c, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * by);
                tmem_st16(my_o + c, o);
              }
              return true;
            }
            return !T::APART || mine == 0 || wait(&ctl.o_done[w], sn - 1, 93);                // (the weights before these have been read)
          };
          // The exponents: scale s - scale m in one FMA. A rounded scale m is the same factor to all of a row's weights, but of scores far beyond
          // what a softmax tells apart (masks of the type's lowest value) it would be a large one: those have m taken off first.
          const f32x2 by2 = pack2(p.scale, p.scale);
          f32x2 sum[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
          auto weigh = [&](const uint32_t (&q)[32], float base, uint32_t (&to)[16]) {
            const f32x2 base2 = pack2(-base, -base);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float a, b;
              unpack2(fma2(pack2(__uint_as_float(q[e]), __uint_as_float(q[e + 1])), by2, base2), a, b);
              a = ex2(a);
              b = ex2(b);
              sum[e / 2 % 2] = add2(sum[e / 2 % 2], pack2(a, b));
              to[e / 2] = pack_weights<BF16>(a, b);
            }
          };
          if (!masked || prefix) {
            uint32_t s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_nowait(my_s + c * 32, s[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_wait_ld(s[c]);
            if (T::APART) {
              tc_fence_before_sync();
              mbar_arrive(smem_u32(&ctl.s_read[w]));
            }
            if (masked) {                  // (a prefix's last keys: the same for all rows)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                if (in >= 32 * c + 32) continue;
                const uint32_t seen = bits_below(in - 32 * c);
#pragma unroll
                for (int e = 0; e < 32; ++e) s[c][e] = seen >> e & 1 ? s[c][e] : 0xff800000u;
              }
            }
            float top[4] = {m, m, m, m};
#pragma unroll
            for (int c = 0; c < 128; c += 2) top[c / 2 % 4] = fmaxf(top[c / 2 % 4], fmaxf(__uint_as_float(s[c / 32][c % 32]), __uint_as_float(s[c / 32][c % 32 + 1])));
            if (!move_sums(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])))) return false;
            float base = (m == -INFINITY ? 0.f : m * p.scale) - PFX_UP<BF16>;
            if (__any_sync(0xffffffffu, there && fabsf(base) > 1e6f)) {
              const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
              for (int c = 0; c < 128; ++c) s[c / 32][c % 32] = __float_as_uint(__uint_as_float(s[c / 32][c % 32]) - off);
              base = -PFX_UP<BF16>;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t weights[16];
              weigh(s[c], base, weights);
              tmem_st16(my_p + c * 16, weights);
            }
          } else {
            // By quarters of 32 keys, read once for the maximum and once for the weights; those in which no row of the warp sees a key are left out, and
            // their weights are zero. A word has a bit a key that the row sees.
            const int c0 = max(lo - key0, 0), c1 = min(hi - key0, in);
            auto quarter = [&](int c) { return bits_below(c1 - 32 * c) & ~bits_below(c0 - 32 * c); };
            float next = m;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              const uint32_t seen = quarter(c);
              if (!__any_sync(0xffffffffu, seen != 0u)) continue;
              uint32_t q[32];
              tmem_ld32_nowait(my_s + c * 32, q);
              tmem_wait_ld(q);
              float top[2] = {next, next};
#pragma unroll
              for (int e = 0; e < 32; ++e) top[e % 2] = fmaxf(top[e % 2], seen >> e & 1 ? __uint_as_float(q[e]) : -INFINITY);
              next = fmaxf(top[0], top[1]);
            }
            if (!move_sums(next)) return false;
            const float off = m == -INFINITY ? 0.f : m;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {                  // (weights over scores: a quarter's lie in columns that have been read)
              const uint32_t seen = quarter(c);
              uint32_t weights[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) weights[e] = 0u;
              if (__any_sync(0xffffffffu, seen != 0u)) {
                uint32_t q[32];
                tmem_ld32_nowait(my_s + c * 32, q);
                tmem_wait_ld(q);
#pragma unroll
                for (int e = 0; e < 32; ++e) q[e] = seen >> e & 1 ? __float_as_uint(__uint_as_float(q[e]) - off) : 0xff800000u;
                weigh(q, -PFX_UP<BF16>, weights);
              }
              tmem_st16(my_p + c * 16, weights);
            }
            if (T::APART) {
              tc_fence_before_sync();
              mbar_arrive(smem_u32(&ctl.s_read[w]));
            }
          }
          float sums[4];
          unpack2(sum[0], sums[0], sums[1]);
          unpack2(sum[1], sums[2], sums[3]);
          l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
          tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(smem_u32(&ctl.p_ready[w]));
          ++sn;
          if (!known) know();
          if (mine == stop) {
            const int last = x.of(w).n - 1;
            if (!keep_sums(smem_u32(&ctl.o_done[w]), sn - 1, my_o, p.kept + (blockIdx.x * (p.d / 4) * 2 + w) * PFX_ROWS + row, p.d, &ctl.ml[w][row].x, m, p.scale,
                           mine >= PFX_KEPT, mine == last))
              return false;
            stop = min(stop + PFX_KEPT, last);
          }
        }
      }
      // What a thread has of its row: all columns of a tile of its own, half of them of a tile that both groups share.
      float f[2] = {1.f, 0.f}, top = m, all = l;
      bool bad = false, have[2] = {mine > 0, false};
      const int qs = pieces % T::Q;
      if (!x.empty) {
        const int theirs = other;
        other += x.of(w ^ 1).n;
        // A group without blocks in a piece stays behind the loader and the other group: what it gives back counts for this piece only when all of the piece before
        // has been given back (both groups count on one barrier), and its queries have come.
        if (mine == 0 && !wait_long(&ctl.q_full[qs], pieces / T::Q, 99)) return false;
        if ((mine == 0 || !x.two) && pieces > 0 && !wait(&ctl.o_free[w], pieces - 1, 98)) return false;
        if (!x.two) {                      // (what stands there of the piece before has been read)
          ctl.ml[w][row] = make_float2(m, l);
          mbar_arrive(smem_u32(&ctl.met));
          if (!wait(&ctl.met, mets, 95)) return false;
          ++mets;
          const float2 t = ctl.ml[w ^ 1][row];
          top = fmaxf(m, t.x);
          f[0] = m == -INFINITY ? 0.f : ex2((m - top) * p.scale);
          f[1] = t.x == -INFINITY ? 0.f : ex2((t.x - top) * p.scale);
          // (the same order in both groups: their columns are divided by the same sum)
          all = w == 0 ? l * f[0] + t.y * f[1] : t.y * f[1] + l * f[0];
          have[1] = other > theirs;
        }
        if (have[0] && !wait(&ctl.o_done[w], sn - 1, 96)) return false;
        if (have[1] && !wait(&ctl.o_done[w ^ 1], other - 1, 97)) return false;
        tc_fence_after_sync();
        bad = x.k1 > x.prefix_blocks && reinterpret_cast<volatile int*>(&ctl.bad_last[pieces & 1])[1] == pieces + 1;
        if (bad && !known) know();
        // A row that sees keys and has no weight: its scores are all -infinity, 0 / 0. In a piece a sum of 1 says so (without a maximum it adds nothing).
        if (__any_sync(0xffffffffu, there && all == 0.f)) {
          if (!known) know();
          // (of the own blocks that its tile went through: offsets that do not ascend name others too)
          const int from = x.two && w == 1 ? max(x.k0, x.hole1) : x.k0, to = x.two && w == 0 ? x.of(0).end : x.k1;
          const int own_lo = max(lo, max(from - x.prefix_blocks, 0) * PFX_KEYS), own_hi = min(hi, max(to - x.prefix_blocks, 0) * PFX_KEYS);
          if (there && all == 0.f && (x.k0 < x.prefix_blocks || own_lo < own_hi)) all = x.whole ? NAN : 1.f;
        }
      }
      const int slot = blockIdx.x * PFX_SLOTS + x.slot, part_row = tile * p.R * p.share + row;
      const float by = !x.whole ? 1.f : all > 0.f ? 1.f / all : all;                          // (no weight: zeros; NaN as it is)
      // Results of 16-byte pieces go through shared memory, so that a warp writes whole rows (a thread's pieces lie in 32 of them: 5000 cycles for 128 rows
      // of 64). The queries' buffer is free for it: the last scores have been made, and the second half of it where there is one tile.
      const bool staged = p.vec_y && x.whole && !x.empty;
      uint4* stage = reinterpret_cast<uint4*>(smem_q + (qs * 2 + w) * T::TILE);
      const int c_begin = x.two ? 0 : w * (DP / 2), c_end = x.two ? DP : (w + 1) * (DP / 2);
#pragma unroll 1
      for (int c0 = c_begin; c0 < c_end; c0 += 32) {
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (!(h ? have[1] : have[0])) continue;
          const float times = (h ? f[1] : f[0]) * by;
          uint32_t a[32];
          tmem_ld32_nowait(tmem + T::O + (w ^ h) * DP + lanes + c0, a);
          tmem_wait_ld(a);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = fmaf(__uint_as_float(a[e]), times, o[e]);
        }
        if (x.whole && (there || staged)) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (c0 + e >= p.d) break;                      // (d is whole pieces of 8)
            uint4 t;
            t.x = pack_weights<BF16>(o[e], o[e + 1]); t.y = pack_weights<BF16>(o[e + 2], o[e + 3]);
            t.z = pack_weights<BF16>(o[e + 4], o[e + 5]); t.w = pack_weights<BF16>(o[e + 6], o[e + 7]);
            if (staged) {
              stage[row * (DP / 8) + (((c0 + e) / 8) ^ (row & 7))] = t;
            } else {
              uint16_t* y = const_cast<uint16_t*>(p.y.get<uint16_t>(q_row, q_head)) + c0;
              const uint32_t h[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
              for (int z = 0; z < 8; ++z) y[e + z] = (uint16_t)(h[z / 2] >> (16 * (z & 1)));
            }
          }
        } else if (there) {
          float4* part = p.part + ((int64_t)slot * (p.d / 4) + c0 / 4) * p.part_rows + part_row;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            if (c0 + e >= p.d) break;
            part[(int64_t)(e / 4) * p.part_rows] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        __syncwarp();                                      // the lanes meet ahead of the next loads from tensor memory
      }
      if (staged) {
        uint16_t* mine_y = const_cast<uint16_t*>(p.y.get<uint16_t>(q_row, q_head));
        auto copy_out = [&](auto width) {
          constexpr int N = decltype(width)::value;        // pieces of a row that are here
          const int from = c_begin / 8, n = (min(c_end, p.d) + 7) / 8 - from, first_row = (warp & 3) * 32;
#pragma unroll 2
          for (int i = 0; i < N; ++i) {
            const int e = i * 32 + lane, r = e / N, c = from + e % N;
            uint16_t* to = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine_y), r));
            const bool is = __shfl_sync(0xffffffffu, (int)there, r) != 0 && c < from + n;
            if (is) *reinterpret_cast<uint4*>(to + c * 8) = stage[(first_row + r) * (DP / 8) + (c ^ (r & 7))];
          }
        };
        __syncwarp();
        if (x.two) copy_out(std::integral_constant<int, DP / 8>());
        else copy_out(std::integral_constant<int, DP / 16>());
      }
      if (bad) {                           // (behind what the warp's lanes have stored)
        __syncwarp();
        const int first = INT32_MAX - reinterpret_cast<volatile int*>(&ctl.bad_first[pieces & 1])[0], last = reinterpret_cast<volatile int*>(&ctl.bad_last[pieces & 1])[0];
        const int k_lo = max(lo, (first - x.prefix_blocks) * PFX_KEYS), k_hi = min(hi, (last + 1 - x.prefix_blocks) * PFX_KEYS);
        if (there && k_lo < k_hi)
          spread_bad<BF16>(p.v, x.t.own0, x.head, c_begin, min(c_end, p.d), k_lo, k_hi, x.whole ? const_cast<uint16_t*>(p.y.get<uint16_t>(q_row, q_head)) : nullptr,
                           reinterpret_cast<float*>(p.part + (int64_t)slot * (p.d / 4) * p.part_rows + part_row), (int64_t)p.part_rows * 4);
        __syncwarp();
      }
      if (!x.whole) {
        if (there && (x.two || w == 0)) p.part_ml[(int64_t)slot * p.part_rows + part_row] = make_float2(top, all);
        if (threadIdx.x == 0) p.records[slot] = {x.item, x.head, x.k0, 0};
        slots = x.slot + 1;
      }
      if (!x.empty) {
        tc_fence_before_sync();
        if (x.two) {
          mbar_arrive_twice(smem_u32(&ctl.o_free[w]));
        } else {
          mbar_arrive(smem_u32(&ctl.o_free[0]));
          mbar_arrive(smem_u32(&ctl.o_free[1]));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl.q_empty[qs]));
        ++pieces;
      }
      return true;
    });
    if (threadIdx.x == 0)
#pragma unroll 1
      for (; slots < PFX_SLOTS; ++slots) p.records[blockIdx.x * PFX_SLOTS + slots] = {-1, 0, 0, 0};
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == PFX_MMA) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
  pdl_release();
}

// The pieces of items that were cut, joined in the order of their keys. Every block reads all records, then takes its share of the cut items' rows and
// columns: 32 rows, a lane each, and 16 columns, four a warp.
constexpr int JOIN_THREADS = 128, JOIN_MOST = 1024, JOIN_AHEAD = 8;
template <bool BF16>
__global__ void __launch_bounds__(JOIN_THREADS) prefix_join_kernel(const PrefixParams p) {
  pdl_begin();
  __shared__ int s_item[JOIN_MOST], s_head[JOIN_MOST], s_unit[JOIN_MOST];
  __shared__ int s_first[JOIN_MOST / 2], s_rows[JOIN_MOST / 2], s_ends[JOIN_MOST / 2];
  __shared__ int s_slot[JOIN_MOST], s_sorted[JOIN_MOST], s_n;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, records = p.ctas * PFX_SLOTS;
#pragma unroll 1
  for (int i = threadIdx.x; i < records; i += JOIN_THREADS) {
    const PrefixRecord o = p.records[i];
    s_item[i] = o.item; s_head[i] = o.head; s_unit[i] = o.unit;
  }
  __syncthreads();
  // the items' first pieces, in the order of their places (the same in every block)
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < records; i += JOIN_THREADS)
    if (s_item[i] >= 0 && s_unit[i] == 0) {
      const int at = atomicAdd(&s_n, 1);
      if (at < JOIN_MOST / 2) s_slot[at] = i;              // (a cut item has two records or more)
    }
  __syncthreads();
  for (int i = threadIdx.x; i < min(s_n, JOIN_MOST / 2); i += JOIN_THREADS) {
    int before = 0;
#pragma unroll 1
    for (int o = 0; o < min(s_n, JOIN_MOST / 2); ++o) before += s_slot[o] < s_slot[i];
    s_first[before] = s_slot[i];
    s_rows[before] = p.items[s_item[s_slot[i]]].rows * p.share;
  }
  __syncthreads();
  if (warp == 0) {
    const int n = min(s_n, JOIN_MOST / 2), cols = (p.d + 15) / 16;
    int ends = 0;
    for (int i = lane; i - lane < n; i += 32) {
      int x = i < n ? (s_rows[i] + 31) / 32 * cols : 0;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int t = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += t;
      }
      if (i < n) s_ends[i] = ends + x;
      ends += __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
  const int firsts = min(s_n, JOIN_MOST / 2), all_units = firsts > 0 ? s_ends[firsts - 1] : 0;
  int held = -1, n = 0;
  for (int u = blockIdx.x; u < all_units; u += gridDim.x) {
    int k = 0;
    while (s_ends[k] <= u) ++k;
    const int first = s_first[k], item = s_item[first], head = s_head[first], in = u - (k > 0 ? s_ends[k - 1] : 0), row_blocks = (s_rows[k] + 31) / 32;
    if (k != held) {
      held = k;
      __syncthreads();
      if (threadIdx.x == 0) s_n = 0;
      __syncthreads();
#pragma unroll 1
      for (int i = threadIdx.x; i < records; i += JOIN_THREADS)
        if (s_item[i] == item && s_head[i] == head) s_slot[atomicAdd(&s_n, 1)] = i;
      __syncthreads();
      n = s_n;
      for (int i = threadIdx.x; i < n; i += JOIN_THREADS) {
        int before = 0;
#pragma unroll 1
        for (int o = 0; o < n; ++o) before += s_unit[s_slot[o]] < s_unit[s_slot[i]];
        s_sorted[before] = s_slot[i];
      }
      __syncthreads();
    }
    const int row = in % row_blocks * 32 + lane, col = in / row_blocks * 16 + warp * 4;
    if (row >= s_rows[k] || col >= p.d) continue;
    // (sums so far, and what the next piece moves them by)
    float top = -INFINITY, all = 0.f;
    bool seen = false;                     // scores of -infinity
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += JOIN_AHEAD) {
      float4 v[JOIN_AHEAD];
      float2 ml[JOIN_AHEAD];
#pragma unroll
      for (int i = 0; i < JOIN_AHEAD; ++i) {
        const int64_t s = s_sorted[min(i0 + i, n - 1)];
        ml[i] = p.part_ml[s * p.part_rows + row];
        v[i] = p.part[(s * (p.d / 4) + col / 4) * p.part_rows + row];
      }
#pragma unroll
      for (int i = 0; i < JOIN_AHEAD; ++i) {
        if (i0 + i >= n) break;
        const float next = fmaxf(top, ml[i].x);
        const float f = ml[i].x == -INFINITY ? 0.f : ex2((ml[i].x - next) * p.scale), back = top == next || top == -INFINITY ? 1.f : ex2((top - next) * p.scale);
        top = next;
        seen |= ml[i].x == -INFINITY && ml[i].y != 0.f;
        all = fmaf(ml[i].y, f, all * back);
        o.x = fmaf(v[i].x, f, o.x * back); o.y = fmaf(v[i].y, f, o.y * back); o.z = fmaf(v[i].z, f, o.z * back); o.w = fmaf(v[i].w, f, o.w * back);
      }
    }
    const float by = all > 0.f ? 1.f / all : seen ? NAN : all;
    uint16_t* y = const_cast<uint16_t*>(p.y.get<uint16_t>((int64_t)p.items[item].row0 + row / p.share, head * p.share + row % p.share)) + col;
    const uint32_t low = pack_weights<BF16>(o.x * by, o.y * by), high = pack_weights<BF16>(o.z * by, o.w * by);
    if (p.vec_y) {
      *reinterpret_cast<uint2*>(y) = make_uint2(low, high);
    } else {
      y[0] = (uint16_t)low; y[1] = (uint16_t)(low >> 16); y[2] = (uint16_t)high; y[3] = (uint16_t)(high >> 16);
    }
  }
}

}  // namespace
}  // namespace xb
