// The tensor-core path of xb_lora_gemm, two kernels:
//   lora_shrink_kernel   U = scale (X A_a^T), every row with its own adapter's A, in fp32; and B as fp32 beside it
//   lora_gemm_kernel     Y = X W + bias + U B_a^T: the tiles of the projection, whose depth goes on through the adapters' products
//
// Rows of a tile belong to any adapters, so neither sorting nor padding is asked of the caller; a tile of one request has one. U is made
// for all 128 rows and up to 64 / rb adapters at once, side by side in tensor memory, and a row takes its own; the product with B
// runs once for each adapter of the tile (ascending), with the lanes of the other rows disabled.
// U is held as two TF32 terms, hi + lo (|U - hi - lo| <= 2^-22 |U|), side by side along the depth, and B, whose
// 16-bit values TF32 holds exactly, is read for both: fp16 would overflow or lose U's range, one term of bf16 would show in the result.
// The products of adapters cost ceil(r / 16) depth blocks of 32 fp32 for each adapter of a tile beside the ceil(K / 64) of the projection.
#pragma once

#include "xb_gemm_tile.cuh"

namespace xb {
namespace {

constexpr uint32_t NO_ADAPTER = 0xffffffffu;

// The adapters of a tile's rows, 32 WORDS of them: lane l has those of rows l, 32 + l, ...
template <int WORDS>
struct TileAdapters {
  uint32_t id[WORDS];
  // as they stand in memory; settle() makes them adapters, so that one tile's may be on their way while another's are used
  __device__ __forceinline__ void fetch(const int32_t* adapter, int m0, int M, int lane) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const int m = m0 + 32 * w + lane;
      id[w] = m < M ? (uint32_t)adapter[m] : NO_ADAPTER;
    }
  }
  __device__ __forceinline__ void settle(int n_adapters) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) id[w] = id[w] < (uint32_t)n_adapters ? id[w] : NO_ADAPTER;
  }
  __device__ __forceinline__ void load(const int32_t* adapter, int n_adapters, int m0, int M, int lane) {
    fetch(adapter, m0, M, lane);
    settle(n_adapters);
  }
  // the least that is `from` or above; NO_ADAPTER: none is left. The same for all lanes.
  __device__ __forceinline__ uint32_t next(uint32_t from) const {
    uint32_t least = NO_ADAPTER;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) least = id[w] >= from ? min(least, id[w]) : least;
    return __reduce_min_sync(0xffffffffu, least);
  }
  // lanes of 32-row word w that an MMA for adapter a leaves as they are
  __device__ __forceinline__ uint32_t others(int w, uint32_t a) const { return ~__ballot_sync(0xffffffffu, id[w] == a); }
};

// 128 x N TF32 MMA that leaves the rows set in m as they are (one bit a row), issued by an elected lane of a warp in uniform control flow
__device__ __forceinline__ void mma_tf32_ss_rows_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, const uint32_t (&m)[4], uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(m[0]), "r"(m[1]), "r"(m[2]), "r"(m[3])
      : "memory");
}
// and one for all rows: the masks of the other cost its issue several times as much
__device__ __forceinline__ void mma_tf32_ss_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc)
      : "memory");
}
constexpr int FMT_TF32 = 2;
// A stage's bytes announced and its copies issued the same way
__device__ __forceinline__ void expect_tx_elect(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_elect(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

__device__ __forceinline__ float round_tf32(float v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return __uint_as_float(r);
}

// The adapters that some row names, in any order: what a call lays out of large tables goes by them and not by what the table holds.
struct LoraNamed {
  int32_t* place;                         // [n_adapters]: the place of an adapter among them, -1 where no row names it; null: all are laid out
  int32_t* count;                         // [1]: how many there are, less one
  int32_t* id;                            // [places]
};
__global__ void __launch_bounds__(256) lora_named_kernel(LoraNamed to, const int32_t* adapter, int M, int n_adapters) {
  pdl_begin();
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t a = m < M ? (uint32_t)adapter[m] : NO_ADAPTER, before = __shfl_up_sync(0xffffffffu, a, 1);
  if (a >= (uint32_t)n_adapters || ((threadIdx.x & 31) && before == a)) return;       // (rows of a request lie side by side)
  if (*reinterpret_cast<volatile int32_t*>(to.place + a) != -1 || atomicCAS(to.place + a, -1, -2) != -1) return;
  const int at = atomicAdd(to.count, 1) + 1;
  to.id[at] = (int32_t)a;
  to.place[a] = at;
}

struct LoraTiles {
  int M, N, K, r, n_adapters;
  int rb;                                 // rank, rounded up to 16, 32, 64 or 128
  int u_cols, b_cols;                     // floats of a row of U (2 rb: hi, lo) and of B (rb, at least 32: with rb = 16 it stands there twice)
  const int32_t* adapter;
  const float* scale;
  float* U;                               // [M, u_cols]
  float* B32;                             // [b_adapters, N, b_cols]
  const void* B; int64_t ldb, stride_b; int dtype;
  int b_adapters;                         // that are laid out in B32, 1 where all share one B (with `named`: no more than these)
  LoraNamed named;                        // the adapters that are laid out, where those are not all
  int a_step, a_named;                    // adapter a's A is number a_step a of what map_a covers, or that of its place among the named
  int vec_b;                              // rows of B in whole 16-byte pieces
  int group;                              // adapters of a pass of the shrink kernel
  int stages, tiles_m;
  uint32_t idesc_a, idesc_ext;
};

// eight 16-bit values as fp32
__device__ __forceinline__ void widen8(const uint4& t, int dtype, float (&v)[8]) {
  const uint32_t x[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (dtype == XB_BF16) {
      v[2 * k] = __uint_as_float(x[k] << 16);
      v[2 * k + 1] = __uint_as_float(x[k] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[k]));
      v[2 * k] = f.x;
      v[2 * k + 1] = f.y;
    }
  }
}
// B as fp32, zeros behind its r columns, of all adapters or of those that are named: pieces of eight from `first` on, every `step`-th
__device__ __forceinline__ void widen_b(const LoraTiles& p, int64_t first, int64_t step) {
  const int pieces = p.b_cols / 8;
  const int64_t all = (int64_t)(p.named.place ? min(p.b_adapters, *p.named.count + 1) : p.b_adapters) * p.N * pieces;
  int j, n, id;
  auto find = [&](int64_t e) {
    const int64_t an = e / pieces;
    const int a = (int)(an / p.N);
    j = (int)(e - an * pieces) * 8 % p.rb;
    n = (int)(an - (int64_t)a * p.N);
    id = p.named.place ? p.named.id[a] : a;
  };
  if (first < all) find(first);
  for (int64_t e = first; e < all; e += step) {
    const int64_t at = (int64_t)id * p.stride_b + (int64_t)n * p.ldb + j;
    const int left = p.r - j;
    const bool whole = p.vec_b && left > 0;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (whole) raw = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.B) + at));
    if (e + step < all) find(e + step);                    // (while those are on their way)
    float v[8];
    if (whole) {
      widen8(raw, p.dtype, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? load_as_f32(p.B, at + i, p.dtype) : 0.f;
    }
    float4* to = reinterpret_cast<float4*>(p.B32) + 2 * e;
    to[0] = make_float4(v[0], v[1], v[2], v[3]);
    to[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}
// v as two TF32 terms, hi + lo = v within 2^-22 |v|, of one sign and neither of them 0 where v is not: times an infinity of B both give the
// infinity that v would (|v| above 2^-100; hi takes v's upper bits as they are, and a lo of 0 becomes 2^-126). An infinity or NaN is in hi.
// Columns behind the rank are zeros whatever X holds: an infinity times the zeros of A would be a NaN there.
__device__ __forceinline__ void split_tf32(float v, float& hi, float& lo) {
  hi = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
  lo = round_tf32(v - hi);
  if (!(fabsf(lo) > 0.f)) lo = fabsf(v) > 0x1p-100f ? copysignf(0x1p-126f, v) : 0.f;
}

// The adapters of a tile, `group` at a time.
constexpr int SHRINK_GROUP = 4;           // adapters of a pass, at most
struct Pass {
  uint32_t id[SHRINK_GROUP];
  int n;
  uint32_t next;                          // the first that this pass does not take
  __device__ __forceinline__ void take(const TileAdapters<4>& t, uint32_t first, int group) {
    n = 0;
    next = first;
#pragma unroll
    for (int i = 0; i < SHRINK_GROUP; ++i) {
      id[i] = i < group ? next : NO_ADAPTER;
      if (id[i] != NO_ADAPTER) {
        ++n;
        next = t.next(next + 1);
      }
    }
  }
};

// The number of an adapter's A among those that map_a covers, of a whole warp's adapter a. (A reduction, so that it stands where the instructions that
// issue copies take their operands from: computed at each copy it cost lora_fused_kernel 3 %.)
__device__ __forceinline__ int a_number(const LoraTiles& p, uint32_t a) {
  return (int)__reduce_max_sync(0xffffffffu, p.a_named ? (uint32_t)p.named.place[a] : a * (uint32_t)p.a_step);
}

constexpr int SHRINK_THREADS = 320;       // producer, MMA, four warps for the results, four for B
constexpr int SHRINK_GROUP_ROWS = 64;     // rows of A (adapters x rb) in a stage, or rb where that is more

// Persistent, 128 rows a tile. Bound by reading X once; the adapters' A come from L2. A pass over the depth takes the A of up to 64 / rb
// adapters with it, one MMA for all of them; tiles of more adapters take more passes, each with an accumulator of its own. (With
// an MMA for each adapter that masks the others' rows out the warp that issues them bounded the kernel: a masked MMA takes it about
// 150 cycles. [65536, 1280], rank 16, 32 adapters: 54 us so, 40 now = 4.5 TB/s, 0.70 of a copy's rate.)
__global__ void __launch_bounds__(SHRINK_THREADS, 1)
lora_shrink_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ LoraTiles p) {
  using namespace umma;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int STAGES = p.stages, box = p.rb * BLOCK_K * 2, stage_bytes = A_STAGE_BYTES + p.group * box;
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ uint32_t tmem_base_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_kb = (p.K + BLOCK_K - 1) / BLOCK_K;
  const uint32_t acc_cols = (uint32_t)(p.group * p.rb), tmem_cols = max(32u, 2 * acc_cols);
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&full_bar[s]), 1); mbar_init(smem_u32(&empty_bar[s]), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&acc_full[s]), 1); mbar_init(smem_u32(&acc_empty[s]), 4); }
    fence_barrier_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_a);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), tmem_cols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  pdl_wait();

  // every role but the last walks the same passes
  if (warp < 6) {
    const int q = warp & 3, row = q * 32 + lane;           // (the result warps' rows)
    int s = 0, it = 0;
    uint32_t ph = 0;
    bool ok = true;
    TileAdapters<4> t, ahead;                              // (the next tile's are read while this one's operands are)
    ahead.fetch(p.adapter, blockIdx.x * BLOCK_M, p.M, lane);
    for (int tile = blockIdx.x; tile < p.tiles_m && ok; tile += gridDim.x) {
      const int m0 = tile * BLOCK_M;
      t = ahead;
      t.settle(p.n_adapters);
      if (tile + (int)gridDim.x < p.tiles_m) ahead.fetch(p.adapter, (tile + (int)gridDim.x) * BLOCK_M, p.M, lane);
      uint32_t mine = NO_ADAPTER;
#pragma unroll
      for (int w = 0; w < 4; ++w) mine = w == q ? t.id[w] : mine;
      const float scale = warp >= 2 && mine != NO_ADAPTER && p.scale ? p.scale[mine] : 1.f;
      Pass pass;
      for (uint32_t first = t.next(0); first != NO_ADAPTER && ok; first = pass.next, ++it) {
        pass.take(t, first, p.group);
        const int as = it & 1;
        const uint32_t acc = tmem_base + as * acc_cols, acc_ph = (uint32_t)(it >> 1) & 1u;
        if (warp == 0) {
          int at[SHRINK_GROUP];
#pragma unroll
          for (int i = 0; i < SHRINK_GROUP; ++i) at[i] = i < pass.n ? a_number(p, pass.id[i]) : 0;
          for (int kb = 0; kb < num_kb; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0 ? 1u : 0u)) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1u, 51));
            if (!ok) break;
            const uint32_t x = smem_u32(smem + s * stage_bytes), bar = smem_u32(&full_bar[s]);
            expect_tx_elect(bar, (uint32_t)(A_STAGE_BYTES + pass.n * box));
            tma_load_3d_elect(x, &map_x, bar, kb * BLOCK_K, m0, 0);
#pragma unroll
            for (int i = 0; i < SHRINK_GROUP; ++i)
              if (i < pass.n) tma_load_3d_elect(x + A_STAGE_BYTES + i * box, &map_a, bar, kb * BLOCK_K, 0, at[i]);
          }
        } else if (warp == 1) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_empty[as]), acc_ph ^ 1u, 54));
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t idesc = p.idesc_a | (uint32_t)(pass.n * p.rb >> 3) << 17;          // (columns: rb of every adapter of the pass)
          for (int kb = 0; kb < num_kb; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0 ? 1u : 0u)) {
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full_bar[s]), ph, 52));
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t x = smem_u32(smem + s * stage_bytes);
#pragma unroll
            for (int k = 0; k < BLOCK_K / 16; ++k)
              mma_f16_ss_elect(acc, make_desc_sw128(x + k * 32, 1024), make_desc_sw128(x + A_STAGE_BYTES + k * 32, 1024), idesc, (kb > 0 || k > 0) ? 1u : 0u);
            mma_commit_elect(smem_u32(&empty_bar[s]));
          }
          if (ok) mma_commit_elect(smem_u32(&acc_full[as]));
        } else {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[as]), acc_ph, 53));
          if (!ok) break;
          tc_fence_after_sync();
          float* u = p.U + (int64_t)(m0 + row) * p.u_cols;
#pragma unroll
          for (int i = 0; i < SHRINK_GROUP; ++i) {
            if (i >= pass.n) break;
            if (!__any_sync(0xffffffffu, mine == pass.id[i])) continue;
            for (int c = 0; c < p.rb; c += 16) {
              uint32_t raw[16];
              tmem_ld16_nowait(acc + i * p.rb + c + ((uint32_t)(q * 32) << 16), raw);
              tmem_wait_ld(raw);
              if (mine == pass.id[i]) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  float hi[4], lo[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) split_tf32(c + j + e < p.r ? scale * __uint_as_float(raw[j + e]) : 0.f, hi[e], lo[e]);
                  *reinterpret_cast<float4*>(u + c + j) = make_float4(hi[0], hi[1], hi[2], hi[3]);
                  *reinterpret_cast<float4*>(u + p.rb + c + j) = make_float4(lo[0], lo[1], lo[2], lo[3]);
                }
              }
              __syncwarp();                                // (the next load of tensor memory is the whole warp's)
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&acc_empty[as]));
        }
      }
    }
  } else {
    widen_b(p, (int64_t)blockIdx.x * 128 + (threadIdx.x - 192), (int64_t)gridDim.x * 128);
  }

  pdl_release();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

// The one-CTA GEMM kernel of xb_gemm_umma.cu without batches and resident weights, whose tiles go on through the adapters' products: the
// stages have the same size (128 rows of 128 bytes of X or U, block_n of W or B), only the maps and the MMAs differ.
// [65536, 1280] x [1280, 1024], 32 adapters of rank 16: 155 us = 1.1 PFLOP/s at 1965 MHz (the call 188; 231 where power holds the clock down), tensor pipe 62 % busy. One-CTA tiles of 128 x 256 read 48 KB
// from L2 for 64 of the depth, which is the bound; xb_gemm's pairs of CTAs halve W's part of it (130-140 us for the projection alone).
enum { LORA_Y_TMA, LORA_Y_ANY };
template <typename TOut, bool B_MN, int Y>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
lora_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_u,
                 const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_y, const __grid_constant__ UmmaGemmParams p,
                 const __grid_constant__ LoraTiles l) {
  using namespace umma;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int w_bytes = (B_MN ? (p.block_n + 63) / 64 * 64 : p.block_n) * BLOCK_K * 2, b_bytes = p.block_n * BLOCK_K * 2;
  const int STAGES = p.stages;
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + STAGES * A_STAGE_BYTES;
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_kb = (p.K + BLOCK_K - 1) / BLOCK_K, u_blocks = l.u_cols / 32, b_blocks = l.b_cols / 32;
  const uint32_t total_tiles = (uint32_t)p.tiles_m * (uint32_t)p.tiles_n;
  const uint32_t acc_stride = (uint32_t)p.tmem_cols / 2;
  auto place = [&](uint32_t tile, int& m0, int& n0) {
    const uint32_t inner = (uint32_t)(p.n_fast ? p.tiles_n : p.tiles_m), o = tile / inner, i = tile - o * inner;
    m0 = (int)(p.n_fast ? o : i) * BLOCK_M;
    n0 = (int)(p.n_fast ? i : o) * p.block_n;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&full_bar[s]), 1); mbar_init(smem_u32(&empty_bar[s]), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(smem_u32(&acc_full[s]), 1); mbar_init(smem_u32(&acc_empty[s]), EPI_WARPS); }
    fence_barrier_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_u);
    prefetch_tensormap(&map_b);
    if (Y == LORA_Y_TMA) prefetch_tensormap(&map_y);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), (uint32_t)p.tmem_cols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  pdl_wait();

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    auto advance = [&]() {
      s = s + 1 == STAGES ? 0 : s + 1;
      ph ^= s == 0 ? 1u : 0u;
    };
    for (uint32_t tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x) {
      int m0, n0;
      place(tile, m0, n0);
      TileAdapters<4> t;
      t.load(l.adapter, l.n_adapters, m0, p.M, lane);      // (used when the projection's loads are under way)
      int place[4] = {0, 0, 0, 0};                         // of the rows' adapters in B32, where that holds the named ones
      if (l.named.place && l.b_adapters > 1) {
#pragma unroll
        for (int w = 0; w < 4; ++w) place[w] = t.id[w] != NO_ADAPTER ? l.named.place[t.id[w]] : 0;
      }
      for (int kb = 0; kb < num_kb && ok; ++kb, advance()) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1u, 61));
        if (ok) {
          const uint32_t bar = smem_u32(&full_bar[s]), w = smem_u32(smem_b + s * w_bytes);
          expect_tx_elect(bar, (uint32_t)(A_STAGE_BYTES + w_bytes));
          tma_load_3d_elect(smem_u32(smem_a + s * A_STAGE_BYTES), &map_x, bar, kb * BLOCK_K, m0, 0);
          if (!B_MN) {
            tma_load_3d_elect(w, &map_w, bar, kb * BLOCK_K, n0, 0);
          } else {
            for (int j = 0; j * 64 < p.block_n; ++j) tma_load_3d_elect(w + j * MN_BOX_BYTES, &map_w, bar, n0 + j * 64, kb * BLOCK_K, 0);
          }
        }
      }
      for (uint32_t a = t.next(0); a != NO_ADAPTER && ok; a = t.next(a + 1)) {
        int at = l.b_adapters > 1 ? (int)a : 0;
        if (l.named.place && l.b_adapters > 1) {
          uint32_t mine = 0;
#pragma unroll
          for (int w = 0; w < 4; ++w) mine = t.id[w] == a ? (uint32_t)place[w] : mine;
          at = (int)__reduce_max_sync(0xffffffffu, mine);
        }
        for (int e = 0; e < u_blocks && ok; ++e, advance()) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1u, 61));
          if (ok) {
            const uint32_t bar = smem_u32(&full_bar[s]);
            expect_tx_elect(bar, (uint32_t)(A_STAGE_BYTES + b_bytes));
            tma_load_3d_elect(smem_u32(smem_a + s * A_STAGE_BYTES), &map_u, bar, e * 32, m0, 0);
            tma_load_3d_elect(smem_u32(smem_b + s * w_bytes), &map_b, bar, e % b_blocks * 32, n0, at);
          }
        }
      }
    }
  } else if (warp == 1) {
    int s = 0, it = 0;
    uint32_t ph = 0;
    bool ok = true;
    auto advance = [&]() {
      s = s + 1 == STAGES ? 0 : s + 1;
      ph ^= s == 0 ? 1u : 0u;
    };
    for (uint32_t tile = blockIdx.x; tile < total_tiles && ok; tile += gridDim.x, ++it) {
      int m0, n0;
      place(tile, m0, n0);
      TileAdapters<4> t;
      t.load(l.adapter, l.n_adapters, m0, p.M, lane);
      const int as = it & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_empty[as]), ((uint32_t)(it >> 1) & 1u) ^ 1u, 64));
      if (!ok) break;
      tc_fence_after_sync();
      const uint32_t tmem_acc = tmem_base + as * acc_stride;
      for (int kb = 0; kb < num_kb; ++kb, advance()) {
        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full_bar[s]), ph, 62));
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t a_addr = smem_u32(smem_a + s * A_STAGE_BYTES), b_addr = smem_u32(smem_b + s * w_bytes);
#pragma unroll
        for (int k = 0; k < BLOCK_K / 16; ++k)
          mma_f16_ss_elect(tmem_acc, make_desc_sw128(a_addr + k * 32, 1024),
                           B_MN ? make_desc_sw128_mn(b_addr + k * 2048, MN_BOX_BYTES) : make_desc_sw128(b_addr + k * 32, 1024), p.idesc,
                           (kb > 0 || k > 0) ? 1u : 0u);
        mma_commit_elect(smem_u32(&empty_bar[s]));
      }
      for (uint32_t a = t.next(0); a != NO_ADAPTER && ok; a = t.next(a + 1)) {
        const uint32_t rows[4] = {t.others(0, a), t.others(1, a), t.others(2, a), t.others(3, a)};
        const bool all = (rows[0] | rows[1] | rows[2] | rows[3]) == 0u;
        for (int e = 0; e < u_blocks; ++e, advance()) {
          ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full_bar[s]), ph, 62));
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t a_addr = smem_u32(smem_a + s * A_STAGE_BYTES), b_addr = smem_u32(smem_b + s * w_bytes);
          // (32 fp32 are four steps of 8)
          if (all) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_tf32_ss_elect(tmem_acc, make_desc_sw128(a_addr + k * 32, 1024), make_desc_sw128(b_addr + k * 32, 1024), l.idesc_ext);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_tf32_ss_rows_elect(tmem_acc, make_desc_sw128(a_addr + k * 32, 1024), make_desc_sw128(b_addr + k * 32, 1024), l.idesc_ext, rows, 1u);
          }
          mma_commit_elect(smem_u32(&empty_bar[s]));
        }
      }
      if (ok) mma_commit_elect(smem_u32(&acc_full[as]));
    }
  } else {
    // (the epilogue of gemm_umma_kernel; the reasons for the order of its barriers stand there)
    const int ew = warp - 2, q = warp & 3, part = ew >> 2, row = q * 32 + lane;
    const int chunks = p.block_n / 16, c_begin = chunks * part / 4, c_end = chunks * (part + 1) / 4;
    const bool vec_base = ((reinterpret_cast<uintptr_t>(p.Y) & 15) == 0) && ((p.ldy * sizeof(TOut)) % 16 == 0);
    float* s_bias = reinterpret_cast<float*>(smem_b + STAGES * w_bytes);                           // [4][256]
    uint4* stage = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(s_bias + 4 * 256) + ew * EPI_STAGE_BYTES);
    float *s_a = s_bias + 256, *s_b = s_a + 256, *s_c = s_b + 256;
    uint8_t* area = reinterpret_cast<uint8_t*>(s_bias + 4 * 256) + ew * p.y_bufs * p.y_unit * 64;
    uint32_t turn = 0;
    int it = 0, cur_n0 = -1;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++it) {
      int m0, n0;
      place(tile, m0, n0);
      const int as = it & 1, gm = m0 + row;
      if (n0 != cur_n0) {
        cur_n0 = n0;
        asm volatile("bar.sync 2, 512;" ::: "memory");
        const int e = ew * 32 + lane;
        if (e < p.block_n) stage_columns(p, 0, n0 + e, e, s_bias, s_a, s_b, s_c);
        asm volatile("bar.sync 2, 512;" ::: "memory");
      }
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[as]), (uint32_t)(it >> 1) & 1u, 63));
      if (!ok) continue;
      tc_fence_after_sync();
      const uint32_t tmem_acc = tmem_base + as * acc_stride + ((uint32_t)(q * 32) << 16);
      TOut* yrow = reinterpret_cast<TOut*>(p.Y) + (int64_t)gm * p.ldy;
      if constexpr (Y == LORA_Y_TMA) {
        const int y = m0 + q * 32, cols = min(p.block_n, p.N - n0);
        if (p.y_unit == 32)
          epi_tile_tma<TOut, XB_EPI_NONE, 32>(map_y, tmem_acc, part, cols, 1.f, s_bias, s_a, s_b, s_c, area, p.y_bufs, turn, n0, y, 0, y < p.M, lane);
        else
          epi_tile_tma<TOut, XB_EPI_NONE, 16>(map_y, tmem_acc, part, cols, 1.f, s_bias, s_a, s_b, s_c, area, p.y_bufs, turn, n0, y, 0, y < p.M, lane);
      } else if (sizeof(TOut) == 4 && vec_base && m0 + BLOCK_M <= p.M && n0 + p.block_n <= p.N) {
        epi_tile_fast<TOut, XB_EPI_NONE, true>(tmem_acc, c_begin, c_end, 1.f, s_bias, s_a, s_b, s_c, yrow + n0, p.ldy, 32, p.block_n, stage, lane);
      } else {
        epi_tile_edge<TOut>(p, tmem_acc, c_begin, c_end, s_bias, s_a, s_b, s_c, yrow, 0, gm, gm, n0, vec_base, reinterpret_cast<uint16_t*>(stage), lane);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&acc_empty[as]));
    }
    if (Y == LORA_Y_TMA && lane == 0) tma_store_wait_read<0>();
  }

  pdl_release();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, (uint32_t)p.tmem_cols);
  }
}

// Products of one column of tiles: both steps in one kernel, X read once. A tile's walk over the depth makes its projection and, in the same
// MMAs, the U of up to `group` adapters beside it in tensor memory (further adapters: U alone, over the depth once more). Four warps
// take U out, scale and split it, widen B to fp32 beside it, and leave both in shared memory as the operands of U B^T, which is issued
// after the next walk, so that nobody waits for them. [74000, 324] x [324, 200], rank 8: 41 us as two kernels, 35
// now. What bounds it is the way from L2, 47 KB of X, W and A for each 64 of the depth, and four tiles a CTA whose first and last
// steps nothing overlaps.
constexpr int FUSED_THREADS = GEMM_THREADS + 128;
constexpr int FUSED_MAX_RB = 32;                           // (the operands of a larger rank would take the ring's space)
struct LoraItem {                                          // one walk
  uint32_t id[SHRINK_GROUP];
  uint32_t row[4];                                         // the tile's adapters (TileAdapters)
  int n, m0, it;                                           // adapters of the walk; first row; which of this CTA's tiles
  bool first, last;                                        // of the tile
};
template <typename TOut, bool B_MN, int Y>
__global__ void __launch_bounds__(FUSED_THREADS, 1)
lora_fused_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                  const __grid_constant__ CUtensorMap map_y, const __grid_constant__ UmmaGemmParams p, const __grid_constant__ LoraTiles l) {
  using namespace umma;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int w_bytes = (B_MN ? (p.block_n + 63) / 64 * 64 : p.block_n) * BLOCK_K * 2, box = l.rb * BLOCK_K * 2;
  const int STAGES = p.stages, stage_bytes = A_STAGE_BYTES + w_bytes + l.group * box;         // X, W, the adapters' A behind it
  uint8_t* smem_u = smem + STAGES * stage_bytes;                                              // U: blocks of 128 rows x 32 floats
  uint8_t* smem_b = smem_u + l.u_cols / 32 * A_STAGE_BYTES;                                   // B: block_n rows x 32 floats
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t empty_bar[MAX_STAGES];
  __shared__ __align__(8) uint64_t acc_full[2];
  __shared__ __align__(8) uint64_t acc_empty[2];
  __shared__ __align__(8) uint64_t u_full[2], ready, used;
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_kb = (p.K + BLOCK_K - 1) / BLOCK_K, u_blocks = l.u_cols / 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(smem_u32(&full_bar[s]), 1); mbar_init(smem_u32(&empty_bar[s]), 1); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&acc_full[s]), 1);
      mbar_init(smem_u32(&acc_empty[s]), EPI_WARPS);
      mbar_init(smem_u32(&u_full[s]), 1);
    }
    mbar_init(smem_u32(&ready), 4);
    mbar_init(smem_u32(&used), 1);
    fence_barrier_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_a);
    if (Y == LORA_Y_TMA) prefetch_tensormap(&map_y);
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), (uint32_t)p.tmem_cols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s, acc_stride = (uint32_t)(p.block_n + l.group * l.rb);        // an accumulator, its U behind it
  pdl_wait();

  // The walks of this CTA's tiles in order; `visit` is false where a wait ran out. The same for every role.
  auto each_item = [&](auto visit) {
    TileAdapters<4> t, ahead;                              // (the next tile's are read while this one's operands are)
    ahead.fetch(l.adapter, blockIdx.x * BLOCK_M, p.M, lane);
    int it = 0;
    for (int tile = blockIdx.x; tile < p.tiles_m; tile += gridDim.x, ++it) {
      t = ahead;
      t.settle(l.n_adapters);
      if (tile + (int)gridDim.x < p.tiles_m) ahead.fetch(l.adapter, (tile + (int)gridDim.x) * BLOCK_M, p.M, lane);
      LoraItem item;
#pragma unroll
      for (int w = 0; w < 4; ++w) item.row[w] = t.id[w];
      item.m0 = tile * BLOCK_M;
      item.it = it;
      item.first = true;
      Pass pass;
      uint32_t next = t.next(0);
      do {
        pass.take(t, next, l.group);
        next = pass.next;
#pragma unroll
        for (int i = 0; i < SHRINK_GROUP; ++i) item.id[i] = pass.id[i];
        item.n = pass.n;
        item.last = next == NO_ADAPTER;
        if (!visit(item)) return false;
        item.first = false;
      } while (!item.last);
    }
    return true;
  };

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 0;
    each_item([&](const LoraItem& item) {
      const uint32_t bytes = (uint32_t)(A_STAGE_BYTES + (item.first ? w_bytes : 0) + item.n * box);
      int at[SHRINK_GROUP];
#pragma unroll
      for (int i = 0; i < SHRINK_GROUP; ++i) at[i] = i < item.n ? a_number(l, item.id[i]) : 0;
      for (int kb = 0; kb < num_kb; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0 ? 1u : 0u)) {
        const uint32_t x = smem_u32(smem + s * stage_bytes), w = x + A_STAGE_BYTES, a = w + w_bytes, bar = smem_u32(&full_bar[s]);
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&empty_bar[s]), ph ^ 1u, 71))) return false;
        expect_tx_elect(bar, bytes);
        tma_load_3d_elect(x, &map_x, bar, kb * BLOCK_K, item.m0, 0);
        if (item.first) {
          if (!B_MN) {
            tma_load_3d_elect(w, &map_w, bar, kb * BLOCK_K, 0, 0);
          } else {
            for (int j = 0; j * 64 < p.block_n; ++j) tma_load_3d_elect(w + j * MN_BOX_BYTES, &map_w, bar, j * 64, kb * BLOCK_K, 0);
          }
        }
#pragma unroll
        for (int i = 0; i < SHRINK_GROUP; ++i)
          if (i < item.n) tma_load_3d_elect(a + i * box, &map_a, bar, kb * BLOCK_K, 0, at[i]);
      }
      return true;
    });
  } else if (warp == 1) {
    int s = 0, walks = 0, product = 0;                     // walks with adapters; products with B
    uint32_t ph = 0;
    LoraItem before;
    before.n = 0;
    auto products = [&](const LoraItem& item) {            // U B^T of a walk's adapters
#pragma unroll
      for (int i = 0; i < SHRINK_GROUP; ++i) {
        if (i >= item.n) break;
        uint32_t rows[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) rows[w] = ~__ballot_sync(0xffffffffu, item.row[w] == item.id[i]);
        const bool all = (rows[0] | rows[1] | rows[2] | rows[3]) == 0u;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&ready), (uint32_t)product & 1u, 75))) return false;
        tc_fence_after_sync();
        ++product;
        const uint32_t b = smem_u32(smem_b), acc = tmem_base + (item.it & 1) * acc_stride;
        for (int e = 0; e < u_blocks; ++e) {
          const uint32_t u = smem_u32(smem_u + e * A_STAGE_BYTES);
          // (32 fp32 are four steps of 8)
          if (all) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_tf32_ss_elect(acc, make_desc_sw128(u + k * 32, 1024), make_desc_sw128(b + k * 32, 1024), l.idesc_ext);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_tf32_ss_rows_elect(acc, make_desc_sw128(u + k * 32, 1024), make_desc_sw128(b + k * 32, 1024), l.idesc_ext, rows, 1u);
          }
        }
        mma_commit_elect(smem_u32(&used));
      }
      if (item.last) mma_commit_elect(smem_u32(&acc_full[item.it & 1]));
      return true;
    };
    const bool ok = each_item([&](const LoraItem& item) {
      const uint32_t acc = tmem_base + (item.it & 1) * acc_stride, u = acc + p.block_n;
      if (!item.first) {                                   // the U before this one, in the same columns, has been taken out
        if (!products(before)) return false;
        before.n = 0;
      } else {
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_empty[item.it & 1]), ((uint32_t)(item.it >> 1) & 1u) ^ 1u, 74))) return false;
        tc_fence_after_sync();
      }
      // the descriptors' columns: those of W, rb of every adapter of the walk, or both where they lie one behind the other
      const uint32_t cols_u = (uint32_t)(item.n * l.rb >> 3) << 17;
      const uint32_t idesc_u = l.idesc_a | cols_u, idesc = p.idesc + (B_MN ? 0u : cols_u);
      for (int kb = 0; kb < num_kb; ++kb, s = (s + 1 == STAGES ? 0 : s + 1), ph ^= (s == 0 ? 1u : 0u)) {
        const uint32_t x = smem_u32(smem + s * stage_bytes), w = x + A_STAGE_BYTES, a = w + w_bytes;
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&full_bar[s]), ph, 72))) return false;
        tc_fence_after_sync();
        if (item.first) {
#pragma unroll
          for (int k = 0; k < BLOCK_K / 16; ++k)
            mma_f16_ss_elect(acc, make_desc_sw128(x + k * 32, 1024),
                             B_MN ? make_desc_sw128_mn(w + k * 2048, MN_BOX_BYTES) : make_desc_sw128(w + k * 32, 1024), idesc, (kb > 0 || k > 0) ? 1u : 0u);
        }
        if (item.n > 0 && (B_MN || !item.first)) {
#pragma unroll
          for (int k = 0; k < BLOCK_K / 16; ++k)
            mma_f16_ss_elect(u, make_desc_sw128(x + k * 32, 1024), make_desc_sw128(a + k * 32, 1024), idesc_u, (kb > 0 || k > 0) ? 1u : 0u);
        }
        mma_commit_elect(smem_u32(&empty_bar[s]));
      }
      if (item.n > 0) mma_commit_elect(smem_u32(&u_full[walks & 1]));
      else mma_commit_elect(smem_u32(&acc_full[item.it & 1]));
      if (item.n > 0) ++walks;
      if (before.n > 0 && !products(before)) return false;
      before = item;
      return true;
    });
    if (ok && before.n > 0) products(before);
  } else if (warp >= 2 + EPI_WARPS) {
    // The operands of U B^T, in rows of 128 bytes whose pieces of 16 are swapped by the row: B as fp32, zeros behind its r columns, and (with
    // the first adapter of a walk) U out of tensor memory, times the row's scale, as hi and lo.
    const int q = warp & 3, row = q * 32 + lane, thread = threadIdx.x - (2 + EPI_WARPS) * 32;
    auto put = [](uint8_t* block, int r, int c, const float (&v)[4]) {
      *reinterpret_cast<float4*>(block + r * 128 + (((c >> 2) ^ (r & 7)) << 4)) = make_float4(v[0], v[1], v[2], v[3]);
    };
    int walks = 0, product = 0;
    each_item([&](const LoraItem& item) {
      uint32_t mine = NO_ADAPTER;
#pragma unroll
      for (int w = 0; w < 4; ++w) mine = w == q ? item.row[w] : mine;
      const float scale = mine != NO_ADAPTER && l.scale ? l.scale[mine] : 1.f;
#pragma unroll 1
      for (int i = 0; i < item.n; ++i) {
        uint32_t id = item.id[0];
#pragma unroll
        for (int k = 1; k < SHRINK_GROUP; ++k) id = i == k ? item.id[k] : id;
        // the product before has read what is overwritten now
        if (!__all_sync(0xffffffffu, product == 0 || mbar_wait(smem_u32(&used), (uint32_t)(product - 1) & 1u, 76))) return false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = thread + 128 * h;
          if (n >= p.block_n) break;
          const int64_t at = (int64_t)id * l.stride_b + (int64_t)n * l.ldb;
#pragma unroll
          for (int j = 0; j < FUSED_MAX_RB; j += 8) {
            if (j >= l.rb) break;
            float v[8];
            if (l.vec_b && n < p.N && j < l.r) {
              widen8(__ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(l.B) + at + j)), l.dtype, v);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = n < p.N && j + k < l.r ? load_as_f32(l.B, at + j + k, l.dtype) : 0.f;
            }
            const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
            put(smem_b, n, j, lo);
            put(smem_b, n, j + 4, hi);
            if (l.rb == 16) {                              // 16 columns stand there twice, for U's hi and lo in one block
              put(smem_b, n, 16 + j, lo);
              put(smem_b, n, 20 + j, hi);
            }
          }
        }
        if (i == 0) {
          if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&u_full[walks & 1]), (uint32_t)(walks >> 1) & 1u, 73))) return false;
          tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < SHRINK_GROUP; ++k) {
            if (k >= item.n) break;
            if (!__any_sync(0xffffffffu, mine == item.id[k])) continue;
            for (int c = 0; c < l.rb; c += 16) {
              uint32_t raw[16];
              tmem_ld16_nowait(tmem_base + (item.it & 1) * acc_stride + p.block_n + k * l.rb + c + ((uint32_t)(q * 32) << 16), raw);
              tmem_wait_ld(raw);
              if (mine == item.id[k]) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  float hi[4], lo[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) split_tf32(c + j + e < l.r ? scale * __uint_as_float(raw[j + e]) : 0.f, hi[e], lo[e]);
                  put(smem_u, row, c + j, hi);             // (hi and lo of 16 columns share the one block there is, of 32 they have one each)
                  put(smem_u + (l.rb >> 5) * A_STAGE_BYTES, row, (l.rb == 16 ? 16 : 0) + c + j, lo);
                }
              }
              __syncwarp();                                // (the next load of tensor memory is the whole warp's)
            }
          }
          tc_fence_before_sync();
          ++walks;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ready));
        ++product;
      }
      return true;
    });
  } else {
    // (the epilogue of gemm_umma_kernel; the reasons for the order of its barriers stand there)
    const int ew = warp - 2, q = warp & 3, part = ew >> 2, row = q * 32 + lane;
    const int chunks = p.block_n / 16, c_begin = chunks * part / 4, c_end = chunks * (part + 1) / 4;
    const bool vec_base = ((reinterpret_cast<uintptr_t>(p.Y) & 15) == 0) && ((p.ldy * sizeof(TOut)) % 16 == 0);
    float* s_bias = reinterpret_cast<float*>(smem_b + p.block_n * 128);                            // [4][256]
    uint4* stage = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(s_bias + 4 * 256) + ew * EPI_STAGE_BYTES);
    float *s_a = s_bias + 256, *s_b = s_a + 256, *s_c = s_b + 256;
    uint8_t* area = reinterpret_cast<uint8_t*>(s_bias + 4 * 256) + ew * p.y_bufs * p.y_unit * 64;
    uint32_t turn = 0;
    const int e = ew * 32 + lane;
    if (e < p.block_n) stage_columns(p, 0, e, e, s_bias, s_a, s_b, s_c);
    asm volatile("bar.sync 2, 512;" ::: "memory");
    int it = 0;
    for (int tile = blockIdx.x; tile < p.tiles_m; tile += gridDim.x, ++it) {
      const int m0 = tile * BLOCK_M, as = it & 1, gm = m0 + row;
      if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&acc_full[as]), (uint32_t)(it >> 1) & 1u, 77))) break;
      tc_fence_after_sync();
      const uint32_t tmem_acc = tmem_base + as * acc_stride + ((uint32_t)(q * 32) << 16);
      TOut* yrow = reinterpret_cast<TOut*>(p.Y) + (int64_t)gm * p.ldy;
      if constexpr (Y == LORA_Y_TMA) {
        const int y = m0 + q * 32;
        if (p.y_unit == 32)
          epi_tile_tma<TOut, XB_EPI_NONE, 32>(map_y, tmem_acc, part, p.N, 1.f, s_bias, s_a, s_b, s_c, area, p.y_bufs, turn, 0, y, 0, y < p.M, lane);
        else
          epi_tile_tma<TOut, XB_EPI_NONE, 16>(map_y, tmem_acc, part, p.N, 1.f, s_bias, s_a, s_b, s_c, area, p.y_bufs, turn, 0, y, 0, y < p.M, lane);
      } else if (sizeof(TOut) == 4 && vec_base && m0 + BLOCK_M <= p.M && p.block_n <= p.N) {
        epi_tile_fast<TOut, XB_EPI_NONE, true>(tmem_acc, c_begin, c_end, 1.f, s_bias, s_a, s_b, s_c, yrow, p.ldy, 32, p.block_n, stage, lane);
      } else {
        epi_tile_edge<TOut>(p, tmem_acc, c_begin, c_end, s_bias, s_a, s_b, s_c, yrow, 0, gm, gm, 0, vec_base, reinterpret_cast<uint16_t*>(stage), lane);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&acc_empty[as]));
    }
    if (Y == LORA_Y_TMA && lane == 0) tma_store_wait_read<0>();
  }

  pdl_release();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, (uint32_t)p.tmem_cols);
  }
}

int make_map_f32(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t batch, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(XB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)cols * 4, (cuuint64_t)cols * rows * 4};
  cuuint32_t box[3] = {32, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(XB_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return 0;
}

template <typename TOut, bool B_MN, int Y>
int launch_lora_gemm(const CUtensorMap (&m)[5], const UmmaGemmParams& p, const LoraTiles& l, unsigned grid, size_t smem, cudaStream_t s) {
  static PerDeviceOnce attr_set;          // per instantiation
  XB_SET_MAX_SMEM_ONCE(attr_set, 226 * 1024, (const void*)lora_gemm_kernel<TOut, B_MN, Y>);
  launch_dependent(lora_gemm_kernel<TOut, B_MN, Y>, grid, GEMM_THREADS, smem, s, m[0], m[1], m[2], m[3], m[4], p, l);
  return check_launch("lora_gemm_kernel");
}

template <typename TOut, bool B_MN, int Y>
int launch_lora_fused(const CUtensorMap (&m)[5], const UmmaGemmParams& p, const LoraTiles& l, unsigned grid, size_t smem, cudaStream_t s) {
  static PerDeviceOnce attr_set;          // per instantiation
  XB_SET_MAX_SMEM_ONCE(attr_set, 226 * 1024, (const void*)lora_fused_kernel<TOut, B_MN, Y>);
  launch_dependent(lora_fused_kernel<TOut, B_MN, Y>, grid, FUSED_THREADS, smem, s, m[0], m[1], m[2], m[4], p, l);
  return check_launch("lora_fused_kernel");
}

// Rows that TMA cannot address (they do not start on 16 bytes) are laid out again in the workspace, as K-major rows of `ld` elements; the same
// for weights in [K, N] whose results are fp32.
struct LoraCopies { bool x, w, a; int64_t ld; };
LoraCopies lora_copies(const xb_lora_args& a) {
  auto odd = [](const void* p, int64_t ld) { return ld % 8 != 0 || (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  LoraCopies c;
  c.ld = ((int64_t)a.K + 7) / 8 * 8;
  c.x = odd(a.X, a.ldx);
  c.w = odd(a.W, a.ldw) || (!a.trans_w && a.y_dtype == XB_F32);
  c.a = odd(a.A, a.lda) || (a.n_adapters > 1 && a.stride_a % 8 != 0);
  return c;
}
// `rows` rows of K elements, element (row, k) at from + row * step_row + k * step_k of block row / rows_a_block, into rows of ld
struct LoraCopy { const uint16_t* from; uint16_t* to; int64_t rows, rows_a_block, step_block, step_row, step_k; };
struct LoraCopyJobs { LoraCopy job[3]; int n, K, ld; int64_t first_block[4]; int named_job; LoraNamed named; };
// A thread takes eight elements of a row; the rows of a block lie side by side where those are what is adjacent in memory ([K, N] weights).
constexpr int COPY_THREADS = 256;
__global__ void __launch_bounds__(COPY_THREADS) lora_copy_kernel(const __grid_constant__ LoraCopyJobs p) {
  pdl_begin();
  int j = 0;
  while (j + 1 < p.n && (int64_t)blockIdx.x >= p.first_block[j + 1]) ++j;
  const LoraCopy c = p.job[j];
  const int64_t at = ((int64_t)blockIdx.x - p.first_block[j]) * COPY_THREADS + threadIdx.x;
  const int pieces = p.ld / 8;
  const int64_t row = c.step_k == 1 ? at / pieces : at % c.rows;
  const int k0 = (int)(c.step_k == 1 ? at - row * pieces : at / c.rows) * 8;
  if (row >= c.rows || k0 >= p.ld) return;
  const int64_t block = row / c.rows_a_block;
  int64_t from_block = block;
  if (j == p.named_job) {                  // (places behind the last of the named adapters stay as they are)
    if (block > *p.named.count) return;
    from_block = p.named.id[block];
  }
  const uint16_t* from = c.from + from_block * c.step_block + (row - block * c.rows_a_block) * c.step_row;
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k0 + i < p.K) w[i / 2] |= (uint32_t)__ldg(from + (k0 + i) * c.step_k) << (16 * (i & 1));
  *reinterpret_cast<uint4*>(c.to + row * p.ld + k0) = make_uint4(w[0], w[1], w[2], w[3]);
}

// What the tensor-core path takes
bool lora_umma_takes(const xb_lora_args& a) { return (a.dtype == XB_F16 || a.dtype == XB_BF16) && a.n_adapters >= 1 && a.r >= 1; }
struct LoraScratch {
  int rb, u_cols, b_cols;
  int fused_group;                        // adapters of a walk where both steps are one kernel, 0 where they are two
  int a_adapters, b_adapters;             // that are laid out, where A or B is: one where all share it
  bool named;                             // only the adapters that rows name are laid out
  size_t u, b, x, w, a, place, bytes;
  bool fits;                              // in what the sizes above count
};
// Where more than 32 MB would be laid out of a table of adapters, only those that some row names are, which a kernel (and the clearing of its
// table) finds out first: 6 to 8 us. us in a graph, 4096 rows, K = 256, N = 1024, rank 16 (131 KB an adapter), all laid out and the named ones:
// every adapter named, 128 of them 20 and 27, 256 32 and 41, 512 78 and 85, 1024 155 and 161; three named, of 128 19 and 17, 256 29 and 17, 512 67 and
// 17, 1024 134 and 14. Scratch for no more of them than there are rows.
constexpr double LORA_HELD = 32 << 20;
LoraScratch lora_scratch(const xb_lora_args& a) {
  LoraScratch w;
  w.rb = a.r <= 16 ? 16 : a.r <= 32 ? 32 : a.r <= 64 ? 64 : 128;
  w.u_cols = 2 * w.rb;
  w.b_cols = std::max(w.rb, 32);
  // One column of tiles, and tensor memory for it and the U of an adapter twice: both steps in one kernel. (Two adapters a walk: a third would
  // be a longer stage for every tile. Fewer tiles than half of the SMs become narrower ones, in two steps.)
  const int whole_n = (a.N + 15) / 16 * 16;
  w.fused_group = whole_n <= 256 && w.rb <= FUSED_MAX_RB && ((int64_t)a.M + BLOCK_M - 1) / BLOCK_M >= sm_count() / 2 ? std::min(2, (256 - whole_n) / w.rb) : 0;
  const LoraCopies c = lora_copies(a);
  const double a_each = c.a ? 2.0 * c.ld * a.r : 0, b_each = w.fused_group ? 0 : 4.0 * a.N * w.b_cols;
  w.a_adapters = a.stride_a ? a.n_adapters : 1;
  w.b_adapters = a.stride_b ? a.n_adapters : 1;
  w.named = a_each * w.a_adapters + b_each * w.b_adapters > LORA_HELD && a.n_adapters > 1;
  if (w.named) {                           // no more than there are rows
    w.a_adapters = std::min(w.a_adapters, a.M);
    w.b_adapters = std::min(w.b_adapters, a.M);
  }
  // (adapters may share their memory, so what is laid out of them has no bound in what the caller holds)
  w.fits = 4.0 * a.M * w.u_cols + b_each * w.b_adapters + a_each * w.a_adapters + 2.0 * c.ld * (c.x * (double)a.M + c.w * (double)a.N) < 1.0e15;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  auto rows = [&](bool copy, int64_t n) { return copy ? up((size_t)n * c.ld * 2) : 0; };
  w.u = 0;
  w.b = w.fused_group ? 0 : up((size_t)a.M * w.u_cols * 4);
  w.x = w.b + (w.fused_group ? 0 : up((size_t)w.b_adapters * a.N * w.b_cols * 4));
  w.w = w.x + rows(c.x, a.M);
  w.a = w.w + rows(c.w, a.N);
  w.place = w.a + rows(c.a, (int64_t)w.a_adapters * a.r);
  w.bytes = w.place + (w.named ? up(((size_t)a.n_adapters + 1 + std::min(a.n_adapters, a.M)) * 4) : 0);
  return w;
}

int run_umma(const xb_lora_args& given, uint8_t* ws, cudaStream_t stream) {
  const LoraScratch w = lora_scratch(given);
  xb_lora_args a = given;
  LoraNamed named = {nullptr, nullptr, nullptr};
  if (w.named) {
    named.place = reinterpret_cast<int32_t*>(ws + w.place);
    named.count = named.place + a.n_adapters;
    named.id = named.count + 1;
    XB_CUDA(cudaMemsetAsync(named.place, 0xff, ((size_t)a.n_adapters + 1) * 4, stream));
    // (not launch_dependent: what it follows is no kernel)
    lora_named_kernel<<<(unsigned)(((int64_t)a.M + 255) / 256), 256, 0, stream>>>(named, a.adapter, a.M, a.n_adapters);
    if (int rc = check_launch("lora_named_kernel")) return rc;
  }
  if (const LoraCopies c = lora_copies(given); c.x || c.w || c.a) {
    LoraCopyJobs jobs;
    memset(&jobs, 0, sizeof(jobs));
    jobs.K = a.K;
    jobs.ld = (int)c.ld;
    jobs.named_job = -1;
    jobs.named = named;
    auto add = [&](const void* from, size_t to, int64_t rows, int64_t rows_a_block, int64_t step_block, int64_t step_row, int64_t step_k) {
      jobs.job[jobs.n] = {static_cast<const uint16_t*>(from), reinterpret_cast<uint16_t*>(ws + to), rows, rows_a_block, step_block, step_row, step_k};
      jobs.first_block[jobs.n + 1] = jobs.first_block[jobs.n] + (rows * (c.ld / 8) + COPY_THREADS - 1) / COPY_THREADS;
      ++jobs.n;
      return ws + to;
    };
    if (c.x) { a.X = add(a.X, w.x, a.M, a.M, 0, a.ldx, 1); a.ldx = c.ld; }
    if (c.w) { a.W = add(a.W, w.w, a.N, a.N, 0, a.trans_w ? a.ldw : 1, a.trans_w ? 1 : a.ldw); a.ldw = c.ld; a.trans_w = 1; }
    if (c.a) {
      if (w.named && a.stride_a) jobs.named_job = jobs.n;
      a.A = add(a.A, w.a, (int64_t)w.a_adapters * a.r, a.r, a.stride_a, a.lda, 1);
      a.lda = c.ld;
      a.stride_a = a.stride_a ? c.ld * a.r : 0;
    }
    const int64_t blocks = jobs.first_block[jobs.n];
    XB_REQUIRE(blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_lora_gemm: %d rows of %d are too many for one call", a.M, a.K);
    launch_dependent(lora_copy_kernel, (unsigned)blocks, COPY_THREADS, 0, stream, jobs);
    if (int rc = check_launch("lora_copy_kernel")) return rc;
  }
  const int bf16 = a.dtype == XB_BF16;
  LoraTiles l;
  memset(&l, 0, sizeof(l));
  l.M = a.M; l.N = a.N; l.K = a.K; l.r = a.r; l.n_adapters = a.n_adapters; l.rb = w.rb; l.u_cols = w.u_cols; l.b_cols = w.b_cols;
  const bool a_laid_out = a.A != given.A;
  l.b_adapters = w.b_adapters; l.named = named; l.a_named = w.named && a_laid_out && a.stride_a; l.a_step = a.stride_a ? 1 : 0;
  l.adapter = a.adapter; l.scale = a.scale; l.U = reinterpret_cast<float*>(ws + w.u); l.B32 = reinterpret_cast<float*>(ws + w.b);
  l.B = a.B; l.ldb = a.ldb; l.stride_b = a.stride_b; l.dtype = a.dtype;
  l.vec_b = a.r % 8 == 0 && a.ldb % 8 == 0 && a.stride_b % 8 == 0 && (reinterpret_cast<uintptr_t>(a.B) & 15) == 0;
  l.group = std::max(1, SHRINK_GROUP_ROWS / l.rb);
  l.tiles_m = (a.M + BLOCK_M - 1) / BLOCK_M;
  l.idesc_a = umma::make_idesc(BLOCK_M, 0, bf16);          // (the columns are the pass's)
  CUtensorMap mx, ma;
  if (int rc = make_map(&mx, a.X, bf16, a.K, a.M, a.ldx, 1, 0, BLOCK_M, BLOCK_K, CU_TENSOR_MAP_SWIZZLE_128B, 1, CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return rc;
  if (int rc = make_map(&ma, a.A, bf16, a.K, a.r, a.lda, a_laid_out ? w.a_adapters : a.stride_a ? a.n_adapters : 1, a.stride_a, l.rb)) return rc;
  const bool fused = w.fused_group > 0;
  if (fused) {
    l.group = w.fused_group;
  } else {
    const int stage = A_STAGE_BYTES + l.group * l.rb * BLOCK_K * 2;
    l.stages = std::min(MAX_STAGES, 220 * 1024 / stage);
    static PerDeviceOnce attr_set;
    XB_SET_MAX_SMEM_ONCE(attr_set, 226 * 1024, (const void*)lora_shrink_kernel);
    // (every SM takes its share of B, with or without tiles: 520 rows, 16 adapters, N = 1024, rank 64, with a block a tile 220 us, 19 now)
    launch_dependent(lora_shrink_kernel, (unsigned)sm_count(), SHRINK_THREADS, (size_t)l.stages * stage + 1024, stream, mx, ma, l);
    if (int rc = check_launch("lora_shrink_kernel")) return rc;
  }
  UmmaGemmParams p;
  memset(&p, 0, sizeof(p));
  p.M = a.M; p.N = a.N; p.K = a.K; p.batch = 1; p.alpha = p.beta = 1.f;
  p.bias = a.bias; p.bias_kind = a.bias ? XB_BIAS_ROW : XB_BIAS_NONE; p.bias_dtype = XB_F32; p.bias_group = 1;
  p.Y = a.Y; p.ldy = a.ldy; p.y_dtype = a.y_dtype;
  p.b_mn = !a.trans_w;
  p.tiles_m = l.tiles_m;
  // all of a product of up to 256 columns, equal shares of a wider one; narrower where the tiles would leave SMs idle
  const int wide = (a.N + 255) / 256, least = a.trans_w ? 32 : 64;
  const int64_t split = fused ? 1 : std::max<int64_t>(wide, std::min<int64_t>(sm_count() / std::max(p.tiles_m, 1), (a.N + least - 1) / least));
  p.block_n = (int)((a.N + split - 1) / split + 15) / 16 * 16;
  p.tiles_n = (a.N + p.block_n - 1) / p.block_n;
  p.tmem_cols = 64;
  while (p.tmem_cols < 2 * (p.block_n + (fused ? l.group * l.rb : 0))) p.tmem_cols <<= 1;
  p.idesc = umma::make_idesc(BLOCK_M, p.block_n, bf16) | (p.b_mn ? umma::IDESC_B_MN : 0u);
  l.idesc_ext = umma::make_idesc(BLOCK_M, p.block_n, FMT_TF32);
  const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
  XB_REQUIRE(total < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_lora_gemm: %lld output tiles are too many for one call", (long long)total);
  p.n_fast = p.tiles_n > 1;               // the n tiles of a row of tiles run together and share its X
  CUtensorMap m[5];
  m[0] = mx;
  if (int rc = p.b_mn ? make_map(&m[1], a.W, bf16, a.N, a.K, a.ldw, 1, 0, BLOCK_K) : make_map(&m[1], a.W, bf16, a.K, a.N, a.ldw, 1, 0, p.block_n)) return rc;
  if (fused) {
    m[2] = m[3] = ma;
  } else {
    if (int rc = make_map_f32(&m[2], l.U, l.u_cols, a.M, 1, BLOCK_M)) return rc;
    if (int rc = make_map_f32(&m[3], l.B32, l.b_cols, a.N, w.b_adapters, p.block_n)) return rc;
  }
  m[4] = m[0];
  const int64_t es = a.y_dtype == XB_F32 ? 4 : 2;
  int y = LORA_Y_ANY, tail = 4 * 256 * (int)sizeof(float) + EPI_WARPS * EPI_STAGE_BYTES;
  p.y_unit = 16; p.y_bufs = 1;
  const int stage = A_STAGE_BYTES + (p.b_mn ? (p.block_n + 63) / 64 * 64 : p.block_n) * BLOCK_K * 2 + (fused ? l.group * l.rb * BLOCK_K * 2 : 0);
  const int operands = fused ? l.u_cols / 32 * A_STAGE_BYTES + p.block_n * 128 : 0;          // of U B^T
  if (es == 2 && (reinterpret_cast<uintptr_t>(a.Y) & 15) == 0 && a.ldy % 8 == 0 && a.N % 8 == 0) {
    // copies of 32 columns, 16 where the tile has few or where 32 would reach into the next tile
    p.y_unit = p.block_n >= 128 && (p.block_n % 32 == 0 || p.tiles_n == 1) ? 32 : 16;
    if (fused && (SMEM_BUDGET - 4096 - operands - EPI_WARPS * 32 * 64) / stage < std::min(MAX_STAGES, (SMEM_BUDGET - 4096 - operands - EPI_WARPS * 16 * 64) / stage))
      p.y_unit = 16;                      // (a stage more)
    p.y_bufs = 1;                         // (a second would cost a stage of the ring)
    if (make_map(&m[4], a.Y, a.y_dtype == XB_BF16, a.N, a.M, a.ldy, 1, 0, 32, p.y_unit,
                 p.y_unit == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B) == 0) {
      y = LORA_Y_TMA;
      tail = 4 * 256 * (int)sizeof(float) + EPI_WARPS * p.y_bufs * p.y_unit * 64;
    }
  }
  tail += operands;
  p.stages = std::max(2, std::min(MAX_STAGES, (SMEM_BUDGET - tail) / stage));
  const size_t smem = (size_t)p.stages * stage + tail + 1024;
  const unsigned grid = (unsigned)std::min<int64_t>(total, sm_count());
  if (a.y_dtype == XB_F32)
    return fused ? launch_lora_fused<float, false, LORA_Y_ANY>(m, p, l, grid, smem, stream) : launch_lora_gemm<float, false, LORA_Y_ANY>(m, p, l, grid, smem, stream);
  auto half = [&](auto type) {
    using T = decltype(type);
    if (fused && p.b_mn) return y == LORA_Y_TMA ? launch_lora_fused<T, true, LORA_Y_TMA>(m, p, l, grid, smem, stream) : launch_lora_fused<T, true, LORA_Y_ANY>(m, p, l, grid, smem, stream);
    if (fused) return y == LORA_Y_TMA ? launch_lora_fused<T, false, LORA_Y_TMA>(m, p, l, grid, smem, stream) : launch_lora_fused<T, false, LORA_Y_ANY>(m, p, l, grid, smem, stream);
    if (p.b_mn) return y == LORA_Y_TMA ? launch_lora_gemm<T, true, LORA_Y_TMA>(m, p, l, grid, smem, stream) : launch_lora_gemm<T, true, LORA_Y_ANY>(m, p, l, grid, smem, stream);
    return y == LORA_Y_TMA ? launch_lora_gemm<T, false, LORA_Y_TMA>(m, p, l, grid, smem, stream) : launch_lora_gemm<T, false, LORA_Y_ANY>(m, p, l, grid, smem, stream);
  };
  return bf16 ? half(__nv_bfloat16()) : half(__half());
}

}  // namespace
}  // namespace xb
