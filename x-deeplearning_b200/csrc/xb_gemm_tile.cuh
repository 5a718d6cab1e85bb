// What the tcgen05 GEMM kernels share (xb_gemm_umma.cu, xb_lora_umma.cuh): tile sizes, parameters, the epilogues and the tensor maps.
#pragma once

#include <cstring>
#include <type_traits>

#include "xb_common.cuh"
#include "xb_umma.cuh"

namespace xb {
namespace {

constexpr int BLOCK_M = 128;
constexpr int BLOCK_K = 64;
constexpr int MAX_STAGES = 8;       // the launch picks as many as fit in shared memory (at least 2)
constexpr int SMEM_BUDGET = 220 * 1024;
constexpr int A_STAGE_BYTES = BLOCK_M * BLOCK_K * 2;
constexpr int MN_BOX_BYTES = 64 * BLOCK_K * 2;      // one N-major box: 64 k rows of 64 columns (128 bytes each)

struct UmmaGemmParams {
  int M, N, K, block_n, tmem_cols, tiles_m, tiles_n, batch, stages;
  int b_resident;        // the B tile (all of K) stays in shared memory while consecutive tiles share it
  int b_mn;              // B is [K,N] row-major: the MMA reads N-major tiles of 64 columns x 64 k
  int n_fast;            // consecutive tiles walk n first
  uint32_t tiles_per_cta;
  float alpha, beta;
  int a_batched, b_batched;
  const void* bias; int64_t ldbias, stride_bias; int bias_kind, bias_dtype, bias_group;
  void* Y; int64_t ldy, stride_y; int y_dtype;
  EpiParams epi; int64_t stride_ep;
  uint32_t idesc;
  int y_unit, y_bufs;    // results stored by TMA: columns of a copy (32 or 16), staging areas of a warp
  int y_beside;          // the batches lie beside one another in a row of Y: its map has the batch before the row
};

template <typename TOut>
__device__ __forceinline__ void store_row16(TOut* dst, const float (&v)[16], int valid, bool vec_ok) {
  if (sizeof(TOut) == 2 && vec_ok && valid == 16) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      TOut lo = from_f32<TOut>(v[2 * i]), hi = from_f32<TOut>(v[2 * i + 1]);
      w[i] = (uint32_t)(*reinterpret_cast<uint16_t*>(&lo)) | ((uint32_t)(*reinterpret_cast<uint16_t*>(&hi)) << 16);
    }
    uint4* d = reinterpret_cast<uint4*>(dst);
    d[0] = make_uint4(w[0], w[1], w[2], w[3]);
    d[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else if (sizeof(TOut) == 4 && vec_ok && valid == 16) {
    float4* d = reinterpret_cast<float4*>(dst);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < valid) dst[i] = from_f32<TOut>(v[i]);
  }
}

// 16 epilogue warps: four per TMEM lane quarter, each owning a quarter of the tile's columns, so every
// scheduler has four of them to hide the TMEM round trip and the store latency behind one another
constexpr int EPI_WARPS = 16;
constexpr int GEMM_THREADS = 64 + EPI_WARPS * 32;

template <typename TOut>
__device__ __forceinline__ uint4 pack8(const float* v);
template <>
__device__ __forceinline__ uint4 pack8<__half>(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack8<__nv_bfloat16>(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <>
__device__ __forceinline__ uint4 pack8<float>(const float*) { return make_uint4(0, 0, 0, 0); }   // not used

// 16 results of one output row as 16-byte stores, those that lie wholly in the `valid` columns left of it
template <typename TOut>
__device__ __forceinline__ void store16_vec(TOut* dst, const float (&v)[16], int valid) {
  if constexpr (sizeof(TOut) == 4) {
    float4* d = reinterpret_cast<float4*>(dst);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * i + 4 <= valid) d[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    uint4* d = reinterpret_cast<uint4*>(dst);
    if (8 <= valid) d[0] = pack8<TOut>(v);
    if (16 <= valid) d[1] = pack8<TOut>(v + 8);
  }
}

// Activation of 16 adjacent columns of one row; the per-column parameters sit in shared memory and are
// read as 16-byte vectors (all lanes read the same address: a broadcast).
template <int KIND>
__device__ __forceinline__ void epi_apply16(float (&v)[16], const float* s_a, const float* s_b, const float* s_c) {
  if constexpr (KIND != XB_EPI_NONE) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (KIND == XB_EPI_PRELU) {
      const float4 a = reinterpret_cast<const float4*>(s_a)[j];
      // x * (x < 0 ? w : 1): the same value as act_prelu for every x, signed zeros and NaN included
      v[4 * j] *= v[4 * j] < 0.f ? a.x : 1.f;
      v[4 * j + 1] *= v[4 * j + 1] < 0.f ? a.y : 1.f;
      v[4 * j + 2] *= v[4 * j + 2] < 0.f ? a.z : 1.f;
      v[4 * j + 3] *= v[4 * j + 3] < 0.f ? a.w : 1.f;
    } else if (KIND == XB_EPI_DICE) {
      const float4 g = reinterpret_cast<const float4*>(s_a)[j];
      const float4 b = reinterpret_cast<const float4*>(s_b)[j];
      const float4 c = reinterpret_cast<const float4*>(s_c)[j];
      const float gg[4] = {g.x, g.y, g.z, g.w}, bb[4] = {b.x, b.y, b.z, b.w}, cc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = v[4 * j + i];
        const float pr = __fdividef(1.f, 1.f + __expf(-fmaf(x, cc[i], bb[i])));
        v[4 * j + i] = x * fmaf(pr, 1.f - gg[i], gg[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * j + i] = act_sigmoid(v[4 * j + i]);
    }
  }
  }
}

constexpr int EPI_STAGE_BYTES = 32 * 64;      // per epilogue warp: 32 rows x 32 two-byte results

// Epilogue of a tile with a per-column bias (or none) and output rows of whole, aligned 16-byte pieces: this thread's row,
// columns [16 * c_begin, 16 * c_end) of the tile, as far as `rows` of the warp's 32 and `cols` of the tile's columns lie in the
// output (a piece is stored or it is not).
// Bound by shared memory's and L1's data path, which carries a result four times here (staging, both ways, beside the accumulator and
// the store). Ragged tiles went through epi_tile_edge before: [1000, 88] x [88, 168] fp16 4.8 us, 3.8 here; 8 x ([300, 256] x [256, 200])
// 5.1, 4.3.
// Two-byte outputs go through a 2 KB staging area of the warp: a thread holds 64 contiguous bytes of its
// own row, and a store instruction of one piece per lane would touch 32 different lines; after the
// exchange the 32 lanes of an instruction write 8 rows x 64 contiguous bytes. Piece j of row l is kept at
// position j ^ ((l >> 1) & 3) of the row, which makes both the writes (lane = row) and the reads (four
// lanes per row) free of bank conflicts.
template <typename TOut, int KIND, bool WHOLE = false>
__device__ __forceinline__ void epi_tile_fast(uint32_t tmem_row, int c_begin, int c_end, float alpha,
                                              const float* s_bias, const float* s_a, const float* s_b,
                                              const float* s_c, TOut* yrow, int64_t ldy, int rows, int cols,
                                              uint4* stage, int lane) {
  using namespace umma;
  for (int cg = c_begin; cg < c_end; cg += 2) {
    // two chunks per TMEM round trip when the thread owns two more
    uint32_t raw[32];
    const bool two = cg + 1 < c_end;                                    // uniform across the warp
    if (two) {
      tmem_ld32_nowait(tmem_row + (uint32_t)(cg * 16), raw);
    } else {
#pragma unroll
      for (int i = 16; i < 32; ++i) raw[i] = 0u;
      tmem_ld16_lo_nowait(tmem_row + (uint32_t)(cg * 16), raw);
    }
    tmem_wait_ld(raw);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && !two) break;
      const int c = (cg + u) * 16;
      float v[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 b = reinterpret_cast<const float4*>(s_bias + c)[j];
        v[4 * j] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j]), b.x);
        v[4 * j + 1] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j + 1]), b.y);
        v[4 * j + 2] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j + 2]), b.z);
        v[4 * j + 3] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j + 3]), b.w);
      }
      epi_apply16<KIND>(v, s_a + c, s_b + c, s_c + c);
      if (sizeof(TOut) == 2 && two) {
        const int sw = (lane >> 1) & 3;
        stage[lane * 4 + ((2 * u) ^ sw)] = pack8<TOut>(v);
        stage[lane * 4 + ((2 * u + 1) ^ sw)] = pack8<TOut>(v + 8);
      } else if (WHOLE || lane < rows) {
        store16_vec<TOut>(yrow + c, v, WHOLE ? 16 : cols - c);
      }
    }
    if (sizeof(TOut) == 2 && two) {
      __syncwarp();
      const int slot = cg * 16 + (lane & 3) * 8;             // this lane's 16-byte column slot
      const int in = slot + 8 <= cols ? rows : 0;
      TOut* base = yrow + slot;                              // (in its own row)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        const uint4 x = stage[r * 4 + ((lane & 3) ^ ((r >> 1) & 3))];
        if (r < in) *reinterpret_cast<uint4*>(base + (int64_t)(r - lane) * ldy) = x;
      }
      __syncwarp();                                          // the next round overwrites the staging area
    }
  }
}

// A unit of W columns of this thread's row into the warp's staging area, as a W-column copy reads it (pieces swizzled as in
// epi_tile_fast; rows of 32 bytes where W = 16).
template <typename TOut, int KIND, int W>
__device__ __forceinline__ void epi_unit(uint32_t tmem_at, float alpha, const float* s_bias, const float* s_a, const float* s_b, const float* s_c,
                                         uint4* area, int lane) {
  using namespace umma;
  uint32_t raw[W];
  if constexpr (W == 32) tmem_ld32_nowait(tmem_at, raw);
  else tmem_ld16_nowait(tmem_at, raw);
  tmem_wait_ld(raw);
  const int sw = W == 32 ? (lane >> 1) & 3 : (lane >> 2) & 1;
#pragma unroll
  for (int u = 0; u < W / 16; ++u) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 b = reinterpret_cast<const float4*>(s_bias + 16 * u)[j];
      v[4 * j] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j]), b.x);
      v[4 * j + 1] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j + 1]), b.y);
      v[4 * j + 2] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j + 2]), b.z);
      v[4 * j + 3] = fmaf(alpha, __uint_as_float(raw[16 * u + 4 * j + 3]), b.w);
    }
    epi_apply16<KIND>(v, s_a + 16 * u, s_b + 16 * u, s_c + 16 * u);
    area[lane * (W / 8) + ((2 * u) ^ sw)] = pack8<TOut>(v);
    area[lane * (W / 8) + ((2 * u + 1) ^ sw)] = pack8<TOut>(v + 8);
  }
}

template <typename F>
__device__ __forceinline__ void with_kind(int kind, F f) {
  switch (kind) {
    case XB_EPI_PRELU: f(std::integral_constant<int, XB_EPI_PRELU>()); break;
    case XB_EPI_DICE: f(std::integral_constant<int, XB_EPI_DICE>()); break;
    case XB_EPI_SIGMOID: f(std::integral_constant<int, XB_EPI_SIGMOID>()); break;
    default: f(std::integral_constant<int, XB_EPI_NONE>()); break;
  }
}

// Epilogue of a tile whose results leave by TMA, a warp's 32 rows x W columns at a time: units `part`, `part` + 4, ... of the tile.
// A warp with two units a tile has two areas, so that it fills one while the other is read. What the threads' own stores and their
// reads of the staging area took of the data path (4900 wavefronts a tile of 128 x 256, 5000 cycles) is the copy engine's work here.
// [65536, 88] x [88, 256] fp16: 16.1 -> 11.8 us, N = 192 14.4 -> 10.5, 8 x ([4096, 256] x [256, 128]) side by side 8.3 -> 7.9.
// A sigmoid's division is most of an epilogue that has one (8 x ([33434, 88] x [88, 32]) 32 us, 20 without an activation).
// A turn is a copy: the wait counts committed groups, so a warp whose rows all lie past the output (`rows` false) takes no turn and
// leaves the areas as they are. (With turns that commit nothing, the wait for all but the latest copy would name the copy of the other
// area, and a later unit could overwrite what that copy still reads.)
template <typename TOut, int KIND, int W>
__device__ __forceinline__ void epi_tile_tma(const CUtensorMap& map_y, uint32_t tmem_row, int part, int cols, float alpha, const float* s_bias,
                                             const float* s_a, const float* s_b, const float* s_c, uint8_t* stage, int bufs, uint32_t& turn,
                                             int x, int y, int z, bool rows, int lane) {
  using namespace umma;
  if (!rows) return;                                         // (the same for the warp)
  for (int c = part * W; c < cols; c += 4 * W) {
    uint8_t* area = stage + (bufs == 2 ? (turn & 1u) * (32 * W * 2) : 0u);
    ++turn;
    if (lane == 0) {                                         // the copy that read this area last has done so
      if (bufs == 2) tma_store_wait_read<1>();
      else tma_store_wait_read<0>();
    }
    __syncwarp();
    epi_unit<TOut, KIND, W>(tmem_row + (uint32_t)c, alpha, s_bias + c, s_a + c, s_b + c, s_c + c, reinterpret_cast<uint4*>(area), lane);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) tma_store_3d(&map_y, smem_u32(area), x + c, y, z);
  }
}

// bias and activation parameters of output column gn into entry e of the staged columns
__device__ __forceinline__ void stage_columns(const UmmaGemmParams& p, int b, int gn, int e, float* s_bias, float* s_a, float* s_b,
                                              float* s_c) {
  const bool in = gn < p.N;
  float bv = 0.f, pa = 0.f, pb = 0.f, pc = 0.f;
  if (in && p.bias_kind == XB_BIAS_ROW) bv = p.beta * load_as_f32(p.bias, (int64_t)b * p.stride_bias + gn, p.bias_dtype);
  if (in && p.epi.kind == XB_EPI_PRELU) pa = p.epi.a[(int64_t)b * p.stride_ep + (p.epi.count == 1 ? 0 : gn)];
  if (in && p.epi.kind == XB_EPI_DICE) {
    const float var = p.epi.c[(int64_t)b * p.stride_ep + gn];
    pa = p.epi.a[(int64_t)b * p.stride_ep + gn];                            // gamma
    pc = p.epi.nosqrt ? 1.f / var : rsqrtf(var + 1e-8f);                    // 1/std
    pb = -p.epi.b[(int64_t)b * p.stride_ep + gn] * pc;                      // -mean/std
  }
  s_bias[e] = bv; s_a[e] = pa; s_b[e] = pb; s_c[e] = pc;
}

// Epilogue of any output: rows that start or end anywhere, a full bias matrix where there is one.
template <typename TOut>
__device__ __forceinline__ void epi_tile_edge(const UmmaGemmParams& p, uint32_t tmem_row, int c_begin, int c_end, const float* s_bias,
                                              const float* s_a, const float* s_b, const float* s_c, TOut* yrow, int b, int gm,
                                              int brow, int n0, bool vec_base, uint16_t* stage, int lane) {
  using namespace umma;
  for (int cg = c_begin; cg < c_end; ++cg) {
    uint32_t raw[16];
    tmem_ld16_nowait(tmem_row + (uint32_t)(cg * 16), raw);
    tmem_wait_ld(raw);
    const int c = cg * 16, gn0 = n0 + c, valid = min(p.N - gn0, 16);
    if (valid <= 0) continue;                                        // uniform across the warp
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = fmaf(p.alpha, __uint_as_float(raw[i]), s_bias[c + i]);
    if (p.bias_kind == XB_BIAS_FULL && gm < p.M) {
      const int64_t base = (int64_t)b * p.stride_bias + (int64_t)brow * p.ldbias + gn0;
      const float* bf = reinterpret_cast<const float*>(p.bias) + base;
      if (p.bias_dtype == XB_F32 && valid == 16 && (reinterpret_cast<uintptr_t>(bf) & 15) == 0) {
        // fp32 rows (the per-group partial product of a pruned GEMM): four 16-byte loads, mostly one
        // address per warp since consecutive output rows share the bias row
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 t = __ldg(reinterpret_cast<const float4*>(bf) + i);
          v[4 * i] += p.beta * t.x; v[4 * i + 1] += p.beta * t.y;
          v[4 * i + 2] += p.beta * t.z; v[4 * i + 3] += p.beta * t.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < valid) v[i] += p.beta * load_as_f32(p.bias, base + i, p.bias_dtype);
      }
    }
    if (p.epi.kind == XB_EPI_PRELU) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = act_prelu(v[i], s_a[c + i]);
    } else if (p.epi.kind == XB_EPI_DICE) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float g = s_a[c + i];
        const float pr = __fdividef(1.f, 1.f + __expf(-fmaf(v[i], s_c[c + i], s_b[c + i])));
        v[i] = v[i] * fmaf(pr, 1.f - g, g);
      }
    } else if (p.epi.kind == XB_EPI_SIGMOID) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = act_sigmoid(v[i]);
    }
    const bool vec = vec_base && ((gn0 * sizeof(TOut)) % 16 == 0);
    if (sizeof(TOut) == 2 && !(vec && valid == 16)) {
      // Rows that start anywhere: a store of one element per lane and row touches 32 lines, so the warp turns its 32 x 16 results
      // and writes two rows at a time. [65536, 256] x [256, 255] fp16: 173 -> 29 us; [40594, 104] x [104, 41] 24 -> 8.3;
      // 8 x ([4198, 48] x [48, 398]) with a sigmoid 170 -> 36.
      const int piece = (lane >> 2) & 1;                              // (swapped in every other four rows: no bank conflicts)
      reinterpret_cast<uint4*>(stage)[lane * 2 + piece] = pack8<TOut>(v);
      reinterpret_cast<uint4*>(stage)[lane * 2 + (piece ^ 1)] = pack8<TOut>(v + 8);
      __syncwarp();
      const int col = lane & 15, rows = p.M - (gm - lane);            // (gm - lane: the warp's first row)
      uint16_t* at = reinterpret_cast<uint16_t*>(yrow + gn0) + (int64_t)((lane >> 4) - lane) * p.ldy + col;
#pragma unroll 4
      for (int i = 0; i < 16; ++i, at += 2 * p.ldy) {
        const int r = 2 * i + (lane >> 4);
        const uint16_t x = stage[r * 16 + ((col >> 3) ^ ((r >> 2) & 1)) * 8 + (col & 7)];
        if (r < rows && col < valid) *at = x;
      }
      __syncwarp();
    } else if (gm < p.M) {
      store_row16<TOut>(yrow + gn0, v, valid, vec);
    }
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  // (looked up once, whichever thread calls first)
  static const EncodeTiledFn fn = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess && qres == cudaDriverEntryPointSuccess;
    return found ? reinterpret_cast<EncodeTiledFn>(sym) : nullptr;
  }();
  return fn;
}

// [batch, rows, K] tensor of 2-byte elements, box {box_cols, box_rows, box_batch}, swizzled over the box's row (an N-major B is the same with
// its k rows as rows and its columns as the inner extent; so is Y)
int make_map(CUtensorMap* map, const void* base, int is_bf16, int64_t K, int64_t rows, int64_t ld, int64_t batch,
             int64_t batch_stride, int box_rows, int box_cols = BLOCK_K, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B, int box_batch = 1,
             CUtensorMapL2promotion promotion = CU_TENSOR_MAP_L2_PROMOTION_L2_128B) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(XB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(batch > 1 ? batch_stride : ld * rows) * 2};
  if (strides[1] == 0) strides[1] = strides[0];
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, (cuuint32_t)box_batch};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(XB_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  return 0;
}

}  // namespace
}  // namespace xb
