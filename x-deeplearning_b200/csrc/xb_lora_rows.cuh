// The projection and U B^T for few rows: one kernel of warp-level matrix instructions (included by xb_lora.cu).
#pragma once

#include "xb_common.cuh"
#include "xb_mma_half.cuh"
#include "xb_umma.cuh"

namespace xb {
namespace {

constexpr int LORA_MAX_RANK = 128;

struct LoraParams {
  int M, N, K, r, n_adapters;
  const void* X; int64_t ldx;
  const void* A; int64_t lda, stride_a;
  const void* B; int64_t ldb, stride_b;
  const float* scale;
  const float* bias;
  const int32_t* adapter;
  float* U;                               // [M, r]: scale[a] X[m] A[a]^T
  float* part;                            // [M, N]: bias + U[m] B[a]^T
};

// the adapter of row m, -1 where it has none (n_adapters is 0 where the call has none: then `adapter` may be null)
__device__ __forceinline__ int adapter_of(const LoraParams& p, int m) {
  const int a = p.n_adapters > 0 ? p.adapter[m] : -1;
  return a >= 0 && a < p.n_adapters ? a : -1;
}

// Y = X W + bias + U B_a^T for tiles of 64 rows x 32 columns. With few tiles a cluster of up to eight CTAs shares one, each with its part of
// the depth: all of what it reads is on its way at once, it makes its own products with B meanwhile, and the partial sums are added out
// of one another's shared memory, every CTA for its share of the rows. Sums as in gemm_half_kernel: 16 products by a matrix
// instruction, added in fp32. What bounds it is the latency of one round to memory, the exchange and the launch.
// The depth is split in equal parts while those are deeper than ROWS_PART and the SMs have room, and a part comes in as few equal slices as ROWS_BK
// allows. The call in a graph, 64 adapters of rank 16, us; slices of 320 as the unit of both (K = 1288 was five of them for four CTAs), 256 for
// both, these: [64, K] x [K, 1024], K = 320 12.4, 10.2, 10.1; 640 11.4, 9.7, 9.7; 1280 11.4, 10.7, 10.6; 1288 15.9, 11.1, 11.2; where two or four
// CTAs are all there is room for: [400, K] x [K, 304], K = 1280 15.6, 17.3, 14.5; 2048 22.4, 21.5, 18.6; [960, K] x [K, 152], K = 640 15.2, 15.9,
// 15.1; 2048 30.2, 27.2, 26.9. ROWS_BK = 448 is no quicker. (xb_gemm with a bias matrix and a kernel that makes that: 17 at K = 1280, N = 1024.)
constexpr int ROWS_BM = 64, ROWS_BN = 32, ROWS_BK = 384, ROWS_PART = 256, ROWS_THREADS = 256;
constexpr int ROWS_XPITCH = ROWS_BK + 8, ROWS_WPITCH = ROWS_BN + 8;          // halves: no bank conflicts of the eight rows that are read together
constexpr int ROWS_X_BYTES = ROWS_BM * ROWS_XPITCH * 2;
constexpr int ROWS_W_BYTES = ROWS_BK * ROWS_WPITCH * 2;                      // (as [K, N]; the other form is smaller)
constexpr int ROWS_SMEM = ROWS_X_BYTES + ROWS_W_BYTES + ROWS_BM * ROWS_BN * 4;
static_assert(ROWS_BN * ROWS_XPITCH * 2 <= ROWS_W_BYTES, "both forms of W fit the same space");

struct LoraRowsParams {
  LoraParams l;
  const void* W; int64_t ldw;
  void* Y; int64_t ldy;
  int split;                              // CTAs of a tile
  int part, slice;                        // of the depth: a CTA's, and what it brings at once (multiples of 16, slice <= ROWS_BK)
  int y_f32;
  int lanes;                              // that share a row of B, 16 bytes each (a power of two); 0: rows in single elements
};

// 16 bytes of which the first `bytes` exist (the rest becomes zeros)
__device__ __forceinline__ void cp_async16_part(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(umma::smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(umma::cluster_addr(addr, rank)) : "memory");
  return v;
}

// u B^T for 32 columns, by a warp: LP lanes share a column's row of B, so that a load takes whole rows of 32 / LP columns, and their sums
// change sides until lane l has those of column (l % LP) 32 / LP + l / LP. With a column a lane every load touches 32 lines: 230 rows,
// N = 608, rank 64, the call in a graph 38 us, 15 now.
template <int LP, typename T>
__device__ __forceinline__ float expand_row(const T* B, int64_t ldb, const float* u, int r, int cols, int lane) {
  const int sub = lane % LP, c0 = lane / LP, j = sub * 8;
  uint4 t[LP];
#pragma unroll
  for (int g = 0; g < LP; ++g) {
    const int c = g * (32 / LP) + c0;
    t[g] = j < r && c < cols ? __ldg(reinterpret_cast<const uint4*>(B + (int64_t)c * ldb + j)) : make_uint4(0u, 0u, 0u, 0u);
  }
  float uv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[LP];
  if (j < r) {
    const float4 u0 = *reinterpret_cast<const float4*>(u + j), u1 = *reinterpret_cast<const float4*>(u + j + 4);
    uv[0] = u0.x; uv[1] = u0.y; uv[2] = u0.z; uv[3] = u0.w; uv[4] = u1.x; uv[5] = u1.y; uv[6] = u1.z; uv[7] = u1.w;
  }
#pragma unroll
  for (int g = 0; g < LP; ++g) {
    const T* e = reinterpret_cast<const T*>(&t[g]);
    v[g] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[g] = fmaf(uv[k], to_f32<T>(e[k]), v[g]);
  }
  int have = LP;
#pragma unroll
  for (int m = LP / 2; m > 0; m >>= 1) {
    have /= 2;
    const bool up = sub & m;
#pragma unroll
    for (int g = 0; g < LP / 2; ++g)
      if (g < have) {
        const float give = up ? v[g] : v[g + have], keep = up ? v[g + have] : v[g];
        v[g] = keep + __shfl_xor_sync(0xffffffffu, give, m);
      }
  }
  return v[0];
}

template <typename T, bool TRANS_W>
__global__ void __launch_bounds__(ROWS_THREADS, 2) lora_rows_gemm_kernel(const __grid_constant__ LoraRowsParams p) {
  pdl_begin();
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(16) uint8_t rows_smem[];
  uint16_t* xs = reinterpret_cast<uint16_t*>(rows_smem);
  uint16_t* ws = reinterpret_cast<uint16_t*>(rows_smem + ROWS_X_BYTES);
  float* part = reinterpret_cast<float*>(rows_smem + ROWS_X_BYTES + ROWS_W_BYTES);       // [64][32]
  const int rank = blockIdx.x % p.split, m0 = blockIdx.y * ROWS_BM, n0 = (int)(blockIdx.x / p.split) * ROWS_BN;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const LoraParams& l = p.l;
  // this CTA's part of the depth
  const int k_begin = (int)min((int64_t)l.K, (int64_t)rank * p.part), k_end = min(l.K, k_begin + p.part);

  auto bring = [&](int k0) {
    const int depth = min(p.slice, k_end - k0), wide = (depth + 15) / 16 * 2;        // pieces of 8, up to whole steps of 16
    const T* X = reinterpret_cast<const T*>(l.X);
    const T* W = reinterpret_cast<const T*>(p.W);
    for (int e = tid; e < ROWS_BM * wide; e += ROWS_THREADS) {
      const int r = e / wide, c = (e - r * wide) * 8, in = m0 + r < l.M ? max(0, min(8, depth - c)) * 2 : 0;
      cp_async16_part(xs + r * ROWS_XPITCH + c, X + (in ? (int64_t)(m0 + r) * l.ldx + k0 + c : 0), in);
    }
    if (TRANS_W) {
      for (int e = tid; e < ROWS_BN * wide; e += ROWS_THREADS) {
        const int r = e / wide, c = (e - r * wide) * 8, in = n0 + r < l.N ? max(0, min(8, depth - c)) * 2 : 0;
        cp_async16_part(ws + r * ROWS_XPITCH + c, W + (in ? (int64_t)(n0 + r) * p.ldw + k0 + c : 0), in);
      }
    } else {
      for (int e = tid; e < wide * 8 * (ROWS_BN / 8); e += ROWS_THREADS) {
        const int r = e / (ROWS_BN / 8), c = e % (ROWS_BN / 8) * 8, in = r < depth ? max(0, min(8, l.N - n0 - c)) * 2 : 0;
        cp_async16_part(ws + r * ROWS_WPITCH + c, W + (in ? (int64_t)(k0 + r) * p.ldw + n0 + c : 0), in);
      }
    }
    umma::cp_async_commit();
  };
  if (k_begin < k_end) bring(k_begin);

  // the outputs that this thread ends with: OUT rows of one column; bias and U B^T for them
  const int share = ROWS_BM / p.split, first = rank * share, step = ROWS_THREADS / 32;
  const int LP = p.lanes, at_col = LP > 1 ? lane % LP * (32 / LP) + lane / LP : lane, col = n0 + at_col;
  constexpr int OUT = ROWS_BM / (ROWS_THREADS / 32);
  float out[OUT];
#pragma unroll
  for (int i = 0; i < OUT; ++i) out[i] = 0.f;
  {
    const float bias = l.bias && col < l.N ? l.bias[col] : 0.f;
    auto adapter_at = [&](int i) {                         // of this warp's i-th row
      const int m = m0 + first + warp + i * step;
      return i * step + warp < share && m < l.M ? adapter_of(l, m) : -1;
    };
    const float* u = l.U + (int64_t)(m0 + first + warp) * l.r;
    const T* B = reinterpret_cast<const T*>(l.B) + (int64_t)n0 * l.ldb;
    // (a loop: eight rows one behind the other are so much code that its fetching shows in a call of 12 us)
    auto products = [&](auto lanes) {
      constexpr int L = decltype(lanes)::value;
      int a = adapter_at(0);
#pragma unroll 1
      for (int i = 0; i * step < share; ++i) {
        const int now = a;
        a = adapter_at(i + 1);
        if (now < 0) continue;
        const float v = expand_row<L, T>(B + (int64_t)now * l.stride_b, l.ldb, u + (int64_t)i * step * l.r, l.r, l.N - n0, lane);
#pragma unroll
        for (int k = 0; k < OUT; ++k) out[k] = k == i ? v : out[k];
      }
    };
    switch (LP) {
      case 1: products(std::integral_constant<int, 1>()); break;
      case 2: products(std::integral_constant<int, 2>()); break;
      case 4: products(std::integral_constant<int, 4>()); break;
      case 8: products(std::integral_constant<int, 8>()); break;
      case 16: products(std::integral_constant<int, 16>()); break;
      default:
        if (col < l.N) {
#pragma unroll
          for (int i = 0; i < OUT; ++i) {
            const int a = adapter_at(i);
            if (a < 0) continue;
            const T* b = B + (int64_t)a * l.stride_b + (int64_t)lane * l.ldb;
            for (int j = 0; j < l.r; ++j) out[i] = fmaf(u[(int64_t)i * step * l.r + j], to_f32<T>(b[j]), out[i]);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < OUT; ++i) out[i] += bias;
  }

  // 4 x 2 warps of 16 x 16 outputs
  const int wm = (warp >> 1) * 16, wn = (warp & 1) * 16, l8 = lane & 7, g1 = (lane >> 3) & 1, g2 = lane >> 4;
  const uint32_t x_at = umma::smem_u32(xs) + 2 * ((wm + g1 * 8 + l8) * ROWS_XPITCH + g2 * 8);
  const uint32_t w_at = umma::smem_u32(ws) + 2 * (TRANS_W ? (wn + g2 * 8 + l8) * ROWS_XPITCH + g1 * 8 : (g1 * 8 + l8) * ROWS_WPITCH + wn + g2 * 8);
  float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  for (int k0 = k_begin; k0 < k_end; k0 += p.slice) {
    umma::cp_async_wait_all();
    __syncthreads();
    const int depth = min(p.slice, k_end - k0);
#pragma unroll 4
    for (int k = 0; k < depth; k += 16) {
      uint32_t af[4], bf[4];
      ldmatrix4<0>(af, x_at + 2 * k);
      ldmatrix4<TRANS_W ? 0 : 1>(bf, w_at + 2 * (TRANS_W ? k : k * ROWS_WPITCH));
      mma_half<BF16>(acc[0], af, bf[0], bf[1]);
      mma_half<BF16>(acc[1], af, bf[2], bf[3]);
    }
    __syncthreads();
    if (k0 + p.slice < k_end) bring(k0 + p.slice);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float2*>(part + (wm + 8 * h + (lane >> 2)) * ROWS_BN + wn + 8 * j + 2 * (lane & 3)) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
  if (p.split > 1) umma::cluster_sync();
  else __syncthreads();
  if (col < l.N) {
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      const int r = warp + i * step, m = m0 + first + r;
      if (r >= share || m >= l.M) continue;
      const uint32_t at = umma::smem_u32(part + (first + r) * ROWS_BN + at_col);
      float v = 0.f;
      if (p.split > 1) {
        for (int c = 0; c < p.split; ++c) v += ld_cluster_f32(at, (uint32_t)c);
      } else {
        v = part[(first + r) * ROWS_BN + at_col];
      }
      v += out[i];
      if (p.y_f32) reinterpret_cast<float*>(p.Y)[(int64_t)m * p.ldy + col] = v;
      else reinterpret_cast<T*>(p.Y)[(int64_t)m * p.ldy + col] = from_f32<T>(v);
    }
  }
  if (p.split > 1) umma::cluster_sync();               // nobody leaves while its sums may be read
}

template <typename T, bool TRANS_W>
int launch_rows_gemm(const LoraRowsParams& p, cudaStream_t s) {
  static PerDeviceOnce attr_set;          // per instantiation
  XB_SET_MAX_SMEM_ONCE(attr_set, ROWS_SMEM, (const void*)lora_rows_gemm_kernel<T, TRANS_W>);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)p.split; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.l.N + ROWS_BN - 1) / ROWS_BN * p.split), (unsigned)((p.l.M + ROWS_BM - 1) / ROWS_BM));
  cfg.blockDim = ROWS_THREADS; cfg.dynamicSmemBytes = ROWS_SMEM; cfg.stream = s; cfg.attrs = at; cfg.numAttrs = p.split > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, lora_rows_gemm_kernel<T, TRANS_W>, p);
  return check_launch("lora_rows_gemm_kernel");
}

}  // namespace
}  // namespace xb
