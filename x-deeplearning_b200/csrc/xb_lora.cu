// A projection with a low-rank adapter of each row's own beside it (formulas in xdlb200.h).
#include <algorithm>
#include <cstring>

#include "xb_common.cuh"
#include "xb_lora_umma.cuh"

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

// A warp a row: its products with the r rows of its adapter, the lanes along K.
template <typename T>
__global__ void __launch_bounds__(256) lora_rows_shrink_kernel(const LoraParams p) {
  pdl_begin();
  const int m = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (m >= p.M) return;
  const int a = adapter_of(p, m);
  if (a < 0) return;
  const T* x = reinterpret_cast<const T*>(p.X) + (int64_t)m * p.ldx;
  const float scale = p.scale ? p.scale[a] : 1.f;
  for (int j = 0; j < p.r; ++j) {
    const T* w = reinterpret_cast<const T*>(p.A) + (int64_t)a * p.stride_a + (int64_t)j * p.lda;
    float s = 0.f;
    for (int k = lane; k < p.K; k += 32) s = fmaf(to_f32<T>(x[k]), to_f32<T>(w[k]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) p.U[(int64_t)m * p.r + j] = s * scale;
  }
}

// A block a row, a thread an output at a time.
template <typename T>
__global__ void __launch_bounds__(128) lora_rows_expand_kernel(const LoraParams p) {
  pdl_begin();
  const int m = blockIdx.x;
  const int a = adapter_of(p, m);
  const bool with = a >= 0;
  for (int n = threadIdx.x; n < p.N; n += 128) {
    float s = p.bias ? p.bias[n] : 0.f;
    if (with) {
      const T* w = reinterpret_cast<const T*>(p.B) + (int64_t)a * p.stride_b + (int64_t)n * p.ldb;
      float d = 0.f;
      for (int j = 0; j < p.r; ++j) d = fmaf(p.U[(int64_t)m * p.r + j], to_f32<T>(w[j]), d);
      s += d;
    }
    p.part[(int64_t)m * p.N + n] = s;
  }
}

// Few rows: the tiles would leave most SMs idle, and a tile of many adapters walks through all of them.
bool takes_tiles(const xb_lora_args& a) { return a.M >= 512 && lora_umma_takes(a); }

constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Rows of a turn: the fp32 addend of a turn (M x N) is at most 64 MB, so that it is still in L2 when the product reads it.
int turn_rows(const xb_lora_args& a) {
  const int64_t rows = std::max<int64_t>(((int64_t)16 << 20) / std::max(a.N, 1) / 128 * 128, 128);
  return (int)std::min<int64_t>(rows, a.M);
}

int check_args(const xb_lora_args* a) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_lora_gemm: null arguments");
  XB_REQUIRE(a->dtype == XB_F32 || a->dtype == XB_F16 || a->dtype == XB_BF16, XB_ERR_UNSUPPORTED, "xb_lora_gemm: dtype %d", a->dtype);
  XB_REQUIRE(a->y_dtype == a->dtype || a->y_dtype == XB_F32, XB_ERR_UNSUPPORTED, "xb_lora_gemm: results of dtype %d from dtype %d", a->y_dtype,
             a->dtype);
  XB_REQUIRE(a->M >= 0 && a->N >= 0 && a->K >= 1 && a->r >= 0 && a->n_adapters >= 0, XB_ERR_ARG, "xb_lora_gemm: bad sizes");
  XB_REQUIRE(a->r <= LORA_MAX_RANK, XB_ERR_LIMIT, "xb_lora_gemm: rank %d, at most %d", a->r, LORA_MAX_RANK);
  if (a->M == 0 || a->N == 0) return 0;
  const bool adapters = a->n_adapters > 0 && a->r > 0;
  XB_REQUIRE(a->Y && a->X && a->W, XB_ERR_ARG, "xb_lora_gemm: null tensor");
  XB_REQUIRE(a->ldx >= a->K && a->ldy >= a->N && a->ldw >= (a->trans_w ? a->K : a->N), XB_ERR_ARG, "xb_lora_gemm: a row stride is too small");
  XB_REQUIRE(!adapters || (a->adapter && a->B && a->A), XB_ERR_ARG, "xb_lora_gemm: null adapter");
  XB_REQUIRE(!adapters || (a->lda >= a->K && a->ldb >= a->r && a->stride_a >= 0 && a->stride_b >= 0), XB_ERR_ARG,
             "xb_lora_gemm: a stride of the adapters is too small");
  return 0;
}

template <typename T>
int run_rows(const xb_lora_args& a, uint8_t* ws, cudaStream_t s) {
  const int turn = turn_rows(a);
  LoraParams p;
  p.N = a.N; p.K = a.K; p.r = a.r; p.n_adapters = a.r > 0 && a.adapter ? a.n_adapters : 0;
  p.A = a.A; p.lda = a.lda; p.stride_a = a.stride_a; p.B = a.B; p.ldb = a.ldb; p.stride_b = a.stride_b;
  p.scale = a.scale; p.bias = a.bias; p.ldx = a.ldx;
  p.U = reinterpret_cast<float*>(ws);
  p.part = reinterpret_cast<float*>(ws + align256((size_t)turn * a.r * 4));
  xb_gemm_args g;
  memset(&g, 0, sizeof(g));
  g.N = a.N; g.K = a.K; g.trans_b = a.trans_w; g.alpha = g.beta = 1.f; g.batch = 1;
  g.lda = a.ldx; g.B = a.W; g.ldb = a.ldw; g.ldy = a.ldy; g.ab_dtype = a.dtype; g.y_dtype = a.y_dtype;
  g.bias = p.part; g.ldbias = a.N; g.bias_kind = XB_BIAS_FULL; g.bias_dtype = XB_F32;
  for (int64_t m0 = 0; m0 < a.M; m0 += turn) {
    p.M = (int)std::min<int64_t>(turn, a.M - m0);
    p.X = reinterpret_cast<const T*>(a.X) + m0 * a.ldx;
    p.adapter = p.n_adapters ? a.adapter + m0 : nullptr;
    if (p.n_adapters) {
      launch_dependent(lora_rows_shrink_kernel<T>, (unsigned)((p.M + 7) / 8), 256, 0, s, p);
      if (int rc = check_launch("lora_rows_shrink_kernel")) return rc;
    }
    launch_dependent(lora_rows_expand_kernel<T>, (unsigned)p.M, 128, 0, s, p);
    if (int rc = check_launch("lora_rows_expand_kernel")) return rc;
    g.M = p.M;
    g.A = p.X;
    g.Y = reinterpret_cast<uint8_t*>(a.Y) + m0 * a.ldy * (int64_t)dtype_size(a.y_dtype);
    if (int rc = xb_gemm(&g, s)) return rc;
  }
  return 0;
}

}  // namespace

int lora_status(int* out) { return umma::read_status_word(out); }
int lora_clear_status() { return umma::clear_status_word(); }
int lora_set_status_mirror(int* p) { return umma::set_status_mirror(p); }
}  // namespace xb

using namespace xb;

extern "C" size_t xb_lora_workspace_bytes(const xb_lora_args* a) {
  if (check_args(a) != 0 || a->M == 0 || a->N == 0) return 0;
  if (takes_tiles(*a)) return lora_scratch(*a).bytes;
  const size_t turn = (size_t)turn_rows(*a);
  return align256(turn * a->r * 4) + turn * a->N * 4;
}

extern "C" int xb_lora_gemm(const xb_lora_args* a, void* workspace, size_t workspace_bytes, xb_stream_t s) {
  if (int rc = check_args(a)) return rc;
  if (a->M == 0 || a->N == 0) return 0;
  const size_t need = xb_lora_workspace_bytes(a);
  XB_REQUIRE(workspace && workspace_bytes >= need, XB_ERR_SCRATCH, "xb_lora_gemm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  XB_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, XB_ERR_ARG, "xb_lora_gemm: the workspace is not on 16 bytes");
  if (takes_tiles(*a)) return run_umma(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
  if (a->dtype == XB_F32) return run_rows<float>(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
  if (a->dtype == XB_F16) return run_rows<__half>(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
  return run_rows<__nv_bfloat16>(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
}
