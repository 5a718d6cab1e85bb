// A projection with a low-rank adapter of each row's own beside it (formulas in xdlb200.h).
#include <algorithm>
#include <cstring>

#include "xb_common.cuh"
#include "xb_lora_rows.cuh"
#include "xb_lora_umma.cuh"

namespace xb {

int gemm_half_sums(const xb_gemm_args& a, cudaStream_t stream);

namespace {

// V adjacent elements as fp32: one load where they lie aligned, which V > 1 says
template <typename T, int V>
__device__ __forceinline__ void load_piece(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32<T>(p[0]);
  } else {
    static_assert(V * sizeof(T) == 16, "");
    const uint4 t = __ldg(reinterpret_cast<const uint4*>(p));
    const T* e = reinterpret_cast<const T*>(&t);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32<T>(e[i]);
  }
}

// A warp takes four products of one row with the rows of its adapter's A, the lanes along K. Bound by the latency of the few rounds over K
// where there are few rows, by A from L2 otherwise. 64 rows of 1280, rank 16: 79 us with a warp for all of a row's products, 4 now;
// 5003 of 250, rank 12, rows that start anywhere: 20, 5.
constexpr int SHRINK_J = 4;
template <typename T, int V>
__global__ void __launch_bounds__(128) lora_rows_shrink_kernel(const LoraParams p) {
  pdl_begin();
  const int parts = (p.r + SHRINK_J - 1) / SHRINK_J, lane = threadIdx.x % 32;
  const int64_t w = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int m = (int)(w / parts), j0 = (int)(w - (int64_t)m * parts) * SHRINK_J;
  if (m >= p.M) return;
  const int a = adapter_of(p, m);
  if (a < 0) return;
  const T* x = reinterpret_cast<const T*>(p.X) + (int64_t)m * p.ldx;
  // (rows of A past the last are the last again, and what they give is dropped: a branch would keep the loads of a round from the next's)
  const T* at[SHRINK_J];
#pragma unroll
  for (int j = 0; j < SHRINK_J; ++j) at[j] = reinterpret_cast<const T*>(p.A) + (int64_t)a * p.stride_a + (int64_t)min(j0 + j, p.r - 1) * p.lda;
  float s[SHRINK_J] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = lane * V; k < p.K; k += 32 * V) {         // (V > 1: whole pieces, K is a multiple of V)
    float xv[V];
    load_piece<T, V>(x + k, xv);
#pragma unroll
    for (int j = 0; j < SHRINK_J; ++j) {
      float av[V];
      load_piece<T, V>(at[j] + k, av);
#pragma unroll
      for (int v = 0; v < V; ++v) s[j] = fmaf(xv[v], av[v], s[j]);
    }
  }
  const float scale = p.scale ? p.scale[a] : 1.f;
#pragma unroll
  for (int j = 0; j < SHRINK_J; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
    if (lane == 0 && j0 + j < p.r) p.U[(int64_t)m * p.r + j0 + j] = s[j] * scale;
  }
}

// A thread has one column of ROWS adjacent rows, whose B it keeps while they have the same adapter; 16 of the rank at a time.
constexpr int EXPAND_J = 16;
template <typename T, bool VEC, int ROWS>
__global__ void __launch_bounds__(128) lora_rows_expand_kernel(const LoraParams p) {
  pdl_begin();
  __shared__ float s_u[ROWS][LORA_MAX_RANK];
  __shared__ int s_a[ROWS];
  const int m0 = blockIdx.x * ROWS, n = blockIdx.y * 128 + threadIdx.x;
  if (threadIdx.x < ROWS) s_a[threadIdx.x] = m0 + (int)threadIdx.x < p.M ? adapter_of(p, m0 + threadIdx.x) : -1;
  __syncthreads();
  for (int i = threadIdx.x; i < ROWS * p.r; i += 128) {
    const int m = i / p.r, j = i - m * p.r;
    s_u[m][j] = s_a[m] >= 0 ? p.U[(int64_t)(m0 + m) * p.r + j] : 0.f;
  }
  __syncthreads();
  if (n >= p.N) return;
  float sum[ROWS];
#pragma unroll
  for (int m = 0; m < ROWS; ++m) sum[m] = 0.f;
  for (int j0 = 0; j0 < p.r; j0 += EXPAND_J) {
    float b[EXPAND_J];
    int held = -1;
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      const int a = s_a[m];
      if (a < 0) continue;
      if (a != held) {
        held = a;
        const T* at = reinterpret_cast<const T*>(p.B) + (int64_t)a * p.stride_b + (int64_t)n * p.ldb + j0;
        if constexpr (VEC) {
          constexpr int V = 16 / sizeof(T);
#pragma unroll
          for (int i = 0; i < EXPAND_J / V; ++i) {
            float t[V];
#pragma unroll
            for (int v = 0; v < V; ++v) t[v] = 0.f;
            if (j0 + i * V < p.r) load_piece<T, V>(at + i * V, t);
#pragma unroll
            for (int v = 0; v < V; ++v) b[i * V + v] = t[v];
          }
        } else {
#pragma unroll
          for (int j = 0; j < EXPAND_J; ++j) b[j] = j0 + j < p.r ? to_f32<T>(at[j]) : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < EXPAND_J; ++j)
        if (j0 + j < p.r) sum[m] = fmaf(s_u[m][j0 + j], b[j], sum[m]);
    }
  }
  const float bias = p.bias ? p.bias[n] : 0.f;
#pragma unroll
  for (int m = 0; m < ROWS; ++m)
    if (m0 + m < p.M) p.part[(int64_t)(m0 + m) * p.N + n] = bias + sum[m];
}

// Few rows: lora_rows_gemm_kernel while its tiles are at most two blocks an SM, which is what runs at once. us in a graph, 16 adapters, K = 1280,
// the tensor-core tiles and this kernel: 960 rows, N = 152, rank 8 31 and 19, rank 64 66 and 28; 1920 rows 31 and 29, 66 and 49; 256 rows,
// N = 2048 28 and 28, 50 and 33; past two blocks: 448 rows, N = 2048 30 and 48; 1472, N = 600 33 and 49. Few columns and more rows:
// 4800, N = 40, rank 64 73 and 79, at K = 64 27 and 38.
// Rows that the kernel cannot take (not on 16 bytes) are laid out for the tensor cores from 512 on, whatever their adapters: us in a graph as rows and
// so, 8 adapters, bf16, [M, 250] x [250, 131], rank 12, M = 64 20.0 and 17.3, 512 21.0 and 11.4, 1024 24.0 and 11.1; [M, 73] x [73, 600], rank 8, 64 14.4
// and 14.4, 512 16.3 and 10.1; but 350 rows of 67 requests with 50 adapters, [350, 19] x [19, 114], rank 8, fp16 13.5 and 21.1: a tile has a product
// for each of its adapters, and few tiles have all of a call's. fp32 results also show that sums in tensor memory are cut off.
constexpr int ROWS_MOST = 2048, ROWS_ODD = 511;
bool on_16_bytes(const xb_lora_args& a) {
  auto lies = [](const void* q, int64_t ld) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0 && ld % 8 == 0; };
  return lies(a.X, a.ldx) && lies(a.W, a.ldw);
}
bool takes_rows_kernel(const xb_lora_args& a) {
  const int64_t tiles = ((int64_t)a.N + ROWS_BN - 1) / ROWS_BN * ((a.M + ROWS_BM - 1) / ROWS_BM);
  return a.dtype != XB_F32 && on_16_bytes(a) && a.M <= ROWS_MOST && tiles <= 2 * sm_count();
}
bool takes_tiles(const xb_lora_args& a) { return lora_umma_takes(a) && !takes_rows_kernel(a) && (on_16_bytes(a) || a.M > ROWS_ODD); }

constexpr size_t align256(size_t n) { return (n + 255) / 256 * 256; }

bool has_adapters(const xb_lora_args& a) { return a.n_adapters > 0 && a.r > 0; }

constexpr int TURN_COLS = 65535 * 128;    // columns of a turn: a grid's second dimension of lora_rows_expand_kernel's blocks
// Rows of a turn: the fp32 addend of a turn (M x N) is at most 64 MB, so that it is still in L2 when the product reads it, and no more than
// xb_gemm's CUDA cores take in a call.
int turn_rows(const xb_lora_args& a) {
  const int64_t rows = std::max<int64_t>(((int64_t)16 << 20) / std::clamp(a.N, 1, TURN_COLS) / 128 * 128, 128);
  return (int)std::min<int64_t>({rows, a.M, 32767 * 128});
}

// fp32 weights as [N, K] are laid out as [K, N] first, for which xb_gemm has a faster kernel. us in a graph without and with, whatever the rows:
// 8 rows, K = 72, N = 168 12 and 10, K = 1280, N = 1024 50 and 39; 3931 rows of the first 51 and 35; 20000 rows, K = 324, N = 200 194 and 168.
bool lays_out_w(const xb_lora_args& a) { return a.dtype == XB_F32 && a.trans_w && has_adapters(a); }
int64_t laid_out_ld(const xb_lora_args& a) { return ((int64_t)a.N + 3) / 4 * 4; }
struct RowsScratch { size_t part, w, bytes; };             // U lies first
RowsScratch rows_scratch(const xb_lora_args& a) {
  if (!has_adapters(a)) return {0, 0, 0};
  const size_t turn = (size_t)turn_rows(a);
  RowsScratch s;
  s.part = align256(turn * a.r * 4);
  s.w = s.part + align256(turn * std::min(a.N, TURN_COLS) * 4);
  s.bytes = s.w + (lays_out_w(a) ? (size_t)a.K * laid_out_ld(a) * 4 : 0);
  return s;
}
__global__ void __launch_bounds__(256) lora_layout_kernel(const float* w, int64_t ldw, float* to, int64_t ld, int N, int K) {
  pdl_begin();
  __shared__ float tile[32][33];
  const int across = (K + 31) / 32, n0 = (int)(blockIdx.x / across) * 32, k0 = (int)(blockIdx.x % across) * 32, x = threadIdx.x % 32, y = threadIdx.x / 32;
#pragma unroll
  for (int i = y; i < 32; i += 8)
    if (n0 + i < N && k0 + x < K) tile[i][x] = w[(int64_t)(n0 + i) * ldw + k0 + x];
  __syncthreads();
#pragma unroll
  for (int i = y; i < 32; i += 8)
    if (k0 + i < K && n0 + x < N) to[(int64_t)(k0 + i) * ld + n0 + x] = tile[x][i];
}

int check_args(const xb_lora_args* a) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_lora_gemm: null arguments");
  XB_REQUIRE(a->dtype == XB_F32 || a->dtype == XB_F16 || a->dtype == XB_BF16, XB_ERR_UNSUPPORTED, "xb_lora_gemm: dtype %d", a->dtype);
  XB_REQUIRE(a->y_dtype == a->dtype || a->y_dtype == XB_F32, XB_ERR_UNSUPPORTED, "xb_lora_gemm: results of dtype %d from dtype %d", a->y_dtype,
             a->dtype);
  XB_REQUIRE(a->M >= 0 && a->N >= 0 && a->K >= 1 && a->r >= 0 && a->n_adapters >= 0, XB_ERR_ARG, "xb_lora_gemm: bad sizes");
  // (sizes rounded up to whole tiles are counted in 32 bits)
  XB_REQUIRE(std::max({a->M, a->N, a->K}) <= INT32_MAX - 1023, XB_ERR_LIMIT, "xb_lora_gemm: %d x %d x %d, at most 2^31 - 1024 each", a->M, a->N, a->K);
  XB_REQUIRE(a->r <= LORA_MAX_RANK, XB_ERR_LIMIT, "xb_lora_gemm: rank %d, at most %d", a->r, LORA_MAX_RANK);
  if (a->M == 0 || a->N == 0) return 0;
  const bool adapters = has_adapters(*a);
  XB_REQUIRE(a->Y && a->X && a->W, XB_ERR_ARG, "xb_lora_gemm: null tensor");
  XB_REQUIRE(a->ldx >= a->K && a->ldy >= a->N && a->ldw >= (a->trans_w ? a->K : a->N), XB_ERR_ARG, "xb_lora_gemm: a row stride is too small");
  XB_REQUIRE(!adapters || (a->adapter && a->B && a->A), XB_ERR_ARG, "xb_lora_gemm: null adapter");
  XB_REQUIRE(!adapters || (a->lda >= a->K && a->ldb >= a->r && a->stride_a >= 0 && a->stride_b >= 0), XB_ERR_ARG,
             "xb_lora_gemm: a stride of the adapters is too small");
  return 0;
}

// the scratch of a call whose arguments have been checked
int scratch_of(const xb_lora_args& a, size_t* bytes) {
  if (!takes_tiles(a)) {
    *bytes = rows_scratch(a).bytes;
    return 0;
  }
  const LoraScratch w = lora_scratch(a);
  XB_REQUIRE(w.fits, XB_ERR_LIMIT, "xb_lora_gemm: %d adapters of rank %d beside %d x %d x %d are too many for one call", a.n_adapters, a.r, a.M, a.N, a.K);
  *bytes = w.bytes;
  return 0;
}

template <typename T>
int launch_shrink(const LoraParams& p, bool vec, cudaStream_t s) {
  if (p.n_adapters == 0) return 0;
  const int64_t warps = (int64_t)p.M * ((p.r + SHRINK_J - 1) / SHRINK_J);
  XB_REQUIRE(warps < ((int64_t)1 << 32), XB_ERR_LIMIT, "xb_lora_gemm: %d rows of rank %d are too many for one call", p.M, p.r);
  if (vec) launch_dependent(lora_rows_shrink_kernel<T, 16 / (int)sizeof(T)>, (unsigned)((warps + 3) / 4), 128, 0, s, p);
  else launch_dependent(lora_rows_shrink_kernel<T, 1>, (unsigned)((warps + 3) / 4), 128, 0, s, p);
  return check_launch("lora_rows_shrink_kernel");
}

template <typename T>
int launch_expand(const LoraParams& p, bool vec, cudaStream_t s) {
  // eight rows a block share what they read of B; two where that would leave SMs idle
  const unsigned cols = (unsigned)((p.N + 127) / 128);
  const bool few = (int64_t)((p.M + 7) / 8) * cols < 4 * sm_count();
  const dim3 grid((unsigned)(few ? (p.M + 1) / 2 : (p.M + 7) / 8), cols);
  if (few) {
    if (vec) launch_dependent(lora_rows_expand_kernel<T, true, 2>, grid, 128, 0, s, p);
    else launch_dependent(lora_rows_expand_kernel<T, false, 2>, grid, 128, 0, s, p);
  } else {
    if (vec) launch_dependent(lora_rows_expand_kernel<T, true, 8>, grid, 128, 0, s, p);
    else launch_dependent(lora_rows_expand_kernel<T, false, 8>, grid, 128, 0, s, p);
  }
  return check_launch("lora_rows_expand_kernel");
}

template <typename T>
int run_rows(const xb_lora_args& a, uint8_t* ws, cudaStream_t s) {
  const int turn = turn_rows(a);
  LoraParams p;
  p.N = a.N; p.K = a.K; p.r = a.r; p.n_adapters = has_adapters(a) ? a.n_adapters : 0;
  p.A = a.A; p.lda = a.lda; p.stride_a = a.stride_a; p.B = a.B; p.ldb = a.ldb; p.stride_b = a.stride_b;
  p.scale = a.scale; p.bias = a.bias; p.ldx = a.ldx;
  p.U = reinterpret_cast<float*>(ws);
  const RowsScratch scratch = rows_scratch(a);
  p.part = reinterpret_cast<float*>(ws + scratch.part);
  // 16-byte pieces of X and A along K, and of B along the rank
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec_k = a.K % V == 0 && a.ldx % V == 0 && a.lda % V == 0 && a.stride_a % V == 0 &&
                     ((reinterpret_cast<uintptr_t>(a.X) | reinterpret_cast<uintptr_t>(a.A)) & 15) == 0;
  const bool vec_r = a.r % V == 0 && a.ldb % V == 0 && a.stride_b % V == 0 && (reinterpret_cast<uintptr_t>(a.B) & 15) == 0;
  xb_gemm_args g;
  memset(&g, 0, sizeof(g));
  g.N = a.N; g.K = a.K; g.trans_b = a.trans_w; g.alpha = g.beta = 1.f; g.batch = 1;
  g.lda = a.ldx; g.B = a.W; g.ldb = a.ldw; g.ldy = a.ldy; g.ab_dtype = a.dtype; g.y_dtype = a.y_dtype;
  g.bias_dtype = XB_F32;
  if (p.n_adapters) { g.bias = p.part; g.bias_kind = XB_BIAS_FULL; }
  else if (a.bias) g.bias_kind = XB_BIAS_ROW;                               // without adapters: the projection alone
  if constexpr (sizeof(T) == 2) {
    // the projection and the products with B in one kernel (its rows are one turn: at most 2 sm_count() tiles of 64 x 32)
    if (takes_rows_kernel(a)) {
      p.M = a.M;
      p.X = a.X;
      p.adapter = p.n_adapters ? a.adapter : nullptr;
      if (int rc = launch_shrink<T>(p, vec_k, s)) return rc;
      LoraRowsParams r;
      r.l = p;
      r.W = a.W; r.ldw = a.ldw; r.Y = a.Y; r.ldy = a.ldy;
      r.y_f32 = a.y_dtype == XB_F32;
      r.lanes = !vec_r ? 0 : a.r <= 8 ? 1 : a.r <= 16 ? 2 : a.r <= 32 ? 4 : a.r <= 64 ? 8 : 16;
      const int64_t tiles = ((int64_t)a.N + ROWS_BN - 1) / ROWS_BN * ((a.M + ROWS_BM - 1) / ROWS_BM);
      r.split = 1;
      while (r.split < 8 && r.split * ROWS_PART < a.K && tiles * 2 * r.split <= 2 * sm_count()) r.split *= 2;
      auto share = [](int64_t k, int64_t n) { return (int)((k + n * 16 - 1) / (n * 16) * 16); };
      r.part = share(a.K, r.split);
      r.slice = share(r.part, (r.part + ROWS_BK - 1) / ROWS_BK);
      return a.trans_w ? launch_rows_gemm<T, true>(r, s) : launch_rows_gemm<T, false>(r, s);
    }
  }
  if (lays_out_w(a)) {
    const int64_t blocks = (((int64_t)a.K + 31) / 32) * (((int64_t)a.N + 31) / 32);
    XB_REQUIRE(blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_lora_gemm: weights of %d x %d are too many for one call", a.K, a.N);
    float* to = reinterpret_cast<float*>(ws + scratch.w);
    launch_dependent(lora_layout_kernel, (unsigned)blocks, 256, 0, s, static_cast<const float*>(a.W), a.ldw, to, laid_out_ld(a), a.N, a.K);
    if (int rc = check_launch("lora_layout_kernel")) return rc;
    g.B = to; g.ldb = laid_out_ld(a); g.trans_b = 0;
  }
  const void* W = g.B;
  for (int64_t m0 = 0; m0 < a.M; m0 += turn) {
    p.M = (int)std::min<int64_t>(turn, a.M - m0);
    p.X = reinterpret_cast<const T*>(a.X) + m0 * a.ldx;
    p.adapter = p.n_adapters ? a.adapter + m0 : nullptr;
    if (int rc = launch_shrink<T>(p, vec_k, s)) return rc;
    for (int64_t n0 = 0; n0 < a.N; n0 += TURN_COLS) {
      p.N = (int)std::min<int64_t>(TURN_COLS, a.N - n0);
      p.B = reinterpret_cast<const T*>(a.B) + n0 * a.ldb;
      p.bias = a.bias ? a.bias + n0 : nullptr;
      if (p.n_adapters) {
        if (int rc = launch_expand<T>(p, vec_r, s)) return rc;
        g.ldbias = p.N;
      } else {
        g.bias = p.bias;
      }
      g.M = p.M;
      g.N = p.N;
      g.A = p.X;
      g.B = reinterpret_cast<const T*>(W) + (g.trans_b ? n0 * g.ldb : n0);
      g.Y = reinterpret_cast<uint8_t*>(a.Y) + (m0 * a.ldy + n0) * (int64_t)dtype_size(a.y_dtype);
      // (fp32 results of rows that TMA cannot address: matrix instructions here, where xb_gemm stays with the CUDA cores for the sake of its bits.
      // [5003, 250] x [250, 131] bf16: 127 us there)
      const bool half = a.dtype != XB_F32 && a.y_dtype == XB_F32 && !xb_gemm_uses_tcgen05(&g);
      if (int rc = half ? gemm_half_sums(g, s) : xb_gemm(&g, s)) return rc;
    }
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
  size_t bytes = 0;
  if (check_args(a) != 0 || a->M == 0 || a->N == 0 || scratch_of(*a, &bytes) != 0) return 0;
  return bytes;
}

extern "C" int xb_lora_gemm(const xb_lora_args* a, void* workspace, size_t workspace_bytes, xb_stream_t s) {
  if (int rc = check_args(a)) return rc;
  if (a->M == 0 || a->N == 0) return 0;
  size_t need = 0;
  if (int rc = scratch_of(*a, &need)) return rc;
  XB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), XB_ERR_SCRATCH, "xb_lora_gemm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  XB_REQUIRE(need == 0 || (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, XB_ERR_ARG, "xb_lora_gemm: the workspace is not on 16 bytes");
  const int64_t x_size = (int64_t)dtype_size(a->dtype), y_size = (int64_t)dtype_size(a->y_dtype);
  XB_REQUIRE(!rows_meet(a->X, a->ldx * x_size, a->K * x_size, a->Y, a->ldy * y_size, a->N * y_size, a->M), XB_ERR_ARG, "xb_lora_gemm: Y overlaps X");
  if (takes_tiles(*a)) return run_umma(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
  if (a->dtype == XB_F32) return run_rows<float>(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
  if (a->dtype == XB_F16) return run_rows<__half>(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
  return run_rows<__nv_bfloat16>(*a, static_cast<uint8_t*>(workspace), (cudaStream_t)s);
}
