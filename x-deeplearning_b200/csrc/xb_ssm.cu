// Selective state-space layer over behaviour lists: the short causal convolution and the scan (formulas in xdlb200.h).
#include <algorithm>

#include "xb_common.cuh"

namespace xb {
namespace {

// The lists of a call and their kept states (see xdlb200.h). Every offset and slot that a kernel takes from memory goes through
// here and is cut to what exists.
struct Lists {
  const int32_t* offsets;
  const int32_t* slots;
  int64_t rows, per;                      // per: rows a list where there are no offsets
  int batch, n_slots;
  __device__ __forceinline__ int64_t begin(int i) const {
    if (!offsets) return (int64_t)i * per;
    const int64_t o = offsets[i];
    return o < 0 ? 0 : (o > rows ? rows : o);
  }
  __device__ __forceinline__ int slot(int i) const {
    const int s = slots ? slots[i] : i;
    return s >= 0 && s < n_slots ? s : -1;
  }
};

template <typename T>
struct ConvParams {
  const T* x; int64_t ldx;
  T* y; int64_t ldy;
  const T* w; const T* bias;
  const T* state_in; T* state_out;
  Lists lists;
  int D, K, silu;
};

__device__ __forceinline__ float silu(float v) { return v / (1.f + expf(-v)); }

// A thread walks one channel of one list.
template <typename T>
__global__ void __launch_bounds__(128) ssm_conv_kernel(const ConvParams<T> p) {
  pdl_begin();
  const int c = blockIdx.y * 128 + threadIdx.x;
  if (c >= p.D) return;
  const int K = p.K;
  float w[8], past[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = j < K ? to_f32<T>(p.w[(int64_t)c * K + j]) : 0.f;
  const float b = p.bias ? to_f32<T>(p.bias[c]) : 0.f;
  for (int i = blockIdx.x; i < p.lists.batch; i += gridDim.x) {
    const int64_t r0 = p.lists.begin(i), r1 = p.lists.begin(i + 1);
    const int slot = p.lists.slot(i);
#pragma unroll
    for (int j = 0; j < 7; ++j)
      past[j] = j < K - 1 && p.state_in && slot >= 0 ? to_f32<T>(p.state_in[((int64_t)slot * (K - 1) + j) * p.D + c]) : 0.f;
    for (int64_t r = r0; r < r1; ++r) {
      const float x = to_f32<T>(p.x[r * p.ldx + c]);
      float v = b;
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < K - 1) v = fmaf(w[j], past[j], v);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j == K - 1) v = fmaf(w[j], x, v);
#pragma unroll
      for (int j = 0; j < 7; ++j) past[j] = j == K - 2 ? x : past[j + 1];
      p.y[r * p.ldy + c] = from_f32<T>(p.silu ? silu(v) : v);
    }
    if (p.state_out && slot >= 0)
      for (int j = 0; j < K - 1; ++j) p.state_out[((int64_t)slot * (K - 1) + j) * p.D + c] = from_f32<T>(past[j]);
  }
}

template <typename T>
struct ScanParams {
  const T* x; int64_t ldx;
  const T* delta; int64_t lddelta;
  const T* z; int64_t ldz;
  const T* B; int64_t ldb;
  const T* C; int64_t ldc;
  T* y; int64_t ldy;
  const float* A; const float* skip; const float* delta_bias;
  const float* h_in; float* h_out;
  Lists lists;
  int D, N, per_group, softplus;
};

constexpr int SPL = 4;                    // states of a lane

// LPC lanes walk one channel of one list, four states a lane.
template <typename T, int LPC>
__global__ void __launch_bounds__(128) ssm_scan_kernel(const ScanParams<T> p, int channel_blocks) {
  pdl_begin();
  const int i = blockIdx.x / channel_blocks;
  const int n0 = threadIdx.x % LPC * SPL;
  const int at = (blockIdx.x % channel_blocks) * (128 / LPC) + threadIdx.x / LPC;
  const bool mine = at < p.D;
  const int c = mine ? at : p.D - 1, g = c / p.per_group;
  const int64_t r0 = p.lists.begin(i), r1 = p.lists.begin(i + 1);
  const int slot = p.lists.slot(i);
  float A[SPL], h[SPL];
#pragma unroll
  for (int s = 0; s < SPL; ++s) {
    const bool in = n0 + s < p.N;
    A[s] = in ? p.A[(int64_t)c * p.N + n0 + s] : 0.f;
    h[s] = in && p.h_in && slot >= 0 ? p.h_in[((int64_t)slot * p.D + c) * p.N + n0 + s] : 0.f;
  }
  const float bias = p.delta_bias ? p.delta_bias[c] : 0.f, skip = p.skip ? p.skip[c] : 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    const float x = to_f32<T>(p.x[r * p.ldx + c]);
    const float v = to_f32<T>(p.delta[r * p.lddelta + c]) + bias;
    const float d = p.softplus ? (v > 0.f ? v + log1pf(expf(-v)) : log1pf(expf(v))) : v;
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      if (n0 + s >= p.N) continue;
      const float Bn = to_f32<T>(p.B[r * p.ldb + g * p.N + n0 + s]), Cn = to_f32<T>(p.C[r * p.ldc + g * p.N + n0 + s]);
      h[s] = fmaf(expf(d * A[s]), h[s], d * x * Bn);
      y = fmaf(Cn, h[s], y);
    }
#pragma unroll
    for (int m = LPC / 2; m > 0; m >>= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
    if (mine && n0 == 0) {
      y = fmaf(skip, x, y);
      if (p.z) y *= silu(to_f32<T>(p.z[r * p.ldz + c]));
      p.y[r * p.ldy + c] = from_f32<T>(y);
    }
  }
  if (p.h_out && slot >= 0 && mine)
#pragma unroll
    for (int s = 0; s < SPL; ++s)
      if (n0 + s < p.N) p.h_out[((int64_t)slot * p.D + c) * p.N + n0 + s] = h[s];
}

int check_lists(const char* what, const int32_t* offsets, const int32_t* slots, bool states, int64_t rows, int32_t batch, int32_t n_slots) {
  XB_REQUIRE(rows >= 0 && batch >= 0, XB_ERR_ARG, "%s: %lld rows, %d lists", what, (long long)rows, batch);
  XB_REQUIRE(rows < ((int64_t)1 << 31), XB_ERR_LIMIT, "%s: %lld rows, fewer than 2^31", what, (long long)rows);
  XB_REQUIRE(offsets || batch == 0 || rows % batch == 0, XB_ERR_ARG, "%s: without offsets %d lists divide %lld rows", what, batch, (long long)rows);
  XB_REQUIRE(!states || n_slots >= 0, XB_ERR_ARG, "%s: n_slots %d", what, n_slots);
  XB_REQUIRE(!states || slots || n_slots >= batch, XB_ERR_ARG, "%s: %d states for %d lists without slots", what, n_slots, batch);
  return 0;
}
Lists lists_of(const int32_t* offsets, const int32_t* slots, int64_t rows, int32_t batch, int32_t n_slots) {
  return {offsets, slots, rows, batch > 0 ? rows / batch : 0, batch, n_slots};
}
bool ssm_dtype(int dtype) { return dtype == XB_F32 || dtype == XB_F16 || dtype == XB_BF16; }

template <typename T>
int launch_conv(const xb_ssm_conv_args& a, cudaStream_t s) {
  ConvParams<T> p = {(const T*)a.x, a.ldx, (T*)a.y, a.ldy, (const T*)a.w, (const T*)a.bias, (const T*)a.state_in, (T*)a.state_out,
                     lists_of(a.offsets, a.slots, a.rows, a.batch, a.n_slots), a.D, a.K, a.silu};
  const dim3 grid((unsigned)a.batch, (unsigned)((a.D + 127) / 128));
  launch_dependent(ssm_conv_kernel<T>, grid, 128, 0, s, p);
  return check_launch("ssm_conv_kernel");
}

template <typename T, int LPC>
int launch_scan_lanes(const ScanParams<T>& p, cudaStream_t s) {
  const int blocks = (p.D + 128 / LPC - 1) / (128 / LPC);
  XB_REQUIRE((int64_t)blocks * p.lists.batch < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_ssm_scan: too many lists and channels");
  launch_dependent(ssm_scan_kernel<T, LPC>, (unsigned)((int64_t)blocks * p.lists.batch), 128, 0, s, p, blocks);
  return check_launch("ssm_scan_kernel");
}
template <typename T>
int launch_scan(const xb_ssm_scan_args& a, cudaStream_t s) {
  ScanParams<T> p = {(const T*)a.x, a.ldx, (const T*)a.delta, a.lddelta, (const T*)a.z, a.ldz, (const T*)a.B, a.ldb, (const T*)a.C, a.ldc,
                     (T*)a.y, a.ldy, a.A, a.skip, a.delta_bias, a.h_in, a.h_out,
                     lists_of(a.offsets, a.slots, a.rows, a.batch, a.n_slots), a.D, a.N, a.D / a.groups, a.softplus};
  if (a.N <= 4) return launch_scan_lanes<T, 1>(p, s);
  if (a.N <= 8) return launch_scan_lanes<T, 2>(p, s);
  if (a.N <= 16) return launch_scan_lanes<T, 4>(p, s);
  if (a.N <= 32) return launch_scan_lanes<T, 8>(p, s);
  return launch_scan_lanes<T, 16>(p, s);
}

}  // namespace
}  // namespace xb

using namespace xb;

extern "C" int xb_ssm_conv(const xb_ssm_conv_args* a, xb_stream_t s) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_ssm_conv: null arguments");
  XB_REQUIRE(ssm_dtype(a->dtype), XB_ERR_UNSUPPORTED, "xb_ssm_conv: dtype %d", a->dtype);
  XB_REQUIRE(a->D >= 1, XB_ERR_ARG, "xb_ssm_conv: %d channels", a->D);
  XB_REQUIRE(a->K >= 2 && a->K <= 8, XB_ERR_LIMIT, "xb_ssm_conv: %d taps, from 2 to 8", a->K);
  if (int rc = check_lists("xb_ssm_conv", a->offsets, a->slots, a->state_in || a->state_out, a->rows, a->batch, a->n_slots)) return rc;
  if (a->batch == 0) return 0;
  XB_REQUIRE(a->w && (a->rows == 0 || (a->x && a->y)), XB_ERR_ARG, "xb_ssm_conv: null tensor");
  XB_REQUIRE(a->rows == 0 || (a->ldx >= a->D && a->ldy >= a->D), XB_ERR_ARG, "xb_ssm_conv: row strides %lld, %lld of %d channels",
             (long long)a->ldx, (long long)a->ldy, a->D);
  if (a->dtype == XB_F32) return launch_conv<float>(*a, (cudaStream_t)s);
  if (a->dtype == XB_F16) return launch_conv<__half>(*a, (cudaStream_t)s);
  return launch_conv<__nv_bfloat16>(*a, (cudaStream_t)s);
}

extern "C" size_t xb_ssm_scan_workspace_bytes(const xb_ssm_scan_args* a) {
  (void)a;
  return 0;
}

extern "C" int xb_ssm_scan(const xb_ssm_scan_args* a, void* workspace, size_t workspace_bytes, xb_stream_t s) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_ssm_scan: null arguments");
  XB_REQUIRE(ssm_dtype(a->dtype), XB_ERR_UNSUPPORTED, "xb_ssm_scan: dtype %d", a->dtype);
  XB_REQUIRE(a->D >= 1 && a->N >= 1 && a->groups >= 1 && a->D % a->groups == 0, XB_ERR_ARG, "xb_ssm_scan: %d channels in %d groups, %d states",
             a->D, a->groups, a->N);
  XB_REQUIRE(a->N <= 64, XB_ERR_LIMIT, "xb_ssm_scan: %d states, at most 64", a->N);
  XB_REQUIRE(a->longest >= 0, XB_ERR_ARG, "xb_ssm_scan: longest %lld", (long long)a->longest);
  if (int rc = check_lists("xb_ssm_scan", a->offsets, a->slots, a->h_in || a->h_out, a->rows, a->batch, a->n_slots)) return rc;
  if (a->batch == 0) return 0;
  XB_REQUIRE(a->A && (a->rows == 0 || (a->x && a->delta && a->B && a->C && a->y)), XB_ERR_ARG, "xb_ssm_scan: null tensor");
  XB_REQUIRE(a->rows == 0 || (a->ldx >= a->D && a->lddelta >= a->D && a->ldy >= a->D && (!a->z || a->ldz >= a->D)), XB_ERR_ARG,
             "xb_ssm_scan: a row stride below %d channels", a->D);
  XB_REQUIRE(a->rows == 0 || (a->ldb >= (int64_t)a->groups * a->N && a->ldc >= (int64_t)a->groups * a->N), XB_ERR_ARG,
             "xb_ssm_scan: a row stride of B or C below %d x %d", a->groups, a->N);
  const size_t need = xb_ssm_scan_workspace_bytes(a);
  XB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), XB_ERR_SCRATCH, "xb_ssm_scan: workspace of %zu bytes, %zu needed",
             workspace_bytes, need);
  if (a->dtype == XB_F32) return launch_scan<float>(*a, (cudaStream_t)s);
  if (a->dtype == XB_F16) return launch_scan<__half>(*a, (cudaStream_t)s);
  return launch_scan<__nv_bfloat16>(*a, (cudaStream_t)s);
}
