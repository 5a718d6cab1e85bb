// Norms of queries and keys for each head and the position rotation, in one pass (formulas in xdlb200.h).
#include <algorithm>

#include "xb_heads.cuh"

namespace xb {
namespace {

constexpr int ROPE_THREADS = 256, ROPE_MAX_D = 256, ROPE_TURNS = 1024;      // (cosines and sines of a block: 8 KB)
struct RopeParams {
  Heads q, k, yq, yk;
  const float* weight[2];
  const int32_t* positions;
  const float* freqs;
  int64_t rows;
  int Hq, Hk, d, rot, norm, adjacent;
  int rows_a_block, lanes, slots;          // lanes of a head; pairs of pieces of a head
  float eps, inv_d;
};

// A piece is 16 bytes (V elements) where all begins on 16 bytes, else one element. The lanes of a head take its pieces in pairs: those that are
// turned into one another (with `adjacent` a piece holds both parts of its pairs, and a pair of pieces is any two), then the rest, two and two.
// SLOTS: pairs of pieces of a lane.
// The cosines and sines of a block's rows are made once for all heads, the angle as a fraction of a turn in 64 bits: positions go up to 2^31,
// and fp32 keeps no more than 2^-24 of the angle. A head is read once and written once: bound by memory.
template <typename T, int V, int SLOTS>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeParams p) {
  pdl_begin();
  __shared__ float2 s_turn[ROPE_TURNS];
  const int half = p.rot / 2;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows_a_block;
  const int rows = (int)min((int64_t)p.rows_a_block, p.rows - r0);
  for (int i = threadIdx.x; i < rows * half; i += ROPE_THREADS) {
    const int r = i / half, j = i - r * half;
    double turn = (double)p.positions[r0 + r] * (double)p.freqs[j] * 0.15915494309189533577;
    turn -= rint(turn);
    float s, c;
    sincospif((float)(2 * turn), &s, &c);
    s_turn[i] = make_float2(c, s);
  }
  __syncthreads();
  const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = ROPE_THREADS / p.lanes;
  const int pieces = p.d / V, turned = p.adjacent ? 0 : half / V, rest = pieces - 2 * turned;      // (adjacent: all are in the rest)
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int H = which ? p.Hk : p.Hq;
    if (H == 0) continue;
    const Heads& from = which ? p.k : p.q;
    const Heads& to = which ? p.yk : p.yq;
    // the lane's pieces (-1: none) and their weights
    int at[SLOTS][2];
    float w[SLOTS][2][V];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int slot = lane + i * p.lanes, other = slot - turned;
      at[i][0] = slot < turned ? slot : 2 * other < rest ? 2 * turned + 2 * other : -1;
      at[i][1] = slot < turned ? slot + turned : 2 * other + 1 < rest ? 2 * turned + 2 * other + 1 : -1;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][b][e] = p.weight[which] && at[i][b] >= 0 ? p.weight[which][at[i][b] * V + e] : 1.f;
      }
    }
    const int items = rows * H;
    // (all lanes of a warp go the same number of rounds: they meet in the sums)
    for (int round = 0; round < items; round += groups) {
      const int item = round + group;
      const bool there = item < items;
      const int r = there ? item / H : 0, h = there ? item - r * H : 0;
      const T* x = from.get<T>(r0 + r, h);
      T* y = const_cast<T*>(to.get<T>(r0 + r, h));
      Raw<T, V> raw[SLOTS][2];
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          raw[i][b].zero();
          // (rows may be turned where they lie: no read through the read-only path)
          if (there && at[i][b] >= 0) raw[i][b].load_kept(x + at[i][b] * V, V, true);
        }
      float v[SLOTS][2][V];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            v[i][b][e] = raw[i][b].get(e);
            sum = fmaf(v[i][b][e], v[i][b][e], sum);
          }
      if (p.norm) {
        for (int o = p.lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float mean = fmaf(sum, p.inv_d, p.eps), by = 1.f / sqrtf(mean);
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][b][e] *= by * w[i][b][e];
      }
      if (!there) continue;
      const float2* turn = s_turn + r * half;
#pragma unroll
      for (int i = 0; i < SLOTS; ++i) {
        const int slot = lane + i * p.lanes;
        if (slot < turned) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 c = turn[slot * V + e];
            const float a = v[i][0][e], b = v[i][1][e];
            v[i][0][e] = fmaf(a, c.x, -b * c.y);
            v[i][1][e] = fmaf(b, c.x, a * c.y);
          }
        } else if (p.adjacent) {
          if constexpr (V > 1) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
              if (at[i][b] >= 0 && at[i][b] * V < p.rot) {              // (rot is whole pieces)
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                  const float2 c = turn[(at[i][b] * V + e) / 2];
                  const float a = v[i][b][e], d = v[i][b][e + 1];
                  v[i][b][e] = fmaf(a, c.x, -d * c.y);
                  v[i][b][e + 1] = fmaf(d, c.x, a * c.y);
                }
              }
          } else if (at[i][1] >= 0 && at[i][0] < p.rot) {
            const float2 c = turn[at[i][0] / 2];
            const float a = v[i][0][0], d = v[i][1][0];
            v[i][0][0] = fmaf(a, c.x, -d * c.y);
            v[i][1][0] = fmaf(d, c.x, a * c.y);
          }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (at[i][b] < 0) continue;
          Raw<T, V> out;
          out.put_all(v[i][b]);
          out.store(y + at[i][b] * V, V, true);
        }
      }
    }
  }
}

template <typename T>
int launch_rope(const xb_qk_norm_rope_args& a, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T), SIZE = sizeof(T);
  RopeParams p = {};
  p.q = {a.q, a.q_row, a.q_head}; p.k = {a.k, a.k_row, a.k_head}; p.yq = {a.yq, a.yq_row, a.yq_head}; p.yk = {a.yk, a.yk_row, a.yk_head};
  p.weight[0] = a.q_weight; p.weight[1] = a.k_weight;
  p.positions = a.positions; p.freqs = a.freqs;
  p.rows = a.rows; p.Hq = a.Hq; p.Hk = a.Hk; p.d = a.d; p.rot = a.rot; p.norm = a.norm; p.adjacent = a.adjacent;
  p.eps = a.eps; p.inv_d = 1.f / (float)a.d;
  const bool vec = a.d % V == 0 && a.rot % (a.adjacent ? V : 2 * V) == 0 && (a.Hq == 0 || (heads_whole(p.q, SIZE, 16) && heads_whole(p.yq, SIZE, 16))) &&
                   (a.Hk == 0 || (heads_whole(p.k, SIZE, 16) && heads_whole(p.yk, SIZE, 16)));
  const int pairs = ((vec ? a.d / V : a.d) + 1) / 2;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes < pairs) p.lanes *= 2;
  // a few rounds a block, whose rows' cosines fit, and blocks for every SM
  const int groups = ROPE_THREADS / p.lanes, half = std::max(a.rot / 2, 1), H = a.Hq + a.Hk;
  const int64_t fill = (a.rows + 4 * (int64_t)sm_count() - 1) / (4 * (int64_t)sm_count());
  p.rows_a_block = (int)std::clamp<int64_t>(std::min<int64_t>(fill, (4 * groups + H - 1) / H), 1, ROPE_TURNS / half);
  const int64_t blocks = (a.rows + p.rows_a_block - 1) / p.rows_a_block;
  XB_REQUIRE(blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_qk_norm_rope: %lld rows are too many for one call", (long long)a.rows);
  if (vec) launch_dependent(rope_kernel<T, V, 1>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else if (pairs <= 32) launch_dependent(rope_kernel<T, 1, 1>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else launch_dependent(rope_kernel<T, 1, 4>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  return check_launch("rope_kernel");
}

}  // namespace
}  // namespace xb

using namespace xb;

extern "C" int xb_qk_norm_rope(const xb_qk_norm_rope_args* a, xb_stream_t s) {
  XB_REQUIRE(a, XB_ERR_ARG, "xb_qk_norm_rope: null arguments");
  XB_REQUIRE(a->dtype == XB_F32 || a->dtype == XB_F16 || a->dtype == XB_BF16, XB_ERR_UNSUPPORTED, "xb_qk_norm_rope: dtype %d", a->dtype);
  XB_REQUIRE(a->rows >= 0 && a->Hq >= 0 && a->Hk >= 0 && a->d >= 1 && a->rot >= 0 && a->rot % 2 == 0 && a->rot <= a->d, XB_ERR_ARG,
             "xb_qk_norm_rope: %lld rows of %d + %d heads, %d wide, of which %d are turned", (long long)a->rows, a->Hq, a->Hk, a->d, a->rot);
  XB_REQUIRE(a->d <= ROPE_MAX_D, XB_ERR_LIMIT, "xb_qk_norm_rope: heads of %d, at most %d", a->d, ROPE_MAX_D);
  XB_REQUIRE(a->Hq <= 65535 && a->Hk <= 65535, XB_ERR_LIMIT, "xb_qk_norm_rope: %d + %d heads, at most 65535", a->Hq, a->Hk);
  XB_REQUIRE(a->rows < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_qk_norm_rope: %lld rows, fewer than 2^31", (long long)a->rows);
  XB_REQUIRE(a->norm || (!a->q_weight && !a->k_weight), XB_ERR_ARG, "xb_qk_norm_rope: weights without a norm");
  XB_REQUIRE(!a->norm || a->eps >= 0, XB_ERR_ARG, "xb_qk_norm_rope: eps %g", (double)a->eps);
  if (a->rows == 0 || a->Hq + a->Hk == 0) return 0;
  XB_REQUIRE((a->Hq == 0 || (a->q && a->yq)) && (a->Hk == 0 || (a->k && a->yk)) && (a->rot == 0 || (a->positions && a->freqs)), XB_ERR_ARG,
             "xb_qk_norm_rope: null tensor");
  XB_REQUIRE(a->q_row >= 0 && a->q_head >= 0 && a->k_row >= 0 && a->k_head >= 0 && a->yq_row >= 0 && a->yq_head >= 0 && a->yk_row >= 0 && a->yk_head >= 0,
             XB_ERR_ARG, "xb_qk_norm_rope: a negative stride");
  const Heads q = {a->q, a->q_row, a->q_head}, k = {a->k, a->k_row, a->k_head}, yq = {a->yq, a->yq_row, a->yq_head}, yk = {a->yk, a->yk_row, a->yk_head};
  const int64_t size = (int64_t)dtype_size(a->dtype);
  XB_REQUIRE((a->Hq == 0 || heads_apart(yq, a->Hq, a->d, a->rows)) && (a->Hk == 0 || heads_apart(yk, a->Hk, a->d, a->rows)), XB_ERR_ARG,
             "xb_qk_norm_rope: rows of an output overlap one another");
  auto same = [&](const Heads& x, const Heads& y) { return x.at == y.at && x.row == y.row && x.head == y.head; };
  auto meet = [&](const Heads& x, int nx, const Heads& y, int ny) { return heads_meet(x, nx, a->d, y, ny, a->d, a->rows, size); };
  XB_REQUIRE(same(q, yq) || !meet(q, a->Hq, yq, a->Hq), XB_ERR_ARG, "xb_qk_norm_rope: yq overlaps q and is not q");
  XB_REQUIRE(same(k, yk) || !meet(k, a->Hk, yk, a->Hk), XB_ERR_ARG, "xb_qk_norm_rope: yk overlaps k and is not k");
  XB_REQUIRE(!meet(q, a->Hq, yk, a->Hk) && !meet(k, a->Hk, yq, a->Hq) && !meet(yq, a->Hq, yk, a->Hk), XB_ERR_ARG,
             "xb_qk_norm_rope: an output overlaps the other's rows");
  if (a->dtype == XB_F32) return launch_rope<float>(*a, (cudaStream_t)s);
  if (a->dtype == XB_F16) return launch_rope<__half>(*a, (cudaStream_t)s);
  return launch_rope<__nv_bfloat16>(*a, (cudaStream_t)s);
}
