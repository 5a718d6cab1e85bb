// Norms of queries and keys for each head and the position rotation, in one pass (formulas in xdlb200.h).
#include <algorithm>

#include "xb_heads.cuh"

namespace xb {
namespace {

constexpr int ROPE_THREADS = 256, ROPE_MAX_D = 256, ROPE_TURNS = 2048;      // (cosines and sines of a block: 16 KB)
struct RopeParams {
  Heads q, k, yq, yk;
  const float* weight[2];
  const int32_t* positions;
  const float* freqs;
  int64_t rows;
  int Hq, Hk, d, rot, norm;
  int rows_a_block, lanes, slots;          // lanes of a head; pairs of pieces of a head
  float eps, inv_d;
};

// A piece is 16 bytes (V elements) where all begins on 16 bytes, else one element. The lanes of a head take its pieces in pairs: those that are
// turned into one another (with ADJACENT a piece holds both parts of its pairs, and a pair of pieces is any two), then the rest, two and two.
// SLOTS: pairs of pieces of a lane.
// The cosines and sines of a block's rows are made once for all heads, the angle as a fraction of a turn in 64 bits: positions go up to 2^31,
// and fp32 keeps no more than 2^-24 of the angle. They lie so that what the lanes of a head read at once is adjacent. A head is read once and written
// once: bound by memory, which is a matter of reads in flight: the next head of a group of lanes is on its way while this one is worked on, the
// first ones while the cosines are made. 70000 rows of 16 heads of 128, bf16: 107 us (5.4 TB/s, of 6.55
// that a copy reaches); 143 with one head at a time; 138 with cosines in their order, where shared memory was the bound (the lanes' reads in the same banks), and 26 instructions an element.
template <typename T, int V, int SLOTS, bool ADJACENT>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeParams p) {
  pdl_begin();
  __shared__ __align__(16) float2 s_turn[ROPE_TURNS];
  const int half = p.rot / 2;
  const int64_t r0 = (int64_t)blockIdx.x * p.rows_a_block;
  const int rows = (int)min((int64_t)p.rows_a_block, p.rows - r0);
  const int lane = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = ROPE_THREADS / p.lanes;
  const int pieces = p.d / V, turned = ADJACENT ? 0 : half / V, rest = pieces - 2 * turned;      // (adjacent: all are in the rest)
  // the lane's pieces (-1: none)
  int at[SLOTS][2];
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int slot = lane + i * p.lanes, other = slot - turned;
    at[i][0] = slot < turned ? slot : 2 * other < rest ? 2 * turned + 2 * other : -1;
    at[i][1] = slot < turned ? slot + turned : 2 * other + 1 < rest ? 2 * turned + 2 * other + 1 : -1;
  }
  constexpr bool PAIRS = V > 1 && !ADJACENT;                 // two elements an instruction, whose cosines and sines lie as {c, c, s, s}
  auto turn_at = [&](int j) { return PAIRS ? (j % V / 2 * turned + j / V) * 2 : j; };
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int H = which ? p.Hk : p.Hq;
    const Heads& from = which ? p.k : p.q;
    const Heads& to = which ? p.yk : p.yq;
    const float* weight = p.weight[which];
    // a group's heads in order, `groups` of the block's apart
    const int step_row = H ? groups / H : 0, step_head = H ? groups - step_row * H : 0;
    int row = H ? group / H : rows, head = H ? group - row * H : 0;
    Raw<T, V> raw[SLOTS][2];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) { raw[i][0].zero(); raw[i][1].zero(); }
    auto fetch = [&](int r, int h) {
      if (r >= rows) return;
      const T* x = from.get<T>(r0 + r, h);
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          // (rows may be turned where they lie: no read through the read-only path)
          if (at[i][b] >= 0) raw[i][b].load_kept(x + at[i][b] * V, V, true);
    };
    fetch(row, head);
    if (which == 0) {
      for (int i = threadIdx.x; i < rows * half; i += ROPE_THREADS) {
        const int r = i / half, j = i - r * half;
        double turn = (double)p.positions[r0 + r] * (double)p.freqs[j] * 0.15915494309189533577;
        turn -= rint(turn);
        float s, c;
        sincospif((float)(2 * turn), &s, &c);
        if constexpr (PAIRS) {
          float* t = reinterpret_cast<float*>(s_turn + r * half + turn_at(j)) + (j & 1);
          t[0] = c;
          t[2] = s;
        } else {
          s_turn[i] = make_float2(c, s);
        }
      }
      __syncthreads();
    }
    f32x2 w[SLOTS][2][(V + 1) / 2];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const bool has = weight && at[i][b] >= 0;
          w[i][b][e / 2] = pack2(has ? weight[at[i][b] * V + e] : 1.f, has && V > 1 ? weight[at[i][b] * V + min(e + 1, V - 1)] : 1.f);
        }
    // (all lanes of a warp go the same number of rounds: they meet in the sums)
    for (int round = 0; round < rows * H; round += groups) {
      const bool there = row < rows;
      f32x2 v[SLOTS][2][(V + 1) / 2], sum2 = pack2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            f32x2& x = v[i][b][e / 2];
            x = pack2(raw[i][b].get(e), V > 1 ? raw[i][b].get((e + 1) % V) : 0.f);
            sum2 = fma2(x, x, sum2);
          }
      int next_row = row + step_row, next_head = head + step_head;
      if (next_head >= H) { next_head -= H; ++next_row; }
      fetch(next_row, next_head);
      if (p.norm) {
        float s0, s1;
        unpack2(sum2, s0, s1);
        float sum = s0 + s1;
        for (int o = p.lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float f = rsqrtf(fmaf(sum, p.inv_d, p.eps));            // (right to 2^-22)
        const f32x2 by = pack2(f, f);
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < (V + 1) / 2; ++e) v[i][b][e] = mul2(v[i][b][e], mul2(by, w[i][b][e]));
      }
      if (there) {
        T* y = const_cast<T*>(to.get<T>(r0 + row, head));
        const float2* turn = s_turn + row * half;
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
          const int slot = lane + i * p.lanes;
          if (!ADJACENT && slot < turned) {
            if constexpr (PAIRS) {
#pragma unroll
              for (int e = 0; e < V / 2; ++e) {
                const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(turn + (e * turned + slot) * 2);
                const f32x2 a = v[i][0][e], b = v[i][1][e];
                v[i][0][e] = fma2(mul2(b, t.y), pack2(-1.f, -1.f), mul2(a, t.x));
                v[i][1][e] = fma2(b, t.x, mul2(a, t.y));
              }
            } else {
              const float2 c = turn[slot];
              float a, b, none;
              unpack2(v[i][0][0], a, none);
              unpack2(v[i][1][0], b, none);
              v[i][0][0] = pack2(fmaf(a, c.x, -b * c.y), 0.f);
              v[i][1][0] = pack2(fmaf(b, c.x, a * c.y), 0.f);
            }
          } else if constexpr (ADJACENT) {
            if constexpr (V > 1) {
#pragma unroll
              for (int b = 0; b < 2; ++b)
                if (at[i][b] >= 0 && at[i][b] * V < p.rot) {            // (rot is whole pieces)
#pragma unroll
                  for (int e = 0; e < V / 2; ++e) {
                    const float2 c = turn[at[i][b] * (V / 2) + e];
                    float a, d;
                    unpack2(v[i][b][e], a, d);
                    v[i][b][e] = pack2(fmaf(a, c.x, -d * c.y), fmaf(d, c.x, a * c.y));
                  }
                }
            } else if (at[i][1] >= 0 && at[i][0] < p.rot) {
              const float2 c = turn[at[i][0] / 2];
              float a, d, none;
              unpack2(v[i][0][0], a, none);
              unpack2(v[i][1][0], d, none);
              v[i][0][0] = pack2(fmaf(a, c.x, -d * c.y), 0.f);
              v[i][1][0] = pack2(fmaf(d, c.x, a * c.y), 0.f);
            }
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (at[i][b] < 0) continue;
            float f[V];
#pragma unroll
            for (int e = 0; e < V; e += 2) {
              float lo, hi;
              unpack2(v[i][b][e / 2], lo, hi);
              f[e] = lo;
              if (V > 1) f[(e + 1) % V] = hi;
            }
            Raw<T, V> out;
            out.put_all(f);
            out.store(y + at[i][b] * V, V, true);
          }
        }
      }
      row = next_row;
      head = next_head;
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
  p.rows = a.rows; p.Hq = a.Hq; p.Hk = a.Hk; p.d = a.d; p.rot = a.rot; p.norm = a.norm;
  p.eps = a.eps; p.inv_d = 1.f / (float)a.d;
  const bool vec = a.d % V == 0 && a.rot % (a.adjacent ? V : 2 * V) == 0 && (a.Hq == 0 || (heads_whole(p.q, SIZE, 16) && heads_whole(p.yq, SIZE, 16))) &&
                   (a.Hk == 0 || (heads_whole(p.k, SIZE, 16) && heads_whole(p.yk, SIZE, 16)));
  const int pairs = ((vec ? a.d / V : a.d) + 1) / 2;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes < pairs) p.lanes *= 2;
  // Rounds enough to make up for what a block does once, rows whose cosines fit, and blocks for every SM. (4 rounds a block instead of up to 16:
  // 70000 rows of 16 heads of 128, bf16 141 us, 107 so.)
  const int groups = ROPE_THREADS / p.lanes, half = std::max(a.rot / 2, 1), H = a.Hq + a.Hk;
  const int64_t fill = (a.rows + 4 * (int64_t)sm_count() - 1) / (4 * (int64_t)sm_count());
  p.rows_a_block = (int)std::clamp<int64_t>(std::min<int64_t>(fill, (16 * groups + H - 1) / H), 1, ROPE_TURNS / half);
  const int64_t blocks = (a.rows + p.rows_a_block - 1) / p.rows_a_block;
  XB_REQUIRE(blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_qk_norm_rope: %lld rows are too many for one call", (long long)a.rows);
  const bool adj = a.adjacent != 0, few = pairs <= 32;
  if (vec && adj) launch_dependent(rope_kernel<T, V, 1, true>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else if (vec) launch_dependent(rope_kernel<T, V, 1, false>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else if (few && adj) launch_dependent(rope_kernel<T, 1, 1, true>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else if (few) launch_dependent(rope_kernel<T, 1, 1, false>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else if (adj) launch_dependent(rope_kernel<T, 1, 4, true>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
  else launch_dependent(rope_kernel<T, 1, 4, false>, (unsigned)blocks, ROPE_THREADS, 0, s, p);
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
