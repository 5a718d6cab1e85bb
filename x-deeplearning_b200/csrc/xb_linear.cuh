// Linear attention with a decay for each head: what its kernels share, and the one that goes row by row (formulas in xdlb200.h).
//
// A long list is cut into segments of `chunk` rows, counted from the list's beginning, where whole lists would leave SMs idle. Three launches:
// every segment but a list's last makes the state at its end as if it began with zeros (the first one: with the list's state); those are carried
// from segment to segment, in order; then all segments run from the state that they begin with.
#pragma once

#include <algorithm>
#include <cmath>

#include "xb_heads.cuh"
#include "xb_mma_half.cuh"

namespace xb {

struct LinearParams {
  Heads q, k, v, y;
  const float* log_decay;
  const float* h_in;
  float* h_out;
  Lists lists;
  int H, share, dk, dv;                    // share: heads that read one head of k and v
  float scale;
  int vec_y;                               // rows of y in pieces of two
  int unit_q, unit_k, unit_v;              // bytes that rows may be read by: 16, 8, 4 or an element
  int vec_h, vec_e;                        // kept states in pairs; the ends of segments in pieces of four
  int* order;                              // [batch]: whole lists, long ones first; null: as they come
  int64_t chunk;                           // 0: whole lists
  int n_ends;                              // rows / chunk
  float* end;                              // [n_ends][H][dk][dv]: states at the ends of segments
  float* first;                            // the same, of lists' first segments: copies of what they begin with
  int ends_only;                           // the first of the three launches
};
struct LinearPlan {
  bool step;                               // one row a list, states in pieces of four columns
  bool tiles;                              // by chunks of 64 rows on the matrix instructions, else row by row
  int64_t chunk;
  bool order;                              // whole lists, long ones first
};
// the kernels of one type (xb_linear_*.cu)
int linear_f32(const LinearParams& p, const LinearPlan& plan, cudaStream_t s);
int linear_f16(const LinearParams& p, const LinearPlan& plan, cudaStream_t s);
int linear_bf16(const LinearParams& p, const LinearPlan& plan, cudaStream_t s);

namespace {

// The rows of a block, and what it begins and ends with.
struct Segment {
  int64_t begin, end;                      // rows
  int slot, number;                        // number: which segment of its list
  int64_t at;                              // the segment's state of p.end (its list's later ones lie behind it)
  bool last;
};
// false: no such segment, or one that this launch leaves out. By the first warp, the others read it off shared memory.
__device__ __forceinline__ bool find_segment(const LinearParams& p, int u, int lane, Segment& g) {
  int i = u;
  int64_t b, e;
  if (p.chunk == 0) {
    if (p.order) i = p.order[u];
    b = p.lists.begin(i);
    e = p.lists.begin(i + 1);
    g.begin = b; g.end = e > b ? e : b; g.number = 0; g.last = true; g.at = 0;
  } else {
    i = p.lists.of_chunk(u, p.chunk, lane);
    b = p.lists.begin(i);
    e = p.lists.begin(i + 1);
    if (e < b) e = b;
    const int64_t number = u - (b / p.chunk + i);
    if (number < 0 || (number > 0 && number * p.chunk >= e - b)) return false;
    g.number = (int)number;
    g.begin = b + number * p.chunk;
    g.last = e - g.begin <= p.chunk;
    g.end = g.last ? e : g.begin + p.chunk;
    g.at = b / p.chunk + number;
    if (!g.last && g.at >= p.n_ends) return false;
  }
  g.slot = p.lists.slot(i);
  return !p.ends_only || !g.last;
}
__device__ __forceinline__ float log_decay_of(const LinearParams& p, int h) {
  const float l = p.log_decay[h];
  return l > 0.f ? 0.f : l;
}
// decay over n rows; n = 0 is 1 whatever the logarithm
__device__ __forceinline__ float decay_over(float log_decay, int n) { return n == 0 ? 1.f : expf((float)n * log_decay); }
// S decay + add. Near 1 the decay itself is known to 2^-25 only, which adds up over the rows that a slow one looks back on: there it is
// S + S (decay - 1) with decay - 1 to 2^-24 of itself.
struct Decay {
  bool slow;
  float by;
  __device__ __forceinline__ explicit Decay(float log_decay) : slow(log_decay > -0.5f), by(slow ? expm1f(log_decay) : expf(log_decay)) {}
  __device__ __forceinline__ float step(float s, float add) const { return slow ? fmaf(s, by, s + add) : fmaf(s, by, add); }
};

// What a segment's state begins with and where it goes to; null: zeros, not kept
__device__ __forceinline__ const float* state_from(const LinearParams& p, const Segment& g, int h) {
  const int64_t size = (int64_t)p.dk * p.dv;
  if (g.number > 0) return p.ends_only ? nullptr : p.end + ((g.at - 1) * p.H + h) * size;
  if (!p.h_in || g.slot < 0) return nullptr;
  // (a split list's last segment may write over the state that its first one begins with)
  if (!g.last && !p.ends_only) return p.first + (g.at * p.H + h) * size;
  return p.h_in + ((int64_t)g.slot * p.H + h) * size;
}
__device__ __forceinline__ float* state_to(const LinearParams& p, const Segment& g, int h) {
  const int64_t size = (int64_t)p.dk * p.dv;
  if (p.ends_only) return p.end + (g.at * p.H + h) * size;
  return g.last && p.h_out && g.slot >= 0 ? p.h_out + ((int64_t)g.slot * p.H + h) * size : nullptr;
}

// ---- row by row ----
// A block has a list (or segment) and a head; a thread NV columns of dv (two where there are more than 64, and see below) and KT of dk, PARTS lanes sharing the
// columns, whose products with q meet in shuffles. KT is 32, or 8 where there are so few lists that the row's latency counts. The state stays in
// registers, in pairs along dk. Rows come eight at a time through shared memory, three such tiles ahead; pieces of four along dk go round the PARTS
// lanes, so that what a warp reads at once lies in adjacent banks. 3 packed FMAs for two values of the state a row, bound by the reads of k and q from
// shared memory (512 bytes an instruction to registers, however few they are in memory). 74 lists of 100 rows, 2 heads of 36, fp32: 22 us; 31 with
// a row's sums made before the next row's (24 shuffles for 8 rows in place of 7), 37 with rows that pass through registers.
constexpr int LIN_ROWS = 8, LIN_TILES = 4, LIN_MAX = 128;
// four adjacent elements of shared memory, as two pairs of fp32
template <typename T>
__device__ __forceinline__ void read_four(const T* p, f32x2& lo, f32x2& hi) {
  if constexpr (sizeof(T) == 4) {
    const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p);
    lo = t.x; hi = t.y;
  } else {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    Raw<T, 4> r;
    r.w[0] = t.x; r.w[1] = t.y;
    lo = pack2(r.get(0), r.get(1)); hi = pack2(r.get(2), r.get(3));
  }
}
template <typename T, int KT, int PARTS, int NV, int DV>
__global__ void __launch_bounds__(DV / NV * PARTS) linear_rows_kernel(const LinearParams p) {
  pdl_wait();
  constexpr int DK = KT * PARTS, TILE = LIN_ROWS * (2 * DK + DV);
  extern __shared__ __align__(128) uint8_t smem[];          // [tiles][q, k, v][rows][DK or DV]
  T* s_rows = reinterpret_cast<T*>(smem);
  __shared__ Segment s_seg;
  __shared__ int s_there;
  const int lane = threadIdx.x & 31, h = (int)(blockIdx.x % (unsigned)p.H), hkv = h / p.share;
  if (threadIdx.x < 32) {
    Segment g;
    const bool there = find_segment(p, (int)(blockIdx.x / (unsigned)p.H), lane, g);
    if (lane == 0) {
      s_seg = g;
      s_there = there;
    }
  }
  __syncthreads();
  if (!s_there) return;
  const Segment g = s_seg;
  const int part = threadIdx.x % PARTS, c = threadIdx.x / PARTS * NV;
  const bool mine = c < p.dv;
  f32x2 S[NV][KT / 2];
  const float* from = state_from(p, g, h);
  auto at_dk = [&](int j) { return ((j / 4) * PARTS + part) * 4 + j % 4; };
#pragma unroll
  for (int j = 0; j < KT; j += 2) {
    float x[2][NV];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int r = at_dk(j + b);
      const float* f = from + (int64_t)r * p.dv + c;
#pragma unroll
      for (int n = 0; n < NV; ++n) x[b][n] = 0.f;
      if (from && r < p.dk && mine) {
        if (NV == 2 && p.vec_h) {
          const float2 t = *reinterpret_cast<const float2*>(f);
          x[b][0] = t.x; x[b][NV - 1] = t.y;
        } else {
#pragma unroll
          for (int n = 0; n < NV; ++n)
            if (c + n < p.dv) x[b][n] = f[n];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) S[n][j / 2] = pack2(x[0][n], x[1][n]);
  }
  auto put_state = [&](float* to) {
#pragma unroll
    for (int j = 0; j < KT; j += 2) {
      float x[2][NV];
#pragma unroll
      for (int n = 0; n < NV; ++n) unpack2(S[n][j / 2], x[0][n], x[1][n]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int r = at_dk(j + b);
        if (r >= p.dk || !mine) continue;
        float* t = to + (int64_t)r * p.dv + c;
        if (NV == 2 && p.vec_h) {
          *reinterpret_cast<float2*>(t) = make_float2(x[b][0], x[b][NV - 1]);
        } else {
#pragma unroll
          for (int n = 0; n < NV; ++n)
            if (c + n < p.dv) t[n] = x[b][n];
        }
      }
    }
  };
  if (from && p.ends_only) put_state(p.first + (g.at * p.H + h) * (int64_t)p.dk * p.dv);
  const Decay decay(log_decay_of(p, h));
  const f32x2 by = pack2(decay.by, decay.by);
  // Rows [r0, r0 + 8) of q, k and v into a tile, in pieces of the bytes that their rows lie on; what lies behind the list and behind the width is zero.
  // Piece e of a tile is the same row, tensor and column in every tile: where a thread's first pieces come from and go to is worked out once.
  const int n_threads = (int)blockDim.x;
  struct Piece {
    const char* src;                       // in tile 0 (null: none)
    int64_t step;                          // bytes from tile to tile
    uint32_t to;                           // in tile 0
    int row, unit, bytes;
  };
  auto pieces_of = [&](int width, int unit) { return (width * (int)sizeof(T) + unit - 1) / unit; };
  const int n_q = p.ends_only ? 0 : pieces_of(p.dk, p.unit_q), n_k = pieces_of(p.dk, p.unit_k), n_v = pieces_of(p.dv, p.unit_v);
  const int row_pieces = n_q + n_k + n_v, tile_pieces = LIN_ROWS * row_pieces;
  auto piece = [&](int e) {
    Piece x;
    x.row = e / row_pieces;
    int c = e - x.row * row_pieces;
    const int which = c < n_q ? 0 : c < n_q + n_k ? 1 : 2;
    c -= which == 0 ? 0 : which == 1 ? n_q : n_q + n_k;
    const Heads& from = which == 0 ? p.q : which == 1 ? p.k : p.v;
    const int D = which == 2 ? DV : DK, width = which == 2 ? p.dv : p.dk;
    x.unit = which == 0 ? p.unit_q : which == 1 ? p.unit_k : p.unit_v;
    x.src = e < tile_pieces ? reinterpret_cast<const char*>(from.get<T>(g.begin + x.row, which == 0 ? h : hkv)) + c * x.unit : nullptr;
    x.step = from.row * (int64_t)sizeof(T) * LIN_ROWS;
    x.to = (uint32_t)__cvta_generic_to_shared(reinterpret_cast<char*>(s_rows + which * LIN_ROWS * DK + x.row * D) + c * x.unit);
    x.bytes = min(x.unit, width * (int)sizeof(T) - c * x.unit);
    return x;
  };
  auto copy = [&](const Piece& x, int tile) {
    if (!x.src) return;
    const bool in = g.begin + (int64_t)tile * LIN_ROWS + x.row < g.end;
    const char* f = in ? x.src + tile * x.step : x.src;    // (nothing is read of a piece behind the end)
    const uint32_t at = x.to + tile % LIN_TILES * (TILE * (uint32_t)sizeof(T));
    const int bytes = in ? x.bytes : 0;
    if (x.unit == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(f), "r"(bytes) : "memory");
    else if (x.unit == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(f), "r"(bytes) : "memory");
    else if (x.unit == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at), "l"(f), "r"(bytes) : "memory");
    else asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(bytes ? *reinterpret_cast<const uint16_t*>(f) : (uint16_t)0) : "memory");
  };
  constexpr int KNOWN = 2;
  Piece known[KNOWN];
#pragma unroll
  for (int i = 0; i < KNOWN; ++i) known[i] = piece(threadIdx.x + i * n_threads);
  auto load_tile = [&](int tile) {
    if (g.begin + (int64_t)tile * LIN_ROWS < g.end) {
#pragma unroll
      for (int i = 0; i < KNOWN; ++i) copy(known[i], tile);
      for (int e = threadIdx.x + KNOWN * n_threads; e < tile_pieces; e += n_threads) copy(piece(e), tile);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (p.dk != DK || p.dv != DV || p.ends_only) {
    for (int e = threadIdx.x; e < LIN_TILES * TILE * (int)sizeof(T) / 16; e += n_threads) reinterpret_cast<uint4*>(smem)[e] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < LIN_TILES - 1; ++t) load_tile(t);
  int tile = 0;
  for (int64_t r0 = g.begin; r0 < g.end; r0 += LIN_ROWS, ++tile) {
    const int rows = (int)min((int64_t)LIN_ROWS, g.end - r0);
    asm volatile("cp.async.wait_group %0;" ::"n"(LIN_TILES - 2) : "memory");
    __syncthreads();                       // (the tile is there, and all have done with the one before)
    load_tile(tile + LIN_TILES - 1);
    const T *s_q = s_rows + tile % LIN_TILES * TILE, *s_k = s_q + LIN_ROWS * DK, *s_v = s_k + LIN_ROWS * DK;
    T* y_at = const_cast<T*>(p.y.get<T>(r0, h)) + c;
    // N rows: the state goes from row to row, their products with q wait for one another only in the sums over the parts. There a part gives half of its
    // rows to its neighbour and takes the neighbour's half of the others, until it has N / PARTS rows of whole sums: 7 shuffles for 8 rows and parts, not
    // 24. (A row alone: all parts have the same sum, made in the same order.)
    auto steps = [&](auto slow, auto count, int first) {
      constexpr int N = decltype(count)::value, HAVE = N < PARTS ? 1 : N / PARTS;
      static_assert(N == 1 || N % PARTS == 0, "");
      float y[N][NV];
#pragma unroll
      for (int r = 0; r < N; ++r) {
        const int row = first + r;
        f32x2 v2[NV], y2[NV][2];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const float v = mine ? to_f32<T>(s_v[row * DV + c + n]) : 0.f;
          v2[n] = pack2(v, v);
          y2[n][0] = y2[n][1] = pack2(0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < KT / 4; ++j) {
          f32x2 k4[2], q4[2];
          read_four(s_k + row * DK + (j * PARTS + part) * 4, k4[0], k4[1]);
          read_four(s_q + row * DK + (j * PARTS + part) * 4, q4[0], q4[1]);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const f32x2 k2 = k4[b], q2 = q4[b];
#pragma unroll
            for (int n = 0; n < NV; ++n) {
              f32x2& a = S[n][2 * j + b];
              a = fma2(a, by, decltype(slow)::value ? fma2(k2, v2[n], a) : mul2(k2, v2[n]));
              y2[n][j & 1] = fma2(q2, a, y2[n][j & 1]);
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          float lo, hi;
          unpack2(add2(y2[n][0], y2[n][1]), lo, hi);
          y[r][n] = lo + hi;
        }
      }
      if (p.ends_only) return;
#pragma unroll
      for (int o = PARTS / 2, m = N / 2; o > 0; o /= 2, m /= 2) {
        if constexpr (N == 1) {
#pragma unroll
          for (int n = 0; n < NV; ++n) y[0][n] += __shfl_xor_sync(0xffffffffu, y[0][n], o);
        } else {
          const bool upper = (part & o) != 0;
#pragma unroll
          for (int r = 0; r < N / 2; ++r) {
            if (r >= m) break;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
              const float other = __shfl_xor_sync(0xffffffffu, upper ? y[r][n] : y[r + m][n], o);
              y[r][n] = (upper ? y[r + m][n] : y[r][n]) + other;
            }
          }
        }
      }
      if (!mine || (N == 1 && part != 0)) return;
#pragma unroll
      for (int i = 0; i < HAVE; ++i) {
        T* to = y_at + (first + (N == 1 ? 0 : part * HAVE + i)) * p.y.row;
#pragma unroll
        for (int n = 0; n < NV; ++n) y[i][n] *= p.scale;
        if (NV == 2 && p.vec_y) {
          const float two[2] = {y[i][0], y[i][NV - 1]};
          Raw<T, 2> out;
          out.put_all(two);
          out.store_piece(to);
        } else {
#pragma unroll
          for (int n = 0; n < NV; ++n)
            if (c + n < p.dv) to[n] = from_f32<T>(y[i][n]);
        }
      }
    };
    auto tile_steps = [&](auto slow) {
      if (rows == LIN_ROWS) {
        steps(slow, std::integral_constant<int, LIN_ROWS>(), 0);
      } else {
#pragma unroll 1
        for (int r = 0; r < rows; ++r) steps(slow, std::integral_constant<int, 1>(), r);
      }
    };
    if (decay.slow) tile_steps(std::true_type());
    else tile_steps(std::false_type());
  }
  float* to = state_to(p, g, h);
  if (to) put_state(to);
}

// ---- single tokens ----
// One row a list, columns of the states in pieces of four: a block has a list and a head, LANES threads a row of the state, each STEP_AHEAD rows
// at a time, whose reads are on their way at once; y is summed over the rows' groups in shared memory. Bound by the states' bytes, which is a matter
// of reads in flight: few registers, eight blocks an SM. 2048 lists, 8 heads of 64 x 64: 216 us row by row with the state in registers.
constexpr int STEP_THREADS = 128, STEP_AHEAD = 8;
template <typename T, int LANES>
__global__ void __launch_bounds__(STEP_THREADS, 8) linear_step_kernel(const LinearParams p) {
  pdl_wait();
  constexpr int GROUPS = STEP_THREADS / LANES;
  __shared__ float s_q[LIN_MAX], s_k[LIN_MAX];
  __shared__ __align__(16) float s_y[GROUPS][LANES * 4];
  const int h = (int)(blockIdx.x % (unsigned)p.H), i = (int)(blockIdx.x / (unsigned)p.H), hkv = h / p.share;
  const int group = threadIdx.x / LANES, c = threadIdx.x % LANES * 4, slot = p.lists.slot(i);
  const bool mine = c < p.dv;
  const int64_t at = ((int64_t)slot * p.H + h) * p.dk * p.dv;
  const float* from = p.h_in && slot >= 0 && mine ? p.h_in + at + c : nullptr;
  float* to = p.h_out && slot >= 0 && mine ? p.h_out + at + c : nullptr;
  float4 s[STEP_AHEAD];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int a = 0; a < STEP_AHEAD; ++a) {
      const int k = k0 + a * GROUPS;
      s[a] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (from && k < p.dk) s[a] = *reinterpret_cast<const float4*>(from + k * p.dv);
    }
  };
  fetch(group);
  for (int k = threadIdx.x; k < p.dk; k += STEP_THREADS) {
    s_q[k] = to_f32<T>(p.q.get<T>(i, h)[k]);
    s_k[k] = to_f32<T>(p.k.get<T>(i, hkv)[k]);
  }
  float v[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
  if (mine) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32<T>(p.v.get<T>(i, hkv)[c + e]);
  }
  const Decay decay(log_decay_of(p, h));
  const float keep = decay.slow ? 1.f : 0.f;
  __syncthreads();
  for (int k0 = group; k0 < p.dk; k0 += STEP_AHEAD * GROUPS) {
    if (k0 > group) fetch(k0);
#pragma unroll
    for (int a = 0; a < STEP_AHEAD; ++a) {
      const int k = k0 + a * GROUPS;
      if (k >= p.dk) break;
      const float kk = s_k[k], q = s_q[k];
      float x[4] = {s[a].x, s[a].y, s[a].z, s[a].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = fmaf(x[e], decay.by, fmaf(kk, v[e], x[e] * keep));
        y[e] = fmaf(q, x[e], y[e]);
      }
      if (to) *reinterpret_cast<float4*>(to + k * p.dv) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  *reinterpret_cast<float4*>(&s_y[group][c]) = make_float4(y[0], y[1], y[2], y[3]);
  __syncthreads();
  for (int j = threadIdx.x; j < p.dv; j += STEP_THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) sum += s_y[g][j];
    const_cast<T*>(p.y.get<T>(i, h))[j] = from_f32<T>(sum * p.scale);
  }
}
template <typename T>
int launch_linear_step(const LinearParams& p, dim3 grid, cudaStream_t s) {
  const int lanes = (p.dv + 3) / 4;
  if (lanes <= 8) launch_dependent(linear_step_kernel<T, 8>, grid, STEP_THREADS, 0, s, p);
  else if (lanes <= 16) launch_dependent(linear_step_kernel<T, 16>, grid, STEP_THREADS, 0, s, p);
  else launch_dependent(linear_step_kernel<T, 32>, grid, STEP_THREADS, 0, s, p);
  return check_launch("linear_step_kernel");
}

// ends[j] += decay over a segment * ends[j - 1], for all segments of a list but the first and the last. A thread has four values of a state.
constexpr int CARRY_THREADS = 128, CARRY_AHEAD = 8;
__global__ void __launch_bounds__(CARRY_THREADS) linear_carry_kernel(const LinearParams p) {
  pdl_begin();
  const int h = blockIdx.y, size = p.dk * p.dv, e = (blockIdx.x * CARRY_THREADS + threadIdx.x) * 4;
  const float log_decay = log_decay_of(p, h);
  const Decay decay((float)p.chunk * log_decay);
  const bool vec = p.vec_e;
  if (e >= size) return;
  for (int i = blockIdx.z; i < p.lists.batch; i += gridDim.z) {
    const int64_t b = p.lists.begin(i), rows = p.lists.begin(i + 1) - b;
    if (rows <= 2 * p.chunk) continue;
    const int64_t at = b / p.chunk, n = min((rows + p.chunk - 1) / p.chunk - 1, (int64_t)p.n_ends - at);      // segments whose end is kept
    float* s = p.end + (at * p.H + h) * (int64_t)size + e;
    const int64_t step = (int64_t)p.H * size;
    float held[4];
    auto get = [&](int64_t j, float (&t)[4]) {
      if (vec) {
        const float4 f = *reinterpret_cast<const float4*>(s + j * step);
        t[0] = f.x; t[1] = f.y; t[2] = f.z; t[3] = f.w;
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) t[x] = e + x < size ? s[j * step + x] : 0.f;
      }
    };
    if (n < 2) continue;
    get(0, held);
    for (int64_t j = 1; j < n; j += CARRY_AHEAD) {
      float t[CARRY_AHEAD][4];
#pragma unroll
      for (int a = 0; a < CARRY_AHEAD; ++a)
        if (j + a < n) get(j + a, t[a]);
#pragma unroll
      for (int a = 0; a < CARRY_AHEAD; ++a) {
        if (j + a >= n) break;
#pragma unroll
        for (int x = 0; x < 4; ++x) held[x] = decay.step(held[x], t[a][x]);
        if (vec) {
          *reinterpret_cast<float4*>(s + (j + a) * step) = make_float4(held[0], held[1], held[2], held[3]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (e + x < size) s[(j + a) * step + x] = held[x];
        }
      }
    }
  }
}

template <typename T, int KT, int PARTS, int NV, int DV>
int launch_linear_columns(const LinearParams& p, dim3 grid, cudaStream_t s) {
  constexpr int SMEM = LIN_TILES * LIN_ROWS * (2 * KT * PARTS + DV) * (int)sizeof(T);
  if constexpr (SMEM > 46 * 1024) {           // (48 KB with what the kernel has besides)
    static PerDeviceOnce once;
    XB_SET_MAX_SMEM_ONCE(once, SMEM, (const void*)linear_rows_kernel<T, KT, PARTS, NV, DV>);
  }
  const unsigned threads = (unsigned)(((p.dv + NV - 1) / NV * PARTS + 31) / 32 * 32);
  launch_dependent(linear_rows_kernel<T, KT, PARTS, NV, DV>, grid, threads, SMEM, s, p);
  return check_launch("linear_rows_kernel");
}
// Up to 64 columns: two a thread where what is read of k and q is widened for them (16 bits), or where few threads of dk read it (fewer of
// dk a thread, more of those). us with one and two, fp32: 74 lists of 100 rows, 2 heads of 64 29 and 24, one of 74000 433 and 273; 1024 lists of 100
// 176 and 208 (32 of dk a thread: fewer warps for the registers). bf16, 4096 lists of 6 rows, 4 heads of 64: 258 and 180.
template <typename T, int KT, int PARTS>
int launch_linear_parts_of(const LinearParams& p, dim3 grid, cudaStream_t s) {
  if (p.dv <= 32) return launch_linear_columns<T, KT, PARTS, 1, 32>(p, grid, s);
  if (p.dv <= 64) return launch_linear_columns<T, KT, PARTS, sizeof(T) == 2 || (KT == 8 && PARTS == 8) ? 2 : 1, 64>(p, grid, s);
  return launch_linear_columns<T, KT, PARTS, 2, 128>(p, grid, s);
}
// Few lists: fewer of dk a thread, so that there are more of them (a row's FMAs of a thread wait for one another). us with 32 and 8 (or 16) of dk a
// thread, 74 lists of 100 rows, 2 heads, fp32: heads of 32 39 and 18, of 36 29 and 22, of 64 27 and 24, of 128 53 and 51. From 4 blocks an SM on
// both take as long (296 lists of 100 rows: 45).
template <typename T>
int launch_linear_rows(const LinearParams& p, dim3 grid, cudaStream_t s) {
  if ((int64_t)grid.x < 4 * (int64_t)sm_count()) {
    if (p.dk <= 32) return launch_linear_parts_of<T, 8, 4>(p, grid, s);
    if (p.dk <= 64) return launch_linear_parts_of<T, 8, 8>(p, grid, s);
    return launch_linear_parts_of<T, 16, 8>(p, grid, s);
  }
  if (p.dk <= 32) return launch_linear_parts_of<T, 32, 1>(p, grid, s);
  if (p.dk <= 64) return launch_linear_parts_of<T, 32, 2>(p, grid, s);
  return launch_linear_parts_of<T, 32, 4>(p, grid, s);
}

// The launches of a call, with `run` for the segments (or lists) of a grid
template <typename F>
int launch_linear_parts(LinearParams p, cudaStream_t s, F run) {
  const int64_t units = p.chunk ? p.n_ends + (int64_t)p.lists.batch : p.lists.batch;
  // (a list's heads side by side: long lists start first in all of them, and heads that share keys and values run at the same time)
  XB_REQUIRE(units * p.H < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_linear_attention: too many rows, lists and heads");
  const dim3 grid((unsigned)(units * p.H));
  if (p.order) {
    launch_dependent(lists_order_kernel, 1, 1024, 0, s, p.lists, p.order);
    if (int rc = check_launch("lists_order_kernel")) return rc;
  }
  if (p.chunk) {
    p.ends_only = 1;
    if (int rc = run(p, grid)) return rc;
    const int quads = (p.dk * p.dv + 3) / 4;
    launch_dependent(linear_carry_kernel, dim3((unsigned)((quads + CARRY_THREADS - 1) / CARRY_THREADS), (unsigned)p.H, (unsigned)std::min(p.lists.batch, 64)),
                     CARRY_THREADS, 0, s, p);
    if (int rc = check_launch("linear_carry_kernel")) return rc;
    p.ends_only = 0;
  }
  return run(p, grid);
}

}  // namespace
}  // namespace xb
