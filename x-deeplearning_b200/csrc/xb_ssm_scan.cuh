// The selective scan's kernels. Formulas in xdlb200.h; what a call runs is chosen in xb_ssm.cu.
//
// A lane keeps SPL = 4 states of K channels in registers, LPC lanes share a channel (4 LPC >= N). The four states of a lane are
// summed by the lane, the LPC partial sums by shuffles that leave K / LPC channels a lane where K > 1, so that a step of K = 4,
// LPC = 4 takes three shuffles for its four channels.
#pragma once

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
  // the first list that begins at row r or behind it (batch: none), found by a whole warp: 32 places a round
  __device__ __forceinline__ int first_from(int64_t r, int lane) const {
    if (!offsets) {
      const int64_t i = per > 0 ? (r + per - 1) / per : 0;
      return (int)(i < batch ? i : batch);
    }
    int lo = 0, n = batch;                // the answer is in [lo, lo + n]
    while (n > 0) {
      const int step = (n + 31) / 32, at = lo + lane * step;
      const unsigned before = __ballot_sync(0xffffffffu, lane * step < n && begin(at) < r);
      if (before == 0u) return lo;
      const int last = 31 - __clz(before);             // the last of the places that begins before r
      const int from = lo + last * step + 1;
      n = min(step - 1, lo + n - from);
      lo = from;
    }
    return lo;
  }
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.f + ex2(-LOG2E * v)); }
// log(1 + exp(v)) = max(v, 0) + log1p(u), u = exp(-|v|), and log1p(u) = 2 atanh(s) with s = u / (2 + u) <= 1/3 by the series of atanh, cut
// after s^13 (the next term is 1.4e-8 of the sum at most): right in relative terms where u is small too, which log(1 + u) is not.
__device__ __forceinline__ float softplus(float v) {
  const float u = ex2(-LOG2E * fabsf(v));
  const float s = __fdividef(u, 2.f + u), t = s * s;
  float p = fmaf(t, 1.f / 13, 1.f / 11);
  p = fmaf(t, p, 1.f / 9);
  p = fmaf(t, p, 1.f / 7);
  p = fmaf(t, p, 1.f / 5);
  p = fmaf(t, p, 1.f / 3);
  p = fmaf(t, p, 1.f);
  return (v > 0.f ? v : 0.f) + 2.f * s * p;
}

struct ScanParams {
  const void* x; int64_t ldx;
  const void* delta; int64_t lddelta;
  const void* z; int64_t ldz;
  const void* B; int64_t ldb;
  const void* C; int64_t ldc;
  void* y; int64_t ldy;
  const float* A; const float* skip; const float* delta_bias;
  const float* h_in; float* h_out;
  Lists lists;
  int D, N, per_group, groups, softplus, bf16;
  int vec, vec_bc, vec_h;                 // rows of x, delta, z, y in whole 16-byte pieces; B and C in pieces of four; states and A in float4
  // the split scan: chunks of `chunk` rows
  int64_t chunk;
  int n_chunks;
  float* end;                             // [n_chunks][D][N]: state behind the chunk's last row as far as the chunk knows, then with the carry
  float* first;                           // [n_chunks][D][N]: copies of the first states of lists that go on in the next chunk
  float* steps;                           // [n_chunks][D]: sum of the chunk's steps
  int* kind;                              // [n_chunks]: 0 no list goes on behind the chunk, 1 one that begins in it, 2 one that covers it
};

// V adjacent elements of SIZE bytes as they lie in memory
template <int SIZE, int V>
struct Raw {
  static constexpr int W = (SIZE * V + 3) / 4;
  static constexpr bool PIECE = SIZE * V >= 4;          // (one 2-byte element is never read or written as a word)
  uint32_t w[W];
  // `in` of them exist (others are 0); in whole where they do and `vec` says that they lie aligned
  __device__ __forceinline__ void load(const void* base, int64_t at, int in, bool vec) {
    const char* p = static_cast<const char*>(base) + at * SIZE;
    if (PIECE && vec && in >= V) {
      if constexpr (W == 4) { const uint4 t = __ldg(reinterpret_cast<const uint4*>(p)); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
      else if constexpr (W == 2) { const uint2 t = __ldg(reinterpret_cast<const uint2*>(p)); w[0] = t.x; w[1] = t.y; }
      else w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = 0u;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < in) {
          if constexpr (SIZE == 4) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
          else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + i) << (16 * (i & 1));
        }
    }
  }
  __device__ __forceinline__ float get(int i, bool bf16) const {
    if constexpr (SIZE == 4) return __uint_as_float(w[i]);
    const uint32_t b = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
    return bf16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half((unsigned short)b));
  }
  __device__ __forceinline__ void put(int i, float v, bool bf16) {
    if constexpr (SIZE == 4) { w[i] = __float_as_uint(v); return; }
    const uint32_t b = bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
    w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | b << 16 : b;
  }
  __device__ __forceinline__ void store(void* base, int64_t at, int in, bool vec) const {
    char* p = static_cast<char*>(base) + at * SIZE;
    if (PIECE && vec && in >= V) {
      if constexpr (W == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      else if constexpr (W == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < in) {
          if constexpr (SIZE == 4) reinterpret_cast<uint32_t*>(p)[i] = w[i];
          else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
  }
};

constexpr int SPL = 4;                    // states of a lane
constexpr int SCAN_THREADS = 128;

// SPL states of channel c from row `row` of a [rows][D][N] array (zeros where there is none), and back
__device__ __forceinline__ void load_states(const float* p, int64_t row, const ScanParams& q, int c, int n0, float (&h)[SPL]) {
  if (!p || row < 0) {
#pragma unroll
    for (int s = 0; s < SPL; ++s) h[s] = 0.f;
    return;
  }
  p += (row * q.D + c) * q.N + n0;
  if (q.vec_h && n0 < q.N) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    h[0] = t.x; h[1] = t.y; h[2] = t.z; h[3] = t.w;
  } else {
#pragma unroll
    for (int s = 0; s < SPL; ++s) h[s] = n0 + s < q.N ? p[s] : 0.f;
  }
}
__device__ __forceinline__ void store_states(float* p, int64_t row, const ScanParams& q, int c, int n0, const float (&h)[SPL]) {
  if (!p || row < 0) return;
  p += (row * q.D + c) * q.N + n0;
  if (q.vec_h && n0 < q.N) {
    *reinterpret_cast<float4*>(p) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int s = 0; s < SPL; ++s)
      if (n0 + s < q.N) p[s] = h[s];
  }
}

// One row a list: the states are the traffic (8 N bytes a channel against 8 of the row), so a lane has the loads of STEP_U channels on
// their way before it uses the first.
constexpr int STEP_U = 4;
template <int SIZE, int LPC>
__global__ void __launch_bounds__(SCAN_THREADS) ssm_step_kernel(const ScanParams p, int channel_blocks) {
  pdl_begin();
  constexpr int CPB = SCAN_THREADS / LPC;               // channels of a round
  const int i = blockIdx.x / channel_blocks;
  const int n0 = threadIdx.x % LPC * SPL;
  const int c0 = (blockIdx.x % channel_blocks) * CPB * STEP_U + threadIdx.x / LPC;
  const int64_t r = i;
  const int slot = p.lists.slot(i);
  float h[STEP_U][SPL], A[STEP_U][SPL], x[STEP_U], v[STEP_U], bias[STEP_U], skip[STEP_U], z[STEP_U];
  Raw<SIZE, SPL> B[STEP_U], C[STEP_U];
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) {
    const int c = min(c0 + u * CPB, p.D - 1);
    load_states(p.h_in, slot, p, c, n0, h[u]);
    Raw<SIZE, 1> t;
    t.load(p.x, r * p.ldx + c, 1, false);
    x[u] = t.get(0, p.bf16);
    t.load(p.delta, r * p.lddelta + c, 1, false);
    v[u] = t.get(0, p.bf16);
    z[u] = 0.f;
    if (p.z) {
      t.load(p.z, r * p.ldz + c, 1, false);
      z[u] = t.get(0, p.bf16);
    }
    bias[u] = p.delta_bias ? p.delta_bias[c] : 0.f;
    skip[u] = p.skip ? p.skip[c] : 0.f;
    load_states(p.A, 0, p, c, n0, A[u]);
    const int in = max(0, min(SPL, p.N - n0));
    const int64_t at = (int64_t)(c / p.per_group) * p.N + n0;
    B[u].load(p.B, r * p.ldb + at, in, p.vec_bc);
    C[u].load(p.C, r * p.ldc + at, in, p.vec_bc);
  }
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) {
    const int c = c0 + u * CPB;
    const float d = p.softplus ? softplus(v[u] + bias[u]) : v[u] + bias[u], dx = d * x[u];
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      h[u][s] = fmaf(ex2(d * (LOG2E * A[u][s])), h[u][s], dx * B[u].get(s, p.bf16));
      y = fmaf(C[u].get(s, p.bf16), h[u][s], y);
    }
#pragma unroll
    for (int m = LPC / 2; m > 0; m >>= 1) y += __shfl_xor_sync(0xffffffffu, y, m);
    if (c < p.D) {
      store_states(p.h_out, slot, p, c, n0, h[u]);
      if (n0 == 0) {
        y = fmaf(skip[u], x[u], y);
        if (p.z) y *= silu(z[u]);
        Raw<SIZE, 1> t;
        t.put(0, y, p.bf16);
        t.store(p.y, r * p.ldy + c, 1, false);
      }
    }
  }
}

// What a block of the tile kernel walks: one list, or the rows of one chunk; or (TAILS) the rows of a chunk that belong to the list
// that goes on in the next one, for its state alone.
enum { SCAN_LISTS, SCAN_CHUNKS, SCAN_TAILS };

__host__ __device__ constexpr int min_c(int a, int b) { return a < b ? a : b; }
template <int LPC, int K>
struct ScanShape {
  static constexpr int CH = SCAN_THREADS / LPC * K;     // channels of a block
  // rows of a tile: 2048 elements of each input, and at most 2048 of B
  static constexpr int ROWS = min_c(2048 / CH, 2048 / (SPL * LPC));
  static constexpr int E = ROWS * CH / SCAN_THREADS;    // elements of an input a thread brings
};

// Tiles of ROWS rows x CH channels: the threads bring x and delta (16-byte pieces, those of the next tile while this one is walked), leave
// the steps d and x in shared memory as fp32 and B and C beside them, walk the rows, leave the sums where d was, and write y. Every
// exponential, softplus and sigmoid of the call is an SFU instruction: N + 4 for a row and channel, 16 a clock and SM.
template <int SIZE, int LPC, int K, int MODE>
__global__ void __launch_bounds__(SCAN_THREADS, 4) ssm_scan_kernel(const ScanParams p, int blocks_a_group) {
  pdl_begin();
  using S = ScanShape<LPC, K>;
  constexpr int CH = S::CH, ROWS = S::ROWS, E = S::E, NP = SPL * LPC;
  constexpr int V = min_c(E, 16 / SIZE), VPR = CH / V, RPI = SCAN_THREADS / VPR, IT = E / V;
  static_assert(VPR <= SCAN_THREADS && IT * RPI == ROWS, "");
  constexpr int BC = 2 * ROWS * LPC, IT_BC = (BC + SCAN_THREADS - 1) / SCAN_THREADS;      // pieces of four of B and of C
  __shared__ __align__(16) float s_d[ROWS][CH];
  __shared__ __align__(16) float s_x[ROWS][CH];
  __shared__ __align__(16) float s_b[2][ROWS][NP];
  const int tid = threadIdx.x, lane = tid & 31;
  const int channel_blocks = blocks_a_group * p.groups, cb = blockIdx.x % channel_blocks, unit = blockIdx.x / channel_blocks;
  const int g = cb / blocks_a_group, c_lo = g * p.per_group + (cb - g * blocks_a_group) * CH, c_hi = min((g + 1) * p.per_group, c_lo + CH);
  const bool bf16 = p.bf16 != 0;

  // the rows, and the list that they begin in
  int64_t row, row_end;
  int cur = -1, nxt = 0;                  // the list under way (-1: none) and the one that begins next
  int64_t cur_end = 0;
  bool last_chunk = false, fresh = true;  // fresh: the list under way begins in these rows
  const int64_t chunk0 = (int64_t)unit * p.chunk, chunk1 = chunk0 + p.chunk;
  if (MODE == SCAN_LISTS) {
    row = p.lists.begin(unit);
    row_end = p.lists.begin(unit + 1);
    nxt = unit;
  } else if (MODE == SCAN_CHUNKS) {
    row = max(chunk0, p.lists.begin(0));
    row_end = min(chunk1, p.lists.begin(p.lists.batch));
    nxt = p.lists.first_from(chunk0, lane);
    last_chunk = unit == p.n_chunks - 1;
    if (nxt > 0 && row < row_end) {
      const int64_t b = nxt < p.lists.batch ? p.lists.begin(nxt) : p.lists.begin(p.lists.batch);
      if (b > row) { cur = nxt - 1; cur_end = b; fresh = false; }
    }
  } else {
    const int j = p.lists.first_from(chunk1, lane);
    row = row_end = chunk1;
    if (j > 0 && p.lists.begin(j) > chunk1) {
      const int64_t b = p.lists.begin(j - 1);
      cur = j - 1;
      fresh = b >= chunk0;
      row = fresh ? b : chunk0;
    }
    if (tid == 0 && cb == 0) p.kind[unit] = cur < 0 ? 0 : (fresh ? 1 : 2);
    if (cur < 0) return;
  }

  // this lane's channels and states
  const int sub = lane % LPC, n0 = sub * SPL;
  const int cl = (tid / LPC) * K;                       // first of them in the block
  float A[K][SPL], h[K][SPL], sum_d[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sum_d[k] = 0.f;
    load_states(p.A, c_lo + cl + k < c_hi ? 0 : -1, p, c_lo + cl + k, n0, A[k]);
#pragma unroll
    for (int s = 0; s < SPL; ++s) { A[k][s] *= LOG2E; h[k][s] = 0.f; }
  }
  auto take = [&](const float* from, int64_t at) {
#pragma unroll
    for (int k = 0; k < K; ++k) load_states(from, c_lo + cl + k < c_hi ? at : -1, p, c_lo + cl + k, n0, h[k]);
  };
  auto leave = [&](float* to, int64_t at) {
#pragma unroll
    for (int k = 0; k < K; ++k) store_states(to, c_lo + cl + k < c_hi ? at : -1, p, c_lo + cl + k, n0, h[k]);
  };
  // the lists that begin at row r: their first states; those of no rows are done at once
  auto begin_at = [&](int64_t r) {
    cur = -1;
    while (nxt < p.lists.batch) {
      const int64_t b = p.lists.begin(nxt), e = p.lists.begin(nxt + 1);
      if (MODE == SCAN_CHUNKS && b >= chunk1 && !last_chunk) break;         // (the next chunk's)
      if (MODE == SCAN_LISTS && nxt > unit) break;
      const int slot = p.lists.slot(nxt);
      // a list that goes on behind the chunk: its end writes the state, perhaps over this one, so the copy is read
      if (MODE == SCAN_CHUNKS && p.h_in && e > chunk1) take(p.first, slot < 0 ? -1 : unit);
      else take(p.h_in, slot);
      ++nxt;
      if (e > r) { cur = nxt - 1; cur_end = e; break; }
      leave(p.h_out, slot);
    }
  };
  if (MODE == SCAN_TAILS) {
    if (fresh && p.h_in) {
      const int slot = p.lists.slot(cur);
      take(p.h_in, slot);
      if (slot >= 0) leave(p.first, unit);
    }
  } else if (!fresh) {
    take(p.end, unit - 1);
  }
  if (MODE != SCAN_TAILS && cur < 0) begin_at(row);

  Raw<SIZE, V> rx[IT], rd[IT], rz[IT];
  Raw<SIZE, SPL> rb[IT_BC];
  const int vr = tid / VPR, vc = tid % VPR * V, ch_in = max(0, min(V, c_hi - c_lo - vc));
  auto bring = [&](int64_t t0) {
    const int64_t n = row_end - t0;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = vr + i * RPI, in = r < n ? ch_in : 0;
      rx[i].load(p.x, (t0 + r) * p.ldx + c_lo + vc, in, p.vec);
      rd[i].load(p.delta, (t0 + r) * p.lddelta + c_lo + vc, in, p.vec);
    }
#pragma unroll
    for (int i = 0; i < IT_BC; ++i) {
      const int e = tid + i * SCAN_THREADS, r = e / LPC % ROWS, m = e % LPC * SPL;
      const bool second = e >= BC / 2;
      if (MODE == SCAN_TAILS && second) continue;
      const int in = e < BC && r < n ? max(0, min(SPL, p.N - m)) : 0;
      const int64_t at = (t0 + r) * (second ? p.ldc : p.ldb) + (int64_t)g * p.N + m;
      rb[i].load(second ? p.C : p.B, at, in, p.vec_bc);
    }
  };
  float bias[V], skip[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool in = v < ch_in;
    bias[v] = in && p.delta_bias ? p.delta_bias[c_lo + vc + v] : 0.f;
    skip[v] = in && p.skip ? p.skip[c_lo + vc + v] : 0.f;
  }

  if (row < row_end) bring(row);
  for (; row < row_end; row += ROWS) {
    const int n = (int)min((int64_t)ROWS, row_end - row);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = vr + i * RPI;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float t = rd[i].get(v, bf16) + bias[v];
        s_d[r][vc + v] = p.softplus ? softplus(t) : t;
        s_x[r][vc + v] = rx[i].get(v, bf16);
      }
    }
#pragma unroll
    for (int i = 0; i < IT_BC; ++i) {
      const int e = tid + i * SCAN_THREADS, r = e / LPC % ROWS, m = e % LPC * SPL;
      if (e < BC && !(MODE == SCAN_TAILS && e >= BC / 2))
        *reinterpret_cast<float4*>(&s_b[e >= BC / 2][r][m]) = make_float4(rb[i].get(0, bf16), rb[i].get(1, bf16), rb[i].get(2, bf16), rb[i].get(3, bf16));
    }
    __syncthreads();
    if (row + ROWS < row_end) bring(row + ROWS);
    if (MODE != SCAN_TAILS && p.z) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = vr + i * RPI;
        rz[i].load(p.z, (row + r) * p.ldz + c_lo + vc, r < n ? ch_in : 0, p.vec);
      }
    }
    // walk the tile, list by list
    for (int t = 0; t < n;) {
      if (MODE == SCAN_CHUNKS && row + t == cur_end) {
        leave(p.h_out, p.lists.slot(cur));
        begin_at(cur_end);
      }
      const int run = MODE == SCAN_CHUNKS && cur >= 0 ? (int)min((int64_t)n, cur_end - row) : n;
#pragma unroll 2
      for (; t < run; ++t) {
        float d[K], x[K], y[K];
        if constexpr (K == 4) {
          const float4 d4 = *reinterpret_cast<const float4*>(&s_d[t][cl]), x4 = *reinterpret_cast<const float4*>(&s_x[t][cl]);
          d[0] = d4.x; d[1] = d4.y; d[2] = d4.z; d[3] = d4.w;
          x[0] = x4.x; x[1] = x4.y; x[2] = x4.z; x[3] = x4.w;
        } else {
#pragma unroll
          for (int k = 0; k < K; ++k) { d[k] = s_d[t][cl + k]; x[k] = s_x[t][cl + k]; }
        }
        const float4 b4 = *reinterpret_cast<const float4*>(&s_b[0][t][n0]);
        const float b[SPL] = {b4.x, b4.y, b4.z, b4.w};
        float4 c4 = make_float4(0.f, 0.f, 0.f, 0.f);
        if (MODE != SCAN_TAILS) c4 = *reinterpret_cast<const float4*>(&s_b[1][t][n0]);
        const float cc[SPL] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float dx = d[k] * x[k];
          y[k] = 0.f;
#pragma unroll
          for (int s = 0; s < SPL; ++s) {
            h[k][s] = fmaf(ex2(d[k] * A[k][s]), h[k][s], dx * b[s]);
            if (MODE != SCAN_TAILS) y[k] = fmaf(cc[s], h[k][s], y[k]);
          }
          if (MODE == SCAN_TAILS) sum_d[k] += d[k];
        }
        if (MODE != SCAN_TAILS) {
          // sums over the LPC lanes: halves of the channels change sides while a lane has several, then whole sums
          int c = cl;
          int have = K;
#pragma unroll
          for (int m = LPC / 2; m > 0; m >>= 1) {
            const bool up = sub & m;
            if (have > 1) {
              have /= 2;
#pragma unroll
              for (int k = 0; k < K / 2; ++k)
                if (k < have) {
                  const float give = up ? y[k] : y[k + have], keep = up ? y[k + have] : y[k];
                  y[k] = keep + __shfl_xor_sync(0xffffffffu, give, m);
                }
              c += up ? have : 0;
            } else {
              y[0] += __shfl_xor_sync(0xffffffffu, y[0], m);
            }
          }
          constexpr int LEFT = K > LPC ? K / LPC : 1, SHARE = LPC > K ? LPC / K : 1;   // channels that a lane, or SHARE of them, end with
          // (this warp alone reads and writes these channels, and every lane has read d of this row before the sums were exchanged)
          if (sub % SHARE == 0)
#pragma unroll
            for (int k = 0; k < LEFT; ++k) s_d[t][c + k] = y[k];
        }
      }
    }
    __syncthreads();
    if (MODE != SCAN_TAILS) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = vr + i * RPI;
        Raw<SIZE, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float y = fmaf(skip[v], s_x[r][vc + v], s_d[r][vc + v]);
          if (p.z) y *= silu(rz[i].get(v, bf16));
          out.put(v, y, bf16);
        }
        out.store(p.y, (row + r) * p.ldy + c_lo + vc, r < n ? ch_in : 0, p.vec);
      }
    }
  }
  if (MODE == SCAN_TAILS) {
    leave(p.end, unit);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (sub == 0 && c_lo + cl + k < c_hi) p.steps[(int64_t)unit * p.D + c_lo + cl + k] = sum_d[k];
  } else if (cur >= 0 && cur_end <= row_end) {
    leave(p.h_out, p.lists.slot(cur));
    if (MODE == SCAN_CHUNKS) begin_at(cur_end);          // (lists without rows behind the last)
  }
}

// The state that comes into every chunk, from the ends that the chunks know: end[j] += exp(A steps[j]) end[j - 1] where one list covers chunk
// j. A block has 32 (channel, state) pairs and splits the chunks among its 8 warps: each makes its own part's product and sum, takes
// what comes in from the parts before it, and walks its part again.
constexpr int CARRY_PARTS = 8;
__global__ void __launch_bounds__(32 * CARRY_PARTS) ssm_carry_kernel(const ScanParams p) {
  pdl_begin();
  __shared__ float s_p[CARRY_PARTS][32], s_e[CARRY_PARTS][32];
  const int part = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t pairs = (int64_t)p.D * p.N, at = (int64_t)blockIdx.x * 32 + lane;
  const bool mine = at < pairs;
  const int c = mine ? (int)(at / p.N) : 0;
  const float A = mine ? LOG2E * p.A[at] : 0.f;
  const int n = p.n_chunks - 1, share = (n + CARRY_PARTS - 1) / CARRY_PARTS, j0 = min(n, part * share), j1 = min(n, j0 + share);
  float P = 1.f, e = 0.f;
  auto one = [&](int j, float& through, float& own) {
    const int kind = p.kind[j];
    own = mine && kind ? p.end[j * pairs + at] : 0.f;
    through = mine && kind == 2 ? ex2(A * p.steps[(int64_t)j * p.D + c]) : 0.f;
  };
#pragma unroll 8
  for (int j = j0; j < j1; ++j) {
    float t, o;
    one(j, t, o);
    e = t == 0.f ? o : fmaf(t, e, o);
    P *= t;
  }
  s_p[part][lane] = P;
  s_e[part][lane] = e;
  __syncthreads();
  e = 0.f;
  for (int k = 0; k < part; ++k) e = s_p[k][lane] == 0.f ? s_e[k][lane] : fmaf(s_p[k][lane], e, s_e[k][lane]);
#pragma unroll 8
  for (int j = j0; j < j1; ++j) {
    float t, o;
    one(j, t, o);
    e = t == 0.f ? o : fmaf(t, e, o);
    if (mine) p.end[j * pairs + at] = e;
  }
}

}  // namespace
}  // namespace xb
