// The selective scan's kernels. Formulas in xdlb200.h; what a call runs is chosen in xb_ssm.cu.
//
// A lane keeps SPL = 4 states of K channels in registers, LPC lanes share a channel (4 LPC >= N). The four states of a lane are
// summed by the lane, the LPC partial sums by shuffles that leave K / LPC channels a lane where K > 1, so that a step of K = 4,
// LPC = 4 takes three shuffles for its four channels.
#pragma once

#include "xb_ssm.cuh"

namespace xb {
namespace {

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

// One row a list: the states are the traffic (8 N bytes a channel against 8 of the row), so a lane has those of STEP_U channels on their
// way before it uses the first. With four lanes a channel or more each of them has one of the four channels for its own: it alone
// reads its x, delta and z, makes its step and its gate, and ends with its sum. 8192 rows of D = 256, N = 16: 117 us with all of that
// in every lane, 61 now = 4.7 TB/s, 0.73 of a copy's rate; the loads in flight bound it (issue slots 57 % busy).
constexpr int STEP_U = 4;
template <typename T, int LPC>
__global__ void __launch_bounds__(SCAN_THREADS) ssm_step_kernel(const ScanParams p, int channel_blocks) {
  pdl_begin();
  constexpr int CPB = SCAN_THREADS / LPC;               // channels of a round
  constexpr int OWN = LPC >= STEP_U ? 1 : STEP_U;       // channels whose row a lane reads
  constexpr int SHARE = LPC >= STEP_U ? LPC / STEP_U : 1;
  const int i = blockIdx.x / channel_blocks;
  const int sub = threadIdx.x % LPC, n0 = sub * SPL, own0 = LPC >= STEP_U ? sub / SHARE : 0;
  const int c0 = (blockIdx.x - i * channel_blocks) * CPB * STEP_U + threadIdx.x / LPC;
  const int64_t r = i;
  const int slot = p.lists.slot(i);
  auto channel = [&](int u) { return c0 + u * CPB; };
  float h[STEP_U][SPL], A[STEP_U][SPL];
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) load_states(channel(u) < p.D ? p.h_in : nullptr, slot, p, channel(u), n0, h[u]);
  const T *px = static_cast<const T*>(p.x) + r * p.ldx, *pd = static_cast<const T*>(p.delta) + r * p.lddelta;
  const T *pz = static_cast<const T*>(p.z) + r * p.ldz, *pb = static_cast<const T*>(p.B) + r * p.ldb, *pc = static_cast<const T*>(p.C) + r * p.ldc;
  const int in = max(0, min(SPL, p.N - n0));
  float x[OWN], d[OWN], z[OWN], skip[OWN];
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int c = min(channel(own0 + o), p.D - 1);
    x[o] = to_f32<T>(px[c]);
    d[o] = to_f32<T>(pd[c]);
    z[o] = p.z ? to_f32<T>(pz[c]) : 0.f;
    if (p.delta_bias) d[o] += p.delta_bias[c];
    skip[o] = p.skip ? p.skip[c] : 0.f;
  }
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) load_states(channel(u) < p.D ? p.A : nullptr, 0, p, channel(u), n0, A[u]);
  Raw<T, SPL> B, C;
  int g = -1;                                           // whose B and C those are
#pragma unroll
  for (int o = 0; o < OWN; ++o)
    if (p.softplus) d[o] = softplus(d[o]);
  float y[STEP_U];
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) {
    const int now = p.groups == 1 ? 0 : min(channel(u), p.D - 1) / p.per_group;
    if (now != g) {
      g = now;
      B.load(pb + (int64_t)g * p.N + n0, in, p.vec_bc);
      C.load(pc + (int64_t)g * p.N + n0, in, p.vec_bc);
    }
    float du = d[LPC >= STEP_U ? 0 : u % OWN], dx = du * x[LPC >= STEP_U ? 0 : u % OWN];
    if constexpr (LPC >= STEP_U) {
      du = __shfl_sync(0xffffffffu, du, u * SHARE, LPC);
      dx = __shfl_sync(0xffffffffu, dx, u * SHARE, LPC);
    }
    y[u] = 0.f;
#pragma unroll
    for (int s = 0; s < SPL; ++s) {
      h[u][s] = fmaf(ex2(du * (LOG2E * A[u][s])), h[u][s], dx * B.get(s));
      y[u] = fmaf(C.get(s), h[u][s], y[u]);
    }
    if (channel(u) < p.D) store_states(p.h_out, slot, p, channel(u), n0, h[u]);
  }
  // sums over the lanes of a channel: while a lane has several channels' the halves change sides
  int have = STEP_U;
#pragma unroll
  for (int m = LPC / 2; m > 0; m >>= 1) {
    if (LPC >= STEP_U && have > 1) {
      have /= 2;
      const bool up = sub & m;
#pragma unroll
      for (int u = 0; u < STEP_U / 2; ++u)
        if (u < have) {
          const float give = up ? y[u] : y[u + have], keep = up ? y[u + have] : y[u];
          y[u] = keep + __shfl_xor_sync(0xffffffffu, give, m);
        }
    } else {
#pragma unroll
      for (int u = 0; u < OWN; ++u) y[u] += __shfl_xor_sync(0xffffffffu, y[u], m);
    }
  }
#pragma unroll
  for (int o = 0; o < OWN; ++o) {
    const int c = channel(own0 + o);
    if (c < p.D && (LPC >= STEP_U ? sub % SHARE == 0 : sub == 0)) {
      float v = fmaf(skip[o], x[o], y[o]);
      if (p.z) v *= silu(z[o]);
      static_cast<T*>(p.y)[r * p.ldy + c] = from_f32<T>(v);
    }
  }
}

// A list of more than `chunk` rows is walked in chunks of so many, counted from its own beginning, by blocks of their own: ENDS walks every
// chunk but a list's last from zeros (its first from the list's own state) for the state at its end alone, ssm_carry_kernel puts the
// ends together, and WALK makes the results with the state that comes into its chunk. Lists of up to `chunk` rows are walked once.
// Chunk j of list i is number begin(i) / chunk + i + j of WALK (every list has one), and number begin(i) / chunk + j of ENDS: a list whose
// chunk j is not its last reaches beyond begin(i) + (j + 1) chunk, so the next list's numbers lie behind.
enum { SCAN_WALK, SCAN_ENDS };

__host__ __device__ constexpr int min_c(int a, int b) { return a < b ? a : b; }
template <int LPC, int K>
struct ScanShape {
  static constexpr int CH = SCAN_THREADS / LPC * K;     // channels of a block
  // rows of a tile: TILE elements of each input, and at most 1024 of B
  static constexpr int TILE = 1024, ROWS = min_c(TILE / CH, 1024 / (SPL * LPC));
  static constexpr int E = ROWS * CH / SCAN_THREADS;    // elements of an input a thread brings
  static constexpr int R = 4 / K;                       // rows that a lane walks at a time
};

// Tiles of ROWS rows x CH channels: the threads bring x and delta (pieces of four, those of the next tile while this one is walked), leave
// the steps d and x in shared memory as fp32 and B and C beside them, walk the rows, leave the sums there too, and write y. Every
// exponential, softplus and sigmoid is an SFU instruction: N + 4 for a row and channel, 16 a clock and SM. 256 lists of 70000 rows in all,
// D = 256, N = 16: 192 us against 78 of the SFUs alone; they are 58 % busy, issue slots 57 %, and the 20 warps that
// 94 registers leave an SM wait for shared memory and shuffles.
template <int K>
constexpr int SCAN_BLOCKS = K == 1 ? 5 : 6;            // of an SM: the registers are shared among so many
template <typename T, int LPC, int K, int MODE>
__global__ void __launch_bounds__(SCAN_THREADS, SCAN_BLOCKS<K>) ssm_scan_kernel(const ScanParams p, int blocks_a_group) {
  pdl_begin();
  using S = ScanShape<LPC, K>;
  constexpr int CH = S::CH, ROWS = S::ROWS, E = S::E, R = S::R, NP = SPL * LPC;
  constexpr int V = min_c(E, 4), VPR = CH / V, RPI = SCAN_THREADS / VPR, IT = E / V;
  static_assert(VPR <= SCAN_THREADS && IT * RPI == ROWS && VPR * V == CH, "");
  constexpr int BC = 2 * ROWS * LPC, IT_BC = (BC + SCAN_THREADS - 1) / SCAN_THREADS;      // pieces of four of B and of C
  __shared__ struct { __align__(16) float d[ROWS][CH], x[ROWS][CH], y[ROWS][CH], b[2][ROWS][NP], bias[CH], skip[CH]; } sm;
  const int tid = threadIdx.x, lane = tid & 31;
  const int channel_blocks = blocks_a_group * p.groups, cb = blockIdx.x % channel_blocks, unit = blockIdx.x / channel_blocks;
  const int g = cb / blocks_a_group, c_lo = g * p.per_group + (cb - g * blocks_a_group) * CH, c_hi = min((g + 1) * p.per_group, c_lo + CH);

  // the list and the rows of it
  int list = p.order ? p.order[unit] : unit, part = 0;
  if (p.chunk > 0) {
    if (MODE == SCAN_WALK) {
      list = p.lists.of_chunk(unit, p.chunk, lane);
      part = unit - (int)(p.lists.begin(list) / p.chunk) - list;
    } else {
      list = p.lists.first_from((int64_t)(unit + 1) * p.chunk, lane) - 1;
      part = list < 0 ? -1 : unit - (int)(p.lists.begin(list) / p.chunk);
    }
  }
  int64_t row = 0, row_end = 0;
  int end_at = 0;                         // number of the chunk among those whose ends are kept
  bool last = true;
  if (part >= 0) {
    const int64_t b = p.lists.begin(list), e = max(b, p.lists.begin(list + 1));
    row = b + part * p.chunk;
    last = p.chunk == 0 || row + p.chunk >= e;
    row_end = last ? e : row + p.chunk;
    end_at = p.chunk > 0 ? (int)(b / p.chunk) + part : 0;
    if (row > e || (part > 0 && row == e)) part = -1;      // behind the list's last chunk
  }
  if (MODE == SCAN_ENDS) {
    if (last) part = -1;
    if (tid == 0 && cb == 0) p.kind[unit] = part < 0 ? 0 : (part == 0 ? 1 : 2);
  }
  if (part < 0) return;
  const int slot = p.lists.slot(list);
  for (int c = tid; c < CH; c += SCAN_THREADS) {
    sm.bias[c] = p.delta_bias && c_lo + c < c_hi ? p.delta_bias[c_lo + c] : 0.f;
    sm.skip[c] = p.skip && c_lo + c < c_hi ? p.skip[c_lo + c] : 0.f;
  }
  __syncthreads();

  // this lane's channels and states
  const int sub = lane % LPC, n0 = sub * SPL;
  const int cl = (tid / LPC) * K;                       // first of them in the block
  f32x2 A[K][2], h[K][2];
  float sum_d[K];
  auto read = [&](const float* from, int64_t at, f32x2 (&to)[K][2], float times) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t[SPL];
      load_states(from, c_lo + cl + k < c_hi ? at : -1, p, c_lo + cl + k, n0, t);
      to[k][0] = pack2(times * t[0], times * t[1]);
      to[k][1] = pack2(times * t[2], times * t[3]);
    }
  };
  auto take = [&](const float* from, int64_t at) { read(from, at, h, 1.f); };
  auto leave = [&](float* to, int64_t at) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t[SPL];
      unpack2(h[k][0], t[0], t[1]);
      unpack2(h[k][1], t[2], t[3]);
      store_states(to, c_lo + cl + k < c_hi ? at : -1, p, c_lo + cl + k, n0, t);
    }
  };
  read(p.A, 0, A, LOG2E);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sum_d[k] = 0.f;
    h[k][0] = h[k][1] = 0;
  }
  if (part == 0) {
    // a list of several chunks: its last writes the state, perhaps over the one that it began with, so ENDS leaves a copy for WALK
    if (MODE == SCAN_WALK && !last && p.h_in) {
      take(p.first, slot < 0 ? -1 : end_at);
    } else {
      take(p.h_in, slot);
      if (MODE == SCAN_ENDS && p.h_in && slot >= 0) leave(p.first, end_at);
    }
  } else if (MODE == SCAN_WALK) {
    take(p.end, end_at - 1);
  }

  // What a thread brings: V channels of the rows vr, vr + RPI, ...; its places move on with the tiles.
  Raw<T, V> rx[IT], rd[IT], rz[IT];
  Raw<T, SPL> rb[IT_BC];
  const int vr = tid / VPR, vc = tid % VPR * V, ch_in = max(0, min(V, c_hi - c_lo - vc));
  const T* px = static_cast<const T*>(p.x) + (row + vr) * p.ldx + c_lo + vc;
  const T* pd = static_cast<const T*>(p.delta) + (row + vr) * p.lddelta + c_lo + vc;
  const T* pz = static_cast<const T*>(p.z) + (row + vr) * p.ldz + c_lo + vc;
  T* py = static_cast<T*>(p.y) + (row + vr) * p.ldy + c_lo + vc;
  const bool whole_ch = p.vec && ch_in == V;
  // pieces of B, then of C: the threads of the second half bring C where a half of them bring B, and in turns otherwise
  constexpr int HALF = BC / 2;
  static_assert(HALF % SCAN_THREADS == 0 || BC <= SCAN_THREADS, "");
  const bool c_half = BC <= SCAN_THREADS && tid >= HALF;
  const int be = c_half ? tid - HALF : tid, br = be / LPC, bc_in = BC <= SCAN_THREADS && tid >= (MODE == SCAN_ENDS ? HALF : BC) ? 0 : max(0, min(SPL, p.N - n0));
  const T* pb = static_cast<const T*>(c_half ? p.C : p.B) + (row + br) * (c_half ? p.ldc : p.ldb) + (int64_t)g * p.N + n0;
  const T* pc = static_cast<const T*>(p.C) + (row + br) * p.ldc + (int64_t)g * p.N + n0;
  auto bring = [&](int64_t n) {                          // n rows are left
    if (whole_ch && n >= ROWS) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        rx[i].load_piece(px + i * RPI * p.ldx);
        rd[i].load_piece(pd + i * RPI * p.lddelta);
      }
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int in = vr + i * RPI < n ? ch_in : 0;
        rx[i].load(px + i * RPI * p.ldx, in, p.vec);
        rd[i].load(pd + i * RPI * p.lddelta, in, p.vec);
      }
    }
    px += ROWS * p.ldx;
    pd += ROWS * p.lddelta;
    if constexpr (BC <= SCAN_THREADS) {
      rb[0].load(pb, br < n ? bc_in : 0, p.vec_bc);
      pb += ROWS * (c_half ? p.ldc : p.ldb);
    } else {
#pragma unroll
      for (int i = 0; i < IT_BC / 2; ++i) {
        const int r = br + i * (SCAN_THREADS / LPC), in = r < n ? bc_in : 0;
        rb[i].load(pb + i * (SCAN_THREADS / LPC) * p.ldb, in, p.vec_bc);
        if (MODE != SCAN_ENDS) rb[i + IT_BC / 2].load(pc + i * (SCAN_THREADS / LPC) * p.ldc, in, p.vec_bc);
      }
      pb += ROWS * p.ldb;
      pc += ROWS * p.ldc;
    }
  };

  // Rows t, ... of the tile. Their operands are read first, and their sums over the LPC lanes are made together: while a lane has several
  // (rows x channels), halves of them change sides, then whole sums are added.
  auto walk = [&](int t, auto rows_c) {
    constexpr int ROWS_NOW = decltype(rows_c)::value, VALUES = ROWS_NOW * K;
    float d[ROWS_NOW][K], x[ROWS_NOW][K], y[VALUES];
    f32x2 b[ROWS_NOW][2], c[ROWS_NOW][2];
#pragma unroll
    for (int r = 0; r < ROWS_NOW; ++r) {
      read_floats<K>(&sm.d[t + r][cl], d[r]);
      read_floats<K>(&sm.x[t + r][cl], x[r]);
      const ulonglong2 b2 = *reinterpret_cast<const ulonglong2*>(&sm.b[0][t + r][n0]);
      b[r][0] = b2.x; b[r][1] = b2.y;
      if (MODE != SCAN_ENDS) {
        const ulonglong2 c2 = *reinterpret_cast<const ulonglong2*>(&sm.b[1][t + r][n0]);
        c[r][0] = c2.x; c[r][1] = c2.y;
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS_NOW; ++r)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float dx = d[r][k] * x[r][k];
        const f32x2 d2 = pack2(d[r][k], d[r][k]), dx2 = pack2(dx, dx);
        f32x2 sum = 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          float lo, hi;
          unpack2(mul2(d2, A[k][s]), lo, hi);
          h[k][s] = fma2(pack2(ex2(lo), ex2(hi)), h[k][s], mul2(dx2, b[r][s]));
          if (MODE != SCAN_ENDS) sum = s ? fma2(c[r][s], h[k][s], sum) : mul2(c[r][s], h[k][s]);
        }
        if (MODE == SCAN_ENDS) sum_d[k] += d[r][k];
        float lo, hi;
        unpack2(sum, lo, hi);
        y[r * K + k] = lo + hi;
      }
    if (MODE != SCAN_ENDS) {
      int have = VALUES, first = 0;                      // values first .. first + have of the rows' K channels each
#pragma unroll
      for (int m = LPC / 2; m > 0; m >>= 1) {
        const bool up = sub & m;
        if (have > 1) {
          have /= 2;
#pragma unroll
          for (int k = 0; k < VALUES / 2; ++k)
            if (k < have) {
              const float give = up ? y[k] : y[k + have], keep = up ? y[k + have] : y[k];
              y[k] = keep + __shfl_xor_sync(0xffffffffu, give, m);
            }
          first += up ? have : 0;
        } else {
          y[0] += __shfl_xor_sync(0xffffffffu, y[0], m);
        }
      }
      constexpr int LEFT = VALUES > LPC ? VALUES / LPC : 1, SHARE = LPC > VALUES ? LPC / VALUES : 1;   // values that a lane, or SHARE of them, end with
      if (sub % SHARE == 0)
#pragma unroll
        for (int k = 0; k < LEFT; ++k) sm.y[t + (first + k) / K][cl + (first + k) % K] = y[k];
    }
  };

  if (row < row_end) bring(row_end - row);
  for (; row < row_end; row += ROWS) {
    const int n = (int)min((int64_t)ROWS, row_end - row);
    float bias[V];
    read_floats<V>(&sm.bias[vc], bias);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float x[V], d[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[v] = rx[i].get(v);
        d[v] = rd[i].get(v) + bias[v];
      }
      if (p.softplus) {
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] = softplus(d[v]);
      }
      write_floats<V>(&sm.x[vr + i * RPI][vc], x);
      write_floats<V>(&sm.d[vr + i * RPI][vc], d);
    }
    if constexpr (BC <= SCAN_THREADS) {
      if (tid < BC) write_floats<SPL>(&sm.b[c_half][br][n0], rb[0].all().v);
    } else {
#pragma unroll
      for (int i = 0; i < IT_BC / 2; ++i) {
        write_floats<SPL>(&sm.b[0][br + i * (SCAN_THREADS / LPC)][n0], rb[i].all().v);
        if (MODE != SCAN_ENDS) write_floats<SPL>(&sm.b[1][br + i * (SCAN_THREADS / LPC)][n0], rb[i + IT_BC / 2].all().v);
      }
    }
    __syncthreads();
    if (row + ROWS < row_end) bring(row_end - row - ROWS);
    if (MODE != SCAN_ENDS && p.z) {
      if (whole_ch && n == ROWS) {
#pragma unroll
        for (int i = 0; i < IT; ++i) rz[i].load_piece(pz + i * RPI * p.ldz);
      } else {
#pragma unroll
        for (int i = 0; i < IT; ++i) rz[i].load(pz + i * RPI * p.ldz, vr + i * RPI < n ? ch_in : 0, p.vec);
      }
      pz += ROWS * p.ldz;
    }
    int t = 0;
    for (; t + R <= n; t += R) walk(t, std::integral_constant<int, R>());
    for (; t < n; ++t) walk(t, std::integral_constant<int, 1>());
    __syncthreads();
    if (MODE != SCAN_ENDS) {
      float skip[V];
      read_floats<V>(&sm.skip[vc], skip);
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        float x[V], y[V];
        read_floats<V>(&sm.x[vr + i * RPI][vc], x);
        read_floats<V>(&sm.y[vr + i * RPI][vc], y);
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = fmaf(skip[v], x[v], y[v]);
        if (p.z) {
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] *= silu(rz[i].get(v));
        }
        Raw<T, V> out;
        out.put_all(y);
        if (whole_ch && n == ROWS) out.store_piece(py + i * RPI * p.ldy);
        else out.store(py + i * RPI * p.ldy, vr + i * RPI < n ? ch_in : 0, p.vec);
      }
      py += ROWS * p.ldy;
    }
  }
  if (MODE == SCAN_ENDS) {
    leave(p.end, unit);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (sub == 0 && c_lo + cl + k < c_hi) p.steps[(int64_t)unit * p.D + c_lo + cl + k] = sum_d[k];
  } else if (last) {
    leave(p.h_out, slot);
  }
}

// The lists with long ones first, by classes of length (a quarter of a power of two each): the blocks of a launch start in this order, and a
// long list that starts last keeps a few SMs busy while the others have nothing left. Within a class the order is any; results do
// not depend on it.
__global__ void __launch_bounds__(1024) ssm_order_kernel(const ScanParams p) {
  pdl_begin();
  constexpr int CLASSES = 33 * 4;
  __shared__ int s_at[CLASSES];
  const int tid = threadIdx.x;
  auto class_of = [&](int i) {
    const int64_t n = p.lists.begin(i + 1) - p.lists.begin(i);
    const unsigned len = n > 0 ? (unsigned)n : 0u;
    const int zeros = __clz(len);
    return len ? zeros * 4 + 3 - (int)(((len << zeros) >> 29) & 3u) : CLASSES - 1;
  };
  for (int c = tid; c < CLASSES; c += 1024) s_at[c] = 0;
  __syncthreads();
  for (int i = tid; i < p.lists.batch; i += 1024) atomicAdd(&s_at[class_of(i)], 1);
  __syncthreads();
  if (tid == 0) {
    int sum = 0;
    for (int c = 0; c < CLASSES; ++c) {
      const int n = s_at[c];
      s_at[c] = sum;
      sum += n;
    }
  }
  __syncthreads();
  for (int i = tid; i < p.lists.batch; i += 1024) p.order[atomicAdd(&s_at[class_of(i)], 1)] = i;
}

// 2^q as two factors: the rows of a chunk each have a decay that fp32 holds where the chunk's need not. Exponents from -252 to 254 leave of any
// state that is not 0 less than 2^-124, or more than fp32 holds. (Where q is infinite or a NaN the chunk's own end is.)
struct Decay {
  float f[2];
  __device__ __forceinline__ void of(float q) {
    auto part = [](float v) { return fminf(fmaxf(v, -126.f), 127.f); };
    const float q0 = part(q);
    f[0] = ex2(q0);
    f[1] = ex2(part(q - q0));
  }
  __device__ __forceinline__ float apply(float e, float own) const { return fmaf(f[0], f[1] * e, own); }
};

// What the ends are with the states that come into their chunks: end[j] += exp(A steps[j]) end[j - 1] where chunk j is not its list's first. A
// block has 32 (channel, state) pairs and splits the chunks among its 32 warps: each makes its own part's decay and sum, takes what
// comes in from the parts before it, and walks its part again. Bound by the latency of its reads: none waits for another (what stands in
// the place of a chunk that is none is dropped). [30011, 202], N = 10, 156 chunks: the call 145 us with 8 warps that asked first what
// a chunk is, 129 now.
constexpr int CARRY_PARTS = 32;
__global__ void __launch_bounds__(32 * CARRY_PARTS, 2) ssm_carry_kernel(const ScanParams p) {
  pdl_begin();
  __shared__ float s_f[2][CARRY_PARTS][32], s_e[CARRY_PARTS][32];
  __shared__ bool s_cut[CARRY_PARTS];                   // a list begins in the part
  const int part = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t pairs = (int64_t)p.D * p.N, at = (int64_t)blockIdx.x * 32 + lane;
  const bool mine = at < pairs;
  const int c = mine ? (int)(at / p.N) : 0;
  const float A = mine ? LOG2E * p.A[at] : 0.f;
  const int n = p.n_ends, share = (n + CARRY_PARTS - 1) / CARRY_PARTS, j0 = min(n, part * share), j1 = min(n, j0 + share);
  float Q = 0.f, e = 0.f;                                // the part: e <- 2^Q e + its own e
  // (a chunk that is its list's first, or none, cuts off what came before it: a product with 0 would keep another list's NaN. A decay that is
  // 0 is none of this: what came in may be a NaN, which stays to its list's end.)
  auto one = [&](int j, float& q, float& own) {
    const int kind = p.kind[j];
    const float end = mine ? p.end[j * pairs + at] : 0.f;
    q = A * p.steps[(int64_t)j * p.D + c];
    own = kind ? end : 0.f;
    return kind == 2;
  };
  bool cut = false;
#pragma unroll 8
  for (int j = j0; j < j1; ++j) {
    float q, own;
    const bool on = one(j, q, own);
    Decay d;
    d.of(q);
    e = on ? d.apply(e, own) : own;
    cut |= !on;
    Q += q;
  }
  if (lane == 0) s_cut[part] = cut;
  Decay all;
  all.of(Q);
  s_f[0][part][lane] = all.f[0];
  s_f[1][part][lane] = all.f[1];
  s_e[part][lane] = e;
  __syncthreads();
  if (j0 == j1) return;
  e = 0.f;
#pragma unroll 8
  for (int k = 0; k < part; ++k) {
    const Decay d = {{s_f[0][k][lane], s_f[1][k][lane]}};
    const float own = s_e[k][lane];
    e = s_cut[k] ? own : d.apply(e, own);
  }
#pragma unroll 8
  for (int j = j0; j < j1; ++j) {
    float q, own;
    const bool on = one(j, q, own);
    Decay d;
    d.of(q);
    e = on ? d.apply(e, own) : own;
    if (mine) p.end[j * pairs + at] = e;
  }
}

template <typename T, int LPC, int K>
int launch_tiles(const ScanParams& p, const ScanPlan& plan, cudaStream_t s) {
  constexpr int ch = ScanShape<LPC, K>::CH;
  const int a_group = (p.per_group + ch - 1) / ch, blocks = a_group * p.groups;
  const int64_t units = p.lists.batch + (int64_t)p.n_ends;
  XB_REQUIRE(units * blocks < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_ssm_scan: too many lists and channels");
  if (p.order) {
    launch_dependent(ssm_order_kernel, 1, 1024, 0, s, p);
    if (int rc = check_launch("ssm_order_kernel")) return rc;
  }
  if (p.chunk > 0) {
    launch_dependent(ssm_scan_kernel<T, LPC, K, SCAN_ENDS>, (unsigned)((int64_t)p.n_ends * blocks), SCAN_THREADS, 0, s, p, a_group);
    if (int rc = check_launch("ssm_scan_kernel")) return rc;
    launch_dependent(ssm_carry_kernel, (unsigned)(((int64_t)p.D * p.N + 31) / 32), 32 * CARRY_PARTS, 0, s, p);
    if (int rc = check_launch("ssm_carry_kernel")) return rc;
  }
  launch_dependent(ssm_scan_kernel<T, LPC, K, SCAN_WALK>, (unsigned)(units * blocks), SCAN_THREADS, 0, s, p, a_group);
  return check_launch("ssm_scan_kernel");
}
template <typename T, int LPC>
int launch_lanes(const ScanParams& p, const ScanPlan& plan, cudaStream_t s) {
  if (plan.step) {
    const int ch = SCAN_THREADS / LPC * STEP_U, blocks = (p.D + ch - 1) / ch;
    XB_REQUIRE((int64_t)blocks * p.lists.batch < ((int64_t)1 << 31), XB_ERR_LIMIT, "xb_ssm_scan: too many lists and channels");
    launch_dependent(ssm_step_kernel<T, LPC>, (unsigned)((int64_t)blocks * p.lists.batch), SCAN_THREADS, 0, s, p, blocks);
    return check_launch("ssm_step_kernel");
  }
  if constexpr (LPC <= 4) {
    if (plan.K == 1) return launch_tiles<T, LPC, 1>(p, plan, s);
  }
  return launch_tiles<T, LPC, 2>(p, plan, s);
}
template <typename T>
int launch_scan(const ScanParams& p, const ScanPlan& plan, cudaStream_t s) {
  switch (plan.lanes) {
    case 1: return launch_lanes<T, 1>(p, plan, s);
    case 2: return launch_lanes<T, 2>(p, plan, s);
    case 4: return launch_lanes<T, 4>(p, plan, s);
    case 8: return launch_lanes<T, 8>(p, plan, s);
    default: return launch_lanes<T, 16>(p, plan, s);
  }
}
}  // namespace
}  // namespace xb
