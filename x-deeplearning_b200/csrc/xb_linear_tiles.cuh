// Linear attention of 16-bit lists by chunks of 64 rows, on warp-level matrix instructions (formulas in xdlb200.h).
//
// With S ahead of a chunk, t and s rows of it (from 0) and g the decay:
//   y_t = scale (g^(t+1) q_t S + sum_{s <= t} g^(t-s) (q_t k_s) v_s),   S' = g^n S + sum_s g^(n-1-s) k_s v_s^T
// A block has a list (or segment) and a head; a warp 16 columns of dv. S^T stays in the accumulators of the matrix instructions that make it, whose
// pairs along dk are the pairs that the other operand of q S is made of: S moves between no lanes. The scores of a chunk are shared by its warps and go
// through shared memory.
//
// Rounding. S is fp32, and what it is made of is known to fp32's last bits: k as it is, g^.. v as three bf16 terms (24 bits) or two fp16 terms (22).
// For y, scores and S are two bf16 terms (2^-17 of each) or one of fp16 (2^-11, as a result's own rounding). What becomes fp16 is first multiplied by
// powers of two that put the largest values at 2^14: nothing is beyond fp16's numbers, and what is below them is off by 2^-39 of the largest at most.
// S and v have one such power for each column of dv, scores for each row of a block, so that no result is off by the size of another.
#pragma once

#include "xb_linear.cuh"
#include "xb_umma.cuh"

namespace xb {
namespace {

constexpr int LT_ROWS = 64;

template <bool BF16>
__device__ __forceinline__ void mma_add(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the two halves of a word as fp32
template <bool BF16>
__device__ __forceinline__ float2 widen(uint32_t h) {
  if constexpr (BF16) return make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
template <bool BF16>
__device__ __forceinline__ uint32_t narrow(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Rows of D elements in shared memory, their pieces of 16 bytes swapped by the row: what eight rows hold of one column of pieces lies in all banks
template <int D>
__device__ __forceinline__ uint32_t tile_at(int row, int piece) { return (uint32_t)(row * D * 2 + ((piece ^ (row & 7)) << 4)); }

// the power of two that puts `top`, the largest of some sizes, at 2^14 (and one over it)
__device__ __forceinline__ void fp16_scale(float top, float& up, float& down) {
  // (0: as it is; small numbers of fp32: the end of what has a reciprocal. Any finite exponent above has one.)
  const int e = top > 0.f ? max((int)(__float_as_uint(top) >> 23) - 127, -100) : 14;
  up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
  down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
}
// the largest of the four lanes that share a row of an accumulator, several at once: their shuffles wait beside one another
template <int N>
__device__ __forceinline__ void quad_tops(float (&v)[N]) {
#pragma unroll
  for (int o = 2; o > 0; o >>= 1)
#pragma unroll
    for (int z = 0; z < N; ++z) v[z] = fmaxf(v[z], __shfl_xor_sync(0xffffffffu, v[z], o));
}

// The largest sizes in an accumulator's rows g8 and g8 + 8, told by `each`, which calls its argument with every value of a lane and which of the two rows
// it is of. Infinities have no say in it: they are what they are at any scale, and the finite values beside them keep theirs.
template <typename F>
__device__ __forceinline__ void tops_of(F each, float (&top)[2]) {
  top[0] = top[1] = 0.f;
  each([&](int row, float v) { top[row] = fmaxf(top[row], fabsf(v)); });
  quad_tops(top);
  if (__any_sync(0xffffffffu, fmaxf(top[0], top[1]) == INFINITY)) {
    top[0] = top[1] = 0.f;
    each([&](int row, float v) { top[row] = fabsf(v) < INFINITY ? fmaxf(top[row], fabsf(v)) : top[row]; });
    quad_tops(top);
  }
}

template <bool BF16, int DK, int DV>
struct LinearTiles {
  static constexpr int WARPS = DV / 16, THREADS = WARPS * 32;
  // Bytes: queries, keys, values. With an SM's registers in one block or two nobody else hides the wait for keys and values: there the next chunk's are
  // on their way while this one is worked on. us with one buffer and with two: one list of 30011
  // rows, 8 heads of 128 on 4, fp16 276 and 249; heads of 64, bf16 (four blocks) 1024 lists of 64 rows, 8 heads 163 and 177, 256 ragged lists of 273 on
  // average 218 and 211.
  static constexpr int BUFFERS = DK == 128 || DV == 128 ? 2 : 1;
  static constexpr int Q = LT_ROWS * DK * 2, V = LT_ROWS * DV * 2, KV = Q + V, BUFFER = Q + BUFFERS * KV;
  static constexpr int SCORES = 10 * 512, TERMS_Y = BF16 ? 2 : 1, TERMS_S = BF16 ? 3 : 2;      // (blocks of 16 x 16 on and below the diagonal)
  static constexpr int SMEM = BUFFER + TERMS_Y * SCORES + (LT_ROWS + 4) * 4 + (BF16 ? 0 : 10 * 16 * 4);
  // Blocks of an SM, as registers and shared memory have it: what hides a block's waits is the others.
  static constexpr int BLOCKS = DV == 128 ? (DK == 128 ? 1 : 2) : DK == 128 ? 2 : 4;
};
// a row's piece (of two) of a block of scores: what eight rows hold of one lies in all banks
__device__ __forceinline__ uint32_t score_at(int block, int row, int piece) { return (uint32_t)(block * 512 + row * 32 + ((piece ^ (row >> 2 & 1)) << 4)); }

template <bool BF16, int DK, int DV>
__global__ void __launch_bounds__(LinearTiles<BF16, DK, DV>::THREADS, LinearTiles<BF16, DK, DV>::BLOCKS) linear_tiles_kernel(const LinearParams p) {
  using L = LinearTiles<BF16, DK, DV>;
  pdl_wait();
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* s_scores = smem + L::BUFFER;                                       // [terms][10][16][16]
  float* s_power = reinterpret_cast<float*>(s_scores + L::TERMS_Y * L::SCORES);      // decay over 0 to 64 rows
  float* s_down = s_power + LT_ROWS + 4;                                      // fp16: what the scores of a block's 16 rows are to be multiplied by, ten blocks
  __shared__ Segment s_seg;
  __shared__ int s_there;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = (int)(blockIdx.x % (unsigned)p.H), hkv = h / p.share;
  const int g8 = lane >> 2, t4 = lane & 3;                                     // an accumulator's row and pair of columns
  if (threadIdx.x < 32) {
    Segment g;
    const bool there = find_segment(p, (int)(blockIdx.x / (unsigned)p.H), lane, g);
    if (lane == 0) {
      s_seg = g;
      s_there = there;
    }
  }
  const float log_decay = log_decay_of(p, h);
  for (int i = threadIdx.x; i <= LT_ROWS; i += L::THREADS) s_power[i] = decay_over(log_decay, i);
  if (p.dk != DK || p.dv != DV)            // what lies behind dk and dv stays zero
    for (int i = threadIdx.x; i < L::BUFFER / 16; i += L::THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  if (!s_there) return;
  const Segment g = s_seg;
  const uint32_t base = umma::smem_u32(smem), scores_at = umma::smem_u32(s_scores);

  // Rows [r0, r0 + 64) of the segment into a buffer; those behind its end as zeros. Pieces of 16 bytes where rows lie on them, a thread one column of
  // pieces; else of what they do lie on.
  auto load = [&](const Heads& from, int head, int width, int unit, uint32_t at, auto d, int64_t r0) {
    constexpr int D = decltype(d)::value, PIECES = D / 8, STEP = L::THREADS / PIECES;
    const int rows = (int)min((int64_t)LT_ROWS, g.end - r0);
    if (unit == 16) {
      const int piece = threadIdx.x % PIECES, first = threadIdx.x / PIECES, bytes = min(max(width * 2 - piece * 16, 0), 16);
      if (bytes == 0) return;
      const char* f = reinterpret_cast<const char*>(from.get<uint16_t>(r0 + first, head)) + piece * 16;
      const int64_t step = from.row * 2 * STEP;
      const uint32_t to = base + at + first * D * 2;
#pragma unroll
      for (int i = 0; i < LT_ROWS / STEP; ++i, f += step) {
        const int r = first + i * STEP;
        const bool in = r < rows;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + i * STEP * D * 2 + ((piece ^ (r & 7)) << 4)), "l"(in ? f : reinterpret_cast<const char*>(from.at)),
                     "r"(in ? bytes : 0)
                     : "memory");
      }
      return;
    }
    const int parts = (width * 2 + unit - 1) / unit;
    const char* src = reinterpret_cast<const char*>(from.get<uint16_t>(r0, head));
    for (int e = threadIdx.x; e < LT_ROWS * parts; e += L::THREADS) {
      const int r = e / parts, b = (e - r * parts) * unit;
      const uint32_t to = base + at + r * D * 2 + (((b >> 4) ^ (r & 7)) << 4) + (b & 15);
      const char* f = src + (r < rows ? (int64_t)r * from.row * 2 + b : 0);
      const int bytes = r < rows ? min(unit, width * 2 - b) : 0;
      if (unit == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(f), "r"(bytes) : "memory");
      else if (unit == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(f), "r"(bytes) : "memory");
      else asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(bytes ? *reinterpret_cast<const uint16_t*>(f) : (uint16_t)0) : "memory");
    }
  };
  // (a group of their own: with two buffers of keys and values nothing is asked for behind the queries that would take them in)
  auto load_q = [&](int64_t r0) {
    if (p.ends_only) return;
    load(p.q, h, p.dk, p.unit_q, 0, std::integral_constant<int, DK>(), r0);
    umma::cp_async_commit();
  };
  auto load_kv = [&](int64_t r0, uint32_t buffer) {
    load(p.k, hkv, p.dk, p.unit_k, L::Q + buffer, std::integral_constant<int, DK>(), r0);
    load(p.v, hkv, p.dv, p.unit_v, 2 * L::Q + buffer, std::integral_constant<int, DV>(), r0);
    umma::cp_async_commit();
  };
  load_q(g.begin);
  load_kv(g.begin, 0);

  // S^T: rows 16 warp + g8 (and + 8) of dv, columns 8 j + 2 t4 (and + 1) of dk
  float S[DK / 8][4];
  const float* from = state_from(p, g, h);
  const int c0 = warp * 16 + g8;
#pragma unroll
  for (int j = 0; j < DK / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = 8 * j + 2 * t4 + (e & 1), c = c0 + (e >> 1) * 8;
      S[j][e] = from && k < p.dk && c < p.dv ? from[k * p.dv + c] : 0.f;
    }
  auto put_state = [&](float* to) {
#pragma unroll
    for (int j = 0; j < DK / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = 8 * j + 2 * t4 + (e & 1), c = c0 + (e >> 1) * 8;
        if (k < p.dk && c < p.dv) to[k * p.dv + c] = S[j][e];
      }
  };
  if (from && p.ends_only) put_state(p.first + (g.at * p.H + h) * (int64_t)p.dk * p.dv);

  // Decays of a block of scores: on the diagonal over t - s rows; below it over the rest of s's block, whole blocks between, and t's rows of its own,
  // each of them at most 1 whatever the decay.
  const float row_f[2] = {s_power[g8], s_power[g8 + 8]};
  float col_f[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int b = 0; b < 2; ++b) col_f[x][b] = s_power[16 - 8 * x - 2 * t4 - b];
  const float last_f[2] = {s_power[7 - 2 * t4], s_power[6 - 2 * t4]};
  const bool vec_y = p.vec_y;
  const uint32_t sq = base;
  uint32_t buffer = 0;                     // bytes to this chunk's keys and values
  for (int64_t r0 = g.begin; r0 < g.end; r0 += LT_ROWS) {
    const uint32_t sk = sq + L::Q + buffer, sv = sk + L::Q;
    const int n = (int)min((int64_t)LT_ROWS, g.end - r0);
    umma::cp_async_wait_all();
    __syncthreads();
    if (L::BUFFERS > 1) {                  // (all have done with the chunk before, whose buffer this is)
      buffer = L::KV - buffer;
      if (r0 + LT_ROWS < g.end) load_kv(r0 + LT_ROWS, buffer);
    }
    if (!p.ends_only) {
      // scores, times the decay: ten blocks of 16 x 16 on and below the diagonal, those of a warp side by side
      const int row_blocks = (n + 15) / 16, blocks = row_blocks * (row_blocks + 1) / 2;
      auto scores = [&](auto count) {
        constexpr int N = decltype(count)::value;
        float c[N][2][4];
        uint32_t at_q[N], at_k[N];
        int back[N];                       // blocks between
#pragma unroll
        for (int z = 0; z < N; ++z) {
          const int b = warp + z * L::WARPS, i = b < 1 ? 0 : b < 3 ? 1 : b < 6 ? 2 : 3, j = b - i * (i + 1) / 2;
          at_q[z] = sq + 16 * i * DK * 2;
          at_k[z] = sk + 16 * j * DK * 2;
          back[z] = i - j;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[z][x][e] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          const uint32_t at = tile_at<DK>(lane & 15, 2 * k + (lane >> 4));
          uint32_t a[N][4], bk[N][4];
#pragma unroll
          for (int z = 0; z < N; ++z) {
            ldmatrix4<0>(a[z], at_q[z] + at);
            ldmatrix4<0>(bk[z], at_k[z] + at);
          }
#pragma unroll
          for (int z = 0; z < N; ++z) {
            mma_add<BF16>(c[z][0], a[z], bk[z][0], bk[z][2]);
            mma_add<BF16>(c[z][1], a[z], bk[z][1], bk[z][3]);
          }
        }
        [[maybe_unused]] float tops[2 * N];
#pragma unroll
        for (int z = 0; z < N; ++z) {
          if (back[z] == 0) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int rows = g8 + (e >> 1) * 8 - 8 * x - 2 * t4 - (e & 1);
                c[z][x][e] = rows >= 0 ? c[z][x][e] * s_power[max(rows, 0)] : 0.f;
              }
          } else {
            const float far = s_power[16 * (back[z] - 1)];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) c[z][x][e] *= row_f[e >> 1] * far * col_f[x][e & 1];
          }
          if constexpr (!BF16) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
              tops[2 * z + r] = fmaxf(fmaxf(fabsf(c[z][0][2 * r]), fabsf(c[z][0][2 * r + 1])), fmaxf(fabsf(c[z][1][2 * r]), fabsf(c[z][1][2 * r + 1])));
          }
        }
        if constexpr (!BF16) quad_tops(tops);
#pragma unroll
        for (int z = 0; z < N; ++z) {
          const int b = warp + z * L::WARPS;
          if constexpr (!BF16) {
            auto each = [&](auto take) {
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) take(e >> 1, c[z][x][e]);
            };
            float top[2] = {tops[2 * z], tops[2 * z + 1]};
            if (__any_sync(0xffffffffu, fmaxf(top[0], top[1]) == INFINITY)) tops_of(each, top);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float up, down;
              fp16_scale(top[r], up, down);
              if (t4 == 0) s_down[b * 16 + g8 + 8 * r] = down;
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                c[z][x][2 * r] *= up;
                c[z][x][2 * r + 1] *= up;
              }
            }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const uint32_t at = score_at(b, g8 + (e >> 1) * 8, x) + 4 * t4;
              const uint32_t hi = narrow<BF16>(c[z][x][e], c[z][x][e + 1]);
              *reinterpret_cast<uint32_t*>(s_scores + at) = hi;
              if constexpr (BF16) {
                const float2 taken = widen<BF16>(hi);
                *reinterpret_cast<uint32_t*>(s_scores + L::SCORES + at) = narrow<BF16>(c[z][x][e] - taken.x, c[z][x][e + 1] - taken.y);
              }
            }
        }
      };
      const int mine = warp < blocks ? (blocks - warp + L::WARPS - 1) / L::WARPS : 0;
      if constexpr (L::WARPS < 5) {
        if (mine == 3) scores(std::integral_constant<int, 3>());
      }
      if (mine == 2) scores(std::integral_constant<int, 2>());
      if (mine == 1) scores(std::integral_constant<int, 1>());
    }
    // the warp's columns of V, for both products: rows 16 i + .., pairs along the rows
    uint32_t v[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ldmatrix4<1>(v[i], sv + tile_at<DV>(16 * i + (lane & 15), 2 * warp + (lane >> 4)));
    if (!p.ends_only) {
      // (a zero score takes no part beside infinities and NaN of rows behind its own: where there are any, blocks on the diagonal go by sums)
      uint32_t sick = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sick = fma_zero<BF16>(v[i][e], sick);
      const bool bad = __any_sync(0xffffffffu, half_is_bad<BF16>(sick) || half_is_bad<BF16>(sick >> 16));
      float o[4][2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][x][e] = 0.f;
      [[maybe_unused]] float up[2], down[2][2];              // (of columns g8 and g8 + 8; of an accumulator's columns)
      if constexpr (!BF16) {
        float top[2], of_column[2];
        tops_of(
            [&](auto take) {
#pragma unroll
              for (int j = 0; j < DK / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) take(e >> 1, S[j][e]);
            },
            top);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          fp16_scale(top[x], up[x], of_column[x]);
#pragma unroll
          for (int b = 0; b < 2; ++b) down[x][b] = __shfl_sync(0xffffffffu, of_column[x], (2 * t4 + b) * 4);
        }
      }
#pragma unroll
      for (int k = 0; k < DK / 16; ++k) {
        uint32_t hi[4], lo[4];                                                 // columns g8 (rows 2 t4.., + 8), columns g8 + 8
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float(&s)[4] = S[2 * k + (w & 1)];
          float a = s[w & 2], b = s[(w & 2) + 1];
          if constexpr (!BF16) { a *= up[w >> 1]; b *= up[w >> 1]; }
          hi[w] = narrow<BF16>(a, b);
          if constexpr (BF16) {
            const float2 taken = widen<BF16>(hi[w]);
            lo[w] = narrow<BF16>(a - taken.x, b - taken.y);
          }
        }
        // (two blocks of rows at a time: those behind the end are zeros)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          if (16 * i >= n) break;
          uint32_t a[2][4];
#pragma unroll
          for (int z = 0; z < 2; ++z) ldmatrix4<0>(a[z], sq + tile_at<DK>(16 * (i + z) + (lane & 15), 2 * k + (lane >> 4)));
          if constexpr (BF16) {
#pragma unroll
            for (int z = 0; z < 4; ++z) mma_add<BF16>(o[i + z / 2][z % 2], a[z / 2], lo[z % 2 * 2], lo[z % 2 * 2 + 1]);
          }
#pragma unroll
          for (int z = 0; z < 4; ++z) mma_add<BF16>(o[i + z / 2][z % 2], a[z / 2], hi[z % 2 * 2], hi[z % 2 * 2 + 1]);
        }
      }
      __syncthreads();
      if (r0 + LT_ROWS < g.end) load_q(r0 + LT_ROWS);                          // (all have read these)
      uint16_t* y = const_cast<uint16_t*>(p.y.get<uint16_t>(r0 + g8, h)) + warp * 16 + 2 * t4;
      const int64_t step_y = p.y.row * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f0 = s_power[16 * i + g8 + 1], f1 = s_power[16 * i + g8 + 9];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if constexpr (!BF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][x][e] *= down[x][e & 1];
          }
          o[i][x][0] *= f0; o[i][x][1] *= f0; o[i][x][2] *= f1; o[i][x][3] *= f1;
        }
      }
      // a column of blocks of scores at a time: their products wait for one another only where they are of the same rows
      auto column = [&](auto place) {
        constexpr int j = decltype(place)::value;
        if (bad) {
          const int block = j * (j + 1) / 2 + j;
#pragma unroll 1
          for (int s = 0; s < 16; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int row = g8 + (e >> 1 & 1) * 8, c = warp * 16 + (e >> 2) * 8 + 2 * t4 + (e & 1);
              const uint32_t at = score_at(block, row, s >> 3) + (s & 7) * 2;
              float w = widen<BF16>(*reinterpret_cast<const uint16_t*>(s_scores + at)).x;
              if constexpr (BF16) w += widen<BF16>(*reinterpret_cast<const uint16_t*>(s_scores + L::SCORES + at)).x;
              const uint16_t u = *reinterpret_cast<const uint16_t*>(smem + (sv - base) + tile_at<DV>(16 * j + s, c >> 3) + (c & 7) * 2);
              if (s <= row) o[j][e >> 2][e & 3] = fmaf(BF16 ? w : w * s_down[block * 16 + row], widen<BF16>(u).x, o[j][e >> 2][e & 3]);
            }
          __syncwarp();
        }
        auto products = [&](auto from) {
          constexpr int I = decltype(from)::value;
          if constexpr (I < 4) {
            uint32_t a[4 - I][4];
            [[maybe_unused]] uint32_t b[4 - I][4];
#pragma unroll
            for (int i = I; i < 4; ++i) {
              const uint32_t at = score_at(i * (i + 1) / 2 + j, lane & 15, lane >> 4);
              ldmatrix4<0>(a[i - I], scores_at + at);
              if constexpr (BF16) ldmatrix4<0>(b[i - I], scores_at + L::SCORES + at);
            }
            if constexpr (BF16) {
#pragma unroll
              for (int i = I; i < 4; ++i) {
                mma_add<BF16>(o[i][0], b[i - I], v[j][0], v[j][1]);
                mma_add<BF16>(o[i][1], b[i - I], v[j][2], v[j][3]);
              }
#pragma unroll
              for (int i = I; i < 4; ++i) {
                mma_add<BF16>(o[i][0], a[i - I], v[j][0], v[j][1]);
                mma_add<BF16>(o[i][1], a[i - I], v[j][2], v[j][3]);
              }
            } else {
              float c[4 - I][2][4];
#pragma unroll
              for (int i = I; i < 4; ++i) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                  for (int e = 0; e < 4; ++e) c[i - I][x][e] = 0.f;
                mma_add<BF16>(c[i - I][0], a[i - I], v[j][0], v[j][1]);
                mma_add<BF16>(c[i - I][1], a[i - I], v[j][2], v[j][3]);
              }
#pragma unroll
              for (int i = I; i < 4; ++i) {
                const float* f = s_down + (i * (i + 1) / 2 + j) * 16 + g8;
                const float of_row[2] = {f[0], f[8]};
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[i][x][e] = fmaf(c[i - I][x][e], of_row[e >> 1], o[i][x][e]);
              }
            }
          }
        };
        if (bad) products(std::integral_constant<int, j + 1>());
        else products(place);
      };
      column(std::integral_constant<int, 0>());
      if (n > 16) column(std::integral_constant<int, 1>());
      if (n > 32) column(std::integral_constant<int, 2>());
      if (n > 48) column(std::integral_constant<int, 3>());
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (16 * i >= n) break;
#pragma unroll
        for (int e = 0; e < 4; e += 2, y += step_y) {
          if (16 * i + g8 + (e >> 1) * 8 >= n) continue;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int c = warp * 16 + 8 * x + 2 * t4;
            const uint32_t two = narrow<BF16>(o[i][x][e] * p.scale, o[i][x][e + 1] * p.scale);
            if (vec_y) {
              if (c < p.dv) *reinterpret_cast<uint32_t*>(y + 8 * x) = two;
            } else {
              if (c < p.dv) y[8 * x] = (uint16_t)two;
              if (c + 1 < p.dv) y[8 * x + 1] = (uint16_t)(two >> 16);
            }
          }
        }
      }
    }
    // S' = g^n S + (g^.. V)^T K
    [[maybe_unused]] float up[2], down[2];                                     // (of columns g8 and g8 + 8)
    if constexpr (!BF16) {
      float top[2];
      tops_of(
          [&](auto take) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x = widen<BF16>(v[i][e]);
                take(e >> 1, x.x);
                take(e >> 1, x.y);
              }
          },
          top);
#pragma unroll
      for (int x = 0; x < 2; ++x) fp16_scale(top[x], up[x], down[x]);
    }
    // decay behind rows 16 i + 8 e + 2 t4 and the next (rows behind the end are zeros)
    float weight[4][2][2];
    if (n == LT_ROWS) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = s_power[LT_ROWS - 8 - 16 * i - 8 * e];
          weight[i][e][0] = f * last_f[0];
          weight[i][e][1] = f * last_f[1];
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) weight[i][e >> 1][e & 1] = s_power[max(n - 1 - 16 * i - (e >> 1) * 8 - 2 * t4 - (e & 1), 0)];
    }
    uint32_t term[L::TERMS_S][4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // (a word is two rows of one column: 16 i + 2 t4, eight further for odd words)
        float2 x = widen<BF16>(v[i][e]);
        if constexpr (!BF16) { x.x *= up[e >> 1]; x.y *= up[e >> 1]; }
        float a = x.x * weight[i][e & 1][0], b = x.y * weight[i][e & 1][1];
        // an operand's words: dv g8, rows first half; dv g8 + 8; dv g8, second half; dv g8 + 8
        const int w = (e & 1) * 2 + (e >> 1);
#pragma unroll
        for (int k = 0; k < L::TERMS_S; ++k) {
          term[k][i][w] = narrow<BF16>(a, b);
          if (k + 1 < L::TERMS_S) {
            const float2 taken = widen<BF16>(term[k][i][w]);
            a -= taken.x;
            b -= taken.y;
          }
        }
      }
    const Decay decay((float)n * log_decay);
    const float keep = decay.slow ? 1.f : 0.f;
#pragma unroll
    for (int j = 0; j < DK / 16; ++j) {
      float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      uint32_t k[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ldmatrix4<1>(k[i], sk + tile_at<DK>(16 * i + (lane & 15), 2 * j + (lane >> 4)));
      // (the small terms first: what is cut off goes by the sum's size)
#pragma unroll
      for (int x = L::TERMS_S - 1; x >= 0; --x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mma_add<BF16>(c[0], term[x][i], k[i][0], k[i][1]);
          mma_add<BF16>(c[1], term[x][i], k[i][2], k[i][3]);
        }
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& s = S[2 * j + x][e];
          s = fmaf(s, decay.by, fmaf(s, keep, BF16 ? c[x][e] : c[x][e] * down[e >> 1]));
        }
    }
    if (L::BUFFERS == 1 && r0 + LT_ROWS < g.end) {
      __syncthreads();
      load_kv(r0 + LT_ROWS, 0);
    }
  }
  float* to = state_to(p, g, h);
  if (to) put_state(to);
}

template <bool BF16, int DK, int DV>
int launch_linear_tile(const LinearParams& p, dim3 grid, cudaStream_t s) {
  using L = LinearTiles<BF16, DK, DV>;
  static PerDeviceOnce once;
  XB_SET_MAX_SMEM_ONCE(once, L::SMEM, (const void*)linear_tiles_kernel<BF16, DK, DV>);
  launch_dependent(linear_tiles_kernel<BF16, DK, DV>, grid, L::THREADS, L::SMEM, s, p);
  return check_launch("linear_tiles_kernel");
}
template <bool BF16>
int launch_linear_tiles(const LinearParams& p, dim3 grid, cudaStream_t s) {
  if (p.dk <= 64) return p.dv <= 64 ? launch_linear_tile<BF16, 64, 64>(p, grid, s) : launch_linear_tile<BF16, 64, 128>(p, grid, s);
  return p.dv <= 64 ? launch_linear_tile<BF16, 128, 64>(p, grid, s) : launch_linear_tile<BF16, 128, 128>(p, grid, s);
}

}  // namespace
}  // namespace xb
