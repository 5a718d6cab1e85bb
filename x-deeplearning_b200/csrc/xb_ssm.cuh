// What the kernels of the state-space layer share: lists and kept states, pieces of rows, the nonlinear functions.
#pragma once

#include <type_traits>

#include "xb_common.cuh"

namespace xb {

// The lists of a call and their kept states (see xdlb200.h). Every offset and slot that a kernel takes from memory goes through
// here and is cut to what exists.
struct Lists {
  const int32_t* offsets;
  const int32_t* slots;
  int64_t rows, per;                      // per: rows a list where there are no offsets
  int batch, n_slots;
  __device__ __forceinline__ int64_t begin(int i) const {              // i = batch: the end of the last
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
    return search(lane, [&](int i) { return begin(i) < r; });
  }
  // the list of chunk number u (of all lists' chunks of `chunk` rows): the last whose first number is u at most
  __device__ __forceinline__ int of_chunk(int u, int64_t chunk, int lane) const {
    const int i = search(lane, [&](int i) { return begin(i) / chunk + i <= u; }) - 1;
    return i < 0 ? 0 : i;
  }
  // how many of the lists `before` holds for, the first ones of them
  template <typename F>
  __device__ __forceinline__ int search(int lane, F before) const {
    int lo = 0, n = batch;                // the answer is in [lo, lo + n]
    while (n > 0) {
      const int step = (n + 31) / 32;
      const unsigned mask = __ballot_sync(0xffffffffu, lane * step < n && before(lo + lane * step));
      if (mask == 0u) return lo;
      const int from = lo + (31 - __clz(mask)) * step + 1;             // behind the last of the places
      n = min(step - 1, lo + n - from);
      lo = from;
    }
    return lo;
  }
};

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
  int D, N, per_group, groups, softplus;
  int vec, vec_bc, vec_h;                 // rows of x, delta, z, y in whole pieces of four; B and C in pieces of four; states and A in float4
  // lists walked in chunks (0: whole): see xb_ssm_scan.cuh
  int64_t chunk;
  int n_ends;                             // rows / chunk
  float* end;                             // [n_ends][D][N]: state at the chunk's end as far as the chunk knows, then with what comes in
  float* first;                           // [n_ends][D][N]: copies of the states that lists of several chunks begin with
  float* steps;                           // [n_ends][D]: sum of the chunk's steps
  int* kind;                              // [n_ends]: 0 no such chunk, 1 its list's first, 2 another
  int* order;                             // [batch]: the lists, long ones first; null: as they come
};

// What a scan runs as.
struct ScanPlan {
  bool step;                              // one row a list
  int lanes, K;                           // lanes of a channel; channels of a lane
  int64_t chunk;                          // lists of more rows are split (0: none)
  bool order;                             // whole lists, long ones first
};
// the scan of one type (xb_ssm_scan_*.cu)
int ssm_scan_f32(const ScanParams& p, const ScanPlan& plan, cudaStream_t s);
int ssm_scan_f16(const ScanParams& p, const ScanPlan& plan, cudaStream_t s);
int ssm_scan_bf16(const ScanParams& p, const ScanPlan& plan, cudaStream_t s);

namespace {

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / v, right to 1 unit in the last place; 0 for numbers of 2^126 and more
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// two fp32 operations an instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float silu(float v) { return v * rcp(1.f + ex2(-LOG2E * v)); }
// two of them. (One reciprocal for both, of the product, has to be kept from overflowing and one's NaN from the other: more instructions than
// the reciprocal saves. 1024 lists of 262144 rows, D = 512, bf16 138 us so with the exponents cut, 135 now.)
__device__ __forceinline__ f32x2 silu2(f32x2 v) {
  float x0, x1;
  unpack2(mul2(v, pack2(-LOG2E, -LOG2E)), x0, x1);
  return mul2(v, pack2(rcp(1.f + ex2(x0)), rcp(1.f + ex2(x1))));
}
// log(1 + exp(v)) = max(v, 0) + log1p(u), u = exp(-|v|), and log1p(u) = 2 atanh(s) with s = u / (2 + u) <= 1/3 by the series of atanh, cut
// after s^13 (the next term is 1.4e-8 of the sum at most): right in relative terms where u is small too, which log(1 + u) is not.
__device__ __forceinline__ float softplus(float v) {
  const float u = ex2(-LOG2E * fabsf(v));
  const float s = u * rcp(2.f + u), t = s * s;
  float p = fmaf(t, 1.f / 13, 1.f / 11);
  p = fmaf(t, p, 1.f / 9);
  p = fmaf(t, p, 1.f / 7);
  p = fmaf(t, p, 1.f / 5);
  p = fmaf(t, p, 1.f / 3);
  p = fmaf(t, p, 1.f);
  return (v > 0.f ? v : 0.f) + 2.f * s * p;
}

// V adjacent elements as they lie in memory
template <typename T, int V>
struct Raw {
  static constexpr int SIZE = sizeof(T), W = (SIZE * V + 3) / 4;
  static constexpr bool PIECE = SIZE * V >= 4;          // (one 2-byte element is never read or written as a word)
  uint32_t w[W];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load_piece(const T* p) {
    if constexpr (W == 4) { const uint4 t = __ldg(reinterpret_cast<const uint4*>(p)); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
    else if constexpr (W == 2) { const uint2 t = __ldg(reinterpret_cast<const uint2*>(p)); w[0] = t.x; w[1] = t.y; }
    else w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
  // the same of memory that this kernel may also write (kept states moved on in place)
  __device__ __forceinline__ void load_kept(const T* p, int in, bool vec) {
    if (PIECE && vec && in >= V) {
      if constexpr (W == 4) { const uint4 t = *reinterpret_cast<const uint4*>(p); w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w; }
      else if constexpr (W == 2) { const uint2 t = *reinterpret_cast<const uint2*>(p); w[0] = t.x; w[1] = t.y; }
      else w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      zero();
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < in) {
          if constexpr (SIZE == 4) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
          else w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
        }
    }
  }
  // `in` of them exist (others are 0); in whole where they do and `vec` says that they lie aligned
  __device__ __forceinline__ void load(const T* p, int in, bool vec) {
    if (PIECE && vec && in >= V) {
      load_piece(p);
    } else {
      zero();
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < in) {
          if constexpr (SIZE == 4) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
          else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + i) << (16 * (i & 1));
        }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (SIZE == 4) return __uint_as_float(w[i]);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i & 1)))));
  }
  struct Floats { float v[V]; };
  __device__ __forceinline__ Floats all() const {
    Floats f;
#pragma unroll
    for (int i = 0; i < V; ++i) f.v[i] = get(i);
    return f;
  }
  __device__ __forceinline__ void put(int i, float v) {
    if constexpr (SIZE == 4) { w[i] = __float_as_uint(v); return; }
    uint32_t b;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) b = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    else b = __half_as_ushort(__float2half_rn(v));
    w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | b << 16 : b;
  }
  // all V, two a conversion
  __device__ __forceinline__ void put_all(const float (&v)[V]) {
    if constexpr (SIZE == 4 || V % 2) {
#pragma unroll
      for (int i = 0; i < V; ++i) put(i, v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&t);
        } else {
          const __half2 t = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&t);
        }
      }
    }
  }
  __device__ __forceinline__ void store_piece(T* p) const {
    if constexpr (W == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (W == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
  __device__ __forceinline__ void store(T* p, int in, bool vec) const {
    if (PIECE && vec && in >= V) {
      store_piece(p);
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

// V adjacent floats of shared memory, V a multiple of four or two of them
template <int V>
__device__ __forceinline__ void read_floats(const float* p, float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 t = reinterpret_cast<const float4*>(p)[i];
      v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
    }
  } else if constexpr (V == 2) {
    const float2 t = *reinterpret_cast<const float2*>(p);
    v[0] = t.x; v[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = p[i];
  }
}
template <int V>
__device__ __forceinline__ void write_floats(float* p, const float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = v[i];
  }
}

constexpr int SPL = 4;                    // states of a lane
constexpr int SCAN_THREADS = 128;

}  // namespace
}  // namespace xb
