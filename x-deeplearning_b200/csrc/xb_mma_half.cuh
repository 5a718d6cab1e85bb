// Warp-level matrix instructions on 16-bit operands in shared memory.
#pragma once

#include <cstdint>

namespace xb {

template <int X4T>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (X4T)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c += a b as sums of 16 products, each added to c by an fp32 addition of its own: what the matrix instruction adds to an accumulator
// is cut off, not rounded, and a long chain of such sums drifts. The products of [16..512]-deep sums against 64 bits, rms relative to
// the result, before the result's rounding (fp32 FMAs; matrix instructions that accumulate): fp16 normal values 6.5e-8 (1.5e-7; 1.6e-7),
// positive ones 5.7e-8 (9.0e-8; 2.9e-7); bf16 4.5e-8 (5.6e-8; 1.0e-7) and 3.5e-8 (4.3e-8; 1.0e-7). Largest error: 0.3 to 0.7 of the FMAs'.
template <bool BF16>
__device__ __forceinline__ void mma_half(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  float d[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += d[e];
}

// halves that are infinite or NaN
template <bool BF16>
__device__ __forceinline__ bool half_is_bad(uint32_t h) {
  constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
  return (h & E) == E;
}

// sum + 0 * t, two halves: NaN once a t was infinite or NaN
template <bool BF16>
__device__ __forceinline__ uint32_t fma_zero(uint32_t t, uint32_t sum) {
  uint32_t r;
  if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(t), "r"(0u), "r"(sum));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(t), "r"(0u), "r"(sum));
  return r;
}

}  // namespace xb
