// Linear attention: the kernels of bf16.
#include "xb_linear_tiles.cuh"

namespace xb {
int linear_bf16(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  return launch_linear_parts(p, s, [&](const LinearParams& q, dim3 grid) {
    if (plan.step) return launch_linear_step<__nv_bfloat16>(q, grid, s);
    return plan.tiles ? launch_linear_tiles<true>(q, grid, s) : launch_linear_rows<__nv_bfloat16>(q, grid, s);
  });
}
}  // namespace xb
