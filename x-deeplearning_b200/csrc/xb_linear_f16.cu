// Linear attention: the kernels of f16.
#include "xb_linear_tiles.cuh"

namespace xb {
int linear_f16(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  return launch_linear_parts(p, s, [&](const LinearParams& q, dim3 grid) {
    if (plan.step) return launch_linear_step<__half>(q, grid, s);
    return plan.tiles ? launch_linear_tiles<false>(q, grid, s) : launch_linear_rows<__half>(q, grid, s);
  });
}
}  // namespace xb
