// Linear attention: the kernels of f32.
#include "xb_linear.cuh"

namespace xb {
int linear_f32(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  return launch_linear_parts(p, s, [&](const LinearParams& q, dim3 grid) { return plan.step ? launch_linear_step<float>(q, grid, s) : launch_linear_rows<float>(q, grid, s); });
}
}  // namespace xb
