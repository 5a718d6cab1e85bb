// Linear attention: the kernels of bf16.
#include "xb_linear.cuh"

namespace xb {
int linear_bf16(const LinearParams& p, const LinearPlan& plan, cudaStream_t s) {
  return launch_linear_parts(p, s, [&](const LinearParams& q, dim3 grid) { return launch_linear_rows<__nv_bfloat16>(q, grid, s); });
}
}  // namespace xb
