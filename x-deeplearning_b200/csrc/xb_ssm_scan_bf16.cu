// The selective scan of bf16 tensors (a unit of its own: the kernels take a while to compile).
#include "xb_ssm_scan.cuh"

namespace xb {
int ssm_scan_bf16(const ScanParams& p, const ScanPlan& plan, cudaStream_t s) { return launch_scan<__nv_bfloat16>(p, plan, s); }
}  // namespace xb
