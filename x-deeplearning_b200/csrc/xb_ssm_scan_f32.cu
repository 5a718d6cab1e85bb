// The selective scan of fp32 tensors (a unit of its own: the kernels take a while to compile).
#include "xb_ssm_scan.cuh"

namespace xb {
int ssm_scan_f32(const ScanParams& p, const ScanPlan& plan, cudaStream_t s) { return launch_scan<float>(p, plan, s); }
}  // namespace xb
