#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_bf16(const ScanParams& q, bool back) {
  return q.gate_f32 ? run_scan<bf16_t, float>(q, back) : run_scan<bf16_t, bf16_t>(q, back);
}
hipError_t launch_scan_step_bf16(const ScanStepParams& q) {
  return q.gate_f32 ? run_scan_step<bf16_t, float>(q) : run_scan_step<bf16_t, bf16_t>(q);
}
}  // namespace mdgl
