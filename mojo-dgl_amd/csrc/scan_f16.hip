#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_f16(const ScanParams& q, bool back) {
  return q.gate_f32 ? run_scan<f16_t, float>(q, back) : run_scan<f16_t, f16_t>(q, back);
}
hipError_t launch_scan_step_f16(const ScanStepParams& q) {
  return q.gate_f32 ? run_scan_step<f16_t, float>(q) : run_scan_step<f16_t, f16_t>(q);
}
}  // namespace mdgl
