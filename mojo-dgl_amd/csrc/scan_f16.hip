#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_f16(const ScanParams& q, const ScanGeometry& geo, bool back) {
  return q.gate_f32 ? run_scan_width<f16_t, float>(q, geo, back) : run_scan_width<f16_t, f16_t>(q, geo, back);
}
hipError_t launch_scan_step_f16(const ScanStepParams& q) {
  return q.gate_f32 ? run_scan_step<f16_t, float>(q) : run_scan_step<f16_t, f16_t>(q);
}
}  // namespace mdgl
