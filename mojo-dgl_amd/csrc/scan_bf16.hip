#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_bf16(const ScanParams& q, const ScanGeometry& geo, bool back) {
  return q.gate_f32 ? run_scan_width<bf16_t, float>(q, geo, back) : run_scan_width<bf16_t, bf16_t>(q, geo, back);
}
hipError_t launch_scan_step_bf16(const ScanStepParams& q) {
  return q.gate_f32 ? run_scan_step<bf16_t, float>(q) : run_scan_step<bf16_t, bf16_t>(q);
}
}  // namespace mdgl
