#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_f32(const ScanParams& q, const ScanGeometry& geo, bool back) {
  return run_scan_width<float, float>(q, geo, back);
}
hipError_t launch_scan_step_f32(const ScanStepParams& q) { return run_scan_step<float, float>(q); }
}  // namespace mdgl
