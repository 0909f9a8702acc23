#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_f32(const ScanParams& q, bool back) {
  return run_scan<float, float>(q, back);
}
hipError_t launch_scan_step_f32(const ScanStepParams& q) { return run_scan_step<float, float>(q); }
}  // namespace mdgl
