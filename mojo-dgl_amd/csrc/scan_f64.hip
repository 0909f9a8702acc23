#include "scan_impl.h"

namespace mdgl {
hipError_t launch_scan_f64(const ScanParams& q, bool back) {
  return run_scan<double, double>(q, back);
}
hipError_t launch_scan_step_f64(const ScanStepParams& q) { return run_scan_step<double, double>(q); }
}  // namespace mdgl
