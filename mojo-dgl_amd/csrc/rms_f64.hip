#include "rms_impl.h"

namespace mdgl {
hipError_t launch_rms_f64(const RmsParams& q) { return run_rms_types<double>(q); }
}  // namespace mdgl
