#include "rms_impl.h"

namespace mdgl {
hipError_t launch_rms_f16(const RmsParams& q) { return run_rms_types<f16_t>(q); }
}  // namespace mdgl
