#include "rms_impl.h"

namespace mdgl {
hipError_t launch_rms_f32(const RmsParams& q) { return run_rms_types<float>(q); }
}  // namespace mdgl
