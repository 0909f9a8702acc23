#include "rms_impl.h"

namespace mdgl {
hipError_t launch_rms_bf16(const RmsParams& q) { return run_rms_types<bf16_t>(q); }
}  // namespace mdgl
