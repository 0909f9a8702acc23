#include "norm_impl.h"

namespace mdgl {
hipError_t launch_norm_f32(const NormParams& q) { return run_norm_width<float, float>(q); }
}  // namespace mdgl
