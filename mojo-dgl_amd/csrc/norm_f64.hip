#include "norm_impl.h"

namespace mdgl {
hipError_t launch_norm_f64(const NormParams& q) { return run_norm_width<double, double>(q); }
}  // namespace mdgl
