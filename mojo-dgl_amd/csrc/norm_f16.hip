#include "norm_impl.h"

namespace mdgl {
hipError_t launch_norm_f16(const NormParams& q) {
  return q.weight_f32 ? run_norm_width<f16_t, float>(q) : run_norm_width<f16_t, f16_t>(q);
}
}  // namespace mdgl
