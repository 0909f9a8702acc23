#include "norm_impl.h"

namespace mdgl {
hipError_t launch_norm_bf16(const NormParams& q) {
  return q.weight_f32 ? run_norm_width<bf16_t, float>(q) : run_norm_width<bf16_t, bf16_t>(q);
}
}  // namespace mdgl
