#include "expert_mm_impl.h"

namespace mdgl {
hipError_t launch_expert_mm_f8(const ExpertMmParams& q) {
  return run_expert_mm_shape<f8_t, true>(q);
}
}  // namespace mdgl
