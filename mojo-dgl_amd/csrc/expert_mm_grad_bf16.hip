#include "expert_mm_impl.h"

namespace mdgl {
hipError_t launch_expert_mm_grad_bf16(const ExpertMmParams& q) {
  return run_expert_mm_grad_shape<bf16_t>(q);
}
}  // namespace mdgl
