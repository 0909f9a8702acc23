#include "expert_mm_impl.h"

namespace mdgl {
hipError_t launch_expert_mm_bf16(const ExpertMmParams& q) {
  return q.along ? run_expert_mm_shape<bf16_t, true>(q) : run_expert_mm_shape<bf16_t, false>(q);
}
}  // namespace mdgl
