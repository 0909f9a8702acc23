#include "route_impl.h"

namespace mdgl {
hipError_t launch_route_bf16(const RouteParams& q) { return run_route<bf16_t>(q); }
}  // namespace mdgl
