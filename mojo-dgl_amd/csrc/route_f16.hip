#include "route_impl.h"

namespace mdgl {
hipError_t launch_route_f16(const RouteParams& q) { return run_route<f16_t>(q); }
}  // namespace mdgl
