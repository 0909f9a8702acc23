#include "route_impl.h"

namespace mdgl {
hipError_t launch_route_f32(const RouteParams& q) { return run_route<float>(q); }
}  // namespace mdgl
