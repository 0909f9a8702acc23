#include "route_impl.h"

namespace mdgl {
hipError_t launch_route_f64(const RouteParams& q) { return run_route<double>(q); }
}  // namespace mdgl
