// How layer norm lays its rows on threads, and the dispatch by type.
#include "mdgl_half.h"
#include "mdgl_kernels.h"

namespace mdgl {

int64_t norm_most_blocks(int threads) { return 256 * (2048 / threads); }

NormGeometry norm_geometry(int64_t n, int64_t d, int size) {
  const int64_t V = 16 / size;
  const int64_t nv = (d + V - 1) / V;
  const struct { int64_t vecs; int threads; } shapes[] = {
      {8, 8}, {8, 8}, {16, 16}, {32, 32}, {64, 64}, {128, 64},
      {256, 256}, {512, 256}, {1024, 512}, {2048, 512},
      {4096, 1024}};
  // 16-bit rows of more than 2,048 vectors have more sums than 1,024 threads' registers
  const int COUNT = (int)(sizeof shapes / sizeof shapes[0]) - (size == 2 ? 1 : 0);
  int shape = d < V ? 0 : 1;
  if (shape) while (shape < COUNT && shapes[shape].vecs < nv) ++shape;
  // workgroups of the gradient, each of which leaves a row of sums
  int64_t parts;
  if (shape == COUNT) {
    // d times parts work-items in a launch
    const int64_t most = d < (int64_t(1) << 25) ? 64 : 32;
    parts = n < most ? n : most;
  } else {
    const int g = shapes[shape].threads, block = g > 256 ? g : 256;
    const int64_t want = (n + block / g - 1) / (block / g), most = 256 * (1024 / block);
    parts = want < most ? want : most;
  }
  return {shape == COUNT ? NORM_WIDE_SHAPE : shape, parts < 1 ? 1 : parts};
}

int64_t norm_workspace_bytes(int64_t n, int64_t d, int dtype) {
  const int size = (int)dtype_bytes(dtype);
  return norm_geometry(n, d, size).parts * d * 2 * (dtype == DT_F64 ? 8 : 4);
}

hipError_t launch_norm(const NormParams& q, int dtype) {
  switch (dtype) {
    case DT_F32: return launch_norm_f32(q);
    case DT_F64: return launch_norm_f64(q);
    case DT_BF16: return launch_norm_bf16(q);
    default: return launch_norm_f16(q);
  }
}

}  // namespace mdgl
