// The segments' marks that the scan walks by, and how it cuts the rows.
#include "mdgl_half.h"
#include "mdgl_kernels.h"

namespace mdgl {

namespace {

// ids[r] = the segment of row r; bit r % 64 of starts[r / 64] / ends[r / 64]:
// row r is the first / last of its segment. One wavefront writes a word of each.
__global__ void __launch_bounds__(BLOCK) segment_marks_kernel(const int32_t* off, int64_t num_seg,
                                                              int64_t n, int32_t* ids,
                                                              uint64_t* starts, uint64_t* ends) {
  const int64_t r = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
  bool first = false, last = false;
  if (r < n) {
    // the last offset at or in front of r belongs to the one segment that holds it
    int64_t lo = 0, hi = num_seg - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) / 2;
      if (off[mid] <= r) lo = mid;
      else hi = mid - 1;
    }
    ids[r] = (int32_t)lo;
    first = off[lo] == r;
    last = off[lo + 1] == r + 1;
  }
  const uint64_t a = __ballot(first), b = __ballot(last);
  if (threadIdx.x % WAVE == 0 && r < n) {
    starts[r / WAVE] = a;
    ends[r / WAVE] = b;
  }
}

}  // namespace

hipError_t launch_segment_marks(const int32_t* offsets, int64_t num_seg, int64_t n, int32_t* ids,
                                uint64_t* starts, uint64_t* ends, hipStream_t s) {
  if (n == 0) return hipSuccess;
  segment_marks_kernel<<<(n + BLOCK - 1) / BLOCK, BLOCK, 0, s>>>(offsets, num_seg, n, ids, starts,
                                                                 ends);
  return hipGetLastError();
}

ScanGeometry scan_geometry(int64_t n, int64_t d, int64_t longest, int dtype) {
  const int64_t vec = dtype == DT_F64 ? 2 : 4;
  const int64_t lanes = d < vec ? d : (d + vec - 1) / vec;
  // rows a walk: the most that leaves 2,048 wavefronts of them
  int64_t len = 16;
  while (len < 1024 && (n / (2 * len)) * lanes >= 2048 * WAVE) len *= 2;
  return {longest <= 256, len};
}

int64_t scan_workspace_bytes(int64_t n, int64_t d, int64_t longest, int dtype) {
  const ScanGeometry geo = scan_geometry(n, d, longest, dtype);
  if (geo.owners) return 0;
  return (n + geo.len - 1) / geo.len * d * 2 * (dtype == DT_F64 ? 8 : 4);
}

hipError_t launch_scan(const ScanParams& q, bool back, int64_t longest, int dtype) {
  const ScanGeometry geo = scan_geometry(q.n, q.d, longest, dtype);
  switch (dtype) {
    case DT_F32: return launch_scan_f32(q, geo, back);
    case DT_F64: return launch_scan_f64(q, geo, back);
    case DT_BF16: return launch_scan_bf16(q, geo, back);
    default: return launch_scan_f16(q, geo, back);
  }
}

hipError_t launch_scan_step(const ScanStepParams& q, int dtype) {
  switch (dtype) {
    case DT_F32: return launch_scan_step_f32(q);
    case DT_F64: return launch_scan_step_f64(q);
    case DT_BF16: return launch_scan_step_bf16(q);
    default: return launch_scan_step_f16(q);
  }
}

}  // namespace mdgl
