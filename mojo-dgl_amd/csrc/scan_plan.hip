// The segments' marks that the scan walks by, and its dispatch by type.
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

// The scan's ticket and the words its chunks publish: 0, and every bit set.
__global__ void __launch_bounds__(BLOCK) scan_reset_kernel(uint32_t* ticket, uint32_t* words,
                                                           int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * 4;
  if (i == 0) *ticket = 0;
  if (i + 4 <= n) *reinterpret_cast<uint4*>(words + i) = make_uint4(~0u, ~0u, ~0u, ~0u);
  else
    for (int64_t j = i; j < n; ++j) words[j] = ~0u;
}

}  // namespace

hipError_t launch_scan_reset(uint32_t* ticket, uint32_t* words, int64_t n, hipStream_t s) {
  scan_reset_kernel<<<(n + 4 * BLOCK - 1) / (4 * BLOCK), BLOCK, 0, s>>>(ticket, words, n);
  return hipGetLastError();
}

hipError_t launch_segment_marks(const int32_t* offsets, int64_t num_seg, int64_t n, int32_t* ids,
                                uint64_t* starts, uint64_t* ends, hipStream_t s) {
  if (n == 0) return hipSuccess;
  segment_marks_kernel<<<(n + BLOCK - 1) / BLOCK, BLOCK, 0, s>>>(offsets, num_seg, n, ids, starts,
                                                                 ends);
  return hipGetLastError();
}

int64_t scan_workspace_bytes(int64_t n, int64_t d, int dtype) {
  // chunks of 128 rows at least; one chunk needs none
  const int64_t chunks = (n + 127) / 128;
  return chunks > 1 ? SCAN_TICKET_BYTES + scan_words(chunks) * d * (dtype == DT_F64 ? 8 : 4) : 0;
}

hipError_t launch_scan(const ScanParams& q, bool back, int dtype) {
  switch (dtype) {
    case DT_F32: return launch_scan_f32(q, back);
    case DT_F64: return launch_scan_f64(q, back);
    case DT_BF16: return launch_scan_bf16(q, back);
    default: return launch_scan_f16(q, back);
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
