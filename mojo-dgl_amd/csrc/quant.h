// Values in 8 bits: e4m3 (4 exponent bits, 3 mantissa bits, largest value 448, no
// infinities) beside a float scale for each block of 128 columns.
//
//   scale = max(amax / 448, 2^-126),  q = value / scale rounded to nearest even
//
// Both quotients are rounded to float first, so that a value lies on the same side
// of a border between two e4m3 values whoever forms it. The least scale keeps a
// block of zeros, or of values below any use, from a division by 0. |value / scale|
// is at most 448 (1 + 2^-23), which rounds to 448. A NaN stays one, alone; an infinity
// makes its block's scale infinite, and with it every value of the block a NaN when it
// is multiplied back.
#pragma once

#include "mdgl_half.h"

namespace mdgl {

constexpr int Q_BLOCK = 128;
constexpr float Q_TOP = 448.0f;

__device__ __forceinline__ float quant_scale(float top) {
  const float s = top / Q_TOP;
  return s < 0x1p-126f ? 0x1p-126f : s;
}

// The divisor s of a block: r = 1 / s is formed once, x r is off by little more than
// half a step, and its residue, exact in one fma, corrects that. The residue of a value
// that matters is at least 2^-34 s: below s = 2^-90 it may leave the normal numbers, so
// such blocks divide.
struct QuantBy {
  float s, r;
  bool small;
  __device__ __forceinline__ explicit QuantBy(float scale)
      : s(scale), r(1.0f / scale), small(scale < 0x1p-90f) {}
  __device__ __forceinline__ float of(float x) const {
    if (small) return x / s;
    const float q = x * r;
    return __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
  }
  // Values of a block as bytes, the first in the low byte.
  __device__ __forceinline__ uint32_t word(float a, float b, float c, float d) const {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(of(a), of(b), 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(of(c), of(d), w, true);
    return (uint32_t)w;
  }
  __device__ __forceinline__ uint8_t byte(float a) const {
    return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(of(a), 0.0f, 0, false);
  }
};

// Largest of a value over groups of `lanes` (a power of two) consecutive lanes. NaNs
// are passed over, as fmaxf does.
__device__ __forceinline__ float group_max(float v, int lanes) {
  if (lanes > 1) v = fmaxf(v, lane_xor_dpp(v, 0));
  if (lanes > 2) v = fmaxf(v, lane_xor_dpp(v, 1));
  if (lanes > 4) v = fmaxf(v, lane_xor_dpp(v, 2));
  if (lanes > 8) v = fmaxf(v, lane_xor_dpp(v, 3));
  if (lanes > 16) v = fmaxf(v, __shfl_xor(v, 16));
  if (lanes > 32) v = fmaxf(v, __shfl_xor(v, 32));
  return v;
}

}  // namespace mdgl
