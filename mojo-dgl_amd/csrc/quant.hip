// Rows and matrices brought to 8 bits (quant.h: the values and their scales).
//
// quant_rows_kernel: 16 lanes hold the 128 columns of a block, 8 each; their maximum
// goes through DPP, and each lane writes its 8 bytes. Bound by memory: 65,536 bfloat16
// rows of 1,536 take 57 us (306 MB, 5.4 TB/s).
//
// quant_blocks_kernel: a workgroup holds 128 by 128 values, 8 rows of 8 columns a
// thread, and writes them with the rows' axis contiguous (the inner axis of the
// products that take them). A thread's 8 rows are 8 consecutive bytes of each of its
// columns, so the transposition needs no LDS: neighbouring lanes take neighbouring
// rows (128 bytes of a column to 16 lanes), and what is read in pieces of 64 bytes
// comes from the caches the second time. Matrices whose rows' axis is contiguous
// already are read the other way round. 64 bfloat16 matrices of 2,048 by 1,536 take
// 130 us (604 MB, 4.7 TB/s).
#include "mdgl_kernels.h"
#include "quant.h"

namespace mdgl {

namespace {

constexpr int Q_LANE = 8;                    // columns a lane
constexpr int Q_LANES = Q_BLOCK / Q_LANE;    // lanes a block
constexpr int Q_WORK = BLOCK / Q_LANES;      // blocks a workgroup

// Columns [0, left) of the 8 at p; the others are zeros.
template <class T>
__device__ __forceinline__ Held<T, Q_LANE> quant_load(const T* p, int64_t left) {
  Held<T, Q_LANE> v;
  if (left >= Q_LANE) {
    v.load(p);
  } else {
    T some[Q_LANE];
#pragma unroll
    for (int i = 0; i < Q_LANE; ++i) some[i] = i < left ? p[i] : (T)0.0f;
    __builtin_memcpy(v.w, some, sizeof some);
  }
  return v;
}

// Bytes [0, left) of two words.
__device__ __forceinline__ void quant_store(uint8_t* p, const uint32_t (&words)[2], int64_t left) {
  if (left >= Q_LANE) {
    __builtin_memcpy(p, words, Q_LANE);
  } else {
#pragma unroll
    for (int i = 0; i < Q_LANE; ++i)
      if (i < left) p[i] = (uint8_t)(words[i / 4] >> 8 * (i % 4));
  }
}

template <class T>
__global__ void __launch_bounds__(BLOCK)
    quant_rows_kernel(const T* src, uint8_t* dst, float* scale, uint32_t units, uint32_t blocks,
                      int64_t d) {
  const uint32_t unit = blockIdx.x * Q_WORK + threadIdx.x / Q_LANES;
  if (unit >= units) return;  // whole groups of lanes
  const uint32_t row = unit / blocks, b = unit - row * blocks;
  const int64_t col = (int64_t)b * Q_BLOCK + threadIdx.x % Q_LANES * Q_LANE;
  const int64_t left = d - col, at = row * d + col;
  Held<T, Q_LANE> v;
  if (left > 0) v = quant_load(src + at, left);
  float x[Q_LANE], top = 0.0f;
#pragma unroll
  for (int i = 0; i < Q_LANE; ++i) {
    x[i] = left > 0 ? (float)v.at(i) : 0.0f;
    top = fmaxf(top, __builtin_fabsf(x[i]));
  }
  const QuantBy by(quant_scale(group_max(top, Q_LANES)));
  if (threadIdx.x % Q_LANES == 0) scale[unit] = by.s;
  const uint32_t words[2] = {by.word(x[0], x[1], x[2], x[3]), by.word(x[4], x[5], x[6], x[7])};
  if (left > 0) quant_store(dst + at, words, left);
}

// One matrix block a workgroup. TURN: src is [rows][cols], dst [cols][rows]; else
// both are [rows][cols]. Scales are [rows / 128][cols / 128], or the other way round
// without TURN.
template <class T, bool TURN>
__global__ void __launch_bounds__(BLOCK)
    quant_blocks_kernel(const T* src, uint8_t* dst, float* scale, int64_t rows, int64_t cols) {
  __shared__ float tops[WAVES_PER_BLOCK];
  const uint32_t rb = (uint32_t)((rows + Q_BLOCK - 1) / Q_BLOCK);
  const uint32_t cb = (uint32_t)((cols + Q_BLOCK - 1) / Q_BLOCK);
  const uint32_t m = blockIdx.x / (rb * cb), at = blockIdx.x - m * (rb * cb);
  const uint32_t br = at / cb, bc = at - br * cb;
  const int fast = threadIdx.x % Q_LANES, slow = threadIdx.x / Q_LANES;
  const int64_t row = (int64_t)br * Q_BLOCK + (TURN ? fast : slow) * Q_LANE;
  const int64_t col = (int64_t)bc * Q_BLOCK + (TURN ? slow : fast) * Q_LANE;
  src += (int64_t)m * rows * cols;
  dst += (int64_t)m * rows * cols;
  Held<T, Q_LANE> v[Q_LANE];
#pragma unroll
  for (int i = 0; i < Q_LANE; ++i) {
#pragma unroll
    for (int k = 0; k < Held<T, Q_LANE>::WORDS; ++k) v[i].w[k] = 0;
    if (row + i < rows && col < cols) v[i] = quant_load(src + (row + i) * cols + col, cols - col);
  }
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < Q_LANE; ++i)
#pragma unroll
    for (int k = 0; k < Q_LANE; ++k) top = fmaxf(top, __builtin_fabsf((float)v[i].at(k)));
  top = group_max(top, WAVE);
  if (threadIdx.x % WAVE == 0) tops[threadIdx.x / WAVE] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES_PER_BLOCK; ++i) top = fmaxf(top, tops[i]);
  const QuantBy by(quant_scale(top));
  if (threadIdx.x == 0)
    scale[(int64_t)m * rb * cb + (TURN ? br * cb + bc : bc * rb + br)] = by.s;
#pragma unroll
  for (int k = 0; k < Q_LANE; ++k) {
    auto x = [&](int i) { return (float)(TURN ? v[i].at(k) : v[k].at(i)); };
    const uint32_t words[2] = {by.word(x(0), x(1), x(2), x(3)), by.word(x(4), x(5), x(6), x(7))};
    if constexpr (TURN) {
      if (row < rows && col + k < cols) quant_store(dst + (col + k) * rows + row, words, rows - row);
    } else {
      if (row + k < rows && col < cols) quant_store(dst + (row + k) * cols + col, words, cols - col);
    }
  }
}

template <class T>
hipError_t run_quant_rows(const void* src, void* dst, float* scale, int64_t n, int64_t d,
                          hipStream_t s) {
  const int64_t blocks = (d + Q_BLOCK - 1) / Q_BLOCK;
  // units of a launch are counted in 32 bits, their work-items too
  const int64_t most = (MAX_LAUNCH_BLOCKS * Q_WORK - Q_WORK) / blocks;
  for (int64_t at = 0; at < n; at += most) {
    const int64_t rows = n - at < most ? n - at : most, units = rows * blocks;
    quant_rows_kernel<T><<<(units + Q_WORK - 1) / Q_WORK, BLOCK, 0, s>>>(
        (const T*)src + at * d, (uint8_t*)dst + at * d, scale + at * blocks, (uint32_t)units,
        (uint32_t)blocks, d);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T>
hipError_t run_quant_blocks(const void* src, void* dst, float* scale, int64_t r, int64_t d1,
                            int64_t d2, bool transposed, hipStream_t s) {
  const int64_t per = ((d1 + Q_BLOCK - 1) / Q_BLOCK) * ((d2 + Q_BLOCK - 1) / Q_BLOCK);
  const int64_t most = MAX_LAUNCH_BLOCKS / per;  // at least 1 (checked before)
  for (int64_t at = 0; at < r; at += most) {
    const int64_t grid = (r - at < most ? r - at : most) * per, skip = at * d1 * d2;
    const T* from = (const T*)src + skip;
    uint8_t* to = (uint8_t*)dst + skip;
    float* sc = scale + at * per;
    if (transposed) quant_blocks_kernel<T, false><<<grid, BLOCK, 0, s>>>(from, to, sc, d2, d1);
    else quant_blocks_kernel<T, true><<<grid, BLOCK, 0, s>>>(from, to, sc, d1, d2);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_quantize_rows(const void* src, void* dst, float* scale, int64_t n, int64_t d,
                                int dtype, hipStream_t s) {
  if (dtype == DT_F32) return run_quant_rows<float>(src, dst, scale, n, d, s);
  if (dtype == DT_BF16) return run_quant_rows<bf16_t>(src, dst, scale, n, d, s);
  return run_quant_rows<f16_t>(src, dst, scale, n, d, s);
}

hipError_t launch_quantize_blocks(const void* src, void* dst, float* scale, int64_t r, int64_t d1,
                                  int64_t d2, bool transposed, int dtype, hipStream_t s) {
  if (dtype == DT_F32)
    return run_quant_blocks<float>(src, dst, scale, r, d1, d2, transposed, s);
  if (dtype == DT_BF16)
    return run_quant_blocks<bf16_t>(src, dst, scale, r, d1, d2, transposed, s);
  return run_quant_blocks<f16_t>(src, dst, scale, r, d1, d2, transposed, s);
}

}  // namespace mdgl
