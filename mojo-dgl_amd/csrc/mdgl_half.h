// Element types of the row operators (layer norm, the segment scan, routing):
// float, double, bfloat16 and float16 in memory; sums, statistics and states in
// float (double for double). A result is rounded to its type once, to nearest.
#pragma once

#include "mdgl_common.h"

namespace mdgl {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T> struct AccOf { using type = float; };
template <> struct AccOf<double> { using type = double; };
template <class T> using acc_t = typename AccOf<T>::type;

// Dtype codes of include/mdgl.h.
enum DType { DT_F32 = 0, DT_F64 = 1, DT_BF16 = 2, DT_F16 = 3 };
inline int64_t dtype_bytes(int dtype) { return dtype == DT_F64 ? 8 : dtype == DT_F32 ? 4 : 2; }

// Values per 16 bytes of the accumulator type: the columns a lane of the
// scan or of the row movers holds.
template <class T> constexpr int acc_vec() { return 16 / (int)sizeof(acc_t<T>); }

__device__ __forceinline__ float fma_of(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return __builtin_fma(a, b, c); }

// N consecutive elements, at element alignment, in the accumulator type.
template <class T, class A, int N, bool STREAM = false>
__device__ __forceinline__ void load_acc(const T* p, A (&out)[N]) {
  T raw[N];
  load_any<STREAM>(p, raw);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (A)raw[i];
}

// N consecutive elements at element alignment.
template <class T, int N>
__device__ __forceinline__ void store_any(T* p, const T (&in)[N]) {
  if constexpr (N == 1) {
    *p = in[0];
  } else {
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    V v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = in[i];
    *reinterpret_cast<V*>(p) = v;
  }
}

template <class T, class A, int N>
__device__ __forceinline__ void store_acc(T* p, const A (&in)[N]) {
  T out[N];
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (T)in[i];
  store_any(p, out);
}

// N consecutive elements held as they came from memory: 16-bit values stay two
// to a register until they are used.
template <class T, int N>
struct Held {
  static constexpr int WORDS = (N * (int)sizeof(T) + 3) / 4;
  static constexpr int ALIGN = sizeof(T) < 4 ? (int)sizeof(T) : 4;
  uint32_t w[WORDS];
  // past the caches: for what is read once
  __device__ __forceinline__ void load_stream(const T* p) {
    if constexpr (WORDS > 1) {
      typedef uint32_t V __attribute__((ext_vector_type(WORDS), aligned(ALIGN)));
      const V v = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = v[i];
    } else {
      load(p);
    }
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) * N < 4) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else if constexpr (WORDS == 1) {
      __builtin_memcpy(w, p, 4);
    } else {
      typedef uint32_t V __attribute__((ext_vector_type(WORDS), aligned(ALIGN)));
      const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
      for (int i = 0; i < WORDS; ++i) w[i] = v[i];
    }
  }
  __device__ __forceinline__ acc_t<T> at(int k) const {
    if constexpr (sizeof(T) == 8) {
      return __builtin_bit_cast(double, (uint64_t)w[2 * k + 1] << 32 | w[2 * k]);
    } else if constexpr (sizeof(T) == 4) {
      return __builtin_bit_cast(float, w[k]);
    } else {
      const uint16_t h = (uint16_t)(k % 2 ? w[k / 2] >> 16 : w[k / 2]);
      return (float)__builtin_bit_cast(T, h);
    }
  }
};

}  // namespace mdgl
