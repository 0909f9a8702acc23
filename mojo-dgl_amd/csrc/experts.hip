// The way of rows to their experts and back.
//
// route_plan puts the m = n k entries (row t's j-th expert is entry t k + j) in
// the order of their experts, each expert's in entry order: a counting sort. A
// wavefront counts a run of entries in LDS (plan_count_kernel), the counts of the
// runs are summed per expert (plan_scan_kernel), and the wavefront goes over its
// run again: lanes with the same expert find each other by one ballot a bit of the
// expert's number, and take places in lane order. Integer sums only, so the order
// is the same each time. Up to PLAN_ONE entries take one launch of one workgroup
// (plan_one_kernel), as launches are what such a call costs. Entries whose expert
// lies outside [0, experts) belong to none: they come last, and `slot` holds the
// complement of their place.
//
// dispatch_kernel reads a row once and writes its k copies; combine_kernel reads
// a row's k entries and writes their weighted sum, added in the order of the
// choices in float; combine_grad_kernel forms both gradients, four of a row's entries
// at a time, from one read of them (and one of the row's gradient for each four). All
// move 16 bytes a lane whatever the width (the last lane of a row shares columns
// with the one before it) and are bound by memory: 32,768 bfloat16 rows of 2,048
// to 8 experts each, dispatch 222 us (1.21 GB, 5.4 TB/s), combine 230 us (5.2 TB/s;
// its reads past the caches: 269 us without), its gradient 490 us (2.28 GB,
// 4.7 TB/s), where a copy of 1 GiB runs at 5.1 TB/s. The plan of those 262,144
// entries takes 6 + 6 + 12 us.
#include "mdgl_half.h"
#include "mdgl_kernels.h"

namespace mdgl {

namespace {

constexpr int PLAN_RUN = 512;   // entries a wavefront
constexpr int PLAN_ONE = 2048;  // entries of a single launch
constexpr int PLAN_WAVES = 4;   // its wavefronts
constexpr int PLAN_BINS = ROUTE_MAX_EXPERTS + 1;  // one for the entries of no expert

__device__ __forceinline__ int plan_bin(const int64_t* ids, int64_t i, int64_t m, int experts) {
  const int64_t e = i < m ? ids[i] : -1;
  return e >= 0 && e < experts ? (int)e : experts;
}

// Lanes of the wavefront whose `bin` is this lane's, among those that are `in`.
__device__ __forceinline__ uint64_t same_bin(int bin, bool in, int bits) {
  uint64_t same = __ballot(in);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot(bin >> b & 1);
    same &= bin >> b & 1 ? set : ~set;
  }
  return same;
}

// Places of the entries [lo, hi) (at most `hi - lo` rounds of 64), with `next`
// (LDS) the first free place of each bin. All lanes of a wavefront take part.
__device__ __forceinline__ void plan_place(const int64_t* ids, int64_t lo, int64_t hi, int64_t m,
                                           int experts, int bits, int* next, int32_t* order,
                                           int32_t* slot) {
  const int lane = threadIdx.x % WAVE;
  for (int64_t at = lo; at < hi; at += WAVE) {
    const int64_t i = at + lane;
    const bool in = i < hi;
    const int bin = plan_bin(ids, in ? i : m, m, experts);
    const uint64_t same = same_bin(bin, in, bits);
    const uint64_t below = same & ((uint64_t(1) << lane) - 1);
    int place = 0;
    if (in) place = next[bin] + __builtin_popcountll(below);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && below == 0) next[bin] += __builtin_popcountll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      order[place] = (int32_t)i;
      slot[i] = bin < experts ? place : ~place;
    }
  }
}

// Exclusive prefix sums of get(0 .. bins - 1) by one wavefront, given to
// put(bin, sum).
template <class Get, class Put>
__device__ __forceinline__ void wave_prefix(int bins, Get get, Put put) {
  const int lane = threadIdx.x % WAVE;
  int before = 0;
  for (int b0 = 0; b0 < bins; b0 += WAVE) {
    const int b = b0 + lane;
    const int v = b < bins ? get(b) : 0;
    int sum = v;
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) {
      const int o = __shfl_up(sum, off);
      if (lane >= off) sum += o;
    }
    if (b < bins) put(b, before + sum - v);
    before += __shfl(sum, WAVE - 1);
  }
}

__global__ void __launch_bounds__(PLAN_WAVES* WAVE)
    plan_one_kernel(const int64_t* ids, int64_t m, int experts, int bits, int64_t* seglen,
                    int32_t* order, int32_t* slot) {
  extern __shared__ int plan_lds[];  // [PLAN_WAVES][experts + 1]
  const int bins = experts + 1, wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  for (int i = threadIdx.x; i < PLAN_WAVES * bins; i += PLAN_WAVES * WAVE) plan_lds[i] = 0;
  __syncthreads();
  const int64_t per = (m + PLAN_WAVES - 1) / PLAN_WAVES;
  const int64_t lo = wave * per < m ? wave * per : m, hi = lo + per < m ? lo + per : m;
  int* mine = plan_lds + wave * bins;
  for (int64_t i = lo + lane; i < hi; i += WAVE) atomicAdd(&mine[plan_bin(ids, i, m, experts)], 1);
  __syncthreads();
  if (wave == 0) {
    wave_prefix(
        bins,
        [&](int b) {
          int total = 0;
          for (int w = 0; w < PLAN_WAVES; ++w) total += plan_lds[w * bins + b];
          if (b < experts) seglen[b] = total;
          return total;
        },
        [&](int b, int first) {
          for (int w = 0; w < PLAN_WAVES; ++w) {
            const int n = plan_lds[w * bins + b];
            plan_lds[w * bins + b] = first;
            first += n;
          }
        });
  }
  __syncthreads();
  plan_place(ids, lo, hi, m, experts, bits, mine, order, slot);
}

__global__ void __launch_bounds__(WAVE) plan_count_kernel(const int64_t* ids, int64_t m,
                                                          int experts, int32_t* counts) {
  __shared__ int bin[PLAN_BINS];
  const int bins = experts + 1;
  for (int i = threadIdx.x; i < bins; i += WAVE) bin[i] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * PLAN_RUN;
  const int64_t hi = lo + PLAN_RUN < m ? lo + PLAN_RUN : m;
  for (int64_t i = lo + threadIdx.x; i < hi; i += WAVE)
    atomicAdd(&bin[plan_bin(ids, i, m, experts)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += WAVE) counts[(int64_t)blockIdx.x * bins + i] = bin[i];
}

// counts[run][bin] becomes the sum over the runs before; total[bin] the sum over all.
constexpr int PLAN_COLS = 32, PLAN_PARTS = 1024 / PLAN_COLS;

__global__ void __launch_bounds__(1024) plan_scan_kernel(int32_t* counts, int64_t runs, int bins,
                                                         int32_t* total) {
  __shared__ int sums[PLAN_PARTS][PLAN_COLS];
  const int c = threadIdx.x % PLAN_COLS, part = threadIdx.x / PLAN_COLS;
  const int bin = blockIdx.x * PLAN_COLS + c;
  const int64_t per = (runs + PLAN_PARTS - 1) / PLAN_PARTS;
  const int64_t lo = part * per < runs ? part * per : runs;
  const int64_t hi = bin < bins ? (lo + per < runs ? lo + per : runs) : lo;
  int sum = 0;
#pragma unroll 8
  for (int64_t r = lo; r < hi; ++r) sum += counts[r * bins + bin];
  sums[part][c] = sum;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < part; ++i) before += sums[i][c];
#pragma unroll 8
  for (int64_t r = lo; r < hi; ++r) {
    const int n = counts[r * bins + bin];
    counts[r * bins + bin] = before;
    before += n;
  }
  if (part == PLAN_PARTS - 1 && bin < bins) total[bin] = before;
}

__global__ void __launch_bounds__(WAVE) plan_place_kernel(const int64_t* ids, int64_t m,
                                                          int experts, int bits,
                                                          const int32_t* counts,
                                                          const int32_t* total, int64_t* seglen,
                                                          int32_t* order, int32_t* slot) {
  __shared__ int next[PLAN_BINS];
  const int bins = experts + 1;
  const int32_t* mine = counts + (int64_t)blockIdx.x * bins;
  wave_prefix(
      bins, [&](int b) { return total[b]; },
      [&](int b, int first) {
        next[b] = first + mine[b];
        if (blockIdx.x == 0 && b < experts) seglen[b] = total[b];
      });
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * PLAN_RUN;
  plan_place(ids, lo, lo + PLAN_RUN < m ? lo + PLAN_RUN : m, m, experts, bits, next, order, slot);
}

template <class T>
struct MoveArgs {
  using A = acc_t<T>;
  const T* src;
  const int32_t* slot;  // [n][k]
  const A* weights;     // [n][k], may be null: 1
  const T* grad;
  T* dst;
  A* dweights;
  int64_t n, d, lanes;
  int k;
};

template <class T> constexpr int move_vec() { return 16 / (int)sizeof(T); }

// A thread's row and first column, flat over rows times lanes; false past the end.
template <class T, int V>
__device__ __forceinline__ bool move_at(const MoveArgs<T>& p, int64_t* row, int64_t* col) {
  const int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
  *row = i / p.lanes;
  const int64_t c = (i - *row * p.lanes) * V;
  *col = c + V <= p.d ? c : p.d - V;
  return *row < p.n;
}

template <class T, int V>
__global__ void __launch_bounds__(BLOCK) dispatch_kernel(MoveArgs<T> p) {
  int64_t row, col;
  if (!move_at<T, V>(p, &row, &col)) return;
  T v[V], none[V];
  load_any<false>(p.src + row * p.d + col, v);
#pragma unroll
  for (int i = 0; i < V; ++i) none[i] = (T)0.0f;
  const int32_t* slot = p.slot + row * p.k;
  for (int j = 0; j < p.k; ++j) {
    const int32_t s = slot[j];
    if (s >= 0) store_any(p.dst + (int64_t)s * p.d + col, v);
    else store_any(p.dst + (int64_t)~s * p.d + col, none);
  }
}

template <class T, int V>
__global__ void __launch_bounds__(BLOCK) combine_kernel(MoveArgs<T> p) {
  using A = acc_t<T>;
  int64_t row, col;
  if (!move_at<T, V>(p, &row, &col)) return;
  A sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = A(0);
  const int32_t* slot = p.slot + row * p.k;
  constexpr int U = 8;  // rows in flight
  for (int j0 = 0; j0 < p.k; j0 += U) {
    Held<T, V> v[U];
    A w[U];
    int32_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = j0 + u < p.k ? slot[j0 + u] : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = A(1);
      if (at[u] < 0) continue;
      v[u].load_stream(p.src + (int64_t)at[u] * p.d + col);
      if (p.weights) w[u] = p.weights[row * p.k + j0 + u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at[u] >= 0)
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = fma_of(w[u], v[u].at(i), sum[i]);
  }
  store_acc<T, A, V>(p.dst + row * p.d + col, sum);
}

// A group of G threads a row: its gradient in registers, U of the row's entries at
// a time, dst = w * grad and dweights = <grad, src>. Entries of no expert get zeros.
template <class T, int V, int G>
__global__ void __launch_bounds__(BLOCK) combine_grad_kernel(MoveArgs<T> p) {
  using A = acc_t<T>;
  constexpr int U = 4;
  __shared__ A lds[G > WAVE ? U * (G / WAVE) : 1];
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G;
  if (row >= p.n) return;  // a whole workgroup, or whole groups of a wavefront
  const int32_t* slot = p.slot + row * p.k;
  for (int j0 = 0; j0 < p.k; j0 += U) {
    int32_t s[U];
    A w[U], dot[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = j0 + u < p.k ? slot[j0 + u] : 0;
      w[u] = j0 + u < p.k && s[u] >= 0 ? p.weights[row * p.k + j0 + u] : A(0);
      dot[u] = A(0);
    }
    for (int64_t v = lane; v < p.lanes; v += G) {
      const int64_t c = v * V, col = c + V <= p.d ? c : p.d - V;
      const int skip = (int)(c - col);  // columns counted by the lane before
      A g[V];
      load_acc<T, A, V>(p.grad + row * p.d + col, g);
      T x[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p.dweights && j0 + u < p.k && s[u] >= 0)
          load_any<true>(p.src + (int64_t)s[u] * p.d + col, x[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j0 + u >= p.k) continue;
        const bool live = s[u] >= 0;
        if (p.dweights && live)
#pragma unroll
          for (int i = 0; i < V; ++i)
            dot[u] = fma_of(i >= skip ? g[i] : A(0), i >= skip ? (A)x[u][i] : A(0), dot[u]);
        if (p.dst) {
          T out[V];
#pragma unroll
          for (int i = 0; i < V; ++i) out[i] = (T)(live ? w[u] * g[i] : A(0));
          store_stream_any(p.dst + (int64_t)(live ? s[u] : ~s[u]) * p.d + col, out);
        }
      }
    }
    if (!p.dweights) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) dot[u] = group_sum(dot[u], G < WAVE ? G : WAVE);
    if constexpr (G > WAVE) {
      __syncthreads();
      if (threadIdx.x % WAVE == 0)
#pragma unroll
        for (int u = 0; u < U; ++u) lds[u * (G / WAVE) + threadIdx.x / WAVE] = dot[u];
      __syncthreads();
      if (lane < U) {
        A sum = A(0);
#pragma unroll
        for (int i = 0; i < G / WAVE; ++i) sum += lds[lane * (G / WAVE) + i];
        if (j0 + lane < p.k) p.dweights[row * p.k + j0 + lane] = sum;
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lane == u && j0 + u < p.k) p.dweights[row * p.k + j0 + u] = dot[u];
    }
  }
}

// Runs launch(first row, rows) for as many rows as one launch takes.
template <class F>
hipError_t by_launches(int64_t n, int64_t rows_most, F launch) {
  if (rows_most < 1) rows_most = 1;
  for (int64_t at = 0; at < n; at += rows_most) {
    launch(at, n - at < rows_most ? n - at : rows_most);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T, int V>
hipError_t run_move(const MoveParams& q, MoveKind kind) {
  using A = acc_t<T>;
  MoveArgs<T> all{};
  all.src = (const T*)q.src;
  all.slot = q.slot;
  all.weights = (const A*)q.weights;
  all.grad = (const T*)q.grad;
  all.dst = (T*)q.dst;
  all.dweights = (A*)q.dweights;
  all.d = q.d;
  all.lanes = (q.d + V - 1) / V;
  all.k = q.k;
  // the launch for rows [at, at + n): the arrays that go row by row move along
  auto part = [&](int64_t at, int64_t n) {
    MoveArgs<T> p = all;
    p.n = n;
    p.slot += at * q.k;
    if (p.weights) p.weights += at * q.k;
    if (kind == MOVE_DISPATCH) p.src += at * q.d;
    if (kind == MOVE_COMBINE) p.dst += at * q.d;
    if (kind == MOVE_COMBINE_GRAD) {
      p.grad += at * q.d;
      if (p.dweights) p.dweights += at * q.k;
    }
    return p;
  };
  if (kind == MOVE_COMBINE_GRAD) {
    const int g = all.lanes <= 16 ? 16 : all.lanes <= 64 ? 64 : 256;
    return by_launches(q.n, MAX_LAUNCH_BLOCKS * (BLOCK / g), [&](int64_t at, int64_t n) {
      const int64_t grid = (n + BLOCK / g - 1) / (BLOCK / g);
      if (g == 16) combine_grad_kernel<T, V, 16><<<grid, BLOCK, 0, q.stream>>>(part(at, n));
      else if (g == 64) combine_grad_kernel<T, V, 64><<<grid, BLOCK, 0, q.stream>>>(part(at, n));
      else combine_grad_kernel<T, V, 256><<<grid, BLOCK, 0, q.stream>>>(part(at, n));
    });
  }
  return by_launches(q.n, MAX_LAUNCH_BLOCKS * BLOCK / all.lanes, [&](int64_t at, int64_t n) {
    const int64_t grid = (n * all.lanes + BLOCK - 1) / BLOCK;
    if (kind == MOVE_DISPATCH) dispatch_kernel<T, V><<<grid, BLOCK, 0, q.stream>>>(part(at, n));
    else combine_kernel<T, V><<<grid, BLOCK, 0, q.stream>>>(part(at, n));
  });
}

// Rows of e4m3 values, whose bytes are copied; they are never summed.
hipError_t run_dispatch_bytes(const MoveParams& q) {
  const int V = q.d >= 16 ? 16 : 1;
  const int64_t lanes = (q.d + V - 1) / V;
  return by_launches(q.n, MAX_LAUNCH_BLOCKS * BLOCK / lanes, [&](int64_t at, int64_t n) {
    MoveArgs<uint8_t> p{};
    p.src = (const uint8_t*)q.src + at * q.d;
    p.slot = q.slot + at * q.k;
    p.dst = (uint8_t*)q.dst;
    p.n = n;
    p.d = q.d;
    p.lanes = lanes;
    p.k = q.k;
    const int64_t grid = (n * lanes + BLOCK - 1) / BLOCK;
    if (V == 16) dispatch_kernel<uint8_t, 16><<<grid, BLOCK, 0, q.stream>>>(p);
    else dispatch_kernel<uint8_t, 1><<<grid, BLOCK, 0, q.stream>>>(p);
  });
}

template <class T>
hipError_t run_move_width(const MoveParams& q, MoveKind kind) {
  if (q.d >= move_vec<T>()) return run_move<T, move_vec<T>()>(q, kind);
  return run_move<T, 1>(q, kind);
}

int plan_bits(int experts) {
  int bits = 0;
  while (experts >> bits) ++bits;
  return bits;
}

}  // namespace

int64_t route_plan_workspace_bytes(int64_t m, int experts) {
  if (m <= PLAN_ONE) return 0;
  return ((m + PLAN_RUN - 1) / PLAN_RUN + 1) * (experts + 1) * 4;
}

hipError_t launch_route_plan(const int64_t* ids, int64_t m, int experts, int64_t* seglen,
                             int32_t* order, int32_t* slot, void* workspace, hipStream_t s) {
  const int bits = plan_bits(experts), bins = experts + 1;
  if (m <= PLAN_ONE) {
    plan_one_kernel<<<1, PLAN_WAVES * WAVE, PLAN_WAVES * bins * sizeof(int), s>>>(
        ids, m, experts, bits, seglen, order, slot);
    return hipGetLastError();
  }
  const int64_t runs = (m + PLAN_RUN - 1) / PLAN_RUN;
  int32_t* total = (int32_t*)workspace;
  int32_t* counts = total + bins;
  plan_count_kernel<<<runs, WAVE, 0, s>>>(ids, m, experts, counts);
  plan_scan_kernel<<<(bins + PLAN_COLS - 1) / PLAN_COLS, 1024, 0, s>>>(counts, runs, bins, total);
  plan_place_kernel<<<runs, WAVE, 0, s>>>(ids, m, experts, bits, counts, total, seglen, order,
                                          slot);
  return hipGetLastError();
}

hipError_t launch_move(const MoveParams& q, MoveKind kind, int dtype) {
  switch (dtype) {
    case DT_F8: return run_dispatch_bytes(q);
    case DT_F32: return run_move_width<float>(q, kind);
    case DT_F64: return run_move_width<double>(q, kind);
    case DT_BF16: return run_move_width<bf16_t>(q, kind);
    default: return run_move_width<f16_t>(q, kind);
  }
}

hipError_t launch_route(const RouteParams& q, int dtype) {
  switch (dtype) {
    case DT_F32: return launch_route_f32(q);
    case DT_F64: return launch_route_f64(q);
    case DT_BF16: return launch_route_bf16(q);
    default: return launch_route_f16(q);
  }
}

}  // namespace mdgl
