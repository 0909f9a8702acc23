// Layer norm over the last axis, and its gradients (included once per type).
//
//   mean = sum x / d,  r = 1 / sqrt(sum (x - mean)^2 / d + eps),  xh = (x - mean) r
//   y = xh w + b
//   dx = r (g - sum g / d - xh sum(g xh) / d),  g = dy w
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Both passes read and write each row once: a group of G threads holds a row in
// registers, K vectors of 16 bytes a thread, so the variance is summed around the
// mean (no difference of large squares) without a second read. G is 8 to 64 lanes
// of a wavefront for rows of up to 128 vectors, a workgroup of 256 to 1,024 for
// wider ones; a group goes on to further rows with the next one's loads in
// flight. The gradient sums its rows' dw and db in registers, adds the groups of
// a workgroup in a fixed order through LDS, leaves one row of sums a workgroup, and
// norm_sum_kernel adds those: no atomics, the same bits each time. Rows too wide
// for a workgroup's registers go through norm_wide_kernel and norm_cols_kernel,
// which read them again instead.
//
// Bound by memory: 32,768 bfloat16 rows of 4,096 take 99 us forward (537 MB, 5.4 TB/s)
// and 172 + 5 us backward (805 MB and 17 MB of partial sums, 4.8 TB/s), a million float32
// rows of 47 75 us (376 MB, 5.0 TB/s) and 115 + 9 us (564 MB, 4.9 TB/s), where a copy of
// 1 GiB runs at 5.1 TB/s. A workgroup a row from 256 vectors on: a wavefront a row would
// hold 512 vectors in 256 registers and leave one wavefront a SIMD in the gradient.
//
// A row whose width is no whole number of vectors ends with a vector that shares
// columns with the one before it: they count once in every sum, and both write
// the same values.
#pragma once

#include "mdgl_half.h"
#include "mdgl_kernels.h"

namespace mdgl {

template <class T, class W>
struct NormArgs {
  using A = acc_t<T>;
  const T* x;
  const W* w;  // may be null: 1
  const W* b;  // may be null: 0
  const T* dy;
  T* y;
  T* dx;    // may be null
  A* mean;  // [n] written forward when not null, read backward
  A* rstd;
  A* part_w;  // [workgroups][d] (may be null)
  A* part_b;
  int64_t n, d;
  double eps;
};

// The columns of vector `v` of a row: from `col` on, the first `skip` of them
// counted in the vector before; false past the row.
template <int V>
__device__ __forceinline__ bool norm_cols(int64_t v, int64_t d, int64_t* col, int* skip) {
  const int64_t c = v * V;
  if (c >= d) return false;
  *col = c + V <= d ? c : d - V;
  *skip = (int)(c - *col);
  return true;
}

// Sum of two values over the G threads of a group. For G > 64 `lds` holds two
// values a wavefront, twice (`turn` alternates, so one barrier is enough).
template <int G, class A>
__device__ __forceinline__ void norm_sum2(A& a, A& b, A* lds, int& turn) {
  if constexpr (G <= WAVE) {
    a = group_sum(a, G);
    b = group_sum(b, G);
  } else {
    constexpr int W = G / WAVE;
    a = group_sum(a, WAVE);
    b = group_sum(b, WAVE);
    A* s = lds + turn * 2 * W;
    turn ^= 1;
    const int wave = threadIdx.x / WAVE;
    if (threadIdx.x % WAVE == 0) {
      s[2 * wave] = a;
      s[2 * wave + 1] = b;
    }
    __syncthreads();
    a = A(0);
    b = A(0);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      a += s[2 * i];
      b += s[2 * i + 1];
    }
  }
}

template <int G> constexpr int norm_block() { return G > 256 ? G : 256; }

__device__ __forceinline__ float norm_rsqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double norm_rsqrt(double v) { return 1.0 / sqrt(v); }

template <class T, class W, int V, int G, int K>
__global__ void __launch_bounds__(norm_block<G>()) norm_kernel(NormArgs<T, W> p) {
  using A = acc_t<T>;
  constexpr int GROUPS = norm_block<G>() / G;
  __shared__ A lds[G > WAVE ? 4 * (G / WAVE) : 1];
  int turn = 0;
  const int t = threadIdx.x % G;
  int64_t col[K];
  int skip[K];
  bool live[K];
  A w[K][V], b[K][V];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    col[j] = 0;
    skip[j] = 0;
    live[j] = norm_cols<V>(t + j * G, p.d, &col[j], &skip[j]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      w[j][k] = A(1);
      b[j][k] = A(0);
    }
    if (live[j] && p.w) load_acc<W, A, V>(p.w + col[j], w[j]);
    if (live[j] && p.b) load_acc<W, A, V>(p.b + col[j], b[j]);
  }
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const A inv = A(1) / (A)p.d;
  int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G;
  // a group of a whole workgroup leaves the loop with all its threads; smaller
  // groups need none of the others
  T raw[K][V];
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (row < p.n && live[j]) load_any<false>(p.x + row * p.d + col[j], raw[j]);
  while (row < p.n) {
    A x[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) x[j][k] = live[j] ? (A)raw[j][k] : A(0);
    const int64_t next = row + step;
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (next < p.n && live[j]) load_any<false>(p.x + next * p.d + col[j], raw[j]);
    A s = A(0), q = A(0);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) s += k >= skip[j] ? x[j][k] : A(0);
    norm_sum2<G>(s, q, lds, turn);
    const A mean = s * inv;
    s = A(0);
    q = A(0);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        x[j][k] -= mean;
        q = fma_of(x[j][k], live[j] && k >= skip[j] ? x[j][k] : A(0), q);
      }
    norm_sum2<G>(q, s, lds, turn);
    const A r = norm_rsqrt(q * inv + (A)p.eps);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (!live[j]) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) x[j][k] = fma_of(x[j][k] * r, w[j][k], b[j][k]);
      store_acc<T, A, V>(p.y + row * p.d + col[j], x[j]);
    }
    if (p.mean && t == 0) {
      p.mean[row] = mean;
      p.rstd[row] = r;
    }
    row = next;
  }
}

template <class T, class W, int V, int G, int K>
__global__ void __launch_bounds__(norm_block<G>()) norm_grad_kernel(NormArgs<T, W> p) {
  using A = acc_t<T>;
  constexpr int GROUPS = norm_block<G>() / G;
  // four vectors a thread leave no registers for w, and with 1,024 threads (128
  // registers each) none for the next row's loads either
  constexpr bool HOLD = K < 4, AHEAD = G < 1024;
  __shared__ A lds[G > WAVE ? 4 * (G / WAVE) : 1];
  __shared__ A sums[GROUPS > 1 ? 2 * G * K * V : 1];
  int turn = 0;
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  int64_t col[K];
  int skip[K];
  bool live[K];
  A w[HOLD ? K : 1][V], dw[K][V], db[K][V];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    col[j] = 0;
    skip[j] = 0;
    live[j] = norm_cols<V>(t + j * G, p.d, &col[j], &skip[j]);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (HOLD) w[HOLD ? j : 0][k] = A(1);
      dw[j][k] = A(0);
      db[j][k] = A(0);
    }
    if (HOLD && live[j] && p.w) load_acc<W, A, V>(p.w + col[j], w[HOLD ? j : 0]);
  }
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const A inv = A(1) / (A)p.d;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  // rows stay as they came from memory, 16-bit values two to a register, and xh and g
  // are formed again for dx: the registers saved leave room for the next row's loads
  Held<T, V> xn[K], gn[K];
  A mean_n = A(0), r_n = A(0);
  auto fetch = [&](int64_t at) {
    if (at >= p.n) return;
    mean_n = p.mean[at];
    r_n = p.rstd[at];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (!live[j]) continue;
      xn[j].load(p.x + at * p.d + col[j]);
      gn[j].load(p.dy + at * p.d + col[j]);
    }
  };
  fetch(row);
  while (row < p.n) {
    Held<T, V> x[K], g[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      x[j] = xn[j];
      g[j] = gn[j];
    }
    const A mean = mean_n, r = r_n;
    const int64_t next = row + step;
    if (AHEAD) fetch(next);
    A s = A(0), q = A(0);
    // xh and g of vector j
    auto form = [&](int j, A (&xh)[V], A (&dy)[V], A (&gw)[V]) {
      if constexpr (!HOLD) {
#pragma unroll
        for (int k = 0; k < V; ++k) w[0][k] = A(1);
        if (p.w) load_acc<W, A, V>(p.w + col[j], w[0]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dy[k] = g[j].at(k);
        xh[k] = (x[j].at(k) - mean) * r;
        gw[k] = dy[k] * w[HOLD ? j : 0][k];
      }
    };
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (!live[j]) continue;
      A xh[V], dy[V], gw[V];
      form(j, xh, dy, gw);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dw[j][k] = fma_of(dy[k], xh[k], dw[j][k]);
        db[j][k] += dy[k];
        const A c = k >= skip[j] ? gw[k] : A(0);
        s += c;
        q = fma_of(c, xh[k], q);
      }
    }
    if (p.dx) {
      norm_sum2<G>(s, q, lds, turn);
      s *= inv;
      q *= inv;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (!live[j]) continue;
        A xh[V], dy[V], gw[V];
        form(j, xh, dy, gw);
#pragma unroll
        for (int k = 0; k < V; ++k) gw[k] = r * (gw[k] - s - xh[k] * q);
        store_acc<T, A, V>(p.dx + row * p.d + col[j], gw);
      }
    }
    if (!AHEAD) fetch(next);
    row = next;
  }
  if (!p.part_w && !p.part_b) return;
  if constexpr (GROUPS > 1) {
    // the groups of the workgroup one after the other
    for (int i = 0; i < GROUPS; ++i) {
      if (group == i) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
          for (int k = 0; k < V; ++k) {
            A* s = sums + 2 * ((t + j * G) * V + k);
            if (i) {
              dw[j][k] += s[0];
              db[j][k] += s[1];
            }
            s[0] = dw[j][k];
            s[1] = db[j][k];
          }
      }
      __syncthreads();
    }
    if (group != GROUPS - 1) return;
  }
#pragma unroll
  for (int j = 0; j < K; ++j) {
    // formed again: held until here they put two of 1,024 threads' registers in memory
    // (double)
    int64_t c;
    int shared;
    if (!norm_cols<V>(t + j * G, p.d, &c, &shared)) continue;
    const int64_t at = (int64_t)blockIdx.x * p.d + c;
    if (p.part_w) store_acc<A, A, V>(p.part_w + at, dw[j]);
    if (p.part_b) store_acc<A, A, V>(p.part_b + at, db[j]);
  }
}

// Rows wider than a workgroup's registers: a workgroup a row, read again from the
// caches for each sum. GRAD: dx instead of y.
constexpr int NORM_WIDE = 1024;

template <class T, class W, bool GRAD>
__global__ void __launch_bounds__(NORM_WIDE) norm_wide_kernel(NormArgs<T, W> p) {
  using A = acc_t<T>;
  __shared__ A lds[4 * (NORM_WIDE / WAVE)];
  int turn = 0;
  const A inv = A(1) / (A)p.d;
  for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
    const T* x = p.x + row * p.d;
    A s = A(0), q = A(0);
    if constexpr (GRAD) {
      const T* dy = p.dy + row * p.d;
      const A mean = p.mean[row], r = p.rstd[row];
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) {
        const A g = (A)dy[c] * (p.w ? (A)p.w[c] : A(1));
        s += g;
        q = fma_of(g, ((A)x[c] - mean) * r, q);
      }
      norm_sum2<NORM_WIDE>(s, q, lds, turn);
      s *= inv;
      q *= inv;
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) {
        const A g = (A)dy[c] * (p.w ? (A)p.w[c] : A(1));
        p.dx[row * p.d + c] = (T)(r * (g - s - ((A)x[c] - mean) * r * q));
      }
    } else {
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) s += (A)x[c];
      norm_sum2<NORM_WIDE>(s, q, lds, turn);
      const A mean = s * inv;
      s = A(0);
      q = A(0);
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) {
        const A v = (A)x[c] - mean;
        q = fma_of(v, v, q);
      }
      norm_sum2<NORM_WIDE>(q, s, lds, turn);
      const A r = norm_rsqrt(q * inv + (A)p.eps);
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE)
        p.y[row * p.d + c] = (T)fma_of(((A)x[c] - mean) * r, p.w ? (A)p.w[c] : A(1),
                                       p.b ? (A)p.b[c] : A(0));
      if (p.mean && threadIdx.x == 0) {
        p.mean[row] = mean;
        p.rstd[row] = r;
      }
    }
  }
}

// dw and db of such rows: a thread a column, blockIdx.y a run of rows.
template <class T, class W>
__global__ void __launch_bounds__(BLOCK) norm_cols_kernel(NormArgs<T, W> p) {
  using A = acc_t<T>;
  const int64_t c = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
  if (c >= p.d) return;
  A dw = A(0), db = A(0);
  for (int64_t row = blockIdx.y; row < p.n; row += gridDim.y) {
    const A dy = (A)p.dy[row * p.d + c];
    dw = fma_of(dy, ((A)p.x[row * p.d + c] - p.mean[row]) * p.rstd[row], dw);
    db += dy;
  }
  const int64_t at = (int64_t)blockIdx.y * p.d + c;
  if (p.part_w) p.part_w[at] = dw;
  if (p.part_b) p.part_b[at] = db;
}

// dw[c] and db[c] from the `parts` rows of sums; 16 threads a column, each its
// rows in order, their sums then added in order.
constexpr int NORM_SUM_COLS = 64;

template <class W, class A>
__global__ void __launch_bounds__(1024) norm_sum_kernel(const A* part_w, const A* part_b, W* dw,
                                                        W* db, int64_t parts, int64_t d) {
  constexpr int S = 1024 / NORM_SUM_COLS;
  __shared__ A lds[S][NORM_SUM_COLS];
  const int c = threadIdx.x % NORM_SUM_COLS, s = threadIdx.x / NORM_SUM_COLS;
  const int64_t col = (int64_t)blockIdx.x * NORM_SUM_COLS + c;
  const A* part = blockIdx.y ? part_b : part_w;
  W* out = blockIdx.y ? db : dw;
  if (!part) return;
  A v = A(0);
  if (col < d) {
#pragma unroll 8
    for (int64_t i = s; i < parts; i += S) v += part[i * d + col];
  }
  lds[s][c] = v;
  __syncthreads();
  if (s || col >= d) return;
#pragma unroll
  for (int i = 1; i < S; ++i) v += lds[i][c];
  out[col] = (W)v;
}

template <class T, class W, int V, int G, int K>
hipError_t run_norm(NormArgs<T, W> p, bool back, int64_t parts, hipStream_t s) {
  constexpr int GROUPS = norm_block<G>() / G;
  if (back) {
    norm_grad_kernel<T, W, V, G, K><<<parts, norm_block<G>(), 0, s>>>(p);
  } else {
    const int64_t want = (p.n + GROUPS - 1) / GROUPS;
    const int64_t most = norm_most_blocks(norm_block<G>());
    norm_kernel<T, W, V, G, K><<<want < most ? want : most, norm_block<G>(), 0, s>>>(p);
  }
  return hipGetLastError();
}

template <class T, class W>
hipError_t run_norm_width(const NormParams& q) {
  using A = acc_t<T>;
  constexpr int V = 16 / (int)sizeof(T);
  const bool back = q.dy != nullptr;
  NormArgs<T, W> p{};
  p.x = (const T*)q.x;
  p.w = (const W*)q.w;
  p.b = (const W*)q.b;
  p.dy = (const T*)q.dy;
  p.y = (T*)q.y;
  p.dx = (T*)q.dx;
  p.mean = (A*)q.mean;
  p.rstd = (A*)q.rstd;
  p.n = q.n;
  p.d = q.d;
  p.eps = q.eps;
  hipStream_t s = q.stream;
  const NormGeometry geo = norm_geometry(q.n, q.d, (int)sizeof(T));
  const int64_t parts = geo.parts;
  if (q.dw) p.part_w = (A*)q.workspace;
  if (q.db) p.part_b = (A*)q.workspace + (q.dw ? parts * q.d : 0);
  hipError_t e = hipSuccess;
  switch (geo.shape) {
    case 0: e = run_norm<T, W, 1, 8, 1>(p, back, parts, s); break;
    case 1: e = run_norm<T, W, V, 8, 1>(p, back, parts, s); break;
    case 2: e = run_norm<T, W, V, 16, 1>(p, back, parts, s); break;
    case 3: e = run_norm<T, W, V, 32, 1>(p, back, parts, s); break;
    case 4: e = run_norm<T, W, V, 64, 1>(p, back, parts, s); break;
    case 5: e = run_norm<T, W, V, 64, 2>(p, back, parts, s); break;
    case 6: e = run_norm<T, W, V, 256, 1>(p, back, parts, s); break;
    case 7: e = run_norm<T, W, V, 256, 2>(p, back, parts, s); break;
    case 8: e = run_norm<T, W, V, 512, 2>(p, back, parts, s); break;
    case 9: e = run_norm<T, W, V, 512, 4>(p, back, parts, s); break;
    case 10:
      if constexpr (V <= 4) {
        e = run_norm<T, W, V, 1024, 4>(p, back, parts, s);
        break;
      }
    default: {
      const int64_t grid = q.n < 1024 ? q.n : 1024;
      if (!back) {
        norm_wide_kernel<T, W, false><<<grid, NORM_WIDE, 0, s>>>(p);
      } else {
        if (p.dx) norm_wide_kernel<T, W, true><<<grid, NORM_WIDE, 0, s>>>(p);
        if (p.part_w || p.part_b)
          norm_cols_kernel<T, W>
              <<<dim3((p.d + BLOCK - 1) / BLOCK, parts), BLOCK, 0, s>>>(p);
      }
      e = hipGetLastError();
    }
  }
  if (e != hipSuccess || !back || !(q.dw || q.db)) return e;
  norm_sum_kernel<W, A><<<dim3((q.d + NORM_SUM_COLS - 1) / NORM_SUM_COLS, 2), 1024, 0, s>>>(
      p.part_w, p.part_b, (W*)q.dw, (W*)q.db, parts, q.d);
  return hipGetLastError();
}

}  // namespace mdgl
