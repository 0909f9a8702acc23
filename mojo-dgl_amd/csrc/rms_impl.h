// Root-mean-square norm over the last axis with the residual's addition in front,
// its gradients, and its output in 8 bits (included once per type).
//
//   t = x + residual (x without one),  r = 1 / sqrt(sum t^2 / d + eps),  xh = t r
//   y = xh w,  total = t rounded to the residual's type
//   dt = r (g - xh sum(g xh) / d) + dtotal,  g = dy w;  dx and dresidual are dt
//   dw = sum over rows of dy xh
//
// y is formed from the unrounded sum, and so are the gradients: from `total` where that
// is float (double for double rows), else from x and the residual once more (dw of
// 32,768 rows is off by 2e-7 of its size so, by 1e-5 from a bfloat16 total). Rows lie on
// threads as layer norm's do (norm_geometry): a group of threads holds a row in
// registers, so each row is read and written once, with the next one's loads in flight;
// the weight's gradient is summed in registers, 16 rows at a time, these sums in LDS, and
// one row of sums a workgroup is added by norm_sum_kernel, all in a fixed order. In 8 bits
// the 128 columns of a block lie on 128 / V neighbouring lanes, whose maximum goes through
// DPP.
//
// Bound by memory: 32,768 bfloat16 rows of 4,096 with a bfloat16 residual take 473 us
// forward and backward (nine rows of 268 MB read and written, 5.1 TB/s), 200,000 float32
// rows of 602 without one 463 us (five of 482 MB, 5.3 TB/s), 32,768 rows of 5,120 with
// a float32 residual in 8 bits 354 us (1.85 GB, 5.2 TB/s), where a copy of 1 GiB runs at
// 5.2 TB/s.
#pragma once

#include "norm_impl.h"
#include "quant.h"

namespace mdgl {

template <class T, class W, class R>
struct RmsArgs {
  using A = acc_t<T>;
  const T* x;
  const R* r;  // may be null; backward it is added to `total`
  const W* w;  // may be null: 1
  T* y;
  uint8_t* y8;   // instead of y
  float* scale;  // [n][ceil(d / 128)] with y8
  R* total;      // may be null forward
  A* rstd;       // may be null forward
  const T* dy;
  const R* dtotal;  // may be null
  T* dx;            // may be null
  R* dr;            // may be null
  A* part_w;        // [workgroups][d] (may be null)
  int64_t n, d;
  double eps;
};

// Vector j of a thread (fewer than 2^26 columns): whether it lies in the row, its
// first column, and how many of its columns the vector before it has, too.
template <int V, int G>
struct RmsCols {
  int t, d;
  // With 1,024 threads nothing of this is carried from row to row: the registers that
  // would take put others in memory.
  __device__ __forceinline__ void renew() {
    if constexpr (G == 1024) asm volatile("" : "+v"(t));
  }
  __device__ __forceinline__ int at(int j) const { return (t + j * G) * V; }
  __device__ __forceinline__ bool live(int j) const { return at(j) < d; }
  __device__ __forceinline__ int col(int j) const { return at(j) + V <= d ? at(j) : d - V; }
  __device__ __forceinline__ int skip(int j) const { return at(j) + V <= d ? 0 : at(j) - (d - V); }
};

// 1 / sqrt(v). In float the root's and the quotient's roundings, exact in one fma each, are
// put right: a row's values all carry this error (y's is 15 % less so).
__device__ __forceinline__ double rms_rsqrt(double v) { return 1.0 / sqrt(v); }
__device__ __forceinline__ float rms_rsqrt(float v) {
  const float s = sqrtf(v), r = 1.0f / s;
  const float e = __builtin_fmaf(-s, s, v), d = __builtin_fmaf(-s, r, 1.0f);
  const float c = r * (d - 0.5f * e * (r * r));
  return __builtin_fabsf(c) < r ? r + c : r;  // not where v is 0 or infinite
}

// One sum over the G threads of a group.
template <int G, class A>
__device__ __forceinline__ A rms_sum(A a, A* lds, int& turn) {
  A none = A(0);
  norm_sum2<G>(a, none, lds, turn);
  return a;
}

template <class T, class W, class R, int V, int G, int K, bool Q>
__global__ void __launch_bounds__(norm_block<G>()) rms_kernel(RmsArgs<T, W, R> p) {
  using A = acc_t<T>;
  constexpr int GROUPS = norm_block<G>() / G;
  __shared__ A lds[G > WAVE ? 4 * (G / WAVE) : 1];
  int turn = 0;
  const int t = threadIdx.x % G;
  RmsCols<V, G> own{t, (int)p.d};
  // 1,024 threads have no registers for w
  constexpr bool HOLD = G < 1024;
  A w[HOLD ? K : 1][V];
#pragma unroll
  for (int j = 0; j < K; ++j) {
#pragma unroll
    for (int k = 0; k < V; ++k) w[HOLD ? j : 0][k] = A(1);
    if (HOLD && own.live(j) && p.w) load_acc<W, A, V>(p.w + own.col(j), w[HOLD ? j : 0]);
  }
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const A inv = A(1) / (A)p.d;
  int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G;
  Held<T, V> xn[K];
  Held<R, V> rn[K];
  auto fetch = [&](int64_t at) {
    if (at >= p.n) return;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (!own.live(j)) continue;
      xn[j].load(p.x + at * p.d + own.col(j));
      if (p.r) rn[j].load(p.r + at * p.d + own.col(j));
    }
  };
  fetch(row);
  while (row < p.n) {
    own.renew();
    A x[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        x[j][k] = own.live(j) ? xn[j].at(k) : A(0);
        if (p.r && own.live(j)) x[j][k] += (A)rn[j].at(k);
      }
    const int64_t next = row + step;
    fetch(next);
    // columns that the vector before has are left out of the sum, not multiplied by 0,
    // which an infinity turns into a NaN
    A q = A(0);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) q = k >= own.skip(j) ? fma_of(x[j][k], x[j][k], q) : q;
    const A r = rms_rsqrt(rms_sum<G>(q, lds, turn) * inv + (A)p.eps);
    if (p.rstd && t == 0) p.rstd[row] = r;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (p.total && own.live(j)) store_acc<R, A, V>(p.total + row * p.d + own.col(j), x[j]);
      if (!HOLD && own.live(j) && p.w) load_acc<W, A, V>(p.w + own.col(j), w[0]);
#pragma unroll
      for (int k = 0; k < V; ++k) x[j][k] = x[j][k] * r * w[HOLD ? j : 0][k];
      if constexpr (!Q) {
        if (own.live(j)) store_acc<T, A, V>(p.y + row * p.d + own.col(j), x[j]);
      } else {
        // every lane of the group takes part in the maximum
        constexpr int LANES = G < Q_BLOCK / V ? G : Q_BLOCK / V;
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k)
          top = fmaxf(top, own.live(j) && k >= own.skip(j) ? __builtin_fabsf((float)x[j][k]) : 0.0f);
        const QuantBy by(quant_scale(group_max(top, LANES)));
        if (!own.live(j)) continue;
        const int64_t c = own.col(j) + own.skip(j);  // the first column that is this lane's
        if (c % Q_BLOCK == 0)
          p.scale[row * ((p.d + Q_BLOCK - 1) / Q_BLOCK) + c / Q_BLOCK] = by.s;
        uint8_t* out = p.y8 + row * p.d + own.col(j);
        bool whole = false;
        if constexpr (V % 4 == 0) {
          whole = own.skip(j) == 0;
          if (whole) {
            uint32_t words[V / 4];
#pragma unroll
            for (int k = 0; k < V; k += 4)
              words[k / 4] = by.word((float)x[j][k], (float)x[j][k + 1], (float)x[j][k + 2],
                                     (float)x[j][k + 3]);
            __builtin_memcpy(out, words, V);
          }
        }
        // columns that another lane has may belong to its block
        if (!whole)
#pragma unroll
          for (int k = 0; k < V; ++k)
            if (k >= own.skip(j)) out[k] = by.byte((float)x[j][k]);
      }
    }
    row = next;
  }
}

template <class T, class W, class R, int V, int G, int K>
__global__ void __launch_bounds__(norm_block<G>()) rms_grad_kernel(RmsArgs<T, W, R> p) {
  using A = acc_t<T>;
  constexpr int GROUPS = norm_block<G>() / G;
  // the registers of four vectors a thread: none for w, and with 1,024 threads or a
  // float32 total beside 16-bit rows none for the next row's loads or dtotal either
  constexpr bool HOLD = K < 4, AHEAD = K < 4 || (G < 1024 && sizeof(R) == sizeof(T));
  __shared__ A lds[G > WAVE ? 4 * (G / WAVE) : 1];
  __shared__ A sums[GROUPS > 1 ? G * K * V : 1];
  // dw's sums of RUN rows each are added up here, a thread's own: one chain over all of its
  // rows loses bits (200,000 float32 rows of 602, 195 in a chain: dw is off by 3.2e-7 of its
  // size, so by 2.1e-7, at the same time)
  constexpr int RUN = 16;
  __shared__ A kept[K * V][norm_block<G>()];
  int turn = 0, run = 0;
  bool some = false;  // in `kept`
  const int t = threadIdx.x % G, group = threadIdx.x / G;
  RmsCols<V, G> own{t, (int)p.d};
  A w[HOLD ? K : 1][V], dw[K][V];
#pragma unroll
  for (int j = 0; j < K; ++j) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (HOLD) w[HOLD ? j : 0][k] = A(1);
      dw[j][k] = A(0);
    }
    if (HOLD && own.live(j) && p.w) load_acc<W, A, V>(p.w + own.col(j), w[HOLD ? j : 0]);
  }
  auto keep = [&](bool take) {
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A& at = kept[j * V + k][threadIdx.x];
        if (some) dw[j][k] += at;
        if (!take) {
          at = dw[j][k];
          dw[j][k] = A(0);
        }
      }
    some = true;
  };
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const A inv = A(1) / (A)p.d;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  // sums that were rounded to 16 bits are formed again
  constexpr bool SUM = sizeof(R) == 2;
  Held<R, V> xn[K], rn[SUM ? K : 1], tn[K];
  Held<T, V> gn[K];
  A r_n = A(0);
  auto fetch = [&](int64_t at) {
    if (at >= p.n) return;
    r_n = p.rstd[at];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (!own.live(j)) continue;
      xn[j].load(p.total + at * p.d + own.col(j));
      if (SUM && p.r) rn[SUM ? j : 0].load(p.r + at * p.d + own.col(j));
      gn[j].load(p.dy + at * p.d + own.col(j));
      if (AHEAD && p.dtotal) tn[j].load(p.dtotal + at * p.d + own.col(j));
    }
  };
  fetch(row);
  while (row < p.n) {
    own.renew();
    Held<R, V> x[K], y[SUM ? K : 1], dt[K];
    Held<T, V> g[K];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      x[j] = xn[j];
      if (SUM) y[SUM ? j : 0] = rn[SUM ? j : 0];
      g[j] = gn[j];
      dt[j] = tn[j];
    }
    const A r = r_n;
    const int64_t next = row + step;
    if (AHEAD) fetch(next);
    A q = A(0);
    auto form = [&](int j, A (&xh)[V], A (&dy)[V], A (&gw)[V]) {
      if constexpr (!HOLD) {
#pragma unroll
        for (int k = 0; k < V; ++k) w[0][k] = A(1);
        if (p.w) load_acc<W, A, V>(p.w + own.col(j), w[0]);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dy[k] = g[j].at(k);
        A t = (A)x[j].at(k);
        if (SUM && p.r) t += (A)y[SUM ? j : 0].at(k);
        xh[k] = t * r;
        gw[k] = dy[k] * w[HOLD ? j : 0][k];
      }
    };
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (!own.live(j)) continue;
      A xh[V], dy[V], gw[V];
      form(j, xh, dy, gw);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dw[j][k] = fma_of(dy[k], xh[k], dw[j][k]);
        q = k >= own.skip(j) ? fma_of(gw[k], xh[k], q) : q;
      }
    }
    if (p.dx || p.dr) {
      q = rms_sum<G>(q, lds, turn) * inv;
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (!own.live(j)) continue;
        if (!AHEAD && p.dtotal) dt[j].load(p.dtotal + row * p.d + own.col(j));
        A xh[V], dy[V], gw[V];
        form(j, xh, dy, gw);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          gw[k] = r * (gw[k] - xh[k] * q);
          if (p.dtotal) gw[k] += (A)dt[j].at(k);
        }
        if (p.dx) store_acc<T, A, V>(p.dx + row * p.d + own.col(j), gw);
        if (p.dr) store_acc<R, A, V>(p.dr + row * p.d + own.col(j), gw);
      }
    }
    if (!AHEAD) fetch(next);
    row = next;
    if (++run == RUN) {
      run = 0;
      keep(false);
    }
  }
  if (!p.part_w) return;
  if (some) keep(true);
  if constexpr (GROUPS > 1) {
    // the groups of the workgroup one after the other
    for (int i = 0; i < GROUPS; ++i) {
      if (group == i) {
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
          for (int k = 0; k < V; ++k) {
            A* s = sums + (t + j * G) * V + k;
            if (i) dw[j][k] += s[0];
            s[0] = dw[j][k];
          }
      }
      __syncthreads();
    }
    if (group != GROUPS - 1) return;
  }
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (own.live(j))
      store_acc<A, A, V>(p.part_w + (int64_t)blockIdx.x * p.d + own.col(j), dw[j]);
  }
}

// The sum whose gradient is wanted, at place `i`.
template <class T, class W, class R>
__device__ __forceinline__ acc_t<T> rms_total(const RmsArgs<T, W, R>& p, int64_t i) {
  using A = acc_t<T>;
  return (A)p.total[i] + (p.r ? (A)p.r[i] : A(0));
}

// Rows wider than a workgroup's registers: a workgroup a row, read again from the
// caches for each use. GRAD: dx and dresidual; Q: y in 8 bits, a wavefront a block.
template <class T, class W, class R, bool GRAD, bool Q>
__global__ void __launch_bounds__(NORM_WIDE) rms_wide_kernel(RmsArgs<T, W, R> p) {
  using A = acc_t<T>;
  __shared__ A lds[4 * (NORM_WIDE / WAVE)];
  int turn = 0;
  const A inv = A(1) / (A)p.d;
  for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
    const int64_t at = row * p.d;
    auto weight = [&](int64_t c) { return p.w ? (A)p.w[c] : A(1); };
    A q = A(0);
    if constexpr (GRAD) {
      const A r = p.rstd[row];
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE)
        q = fma_of((A)p.dy[at + c] * weight(c), rms_total(p, at + c) * r, q);
      q = rms_sum<NORM_WIDE>(q, lds, turn) * inv;
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) {
        A dt = r * ((A)p.dy[at + c] * weight(c) - rms_total(p, at + c) * r * q);
        if (p.dtotal) dt += (A)p.dtotal[at + c];
        if (p.dx) p.dx[at + c] = (T)dt;
        if (p.dr) p.dr[at + c] = (R)dt;
      }
    } else {
      auto value = [&](int64_t c) { return (A)p.x[at + c] + (p.r ? (A)p.r[at + c] : A(0)); };
      for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) {
        const A v = value(c);
        q = fma_of(v, v, q);
      }
      const A r = rms_rsqrt(rms_sum<NORM_WIDE>(q, lds, turn) * inv + (A)p.eps);
      if (p.rstd && threadIdx.x == 0) p.rstd[row] = r;
      if constexpr (!Q) {
        for (int64_t c = threadIdx.x; c < p.d; c += NORM_WIDE) {
          const A v = value(c);
          if (p.total) p.total[at + c] = (R)v;
          p.y[at + c] = (T)(v * r * weight(c));
        }
      } else {
        const int64_t blocks = (p.d + Q_BLOCK - 1) / Q_BLOCK;
        const int lane = threadIdx.x % WAVE;
        for (int64_t b = threadIdx.x / WAVE; b < blocks; b += NORM_WIDE / WAVE) {
          float y[2], top = 0.0f;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int64_t c = b * Q_BLOCK + i * WAVE + lane;
            y[i] = 0.0f;
            if (c >= p.d) continue;
            const A v = value(c);
            if (p.total) p.total[at + c] = (R)v;
            y[i] = (float)(v * r * weight(c));
            top = fmaxf(top, __builtin_fabsf(y[i]));
          }
          const QuantBy by(quant_scale(group_max(top, WAVE)));
          if (lane == 0) p.scale[row * blocks + b] = by.s;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int64_t c = b * Q_BLOCK + i * WAVE + lane;
            if (c < p.d) p.y8[at + c] = by.byte(y[i]);
          }
        }
      }
    }
  }
}

// dw of such rows: a thread a column, blockIdx.y a run of rows.
template <class T, class W, class R>
__global__ void __launch_bounds__(BLOCK) rms_cols_kernel(RmsArgs<T, W, R> p) {
  using A = acc_t<T>;
  const int64_t c = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
  if (c >= p.d) return;
  A dw = A(0);
  for (int64_t row = blockIdx.y; row < p.n;) {
    A some = A(0);  // of 16 rows (as in rms_grad_kernel)
#pragma unroll 1
    for (int i = 0; i < 16 && row < p.n; ++i, row += gridDim.y)
      some = fma_of((A)p.dy[row * p.d + c], rms_total(p, row * p.d + c) * p.rstd[row], some);
    dw += some;
  }
  p.part_w[(int64_t)blockIdx.y * p.d + c] = dw;
}

template <class T, class W, class R, int V, int G, int K>
hipError_t run_rms(const RmsArgs<T, W, R>& p, bool back, int64_t parts, hipStream_t s) {
  constexpr int GROUPS = norm_block<G>() / G;
  const int64_t want = (p.n + GROUPS - 1) / GROUPS;
  const int64_t most = norm_most_blocks(norm_block<G>());
  const int64_t grid = want < most ? want : most;
  if (back) {
    rms_grad_kernel<T, W, R, V, G, K><<<parts, norm_block<G>(), 0, s>>>(p);
  } else if (!p.y8) {
    rms_kernel<T, W, R, V, G, K, false><<<grid, norm_block<G>(), 0, s>>>(p);
  } else {
    // float64 rows have no output in 8 bits (refused before)
    if constexpr (sizeof(T) < 8)
      rms_kernel<T, W, R, V, G, K, true><<<grid, norm_block<G>(), 0, s>>>(p);
  }
  return hipGetLastError();
}

template <class T, class W, class R>
hipError_t run_rms_width(const RmsParams& q) {
  using A = acc_t<T>;
  constexpr int V = 16 / (int)sizeof(T);
  const bool back = q.dy != nullptr;
  RmsArgs<T, W, R> p{};
  p.x = (const T*)q.x;
  p.r = (const R*)q.residual;
  p.w = (const W*)q.w;
  p.y = q.scale ? nullptr : (T*)q.y;
  p.y8 = q.scale ? (uint8_t*)q.y : nullptr;
  p.scale = (float*)q.scale;
  p.total = (R*)q.total;
  p.rstd = (A*)q.rstd;
  p.dy = (const T*)q.dy;
  p.dtotal = (const R*)q.dtotal;
  p.dx = (T*)q.dx;
  p.dr = (R*)q.dresidual;
  p.part_w = q.dw ? (A*)q.workspace : nullptr;
  p.n = q.n;
  p.d = q.d;
  p.eps = q.eps;
  hipStream_t s = q.stream;
  const NormGeometry geo = norm_geometry(q.n, q.d, (int)sizeof(T));
  const int64_t parts = geo.parts;
  hipError_t e = hipSuccess;
  switch (geo.shape) {
    case 0: e = run_rms<T, W, R, 1, 8, 1>(p, back, parts, s); break;
    case 1: e = run_rms<T, W, R, V, 8, 1>(p, back, parts, s); break;
    case 2: e = run_rms<T, W, R, V, 16, 1>(p, back, parts, s); break;
    case 3: e = run_rms<T, W, R, V, 32, 1>(p, back, parts, s); break;
    case 4: e = run_rms<T, W, R, V, 64, 1>(p, back, parts, s); break;
    case 5: e = run_rms<T, W, R, V, 64, 2>(p, back, parts, s); break;
    case 6: e = run_rms<T, W, R, V, 256, 1>(p, back, parts, s); break;
    case 7: e = run_rms<T, W, R, V, 256, 2>(p, back, parts, s); break;
    case 8: e = run_rms<T, W, R, V, 512, 2>(p, back, parts, s); break;
    case 9: e = run_rms<T, W, R, V, 512, 4>(p, back, parts, s); break;
    case 10:
      if constexpr (V <= 4) {
        e = run_rms<T, W, R, V, 1024, 4>(p, back, parts, s);
        break;
      }
    default: {
      const int64_t grid = q.n < 1024 ? q.n : 1024;
      if (!back) {
        if (!p.y8) {
          rms_wide_kernel<T, W, R, false, false><<<grid, NORM_WIDE, 0, s>>>(p);
        } else {
          if constexpr (sizeof(T) < 8)
            rms_wide_kernel<T, W, R, false, true><<<grid, NORM_WIDE, 0, s>>>(p);
        }
      } else {
        if (p.dx || p.dr) rms_wide_kernel<T, W, R, true, false><<<grid, NORM_WIDE, 0, s>>>(p);
        if (p.part_w)
          rms_cols_kernel<T, W, R>
              <<<dim3((p.d + BLOCK - 1) / BLOCK, parts), BLOCK, 0, s>>>(p);
      }
      e = hipGetLastError();
    }
  }
  if (e != hipSuccess || !back || !q.dw) return e;
  norm_sum_kernel<W, A><<<dim3((q.d + NORM_SUM_COLS - 1) / NORM_SUM_COLS, 1), 1024, 0, s>>>(
      p.part_w, nullptr, (W*)q.dw, nullptr, parts, q.d);
  return hipGetLastError();
}

// The instance of a call: weights and residuals in the rows' type or, beside 16-bit
// rows, in float32.
template <class T>
hipError_t run_rms_types(const RmsParams& q) {
  if constexpr (sizeof(T) == 2) {
    if (q.weight_f32)
      return q.residual_f32 ? run_rms_width<T, float, float>(q) : run_rms_width<T, float, T>(q);
    return q.residual_f32 ? run_rms_width<T, T, float>(q) : run_rms_width<T, T, T>(q);
  } else {
    return run_rms_width<T, T, T>(q);
  }
}

}  // namespace mdgl
