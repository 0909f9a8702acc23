// Gated linear recurrence over the rows of segments (included once per type).
//
//   h[t] = gate[t] * h[t-1] + value[t]         per column, h[-1] = initial or 0
//
// and its gradients, with G the gradient of h (and Gl that of a segment's last
// state), from the last row of a segment to its first:
//
//   D[t] = G[t] + gate[t+1] * D[t+1]           (G + Gl in the last row)
//   dvalue[t] = D[t],  dgate[t] = D[t] * h[t-1],  dinitial = gate[0] * D[0]
//
// Both are chains of affine maps x -> A x + B, which compose: (A1, B1) then
// (A2, B2) is (A1 A2, A2 B1 + B2). No column needs another one, so a lane holds
// 16 bytes' worth of accumulators (4 columns, 2 of double) and walks down its
// rows. The rows of all segments are one axis; bit r of `starts` / `ends` says
// that row r is the first / last of its segment, so a walk resets its state
// there and lengths never leave lanes idle. Two ways to cut that axis, by a rule
// of scan_geometry:
//
//  * owners: a walk takes the segments that start in its `len` rows, to the
//    end of the last one. It needs nothing from another walk: one launch, and
//    each row is read once;
//  * chunks, where a segment is too long for that: scan_fold_kernel reads the
//    rows and leaves each chunk's (A, B), scan_carry_kernel composes them along
//    the chunks, and the walk starts from its chunk's carry.
//
// The gradient walks 16 rows at a time: forward to have h again, in float
// whatever the rows' type (a float gate's gradient would otherwise carry the
// rounding of bfloat16 rows), from the state that the forward pass left in
// `marks` in front of every 16th row (1/16 float a value, where the states h
// themselves would be a whole one), then backward with both in registers.
//
// Across a segment's border nothing is multiplied by zero: the state is replaced,
// so an infinity or a NaN stays in its segment.
#pragma once

#include "mdgl_half.h"
#include "mdgl_kernels.h"

namespace mdgl {

constexpr int SCAN_BLOCK = 16;  // rows per block of a walk, and between marks

template <class T, class G>
struct ScanArgs {
  using A = acc_t<T>;
  const G* gate;
  const T* value;
  const A* initial;  // [segments][d], may be null: zeros
  const T* grad;     // gradient of h (backward)
  const A* grad_last;
  const int32_t* ids;
  const uint16_t* starts;
  const uint16_t* ends;
  const A* carry;  // [chunks][d] state in front of a chunk (behind it, backward); null for owners
  T* out;
  A* last;
  A* marks;  // [ceil(n / 16)][d]: written forward (may be null), read backward
  G* dgate;
  T* dvalue;
  A* dinitial;
  A* fold_a;
  A* fold_b;
  int64_t n, d, lanes, len, walks;
};

// First segment start at or behind row p (n when there is none).
__device__ __forceinline__ int64_t next_start(const uint16_t* starts, int64_t p, int64_t n) {
  if (p >= n) return n;
  int64_t b = p / SCAN_BLOCK;
  uint32_t w = starts[b] & (0xffffu << (p % SCAN_BLOCK));
  const int64_t blocks = (n + SCAN_BLOCK - 1) / SCAN_BLOCK;
  while (w == 0 && ++b < blocks) w = starts[b];
  return b < blocks ? b * SCAN_BLOCK + __builtin_ctz(w) : n;
}

// The rows [r0, r1) of a lane's walk and its first column.
template <class X, int V>
__device__ __forceinline__ bool scan_walk(const X& p, int64_t* walk, int64_t* col, int64_t* r0,
                                          int64_t* r1, bool owners) {
  const int64_t t = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
  const int64_t w = t / p.lanes;
  if (w >= p.walks) return false;
  const int64_t c = (t - w * p.lanes) * V;
  *walk = w;
  // the last lane of a row ends with it, sharing columns with the lane before
  // (both compute and write the same values)
  *col = c + V <= p.d ? c : p.d - V;
  *r0 = w * p.len;
  *r1 = *r0 + p.len < p.n ? *r0 + p.len : p.n;
  if (owners) {
    *r0 = next_start(p.starts, *r0, p.n);
    *r1 = next_start(p.starts, *r1, p.n);
  }
  return true;
}

// The block of rows from `base` that lies in [r0, r1): reads are kept inside by
// repeating the walk's first or last row.
__device__ __forceinline__ int64_t scan_row(int64_t row, int64_t r0, int64_t r1) {
  return row < r0 ? r0 : row >= r1 ? r1 - 1 : row;
}

template <class T, class G, int V>
__global__ void __launch_bounds__(BLOCK) scan_kernel(ScanArgs<T, G> p) {
  using A = acc_t<T>;
  int64_t walk, col, r0, r1;
  if (!scan_walk<ScanArgs<T, G>, V>(p, &walk, &col, &r0, &r1, !p.carry)) return;
  A h[V];
#pragma unroll
  for (int k = 0; k < V; ++k) h[k] = A(0);
  if (p.carry && r0 < r1) load_acc<A, A, V>(p.carry + walk * p.d + col, h);
  constexpr int U = SCAN_BLOCK / 2;  // rows in flight
  for (int64_t base = r0 / SCAN_BLOCK * SCAN_BLOCK; base < r1; base += SCAN_BLOCK) {
    const uint32_t first = p.starts[base / SCAN_BLOCK], end = p.ends[base / SCAN_BLOCK];
    if (p.marks && base >= r0) store_acc<A, A, V>(p.marks + base / SCAN_BLOCK * p.d + col, h);
#pragma unroll
    for (int part = 0; part < SCAN_BLOCK; part += U) {
      if (base + part >= r1 || base + part + U <= r0) continue;
      A a[U][V], v[U][V];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t at = scan_row(base + part + i, r0, r1) * p.d + col;
        load_acc<G, A, V>(p.gate + at, a[i]);
        load_acc<T, A, V>(p.value + at, v[i]);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t row = base + part + i;
        if (row < r0 || row >= r1) continue;
        if (first >> (part + i) & 1) {
          if (p.initial) load_acc<A, A, V>(p.initial + (int64_t)p.ids[row] * p.d + col, h);
          else
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = A(0);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = fma_of(a[i][k], h[k], v[i][k]);
        store_acc<T, A, V>(p.out + row * p.d + col, h);
        if (p.last && (end >> (part + i) & 1))
          store_acc<A, A, V>(p.last + (int64_t)p.ids[row] * p.d + col, h);
      }
    }
  }
}

template <class T, class G, int V>
__global__ void __launch_bounds__(BLOCK) scan_grad_kernel(ScanArgs<T, G> p) {
  using A = acc_t<T>;
  constexpr int U = SCAN_BLOCK;
  int64_t walk, col, r0, r1;
  if (!scan_walk<ScanArgs<T, G>, V>(p, &walk, &col, &r0, &r1, !p.carry)) return;
  if (r0 >= r1) return;
  A c[V];  // gate[t + 1] * D[t + 1]
#pragma unroll
  for (int k = 0; k < V; ++k) c[k] = A(0);
  if (p.carry) load_acc<A, A, V>(p.carry + walk * p.d + col, c);
  const int64_t lowest = r0 / SCAN_BLOCK * SCAN_BLOCK;
  for (int64_t base = (r1 - 1) / SCAN_BLOCK * SCAN_BLOCK; base >= lowest; base -= SCAN_BLOCK) {
    const uint32_t first = p.starts[base / SCAN_BLOCK], end = p.ends[base / SCAN_BLOCK];
    A a[U][V], before[U][V], g[U][V];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = scan_row(base + i, r0, r1) * p.d + col;
      load_acc<G, A, V>(p.gate + at, a[i]);
      load_acc<T, A, V>(p.grad + at, g[i]);
      if (p.dgate) load_acc<T, A, V>(p.value + at, before[i]);
    }
    if (p.dgate) {  // the states in front of each row
      A h[V];
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = A(0);
      // a walk that does not hold the block's first row starts at a segment's
      if (base >= r0) load_acc<A, A, V>(p.marks + base / SCAN_BLOCK * p.d + col, h);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t row = base + i;
        if (row < r0 || row >= r1) continue;
        if (first >> i & 1) {
          if (p.initial) load_acc<A, A, V>(p.initial + (int64_t)p.ids[row] * p.d + col, h);
          else
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = A(0);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const A next = fma_of(a[i][k], h[k], before[i][k]);
          before[i][k] = h[k];
          h[k] = next;
        }
      }
    }
#pragma unroll
    for (int i = U - 1; i >= 0; --i) {
      const int64_t row = base + i;
      if (row < r0 || row >= r1) continue;
      if (end >> i & 1) {
        if (p.grad_last) load_acc<A, A, V>(p.grad_last + (int64_t)p.ids[row] * p.d + col, c);
        else
#pragma unroll
          for (int k = 0; k < V; ++k) c[k] = A(0);
      }
      A da[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        g[i][k] = g[i][k] + c[k];
        c[k] = a[i][k] * g[i][k];
      }
      if (p.dvalue) store_acc<T, A, V>(p.dvalue + row * p.d + col, g[i]);
      if (p.dgate) {
#pragma unroll
        for (int k = 0; k < V; ++k) da[k] = g[i][k] * before[i][k];
        store_acc<G, A, V>(p.dgate + row * p.d + col, da);
      }
      if (p.dinitial && (first >> i & 1))
        store_acc<A, A, V>(p.dinitial + (int64_t)p.ids[row] * p.d + col, c);
    }
  }
}

// A chunk's map of the state in front of it to the state behind it (BACK: of the
// gradient behind it to the one in front). A chunk that holds a segment's border
// has a B only (its A is not read).
template <class T, class G, int V, bool BACK>
__global__ void __launch_bounds__(BLOCK) scan_fold_kernel(ScanArgs<T, G> p) {
  using A = acc_t<T>;
  constexpr int U = SCAN_BLOCK;
  int64_t walk, col, r0, r1;
  if (!scan_walk<ScanArgs<T, G>, V>(p, &walk, &col, &r0, &r1, false)) return;
  A fa[V], fb[V];
#pragma unroll
  for (int k = 0; k < V; ++k) { fa[k] = A(1); fb[k] = A(0); }
  const T* x = BACK ? p.grad : p.value;
  const A* edge = BACK ? p.grad_last : p.initial;
  const int64_t blocks = (r1 - r0 + SCAN_BLOCK - 1) / SCAN_BLOCK;
  for (int64_t b = 0; b < blocks; ++b) {
    const int64_t base = r0 + (BACK ? blocks - 1 - b : b) * SCAN_BLOCK;
    const uint32_t edges = (BACK ? p.ends : p.starts)[base / SCAN_BLOCK];
    A a[U][V], v[U][V];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = scan_row(base + i, r0, r1) * p.d + col;
      load_acc<G, A, V>(p.gate + at, a[i]);
      load_acc<T, A, V>(x + at, v[i]);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = BACK ? U - 1 - j : j;
      const int64_t row = base + i;
      if (row >= r1) continue;
      if (edges >> i & 1) {
        if (edge) load_acc<A, A, V>(edge + (int64_t)p.ids[row] * p.d + col, fb);
        else
#pragma unroll
          for (int k = 0; k < V; ++k) fb[k] = A(0);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        fa[k] = fa[k] * a[i][k];
        fb[k] = BACK ? a[i][k] * (v[i][k] + fb[k]) : fma_of(a[i][k], fb[k], v[i][k]);
      }
    }
  }
  store_acc<A, A, V>(p.fold_a + walk * p.d + col, fa);
  store_acc<A, A, V>(p.fold_b + walk * p.d + col, fb);
}

// x through the map (a, b): a state of 0 leaves b whatever a is (a product of
// gates that overflowed stays out of a segment that starts from nothing).
template <class A>
__device__ __forceinline__ A scan_apply(A a, A b, A x) {
  return x == A(0) ? b : fma_of(a, x, b);
}

// carry[c] = the state in front of chunk c (BACK: the gradient behind it), from
// the chunks' maps. A workgroup takes `wide` lanes of columns; its threads are
// wide lanes times parts of the chunks. Each part composes its chunks' maps, the
// parts' maps are scanned in LDS, and each part goes over its chunks again with
// its carry, which replaces fold_a.
constexpr int CARRY_BLOCK = 1024;

template <class A, int V, bool BACK>
__global__ void __launch_bounds__(CARRY_BLOCK) scan_carry_kernel(
    A* fold_a, const A* fold_b, const uint16_t* edges, int64_t n, int64_t d, int64_t lanes,
    int64_t chunks, int64_t len, int wide) {
  __shared__ A sa[CARRY_BLOCK][V], sb[CARRY_BLOCK][V];
  __shared__ uint8_t sk[CARRY_BLOCK];
  const int parts = CARRY_BLOCK / wide, part = threadIdx.x / wide;
  const int64_t lane = (int64_t)blockIdx.x * wide + threadIdx.x % wide;
  const int64_t c0 = lane * V, col = c0 + V <= d ? c0 : d - V;
  const bool live = lane < lanes;
  const int64_t per = (chunks + parts - 1) / parts;
  const int64_t lo = part * per < chunks ? part * per : chunks;
  const int64_t hi = live ? (lo + per < chunks ? lo + per : chunks) : lo;
  const int64_t blocks = (n + SCAN_BLOCK - 1) / SCAN_BLOCK, step = len / SCAN_BLOCK;
  auto chunk = [&](int64_t i) { return BACK ? chunks - 1 - i : i; };
  auto broken = [&](int64_t c) {
    uint32_t any = 0;
    for (int64_t b = c * step; b < (c + 1) * step && b < blocks; ++b) any |= edges[b];
    return any != 0;
  };
  A fa[V], fb[V];
#pragma unroll
  for (int k = 0; k < V; ++k) { fa[k] = A(1); fb[k] = A(0); }
  bool cut = false;
  for (int64_t i = lo; i < hi; ++i) {
    const int64_t c = chunk(i);
    A a[V], b[V];
    load_acc<A, A, V>(fold_a + c * d + col, a);
    load_acc<A, A, V>(fold_b + c * d + col, b);
    const bool k1 = broken(c);
    cut |= k1;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      fa[k] = fa[k] * a[k];
      fb[k] = k1 ? b[k] : scan_apply(a[k], b[k], fb[k]);
    }
  }
  // inclusive scan of the parts' maps
  const int me = threadIdx.x;
  for (int off = 1; off < parts; off <<= 1) {
#pragma unroll
    for (int k = 0; k < V; ++k) { sa[me][k] = fa[k]; sb[me][k] = fb[k]; }
    sk[me] = cut;
    __syncthreads();
    if (part >= off) {
      const int o = me - off * wide;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        fb[k] = cut ? fb[k] : scan_apply(fa[k], fb[k], sb[o][k]);
        fa[k] = sa[o][k] * fa[k];
      }
      cut |= sk[o] != 0;
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < V; ++k) sb[me][k] = fb[k];
  __syncthreads();
  A x[V];
#pragma unroll
  for (int k = 0; k < V; ++k) x[k] = part ? sb[me - wide][k] : A(0);
  for (int64_t i = lo; i < hi; ++i) {
    const int64_t c = chunk(i);
    A a[V], b[V];
    load_acc<A, A, V>(fold_a + c * d + col, a);
    load_acc<A, A, V>(fold_b + c * d + col, b);
    const bool k1 = broken(c);
    store_acc<A, A, V>(fold_a + c * d + col, x);
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = k1 ? b[k] : scan_apply(a[k], b[k], x[k]);
  }
}

// Rows of `to` of the empty segments: a copy of `from`, zeros where it is null.
template <class A>
__global__ void __launch_bounds__(BLOCK) scan_empty_kernel(const int32_t* off, const A* from,
                                                           A* to, int64_t num_seg, int64_t d) {
  const int64_t step = (int64_t)gridDim.x * BLOCK;
  for (int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x; i < num_seg * d; i += step) {
    const int64_t s = i / d;
    if (off[s] == off[s + 1]) to[i] = from ? from[i] : A(0);
  }
}

// One row of every sequence: state' = gate * state + value, out = state' rounded
// to the rows' type. `next` may be `state` itself.
template <class T, class G, int V>
__global__ void __launch_bounds__(BLOCK) scan_step_kernel(const G* gate, const T* value,
                                                          const acc_t<T>* state, T* out,
                                                          acc_t<T>* next, int64_t n) {
  using A = acc_t<T>;
  const int64_t i = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * V;
  if (i + V <= n) {
    A a[V], v[V], h[V];
    load_acc<G, A, V>(gate + i, a);
    load_acc<T, A, V>(value + i, v);
    load_acc<A, A, V>(state + i, h);
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = fma_of(a[k], h[k], v[k]);
    store_acc<T, A, V>(out + i, h);
    store_acc<A, A, V>(next + i, h);
  } else {
    for (int64_t j = i; j < n; ++j) {
      const A h = fma_of((A)gate[j], state[j], (A)value[j]);
      out[j] = (T)h;
      next[j] = h;
    }
  }
}

inline int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <class T, class G, int V>
hipError_t run_scan(const ScanParams& q, const ScanGeometry& geo, bool back) {
  using A = acc_t<T>;
  hipStream_t s = q.stream;
  ScanArgs<T, G> p{};
  p.gate = (const G*)q.gate;
  p.value = (const T*)q.value;
  p.initial = (const A*)q.initial;
  p.grad = (const T*)q.grad;
  p.grad_last = (const A*)q.grad_last;
  p.ids = q.ids;
  p.starts = (const uint16_t*)q.starts;
  p.ends = (const uint16_t*)q.ends;
  p.out = (T*)q.out;
  p.last = (A*)q.last;
  p.marks = (A*)q.marks;
  p.dgate = (G*)q.dgate;
  p.dvalue = (T*)q.dvalue;
  p.dinitial = (A*)q.dinitial;
  p.n = q.n;
  p.d = q.d;
  p.lanes = ceil_div64(q.d, V);
  p.len = geo.len;
  p.walks = ceil_div64(q.n, geo.len);
  if (q.n > 0) {
    const int64_t grid = ceil_div64(p.walks * p.lanes, BLOCK);
    if (!geo.owners) {
      A* fa = (A*)q.workspace;
      A* fb = fa + p.walks * p.d;
      p.fold_a = fa;
      p.fold_b = fb;
      p.carry = fa;
      int wide = 16;
      while (wide > 1 && wide / 2 >= p.lanes) wide /= 2;
      const int64_t cgrid = ceil_div64(p.lanes, wide);
      if (back) {
        scan_fold_kernel<T, G, V, true><<<grid, BLOCK, 0, s>>>(p);
        scan_carry_kernel<A, V, true><<<cgrid, CARRY_BLOCK, 0, s>>>(
            fa, fb, p.ends, p.n, p.d, p.lanes, p.walks, p.len, wide);
      } else {
        scan_fold_kernel<T, G, V, false><<<grid, BLOCK, 0, s>>>(p);
        scan_carry_kernel<A, V, false><<<cgrid, CARRY_BLOCK, 0, s>>>(
            fa, fb, p.starts, p.n, p.d, p.lanes, p.walks, p.len, wide);
      }
    }
    if (back) scan_grad_kernel<T, G, V><<<grid, BLOCK, 0, s>>>(p);
    else scan_kernel<T, G, V><<<grid, BLOCK, 0, s>>>(p);
  }
  A* edge_to = back ? p.dinitial : p.last;
  if (q.has_empty && edge_to) {
    const int64_t want = ceil_div64(q.num_seg * q.d, BLOCK);
    scan_empty_kernel<A><<<want < 2048 ? want : 2048, BLOCK, 0, s>>>(
        q.offsets, back ? p.grad_last : p.initial, edge_to, q.num_seg, q.d);
  }
  return hipGetLastError();
}

template <class T, class G>
hipError_t run_scan_width(const ScanParams& q, const ScanGeometry& geo, bool back) {
  if (q.d >= acc_vec<T>()) return run_scan<T, G, acc_vec<T>()>(q, geo, back);
  return run_scan<T, G, 1>(q, geo, back);
}

template <class T, class G>
hipError_t run_scan_step(const ScanStepParams& q) {
  constexpr int V = acc_vec<T>();
  scan_step_kernel<T, G, V><<<ceil_div64(q.n, (int64_t)BLOCK * V), BLOCK, 0, q.stream>>>(
      (const G*)q.gate, (const T*)q.value, (const acc_t<T>*)q.state, (T*)q.out,
      (acc_t<T>*)q.next, q.n);
  return hipGetLastError();
}

}  // namespace mdgl
