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
// (A2, B2) is (A1 A2, A2 B1 + B2). The rows of all segments are one axis, cut into
// chunks of equal size whatever the lengths: bit r of `starts` / `ends` says that
// row r is the first / last of its segment, and a walk replaces its state there
// (nothing is multiplied by zero, so an infinity or a NaN stays in its segment).
// Within it an infinite state times a product of gates that underflowed to 0 is a NaN.
// Telling that product from one with a gate of 0, where a NaN is right, took 5 to 10 %
// of every scan's time, and 30 % of a long one with gates of 0.
//
// scan_pass_kernel reads each row once. A workgroup holds its chunk's rows in
// registers, 16 rows of two columns a thread, composes their maps (in the thread,
// then over the threads of a column in LDS), publishes the chunk's map, and looks
// back along the chunks in front of it for the state it starts from (a scan by
// decoupled look-back; by groups of chunks, look_back() says why). With that state
// it goes over its registers again and writes. The one other launch resets what
// chunks publish; a single chunk needs neither.
//
// The gradient's walk runs the other way. It has h again from gate and value, in
// float whatever the rows' type (a float gate's gradient would otherwise carry the
// rounding of bfloat16 rows), and from the state that the forward pass left in
// `marks` in front of every 16th row: 1/16 float a value, where h itself would be
// a whole one.
#pragma once

#include <type_traits>

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
  T* out;
  A* last;
  A* marks;  // [ceil(n / 16)][d]: written forward (may be null), read backward
  G* dgate;
  T* dvalue;
  A* dinitial;
  int64_t n, d, lanes, chunks;
  uint32_t* ticket;
  A* words;       // [chunks][2][d]: A, B; then those of groups, and groups' states
  int64_t tiles;  // of `wide` lanes of columns
  int wide;       // a power of two, 1 to 64
};

// x through the map (a, b): a state of 0 leaves b whatever a is (a product of
// gates that overflowed stays out of a segment that starts from nothing).
template <class A>
__device__ __forceinline__ A scan_apply(A a, A b, A x) {
  return x == A(0) ? b : fma_of(a, x, b);
}

// What chunks publish is one word a value, written and read whole and past the
// caches that one XCD does not share with another (relaxed atomics of the agent's
// scope). Every bit set means "not yet": a word says by itself that it is there, so
// no flag and no fence orders it. A value with that pattern (a NaN) becomes
// another NaN.
template <class A> struct WordOf { using type = uint32_t; };
template <> struct WordOf<double> { using type = unsigned long long; };

template <class A>
__device__ __forceinline__ void publish(A* p, A v) {
  using W = typename WordOf<A>::type;
  if (__builtin_bit_cast(W, v) >= W(~W(0) - 1)) v = A(__builtin_nan(""));
  __hip_atomic_store(reinterpret_cast<W*>(p), __builtin_bit_cast(W, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

// The A of a chunk that holds a segment's border: its B replaces the state. (No other
// A has this pattern: publish() rids values of it too.)
template <class A>
__device__ __forceinline__ bool scan_is_cut(A a) {
  using W = typename WordOf<A>::type;
  return __builtin_bit_cast(W, a) == W(~W(0) - 1);
}

template <class A>
__device__ __forceinline__ void publish_cut(A* p) {
  using W = typename WordOf<A>::type;
  __hip_atomic_store(reinterpret_cast<W*>(p), W(~W(0) - 1), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}

template <class A>
__device__ __forceinline__ bool observe(const A* p, A* v) {
  using W = typename WordOf<A>::type;
  const W w = __hip_atomic_load(reinterpret_cast<const W*>(p), __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_AGENT);
  *v = __builtin_bit_cast(A, w);
  return w != ~W(0);
}

// The published maps [i, end) at `words` (two words a column an item) in order,
// SCAN_LOOK read at a time, which hides all but the first one's latency; waits for
// each. TAKE is given them one by one.
constexpr int SCAN_LOOK = 4;

template <class A, int V, class Take>
__device__ __forceinline__ void scan_maps(const A* words, int64_t d, int64_t col, int64_t i,
                                          int64_t end, Take take) {
  while (i < end) {
    A a[SCAN_LOOK][V], b[SCAN_LOOK][V];
    bool there[SCAN_LOOK];
#pragma unroll
    for (int q = 0; q < SCAN_LOOK; ++q) {
      const A* w = words + (i + q < end ? i + q : end - 1) * 2 * d + col;
      there[q] = true;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        there[q] &= observe(w + k, &a[q][k]);
        there[q] &= observe(w + d + k, &b[q][k]);
      }
    }
    int taken = 0;
#pragma unroll
    for (int q = 0; q < SCAN_LOOK; ++q) {
      const bool step = taken == q && i + q < end && __all(there[q]);
      take(a[q], b[q], step);
      taken += step;
    }
    i += taken;
    if (!taken) __builtin_amdgcn_s_sleep(1);
  }
}

// The state in front of chunk `c` in the order of the walk, into x; (fa, fb, cut) is
// the chunk's own map, already published. Only the lanes that are `mine` publish.
//
// SCAN_GROUP chunks form a group. A chunk composes the maps of its group's chunks in
// front of it, and applies that to the state in front of the group, unless a border
// lies between; the group's last chunk composes the group's map and, with the same
// state, the state behind it. The state in front of a group is looked for group by
// group, back to the nearest that is there and forward again through the groups' maps.
// What is found does not depend on how far that was: each state is one map applied
// to one other, always the same two. Results are the same bits each time.
//
// Every wait ends: chunks are handed out by ticket in this order, so the workgroups
// of all chunks in front have started. Each publishes its map without waiting for
// anything, and the last of a group the group's map after waiting for such maps only.
template <class A, int V>
__device__ __forceinline__ void look_back(A* words, int64_t chunks, int64_t d, int64_t col,
                                          int64_t c, const A (&fa)[V], const A (&fb)[V], bool cut,
                                          bool mine, A (&x)[V]) {
  const int64_t groups = chunks / SCAN_GROUP, g = c / SCAN_GROUP;
  A* maps = words + chunks * 2 * d;       // [groups][2][d]
  A* states = maps + groups * 2 * d;      // [groups][d]: behind each group
  const bool closing = c % SCAN_GROUP == SCAN_GROUP - 1;
  A ma[V], mb[V];
  bool border = false;
#pragma unroll
  for (int k = 0; k < V; ++k) { ma[k] = A(1); mb[k] = A(0); }
  scan_maps<A, V>(words, d, col, g * SCAN_GROUP, c, [&](A (&a)[V], A (&b)[V], bool step) {
    const bool here = scan_is_cut(a[0]);
    border |= step && here;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const A to = here ? b[k] : scan_apply(a[k], b[k], mb[k]);
      mb[k] = step ? to : mb[k];
      ma[k] = step ? ma[k] * a[k] : ma[k];
    }
  });
  A ga[V], gb[V];
  if (closing) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      gb[k] = cut ? fb[k] : scan_apply(fa[k], fb[k], mb[k]);
      ga[k] = ma[k] * fa[k];
      if (!mine) continue;
      A* w = maps + g * 2 * d + col + k;
      if (cut || border) publish_cut(w);
      else publish(w, ga[k]);
      publish(w + d, gb[k]);
      if (cut || border) publish(states + g * d + col + k, gb[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) x[k] = mb[k];
  if (border) return;
  // the nearest group in front whose state is there; none: zeros
  A s[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s[k] = A(0);
  int64_t j = g - 1;
  for (bool found = false; j >= 0 && !found;) {
    A t[SCAN_LOOK][V];
    bool there[SCAN_LOOK];
#pragma unroll
    for (int q = 0; q < SCAN_LOOK; ++q) {
      const A* w = states + (j - q > 0 ? j - q : 0) * d + col;
      there[q] = true;
#pragma unroll
      for (int k = 0; k < V; ++k) there[q] &= observe(w + k, &t[q][k]);
    }
#pragma unroll
    for (int q = 0; q < SCAN_LOOK; ++q) {
      const bool last = !found && j >= 0 && __all(there[q]);
#pragma unroll
      for (int k = 0; k < V; ++k) s[k] = last ? t[q][k] : s[k];
      found |= last;
      j -= !found && j >= 0;
    }
  }
  scan_maps<A, V>(maps, d, col, j + 1, g, [&](A (&a)[V], A (&b)[V], bool step) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const A to = scan_is_cut(a[k]) ? b[k] : scan_apply(a[k], b[k], s[k]);
      s[k] = step ? to : s[k];
    }
  });
#pragma unroll
  for (int k = 0; k < V; ++k) {
    x[k] = scan_apply(ma[k], mb[k], s[k]);
    if (closing && !cut && mine)
      publish(states + g * d + col + k, scan_apply(ga[k], gb[k], s[k]));
  }
}

// A chunk's rows, SCAN_BLOCK a thread: threads of `wide` lanes of columns form a
// strip, the workgroup's strips lie one behind the other, and its maps are scanned
// over the strips in LDS.
//
// Bound by memory; 32,768 rows of 2,048 bfloat16 values with float gates, in four
// sequences: forward 125 us (570 MB, 4.6 TB/s), gradient 187 us (955 MB,
// 5.1 TB/s), where a copy of 1 GiB runs at 5.1 TB/s; 100,000 rows of 1,024 float16
// values in one sequence, whose 782 chunks are one chain: 145 us (614 MB, 4.2 TB/s).
// Two columns a lane: four took 10% longer, as registers then leave room for half
// the wavefronts. Rows that are not used yet stay as they came, two 16-bit values to
// a register: the gradient's 260 us became 195 us. 512 threads: 256 make the chain
// twice as long (the one sequence 190 us). Groups of 4 chunks: 8 take 146 us for it,
// 16 163 us, and no groups, with the state handed from chunk to chunk, 217 us.
// The gradient of 16-bit rows keeps to 128 registers, two workgroups on a compute
// unit; that of float rows takes 148, so there one waits alone (150,001 float rows of
// 100 in 5,000 segments: 96 us, 310 MB, 3.2 TB/s).
constexpr int PASS_BLOCK = 512;

template <class T, class G, int V, bool BACK>
__global__ void __launch_bounds__(PASS_BLOCK) scan_pass_kernel(ScanArgs<T, G> p) {
  using A = acc_t<T>;
  constexpr int U = SCAN_BLOCK;
  __shared__ A sa[PASS_BLOCK][V], sb[PASS_BLOCK][V];
  __shared__ uint8_t sk[PASS_BLOCK];
  __shared__ uint32_t turn;
  const int me = threadIdx.x;
  if (me == 0) turn = p.chunks > 1 ? atomicAdd(p.ticket, 1u) : blockIdx.x;
  __syncthreads();
  const int64_t order = turn / p.tiles, tile = turn % p.tiles;
  const int64_t chunk = BACK ? p.chunks - 1 - order : order;
  const int strips = PASS_BLOCK / p.wide, strip = me / p.wide;
  int64_t lane = tile * p.wide + me % p.wide;
  if (lane >= p.lanes) lane = p.lanes - 1;  // spare lanes do what the last one does
  const int64_t c0 = lane * V, col = c0 + V <= p.d ? c0 : p.d - V;
  const int64_t r0 = (chunk * strips + strip) * U;
  const int64_t r1 = r0 + U < p.n ? r0 + U : p.n;
  const bool any = r0 < r1;
  const int64_t from = r0 * p.d + col;
  const uint32_t first = any ? p.starts[r0 / U] : 0, end = any ? p.ends[r0 / U] : 0;
  const T* x = BACK ? p.grad : p.value;
  Held<G, V> a[U];
  Held<T, V> v[U], value[BACK ? U : 1];
  A fa[V], fb[V];
#pragma unroll
  for (int k = 0; k < V; ++k) { fa[k] = A(1); fb[k] = A(0); }
  bool cut = false;
  const bool plain = __all(r0 + U <= p.n && (first | end) == 0);
  auto read = [&](auto all) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = from + (decltype(all)::value || r0 + i < r1 ? i : r1 - 1 - r0) * p.d;
      a[i].load(p.gate + at);
      v[i].load(x + at);
      if (BACK && p.dgate) value[BACK ? i : 0].load(p.value + at);
    }
  };
  // the state that row i starts from where it is its segment's first
  // (BACK: last), in `to`
  const uint32_t edges = BACK ? end : first;
  const A* edge = BACK ? p.grad_last : p.initial;
  auto border = [&](int i, A (&to)[V]) {
    if (edge) load_acc<A, A, V>(edge + (int64_t)p.ids[r0 + i] * p.d + col, to);
    else
#pragma unroll
      for (int k = 0; k < V; ++k) to[k] = A(0);
  };
  auto fold = [&](auto all) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = BACK ? U - 1 - j : j;
      if constexpr (!decltype(all)::value) {
        if (r0 + i >= r1) continue;
        if (edges >> i & 1) {
          border(i, fb);
          cut = true;
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const A g = a[i].at(k), y = v[i].at(k);
        fa[k] = fa[k] * g;
        fb[k] = BACK ? g * (y + fb[k]) : fma_of(g, fb[k], y);
      }
    }
  };
  if (plain) {
    read(std::true_type{});
    fold(std::true_type{});
  } else if (any) {
    read(std::false_type{});
    fold(std::false_type{});
  }

  // inclusive scan of the strips' maps, in the order of the walk
  const int pos = BACK ? strips - 1 - strip : strip;
  for (int off = 1; off < strips; off <<= 1) {
#pragma unroll
    for (int k = 0; k < V; ++k) { sa[me][k] = fa[k]; sb[me][k] = fb[k]; }
    sk[me] = cut;
    __syncthreads();
    if (pos >= off) {
      const int o = BACK ? me + off * p.wide : me - off * p.wide;
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
  for (int k = 0; k < V; ++k) { sa[me][k] = fa[k]; sb[me][k] = fb[k]; }
  sk[me] = cut;
  __shared__ A carry[WAVE][V];
  // the last strip of the walk holds the chunk's map; its wavefront looks back
  if (p.chunks == 1) {
    if (me < p.wide)
#pragma unroll
      for (int k = 0; k < V; ++k) carry[me][k] = A(0);
  } else if (me / WAVE == (BACK ? 0 : PASS_BLOCK / WAVE - 1)) {
    const bool mine = pos == strips - 1;  // narrow rows: several strips a wavefront
    if (mine) {
      A* w = p.words + order * 2 * p.d + col;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (cut) publish_cut(w + k);
        else publish(w + k, fa[k]);
        publish(w + p.d + k, fb[k]);
      }
    }
    // every strip of this wavefront looks back with the last one's map
    const int last = BACK ? threadIdx.x % p.wide : WAVE - p.wide + threadIdx.x % p.wide;
    A la[V], lb[V], s[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      la[k] = __shfl(fa[k], last);
      lb[k] = __shfl(fb[k], last);
    }
    look_back<A, V>(p.words, p.chunks, p.d, col, order, la, lb, __shfl((int)cut, last) != 0, mine,
                    s);
    if (mine)
#pragma unroll
      for (int k = 0; k < V; ++k) carry[me % p.wide][k] = s[k];
  }
  __syncthreads();
  if (!any) return;
  A h[V];  // the state this strip starts from
#pragma unroll
  for (int k = 0; k < V; ++k) h[k] = carry[me % p.wide][k];
  if (pos) {
    const int o = BACK ? me + p.wide : me - p.wide;
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = sk[o] ? sb[o][k] : scan_apply(sa[o][k], sb[o][k], h[k]);
  }

  if constexpr (!BACK) {
    if (p.marks) store_acc<A, A, V>(p.marks + r0 / U * p.d + col, h);
    auto write = [&](auto all) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if constexpr (!decltype(all)::value) {
          if (r0 + i >= r1) continue;
          if (edges >> i & 1) border(i, h);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = fma_of(a[i].at(k), h[k], v[i].at(k));
        store_acc<T, A, V>(p.out + from + i * p.d, h);
        if constexpr (!decltype(all)::value)
          if (p.last && (end >> i & 1))
            store_acc<A, A, V>(p.last + (int64_t)p.ids[r0 + i] * p.d + col, h);
      }
    };
    if (plain) write(std::true_type{});
    else write(std::false_type{});
  } else {
    auto write = [&](auto all) {
      constexpr bool ALL = decltype(all)::value;
      A before[U][V];
      if (p.dgate) {  // the states in front of each row
        A f[V];
        load_acc<A, A, V>(p.marks + r0 / U * p.d + col, f);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if constexpr (!ALL) {
            if (r0 + i >= r1) continue;
            if (first >> i & 1) {
              if (p.initial) load_acc<A, A, V>(p.initial + (int64_t)p.ids[r0 + i] * p.d + col, f);
              else
#pragma unroll
                for (int k = 0; k < V; ++k) f[k] = A(0);
            }
          }
#pragma unroll
          for (int k = 0; k < V; ++k) {
            before[i][k] = f[k];
            f[k] = fma_of(a[i].at(k), f[k], value[BACK ? i : 0].at(k));
          }
        }
      }
#pragma unroll
      for (int i = U - 1; i >= 0; --i) {
        if constexpr (!ALL) {
          if (r0 + i >= r1) continue;
          if (edges >> i & 1) border(i, h);
        }
        A da[V], dv[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          dv[k] = v[i].at(k) + h[k];
          h[k] = a[i].at(k) * dv[k];
        }
        if (p.dvalue) store_acc<T, A, V>(p.dvalue + from + i * p.d, dv);
        if (p.dgate) {
#pragma unroll
          for (int k = 0; k < V; ++k) da[k] = dv[k] * before[i][k];
          store_acc<G, A, V>(p.dgate + from + i * p.d, da);
        }
        if constexpr (!ALL)
          if (p.dinitial && (first >> i & 1))
            store_acc<A, A, V>(p.dinitial + (int64_t)p.ids[r0 + i] * p.d + col, h);
      }
    };
    if (plain) write(std::true_type{});
    else write(std::false_type{});
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
hipError_t run_scan_pass(ScanArgs<T, G> p, void* workspace, bool back, hipStream_t s) {
  using A = acc_t<T>;
  p.lanes = ceil_div64(p.d, V);
  p.wide = WAVE;
  while (p.wide > 1 && p.wide / 2 >= p.lanes) p.wide /= 2;
  p.tiles = ceil_div64(p.lanes, p.wide);
  p.chunks = ceil_div64(p.n, (int64_t)SCAN_BLOCK * (PASS_BLOCK / p.wide));
  if (p.chunks > 1) {
    p.ticket = (uint32_t*)workspace;
    p.words = (A*)((char*)workspace + SCAN_TICKET_BYTES);
    const int64_t words = scan_words(p.chunks) * p.d * (int64_t)(sizeof(A) / 4);
    const hipError_t e = launch_scan_reset(p.ticket, (uint32_t*)p.words, words, s);
    if (e != hipSuccess) return e;
  }
  const int64_t grid = p.chunks * p.tiles;
  if (back) scan_pass_kernel<T, G, V, true><<<grid, PASS_BLOCK, 0, s>>>(p);
  else scan_pass_kernel<T, G, V, false><<<grid, PASS_BLOCK, 0, s>>>(p);
  return hipGetLastError();
}

template <class T, class G>
hipError_t run_scan(const ScanParams& q, bool back) {
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
  hipError_t e = hipSuccess;
  if (q.n > 0) {
    // a lane's columns are 8 bytes of accumulators: 16 would halve the wavefronts
    // that its registers leave room for
    constexpr int V = acc_vec<T>() / 2;
    e = q.d < V ? run_scan_pass<T, G, 1>(p, q.workspace, back, s)
                : run_scan_pass<T, G, V>(p, q.workspace, back, s);
    if (e != hipSuccess) return e;
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
hipError_t run_scan_step(const ScanStepParams& q) {
  constexpr int V = acc_vec<T>();
  scan_step_kernel<T, G, V><<<ceil_div64(q.n, (int64_t)BLOCK * V), BLOCK, 0, q.stream>>>(
      (const G*)q.gate, (const T*)q.value, (const acc_t<T>*)q.state, (T*)q.out,
      (acc_t<T>*)q.next, q.n);
  return hipGetLastError();
}

}  // namespace mdgl
