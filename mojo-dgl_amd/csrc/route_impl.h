// Routing rows to experts (included once per type): scores, the choice of k
// experts a row, their weights, and the weights' gradient.
//
//   s = softmax(x) or sigmoid(x) over a row's E logits x
//   key = s + bias, or x itself without a bias (both scores grow with x)
//   groups of E / groups neighbouring experts: the topk_groups best by their
//   largest key, or by the sum of their two best experts' s + bias, stay (a sum of
//   scores, with or without a bias: one of logits has another order)
//   ids = the k largest keys in falling order, the lowest index among equals
//   w = scale * s[ids], divided by their sum when renormalised
//
// A logit of -inf masks its expert: its key is below every other (as is that of a
// NaN), and its weight is 0. A row needs G lanes (16, or 32 and 64 for many
// experts or choices), each holding R neighbouring experts, so the lowest index
// among equals is the lowest lane's. A round of the choice is a maximum over the
// lane, over the group by DPP, and the lowest index that has it; lane j keeps the
// j-th choice.
//
// With a bias the order of two keys can hang on their last bits. The float pass
// therefore makes one choice more than asked for, and a row two of whose
// neighbouring keys (or whose last kept and first dropped group) lie closer than
// the float keys can be wrong is chosen again in double, by a whole wavefront.
// Keys of equal logits and biases need no second look: they are equal however they
// are formed. Behind the first that is not chosen lie others, perhaps with larger
// scores, and errors, under lower biases: where it lies closer to the last chosen than
// the largest error of the row, the row is chosen again (sigmoid: few scores are much
// smaller than the largest), or each of them is compared first (softmax; 65,536 rows of
// 256 with a bias: 43 us, 46 without that, and with it 53 instead of 50 for sigmoid).
//
// 65,536 rows of 256 float32 logits in 8 groups, 8 of 4 groups chosen, with a bias:
// 56 us, and 18 us for the gradient, where reading and writing take 14 and 14. The
// choice is bound by its instructions: 1,520 of the vector unit's a wavefront of four
// rows, half of them the nine rounds (98 us with compares and selects on floats
// instead of integer maxima, a second search in double of whole wavefronts, exact
// exponentials for the keys). 16 lanes a row: with 64 a round's two reductions over
// the lanes serve one row instead of four.
#pragma once

#include "mdgl_half.h"
#include "mdgl_kernels.h"

namespace mdgl {

template <class T>
struct RouteArgs {
  using A = acc_t<T>;
  const T* logits;  // [n][e]
  const A* bias;    // [e], may be null
  A* weights;       // [n][k]
  int64_t* ids;     // [n][k]
  int64_t n;
  int e, k, groups, topk_groups;  // groups = 1: no choice of groups
  int sigmoid, top2, renorm;
  A scale;
  const A* dweights;  // backward
  T* dlogits;
};

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float abs_of(float x) { return fabsf(x); }
__device__ __forceinline__ double abs_of(double x) { return fabs(x); }
template <class K> __device__ __forceinline__ K lowest() { return -K(__builtin_huge_val()); }

template <class K>
__device__ __forceinline__ K sigmoid_of(K x) { return K(1) / (K(1) + exp_of(-x)); }

// A score in float by the hardware's exponential and reciprocal; of softmax, as a
// multiple of the score of `top`, the row's largest logit.
constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float sigmoid_near(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * x));
}
__device__ __forceinline__ float softmax_near(float x, float top) {
  return x == top ? 1.0f : __builtin_amdgcn_exp2f(LOG2E * (x - top));  // both may be +inf
}

// Maximum / minimum over G lanes, in all of them. No value is NaN.
template <int G, class K>
__device__ __forceinline__ K lanes_max(K v) {
  auto up = [](K a, K b) { return a > b ? a : b; };
  v = up(v, lane_xor_dpp(v, 0));
  v = up(v, lane_xor_dpp(v, 1));
  v = up(v, lane_xor_dpp(v, 2));
  v = up(v, lane_xor_dpp(v, 3));
  if constexpr (G > 16) v = up(v, __shfl_xor(v, 16));
  if constexpr (G > 32) v = up(v, __shfl_xor(v, 32));
  return v;
}

template <int G>
__device__ __forceinline__ int lanes_min(int v) { return -lanes_max<G>(-v); }

// The larger two of two pairs (a >= b in each).
template <class K>
__device__ __forceinline__ void join_two(K& a, K& b, K c, K d) {
  const K lo = a < c ? a : c;
  a = a > c ? a : c;
  b = b > d ? b : d;
  b = b > lo ? b : lo;
}

// How far a score of the float pass can be off, in half steps (2^-24) of itself. The
// argument of the exponential is rounded, up to three times: sigmoid's error grows
// with -x, softmax's with the distance to the row's largest logit. Beside that a few
// steps of the exponential, the reciprocal, and softmax's sum over a lane's experts,
// up to 32 of them, and over the lanes. Scores below 2^-126 are 0: callers add 2^-100.
__device__ __forceinline__ float route_off(float x, float top, bool sigmoid) {
  return sigmoid ? 16.0f + 2.0f * fmaxf(-x, 0.0f) : 64.0f + 3.0f * (top - x);
}

template <class K>
struct Choice {
  int id;    // lane j: the j-th choice
  K key;     // and its key
  K top, sum;  // softmax: the row's largest logit, the sum of exp(x - top)
  bool near;   // the choice of groups hangs on the last bits
  K limit;     // how far any of the row's scores can be off (float pass), in 2^-24
};

// The group of the lane's experts where every lane's lie in one, by its first
// lanes; `span` lanes form a group (0: groups end inside lanes).
__device__ __forceinline__ int route_span(int e, int groups, int per) {
  const int size = e / groups, span = size / per;
  return size == span * per && (span & (span - 1)) == 0 ? span : 0;
}

// Floats as integers of the same order; 0 is below all of them, NaN stands with
// -inf.
constexpr uint32_t KEY_LOWEST = 0x007fffffu;  // -inf

__device__ __forceinline__ uint32_t ordered(float x) {  // not a NaN, not -0
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float unordered(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Maximum over G lanes, in all of them; the moves inside 16 lanes are part of the
// maximum's own instruction.
template <int G>
__device__ __forceinline__ uint32_t lanes_umax(uint32_t v) {
  auto up = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
  v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));   // quad [1,0,3,2]
  v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));   // quad [2,3,0,1]
  v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));  // row_half_mirror
  v = up(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));  // row_mirror
  if constexpr (G > 16) v = up(v, __shfl_xor((int)v, 16));
  if constexpr (G > 32) v = up(v, __shfl_xor((int)v, 32));
  return v;
}

// The first `count` choices of a row (count <= G) by float keys. An expert that
// is not there, or no longer, has key 0. The keys' exponentials and reciprocals are
// the hardware's: they are good to what the caller's bounds on keys allow, and a
// closer call is chosen again in double.
template <class T, int G, int R>
__device__ __forceinline__ Choice<float> route_choose_float(const RouteArgs<T>& p, const T* x,
                                                            int count) {
  const int lane = threadIdx.x % G;
  const int per = (p.e + G - 1) / G, base = lane * per;
  const int have = base >= p.e ? 0 : (p.e - base < per ? p.e - base : per);
  float v[R];
#pragma unroll
  for (int i = 0; i < R; i += 4) {
    if (i + 4 <= have) {
      T raw[4];
      load_any<false>(x + base + i, raw);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i + q] = (float)raw[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[i + q] = i + q < have ? (float)x[base + i + q] : -__builtin_huge_valf();
    }
  }
  Choice<float> c;
  c.top = lowest<float>();
  c.sum = 0.0f;
  c.near = false;
  c.limit = 0.0f;
  c.id = 0;
  c.key = lowest<float>();
  // without a bias, the marks of groups by two experts need scores that no key has
  const bool marks = p.groups > 1 && p.top2 && !p.bias;
  const bool sums = !p.sigmoid && (p.bias || !p.renorm);
  if (sums || marks) {
#pragma unroll
    for (int i = 0; i < R; ++i) c.top = v[i] > c.top ? v[i] : c.top;
    c.top = lanes_max<G>(c.top);
  }
  if (sums) {
    // the sum of softmax; a NaN goes into it
#pragma unroll
    for (int i = 0; i < R; ++i)  // 0 where no expert is, and in a row of masks
      c.sum += v[i] == lowest<float>() ? 0.0f : expf(v[i] - c.top);
    c.sum = group_sum(c.sum, G);
  }
  uint32_t key[R];
  // the larger a score the more it can be off: no more than the row's largest
  if (marks)  // formed from multiples of softmax's largest
    c.limit = (p.sigmoid ? sigmoid_near(c.top) : 1.0f) * route_off(c.top, c.top, p.sigmoid);
  if (p.bias) {
    const float part = c.sum > 0.0f ? 1.0f / c.sum : 0.0f;
    uint32_t most = 0u;  // the largest score's bits; scores are not negative
#pragma unroll
    for (int i = 0; i < R; i += 4) {
      float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (i + 4 <= have) {
        load_any<false>(p.bias + base + i, b);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i + q < have) b[q] = p.bias[base + i + q];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float y = v[i + q];
        const float s = p.sigmoid ? sigmoid_near(y)
                                  : __builtin_amdgcn_exp2f(LOG2E * (y - c.top)) * part;
        const uint32_t k = ordered(s + b[q]);  // no -0: s is not negative
        const uint32_t bits = __builtin_bit_cast(uint32_t, s);
        most = bits > most ? bits : most;
        key[i + q] = i + q >= have ? 0u : y > lowest<float>() ? k : KEY_LOWEST;
      }
    }
    // (1 beside a NaN; the logit of a sigmoid lies above its logarithm)
    const float big = fminf(__builtin_bit_cast(float, lanes_umax<G>(most)), 1.0f);
    const float at = p.sigmoid ? 0.6931472f * __builtin_amdgcn_logf(big + 0x1p-100f) : c.top;
    c.limit = big * route_off(at, c.top, p.sigmoid);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const uint32_t k = v[i] == v[i] ? ordered(v[i] + 0.0f) : KEY_LOWEST;
      key[i] = i < have ? k : 0u;
    }
  }

  if (p.groups > 1) {
    const int size = p.e / p.groups, span = route_span(p.e, p.groups, per);
    auto score = [&](uint32_t k) {
      const float y = unordered(k);
      return p.sigmoid ? sigmoid_near(y) : softmax_near(y, c.top);
    };
    // a group's mark, from its two largest keys: -inf where all are masked
    // (a sum that overflows stays finite, above a masked group's, and its row is near)
    auto grade = [&](uint32_t a, uint32_t b) {
      if (marks && a > KEY_LOWEST) return b > KEY_LOWEST ? score(a) + score(b) : score(a);
      const float f = unordered(a);
      if (!p.top2 || b <= KEY_LOWEST) return f;
      return fminf(fmaxf(f + unordered(b), -__FLT_MAX__), __FLT_MAX__);
    };
    auto two = [](uint32_t& a, uint32_t& b, uint32_t k) {  // a >= b the larger two
      const uint32_t lo = k < a ? k : a;
      a = k > a ? k : a;
      b = lo > b ? lo : b;
    };
    auto join = [](uint32_t& a, uint32_t& b, int off) {
      const uint32_t oa = __shfl_xor(a, off), ob = __shfl_xor(b, off);
      join_two(a, b, oa, ob);
    };
    // lane j: the mark of group j, and how large what is summed in it is
    float mark = lowest<float>(), size_of = 0.0f;
    auto large = [&](uint32_t a, uint32_t b) {
      if (marks) return a > KEY_LOWEST ? grade(a, b) : 0.0f;
      const float f = a > KEY_LOWEST ? abs_of(unordered(a)) : 0.0f;
      return p.top2 && b > KEY_LOWEST ? f + abs_of(unordered(b)) : f;
    };
    if (span) {
      uint32_t a = KEY_LOWEST, b = KEY_LOWEST;
#pragma unroll
      for (int i = 0; i < R; ++i) two(a, b, key[i]);
      for (int off = 1; off < span; off <<= 1) join(a, b, off);
      const int from = lane * span < G ? lane * span : 0;
      mark = __shfl(grade(a, b), from, G);
      size_of = __shfl(large(a, b), from, G);
    } else {
      for (int g = 0; g < p.groups; ++g) {
        uint32_t a = KEY_LOWEST, b = KEY_LOWEST;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int e = base + i - g * size;
          two(a, b, e >= 0 && e < size ? key[i] : 0u);
        }
#pragma unroll
        for (int off = 1; off < G; off <<= 1) join(a, b, off);
        if (lane == g) {
          mark = grade(a, b);
          size_of = large(a, b);
        }
      }
    }
    // a group stays when fewer than topk_groups are ranked before it
    const bool real = lane < p.groups;
    int before = 0;
    for (int g = 0; g < p.groups; ++g) {
      const float m = __shfl(mark, g, G);
      before += m > mark || (m == mark && g < lane);
    }
    const bool stays = real && before < p.topk_groups;
    const float kept_low = -lanes_max<G>(stays ? -mark : lowest<float>());
    const float lost_top = lanes_max<G>(real && !stays ? mark : lowest<float>());
    // both marks are sums of up to two scores or keys, which round, too
    const float big = lanes_max<G>(real ? size_of : 0.0f);
    const float wrong = 4.0f * c.limit + 8.0f * big;
    c.near = kept_low - lost_top <= wrong * 0x1p-24f + 0x1p-100f && lost_top > lowest<float>();
    const uint64_t all = __ballot(stays) >> (threadIdx.x % WAVE / G * G);
    if (span) {
      const int mine = lane / span;
      const bool out = mine >= p.groups || !(all >> mine & 1);
#pragma unroll
      for (int i = 0; i < R; ++i) key[i] = out ? 0u : key[i];
    } else {
      int g = base / size, at = base % size;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (i < have && !(all >> g & 1)) key[i] = 0u;
        if (++at == size) {
          at = 0;
          ++g;
        }
      }
    }
  }

  for (int j = 0; j < count; ++j) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < R; ++i) top = key[i] > top ? key[i] : top;
    top = lanes_umax<G>(top);
    int at = p.e;
    bool hit[R];
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      hit[i] = key[i] == top;
      at = hit[i] ? base + i : at;
    }
    const int first = top ? (int)~lanes_umax<G>(~(uint32_t)at) : p.e;
    if (lane == j) {
      c.id = first;
      c.key = top ? unordered(top) : lowest<float>();
    }
    // of equal keys only the first is taken
    const int t = at == first ? first - base : -1;
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = t == i ? 0u : key[i];
  }
  return c;
}

// Softmax: whether an expert that was not chosen may belong in front of the last that
// was, `id` (with its key, logit and bias, and how far its score can be off): the row's
// keys once more, each with its own error. (Experts of dropped groups may answer, too.)
template <class T, int G, int R>
__device__ __forceinline__ bool route_rival(const RouteArgs<T>& p, const T* x, float top, float sum,
                                            int id, float key, float logit, float bias,
                                            float off) {
  const int lane = threadIdx.x % G;
  const int per = (p.e + G - 1) / G, base = lane * per;
  const float part = sum > 0.0f ? 1.0f / sum : 0.0f;
  const int have = base >= p.e ? 0 : (p.e - base < per ? p.e - base : per);
  bool found = false;
#pragma unroll
  for (int i = 0; i < R; i += 4) {
    T raw[4];
    float b[4];
    if (i + 4 <= have) {
      load_any<false>(x + base + i, raw);
      load_any<false>(p.bias + base + i, b);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        raw[q] = i + q < have ? x[base + i + q] : (T)lowest<float>();
        b[q] = i + q < have ? p.bias[base + i + q] : 0.0f;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float y = (float)raw[q];
      const float s = __builtin_amdgcn_exp2f(LOG2E * (y - top)) * part;
      const float k = s + b[q];
      const int e = base + i + q;
      const bool behind = y > lowest<float>() && (k < key || (k == key && e > id));
      const float wrong = off + s * route_off(y, top, false) + 2.0f * (abs_of(k) + abs_of(key));
      found |= behind && key - k <= wrong * 0x1p-24f + 0x1p-100f && !(y == logit && b[q] == bias);
    }
  }
  return (__ballot(found) >> (threadIdx.x % WAVE / G * G) & (~uint64_t(0) >> (WAVE - G))) != 0;
}

// The first `count` choices of a row (count <= G), keys formed in K.
template <class K, class T, int G, int R>
__device__ __forceinline__ Choice<K> route_choose(const RouteArgs<T>& p, const T* x, int count) {
  const int lane = threadIdx.x % G;
  const int per = (p.e + G - 1) / G, base = lane * per;
  const int have = base >= p.e ? 0 : (p.e - base < per ? p.e - base : per);
  K key[R];
  uint32_t gone = 0;  // experts not to be chosen (any more)
#pragma unroll
  for (int i = 0; i < R; i += 4) {
    if (i + 4 <= have) {
      T v[4];
      load_any<false>(x + base + i, v);
#pragma unroll
      for (int q = 0; q < 4; ++q) key[i + q] = (K)v[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        key[i + q] = i + q < have ? (K)x[base + i + q] : lowest<K>();
        if (i + q >= have) gone |= 1u << (i + q);
      }
    }
  }
  Choice<K> c;
  c.top = lowest<K>();
  c.sum = K(0);
  c.near = false;
  c.limit = K(0);
  c.id = 0;
  c.key = lowest<K>();
  const bool marks = p.groups > 1 && p.top2 && !p.bias;
  const bool sums = !p.sigmoid && (p.bias || !p.renorm);
  if (sums || marks) {
#pragma unroll
    for (int i = 0; i < R; ++i) c.top = key[i] > c.top ? key[i] : c.top;
    c.top = lanes_max<G>(c.top);
  }
  if (sums) {
    // the sum of softmax; a NaN goes into it
#pragma unroll
    for (int i = 0; i < R; ++i)
      c.sum += gone >> i & 1 || key[i] == lowest<K>() ? K(0) : exp_of(key[i] - c.top);
    c.sum = group_sum(c.sum, G);
  }
  if (p.bias) {
    const K part = c.sum > K(0) ? K(1) / c.sum : K(0);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (gone >> i & 1 || key[i] == lowest<K>()) continue;
      const K s = p.sigmoid ? sigmoid_of(key[i]) : exp_of(key[i] - c.top) * part;
      key[i] = s + (K)p.bias[base + i];
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = key[i] != key[i] ? lowest<K>() : key[i];

  if (p.groups > 1) {
    const int size = p.e / p.groups;
    K mark = lowest<K>();  // lane j: the mark of group j
    auto score = [&](K y) {
      return p.sigmoid ? sigmoid_of(y) : y == c.top ? K(1) : exp_of(y - c.top);
    };
    auto grade = [&](K a, K b) {
      if (marks && a > lowest<K>()) return b > lowest<K>() ? score(a) + score(b) : score(a);
      // (a sum of biases that overflows stays above a masked group's)
      return p.top2 && b > lowest<K>() ? fmax(a + b, -__DBL_MAX__) : a;
    };
    const int span = route_span(p.e, p.groups, per);
    const bool whole = span != 0;
    int mine = lane / (whole ? span : 1);  // the group of all of the lane's experts
    if (whole) {
      K a = lowest<K>(), b = lowest<K>();
#pragma unroll
      for (int i = 0; i < R; ++i) join_two(a, b, key[i], lowest<K>());
      for (int off = 1; off < span; off <<= 1) {
        const K oa = __shfl_xor(a, off), ob = __shfl_xor(b, off);
        join_two(a, b, oa, ob);
      }
      mark = grade(a, b);
      mark = __shfl(mark, lane * span < G ? lane * span : 0, G);
      if (lane >= p.groups) mark = lowest<K>();
    } else {
      for (int g = 0; g < p.groups; ++g) {
        K a = lowest<K>(), b = lowest<K>();
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int e = base + i - g * size;
          join_two(a, b, i < have && e >= 0 && e < size ? key[i] : lowest<K>(), lowest<K>());
        }
#pragma unroll
        for (int off = 1; off < G; off <<= 1) {
          const K oa = __shfl_xor(a, off), ob = __shfl_xor(b, off);
          join_two(a, b, oa, ob);
        }
        if (lane == g) mark = grade(a, b);
      }
    }
    uint64_t kept = 0;
    bool open = lane < p.groups;
    for (int j = 0; j < p.topk_groups; ++j) {
      const K top = lanes_max<G>(open ? mark : lowest<K>());
      const int g = lanes_min<G>(open && mark == top ? lane : G);
      if (g < G) kept |= uint64_t(1) << g;
      if (lane == g) open = false;
    }
    if (whole) {
      if (!(kept >> mine & 1)) gone = ~0u;
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i < have && !(kept >> ((base + i) / size) & 1)) gone |= 1u << i;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = gone >> i & 1 ? lowest<K>() : key[i];
  }

  for (int j = 0; j < count; ++j) {
    K top = lowest<K>();
#pragma unroll
    for (int i = 0; i < R; ++i) top = key[i] > top ? key[i] : top;
    top = lanes_max<G>(top);
    int at = p.e;
#pragma unroll
    for (int i = R - 1; i >= 0; --i) at = key[i] == top && !(gone >> i & 1) ? base + i : at;
    at = lanes_min<G>(at);
    if (lane == j) {
      c.id = at;
      c.key = top;
    }
    const int t = at - base;
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = t == i ? lowest<K>() : key[i];
    if (t >= 0 && t < R) gone |= 1u << t;
  }
  return c;
}

// A chosen expert's weight before scaling, on lane j < k with its logit x:
// normalised over the row's choices, or its score.
template <int G, class A>
__device__ __forceinline__ A route_weight(A x, bool live, bool sigmoid, bool renorm, A top, A sum) {
  if (!renorm) {
    if (sigmoid) return sigmoid_of(x);
    return top > lowest<A>() ? exp_of(x - top) / sum : sum;  // masks, NaN: 0 or NaN
  }
  const A most = lanes_max<G>(live && x == x ? x : lowest<A>());
  // scores that would underflow are in the ratio of exp(x) in any case
  A v = sigmoid && most > A(-60) ? sigmoid_of(x) : exp_of(x - most);
  if (most == lowest<A>() && x == x) v = A(0);
  if (!sigmoid && sum != sum) v = sum;  // the row's softmax is NaN
  const A total = group_sum(live ? v : A(0), G);
  return total == A(0) ? A(0) : v / total;
}

template <class T, int G, int R>
__global__ void __launch_bounds__(BLOCK) route_kernel(RouteArgs<T> p) {
  using A = acc_t<T>;
  const int lane = threadIdx.x % G;
  const int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G;
  const int64_t row = r < p.n ? r : p.n - 1;  // the last rows' spare lanes go along
  const T* x = p.logits + row * p.e;
  const bool live = lane < p.k;
  int id;
  A logit, top, sum;
  if constexpr (sizeof(A) == 8) {
    const Choice<double> c = route_choose<double, T, G, R>(p, x, p.k);
    id = c.id;
    top = c.top;
    sum = c.sum;
    logit = lane < p.k && id < p.e ? (A)x[id] : lowest<A>();
  } else {
    const bool more = p.bias && p.k < p.e;  // the first that is not chosen, too
    const Choice<float> c = route_choose_float<T, G, R>(p, x, p.k + (more ? 1 : 0));
    const bool kept = lane < p.k + (more ? 1 : 0) && c.id < p.e;
    id = c.id;
    top = c.top;
    sum = c.sum;
    logit = kept ? (A)x[id] : lowest<A>();
    bool again = false;
    if (p.bias) {
      const A bias = kept ? p.bias[id] : A(0);
      const A s = abs_of(c.key - bias);  // the score, near enough
      const A off = s * route_off(logit, c.top, p.sigmoid);
      const A key1 = __shfl_up(c.key, 1, G), x1 = __shfl_up(logit, 1, G);
      const A b1 = __shfl_up(bias, 1, G), off1 = __shfl_up(off, 1, G);
      // the last lane's is the first that is not chosen: any other of these may be the
      // one that belongs in front of it, whatever its score
      const A wrong = (lane < p.k ? off : c.limit) + off1 + A(2) * (abs_of(c.key) + abs_of(key1));
      const bool near = lane > 0 && kept && c.key > lowest<A>() &&
                        key1 - c.key <= wrong * A(0x1p-24) + A(0x1p-100) &&
                        !(lane < p.k && x1 == logit && b1 == bias);
      again = near && (p.sigmoid || lane < p.k);
      if (!p.sigmoid && __ballot(near && lane == p.k)) {
        const int last = p.k - 1;
        const bool rival = route_rival<T, G, R>(
            p, x, top, sum, __shfl(id, last, G), __shfl(c.key, last, G), __shfl(logit, last, G),
            __shfl(bias, last, G), __shfl(off, last, G));
        again = again || (near && rival);
      }
    }
    // without a bias only marks that are sums of scores can round
    again = again || (c.near && (p.bias || p.top2));
    for (uint64_t flags = __ballot(again); flags;) {
      const int g = __builtin_ctzll(flags) / G;  // the wavefront's g-th row
      const int64_t other = __shfl(row, g * G);
      const int sure = route_choose<double, T, WAVE, R * G / WAVE < 4 ? 4 : R * G / WAVE>(
                           p, p.logits + other * p.e, p.k).id;
      const int mine = __shfl(sure, lane);
      if ((int)(threadIdx.x % WAVE) / G == g) id = mine;
      flags &= ~(~uint64_t(0) >> (WAVE - G) << (g * G));
    }
    if (live) logit = id < p.e ? (A)x[id] : lowest<A>();
  }
  const A w = route_weight<G, A>(logit, live, p.sigmoid, p.renorm, top, sum);
  if (live && r < p.n) {
    p.ids[row * p.k + lane] = id;
    p.weights[row * p.k + lane] = w * p.scale;
  }
}

// dlogits of a row, formed in LDS: zeros (or, where every score counts, the
// softmax's share) with the choices' terms added, then written, a value a lane.
template <class T, int G>
__global__ void __launch_bounds__(BLOCK) route_grad_kernel(RouteArgs<T> p) {
  using A = acc_t<T>;
  extern __shared__ __align__(16) char route_lds[];
  const int lane = threadIdx.x % G;
  const int64_t r = (int64_t)blockIdx.x * (BLOCK / G) + threadIdx.x / G;
  const int64_t row = r < p.n ? r : p.n - 1;
  A* buf = reinterpret_cast<A*>(route_lds) + (int64_t)(threadIdx.x / G) * p.e;
  const T* x = p.logits + row * p.e;
  const bool live = lane < p.k;
  const int64_t id = live ? p.ids[row * p.k + lane] : -1;
  const bool ok = id >= 0 && id < p.e;
  const A logit = ok ? (A)x[id] : lowest<A>();
  const A dw = ok ? p.dweights[row * p.k + lane] * p.scale : A(0);
  const bool full = !p.sigmoid && !p.renorm;
  A top = lowest<A>(), sum = A(0);
  if (full) {
    for (int i = lane; i < p.e; i += G) {
      const A v = (A)x[i];
      buf[i] = v;
      top = v > top ? v : top;
    }
    top = lanes_max<G>(top);
    for (int i = lane; i < p.e; i += G) {
      const A v = buf[i] == lowest<A>() ? A(0) : exp_of(buf[i] - top);
      buf[i] = v;
      sum += v;
    }
    sum = group_sum(sum, G);
  }
  const A w = route_weight<G, A>(logit, ok, p.sigmoid, p.renorm, top, sum);
  const A inner = group_sum(ok ? dw * w : A(0), G);
  A dx;
  if (full) {
    const A part = sum == A(0) ? A(0) : A(1) / sum;
    for (int i = lane; i < p.e; i += G) buf[i] = -(buf[i] * part) * inner;
    dx = w * (dw - inner);
  } else {
    for (int i = lane; i < p.e; i += G) buf[i] = A(0);
    dx = w * (p.renorm ? dw - inner : dw);
    if (p.sigmoid) dx *= sigmoid_of(-logit);
    if (logit == lowest<A>()) dx = A(0);
  }
  __syncthreads();
  if (ok) buf[id] = dx;
  __syncthreads();
  if (r >= p.n) return;
  for (int i = lane; i < p.e; i += G) p.dlogits[row * p.e + i] = (T)buf[i];
}

// Rows [at, at + n) of a call.
template <class T>
hipError_t run_route_rows(RouteArgs<T> p, int64_t at, int64_t n, hipStream_t s) {
  using A = acc_t<T>;
  p.logits += at * p.e;
  p.ids += at * p.k;
  p.n = n;
  auto grid = [&](int g) { return (n + BLOCK / g - 1) / (BLOCK / g); };
  if (p.dlogits) {
    p.dlogits += at * p.e;
    p.dweights += at * p.k;
    const int g = p.k <= 16 && p.e <= 256 ? 16 : 64;
    const size_t lds = (size_t)(BLOCK / g) * p.e * sizeof(A);
    if (g == 16) route_grad_kernel<T, 16><<<grid(16), BLOCK, lds, s>>>(p);
    else route_grad_kernel<T, 64><<<grid(64), BLOCK, lds, s>>>(p);
    return hipGetLastError();
  }
  p.weights += at * p.k;
  // lanes for the choices (and the one more), and for the groups' marks
  const int need = p.k + 1 > p.groups ? p.k + 1 : p.groups;
  if (need <= 16 && p.e <= 64) route_kernel<T, 16, 4><<<grid(16), BLOCK, 0, s>>>(p);
  else if (need <= 16 && p.e <= 256) route_kernel<T, 16, 16><<<grid(16), BLOCK, 0, s>>>(p);
  else if (need <= 32 && p.e <= 512) route_kernel<T, 32, 16><<<grid(32), BLOCK, 0, s>>>(p);
  else if (p.e <= 1024) route_kernel<T, 64, 16><<<grid(64), BLOCK, 0, s>>>(p);
  else route_kernel<T, 64, 32><<<grid(64), BLOCK, 0, s>>>(p);
  return hipGetLastError();
}

template <class T>
hipError_t run_route(const RouteParams& q) {
  using A = acc_t<T>;
  RouteArgs<T> p{};
  p.logits = (const T*)q.logits;
  p.bias = (const A*)q.bias;
  p.weights = (A*)q.weights;
  p.ids = q.ids;
  p.n = q.n;
  p.e = q.e;
  p.k = q.k;
  p.groups = q.topk_groups == q.groups ? 1 : q.groups;
  p.topk_groups = q.topk_groups;
  p.sigmoid = q.sigmoid;
  p.top2 = q.top2;
  p.renorm = q.renorm;
  p.scale = (A)q.scale;
  p.dweights = (const A*)q.dweights;
  p.dlogits = (T*)q.dlogits;
  hipStream_t s = q.stream;
  // a launch takes MAX_LAUNCH_BLOCKS workgroups of four rows at least
  for (int64_t at = 0; at < q.n; at += 4 * MAX_LAUNCH_BLOCKS) {
    const hipError_t e = run_route_rows(p, at, q.n - at < 4 * MAX_LAUNCH_BLOCKS
                                                   ? q.n - at : 4 * MAX_LAUNCH_BLOCKS, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mdgl
