// Products of rows with their experts' matrices on the matrix cores, in 16 bits and in
// 8 bits with scales (included once per type).
//
//   forward      out[i] = a[i] @ b[g(i)]                 (rows in the experts' order)
//   gradient     of a: the same with the blocks' transposes; of b: for each expert
//                db[g] = sum over its rows of a[i]^T grad[i]
//   8 bits       out[i][n] = sum over blocks c of 128 columns of
//                sa[i][c] sb[g][c][n / 128] (sum over c's columns of a[i][k] b[g][k][n])
//
// A workgroup forms tiles of BM rows by BN columns. The inner axis goes in stages of
// 128 bytes a row (64 values of 16 bits, 128 of 8), which travel from memory to LDS
// without passing registers (buffer loads to LDS, 16 bytes a lane), in a ring of ST
// buffers: while one is multiplied the next ST - 1 are on their way. The ring runs on
// over the border of two tiles, so a tile's first stages load while the one before it
// is finished and written. Each wavefront holds BM / WM by BN / WN sums in registers.
//
// Layout in LDS. An operand whose memory runs along the inner axis is kept as rows of
// 128 bytes; the 16-byte pieces of row r lie at piece ^ swizzle(r), so that the eight
// rows that eight lanes read at a time use all banks. The loads to LDS write in lane
// order, so it is the lane's source address that is permuted. An operand whose memory
// runs along the other axis (b as segment_mm has it; both operands of the gradient of
// b) is kept as 64 rows, and read with the transposing LDS loads: 16 lanes read four
// inner places of 16 columns and each gets the four values of its column; its pieces
// of 64 bytes lie at piece ^ (row & 3).
//
// The product is formed transposed (b's values as the first operand), which leaves a
// lane with four neighbouring columns of one row; two blocks of 16 columns are dealt
// out so that a lane's two fours are eight neighbours: results leave in stores of 16
// bytes.
//
// Past the edges: rows past the tile's group and inner places past the end are read as
// zeros by the buffer's own bounds check (a lane past the inner end is given an offset
// behind the buffer), so no stage has a case of its own. Rows that start off a 16-byte
// boundary (an odd width) go through registers instead, element by element at the ends.
//
// Tiles are counted on the GPU from the experts' lengths, which the host need not know:
// every wavefront walks them 64 experts at a time. A tile index in the order of the
// experts, each in bands of 8 column tiles; an XCD takes one contiguous run of tiles,
// so that the rows and blocks its workgroups share lie in its own L2. Rows behind the
// last expert's form a group without an inner axis: they are written as zeros.
#pragma once

#include "mdgl_half.h"
#include "mdgl_kernels.h"

#include <type_traits>

#pragma clang diagnostic ignored "-Winline-asm"

namespace mdgl {

typedef float mm_f32x4 __attribute__((ext_vector_type(4)));
typedef int mm_i32x4 __attribute__((ext_vector_type(4)));
typedef int mm_i32x8 __attribute__((ext_vector_type(8)));
typedef short mm_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

struct f8_t { uint8_t v; };  // e4m3

constexpr int MM_STAGE = 128;  // bytes of a row's inner axis a stage
constexpr uint32_t MM_PAST = 0x80000000u;  // an offset behind every buffer

// ---------------------------------------------------------------- walking the experts

// Inclusive sums over the wavefront, saturating.
__device__ __forceinline__ uint32_t mm_scan(uint32_t v) {
  auto add = [&](int from) { v = __builtin_elementwise_add_sat(v, (uint32_t)from); };
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return v;
}

// The groups' rows cut into pieces of `size`: 64 groups at a time, one a lane. REST: the
// rows behind the last group are group `groups`; else every group has a piece at least.
template <bool REST>
struct MmWalk {
  const int64_t* seglen;  // null: one group of all rows
  int groups;
  uint32_t rows, size;
  int base;                          // first group of the 64
  uint32_t rows_before, piece_before;  // in front of them
  uint32_t start, end, first, last;  // a lane's group: its rows, its pieces

  __device__ __forceinline__ void init(const int64_t* lens, int n, int64_t m, uint32_t piece) {
    seglen = lens;
    groups = n;
    rows = (uint32_t)m;
    size = piece;
    base = 0;
    rows_before = piece_before = 0;
    load();
  }
  __device__ __forceinline__ void load() {
    const int g = base + (int)(threadIdx.x % WAVE);
    uint32_t len = 0;
    if (g < groups) {
      // lengths that do not fit the rows are cut: every access stays in bounds
      const int64_t given = seglen ? seglen[g] : (int64_t)rows;
      len = given < 0 ? 0 : given > (int64_t)rows ? rows : (uint32_t)given;
    } else if (REST && g == groups) {
      len = rows;
    }
    const uint32_t sum = __builtin_elementwise_add_sat(rows_before, mm_scan(len));
    end = sum < rows ? sum : rows;
    start = sum - len < rows ? sum - len : rows;
    uint32_t pieces = (end - start) / size + ((end - start) % size != 0);
    if (!REST && g < groups && pieces == 0) pieces = 1;
    last = piece_before + mm_scan(pieces);
    first = last - pieces;
  }
  // The next 64 groups; false behind the last.
  __device__ __forceinline__ bool next() {
    if (base + WAVE >= groups + (REST ? 1 : 0)) return false;
    rows_before = (uint32_t)readlane_int((int)end, WAVE - 1);
    piece_before = (uint32_t)readlane_int((int)last, WAVE - 1);
    base += WAVE;
    load();
    return true;
  }
  // All pieces.
  __device__ __forceinline__ uint32_t total() {
    while (next()) {
    }
    const uint32_t n = (uint32_t)readlane_int((int)last, WAVE - 1);
    if (base) init(seglen, groups, rows, size);
    return n;
  }
  // The group of a piece (not before the last one asked for); false past the end.
  __device__ __forceinline__ bool find(uint32_t piece, int* group, uint32_t* s, uint32_t* e,
                                       uint32_t* p0, uint32_t* p1) {
    while (piece >= (uint32_t)readlane_int((int)last, WAVE - 1))
      if (!next()) return false;
    const uint64_t at = __ballot(piece >= first && piece < last);
    const int lane = __builtin_ctzll(at);
    *group = base + lane;
    *s = (uint32_t)readlane_int((int)start, lane);
    *e = (uint32_t)readlane_int((int)end, lane);
    *p0 = (uint32_t)readlane_int((int)first, lane);
    *p1 = (uint32_t)readlane_int((int)last, lane);
    return true;
  }
};

// Place `l` among `down` by `across` tiles: bands of 8 across, each from the top down.
__device__ __forceinline__ void mm_band(uint32_t l, uint32_t down, uint32_t across, uint32_t* i,
                                        uint32_t* j) {
  constexpr uint32_t W = 8;
  const uint32_t band = l / (down * W), in = l - band * (down * W);
  const uint32_t w = across - band * W < W ? across - band * W : W;
  *i = in / w;
  *j = band * W + (in - *i * w);
}

// The tiles of a workgroup: the run of its XCD, in steps of the XCD's workgroups.
struct MmOrder {
  uint32_t at, end, step;
  __device__ __forceinline__ void init(uint32_t total) {
    const uint32_t x = blockIdx.x % 8;
    at = (uint32_t)((uint64_t)total * x / 8) + blockIdx.x / 8;
    end = (uint32_t)((uint64_t)total * (x + 1) / 8);
    step = gridDim.x / 8;  // a multiple of 8 workgroups are launched
  }
};

// ---------------------------------------------------------------- memory to LDS

// A buffer of `bytes` from p on, uniform over the wavefront.
__device__ __forceinline__ mm_i32x4 mm_buffer(const char* p, int64_t bytes) {
  const uint64_t a = (uint64_t)p;
  const uint32_t n = bytes <= 0 ? 0u : bytes < (int64_t)MM_PAST ? (uint32_t)bytes : MM_PAST;
  mm_i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)n);
  r[3] = 0x00020000;
  return r;
}

// 16 (4) bytes a lane from the buffer to consecutive LDS places from `lds` on; zeros
// where the offset lies behind the buffer. It is waited for with the vector memory
// counter, which the compiler does not do for it.
__device__ __forceinline__ void mm_load16(mm_i32x4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(buf), "s"(lds)
               : "m0");
}
__device__ __forceinline__ void mm_load4(mm_i32x4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dword %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(buf), "s"(lds)
               : "m0");
}

// The first `left` bytes of the 16 at p (of values of SIZE bytes), zeros behind them.
template <int SIZE>
__device__ __forceinline__ mm_i32x4 mm_read16(const char* p, int64_t left) {
  using U = std::conditional_t<SIZE == 2, uint16_t, uint8_t>;
  mm_i32x4 v = {0, 0, 0, 0};
  if (left >= 16) {
    U raw[16 / SIZE];
    load_any<false>(reinterpret_cast<const U*>(p), raw);
    __builtin_memcpy(&v, raw, 16);
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < 16; i += SIZE) {
      if (i >= left) continue;
      v[i / 4] |= (int)((uint32_t)*reinterpret_cast<const U*>(p + i) << 8 * (i % 4));
    }
  }
  return v;
}

// At most `n` of the wavefront's loads to LDS outstanding, and none of its LDS reads,
// then all wavefronts of the workgroup here.
template <int N>
__device__ __forceinline__ void mm_wait() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 & 3) << 14 | 7 << 4);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// An operand whose inner axis is contiguous: ROWS rows of a stage's 128 bytes.
// SECOND: the operand whose rows are dealt out to lanes in fours of eight (b).
template <int ROWS, int THREADS, int SIZE, bool SECOND, bool DIRECT>
struct MmAlong {
  static constexpr int BYTES = ROWS * MM_STAGE;
  static constexpr int PIECES = ROWS * 8;
  static constexpr int LOADS = PIECES < THREADS ? 1 : PIECES / THREADS;
  static constexpr int STEP = THREADS / 8;  // rows a load of the workgroup
  mm_i32x4 buf;
  const char* p;
  mm_i32x4 held[DIRECT ? 1 : LOADS];
  uint32_t off, lds;  // this lane's source; this wavefront's place
  uint32_t stride;    // bytes of a row
  int col;            // bytes to its place in a row
  int row, live;

  __device__ static __forceinline__ int swizzle(int r) {
    return SECOND ? (r & 3) | (r >> 1 & 4) : r & 7;
  }
  __device__ __forceinline__ void init(uint32_t row_bytes) {
    // with fewer pieces than threads some wavefronts load the same ones again
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE) % (PIECES / WAVE);
    const int piece = wave * WAVE + (int)(threadIdx.x % WAVE);
    row = piece / 8;
    col = ((piece & 7) ^ swizzle(row)) * 16;
    stride = row_bytes;
    off = (uint32_t)row * stride + (uint32_t)col;
    lds = (uint32_t)wave * (WAVE * 16);
  }
  // `rows` rows from `from` on.
  __device__ __forceinline__ void tile(const char* from, int rows) {
    live = rows < ROWS ? rows : ROWS;
    p = from;
    if constexpr (DIRECT) buf = mm_buffer(from, (int64_t)live * stride);
  }
  __device__ __forceinline__ void issue(uint32_t at, uint32_t stage) {
    const uint32_t in = stage * MM_STAGE;
    if constexpr (DIRECT) {
      const uint32_t o = in + (uint32_t)col < stride ? off + in : MM_PAST;
      const uint32_t more = in + (uint32_t)col < stride ? STEP * stride : 0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) mm_load16(buf, o + i * more, at + lds + i * (THREADS * 16));
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int r = row + i * STEP;
        held[i] = mm_read16<SIZE>(p + (int64_t)r * stride + in + col,
                                  r < live ? (int64_t)stride - in - col : 0);
      }
    }
  }
  __device__ __forceinline__ void commit(uint32_t at) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *(__attribute__((address_space(3))) mm_i32x4*)(lds_char*)(uintptr_t)(
          at + lds + (threadIdx.x % WAVE) * 16 + i * (THREADS * 16)) = held[i];
  }
  // Where this lane reads its pieces of row block 0 of its wavefront: [kk] of 16 bits,
  // [half] of 8.
  __device__ static __forceinline__ uint32_t read_at(int piece) {
    const int l = threadIdx.x % 16;
    const int r = SECOND ? 8 * (l / 4) + l % 4 : l;
    return (uint32_t)(r * MM_STAGE + ((piece ^ swizzle(r)) * 16));
  }
};

// An operand whose other axis is contiguous (16 bits): 64 inner places of COLS columns.
template <int COLS, int THREADS, bool DIRECT>
struct MmAcross {
  static constexpr int BYTES = COLS * MM_STAGE;
  static constexpr int ROW = COLS * 2;  // bytes
  static constexpr int PER = COLS / 8;  // pieces a row
  static constexpr int LOADS = 64 * PER / THREADS;
  static constexpr int STEP = THREADS / PER;
  static_assert(STEP % 4 == 0 && COLS >= 64, "");
  mm_i32x4 buf;
  const char* p;
  mm_i32x4 held[DIRECT ? 1 : LOADS];
  uint32_t off, lds, stride;
  int row, col;
  int64_t left;   // inner places from the tile's first on
  int64_t width;  // bytes of a row from the tile's first column on

  __device__ static __forceinline__ int swizzle(int r) { return COLS >= 128 ? r & 3 : r & 1; }
  __device__ __forceinline__ void init(uint32_t row_bytes) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
    const int piece = wave * WAVE + (int)(threadIdx.x % WAVE);
    row = piece / PER;
    const int at = piece % PER;
    col = (((at >> 2) ^ swizzle(row)) * 4 + (at & 3)) * 16;
    stride = row_bytes;
    off = (uint32_t)row * stride + (uint32_t)col;
    lds = (uint32_t)wave * (WAVE * 16);
  }
  // `places` inner places from `from` on, `columns` (bytes) of each wanted.
  __device__ __forceinline__ void tile(const char* from, int64_t places, int64_t columns) {
    p = from;
    left = places;
    width = columns;
  }
  __device__ __forceinline__ void issue(uint32_t at, uint32_t stage) {
    const int64_t first = (int64_t)stage * 64;
    const char* from = p + first * stride;
    if constexpr (DIRECT) {
      // columns past the width hold what follows in memory: they meet only results
      // that are not written
      buf = mm_buffer(from, (left - first - 1) * stride + width);
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        mm_load16(buf, off + i * (STEP * stride), at + lds + i * (THREADS * 16));
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int r = row + i * STEP;
        held[i] = mm_read16<2>(from + (int64_t)r * stride + col, first + r < left ? width - col : 0);
      }
    }
  }
  __device__ __forceinline__ void commit(uint32_t at) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      *(__attribute__((address_space(3))) mm_i32x4*)(lds_char*)(uintptr_t)(
          at + lds + (threadIdx.x % WAVE) * 16 + i * (THREADS * 16)) = held[i];
  }
  // Where this lane reads block `unit` of 32 columns: inner places 8 q + l / 4. FOURS:
  // the lane's four columns of eight (b), else 16 columns after one another.
  template <bool FOURS>
  __device__ static __forceinline__ uint32_t read_at(int unit) {
    const int l = threadIdx.x % 16, q = threadIdx.x % WAVE / 16, r = 8 * q + l / 4;
    return (uint32_t)(r * ROW + (unit ^ swizzle(r)) * 64 + (l % 4) * (FOURS ? 16 : 8));
  }
};

// ---------------------------------------------------------------- operands and products

__device__ __forceinline__ mm_i32x4 mm_lds16(uint32_t at) {
  return *(__attribute__((address_space(3))) mm_i32x4*)(lds_char*)(uintptr_t)at;
}
__device__ __forceinline__ float mm_lds4(uint32_t at) {
  return *(__attribute__((address_space(3))) float*)(lds_char*)(uintptr_t)at;
}
// Eight inner places of this lane's column: two transposing loads, four rows apart.
__device__ __forceinline__ mm_i32x4 mm_lds_turned(uint32_t at, uint32_t four_rows) {
  typedef __attribute__((address_space(3))) mm_i16x4 L;
  const mm_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(lds_char*)(uintptr_t)at);
  const mm_i16x4 hi =
      __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(lds_char*)(uintptr_t)(at + four_rows));
  return __builtin_bit_cast(mm_i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ mm_f32x4 mm_mul(bf16_t, mm_i32x4 x, mm_i32x4 y, mm_f32x4 c) {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y),
                                                 c, 0, 0, 0);
}
__device__ __forceinline__ mm_f32x4 mm_mul(f16_t, mm_i32x4 x, mm_i32x4 y, mm_f32x4 c) {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y),
                                                c, 0, 0, 0);
}
// 128 inner places of 8 bits, no scales of the instruction's own. The matrix cores add
// the products of eight neighbouring places cut off 13 binary places below the largest of
// them (measured: 2^16 + 2^3 is whole, 2^16 + 2^2 is 2^16; what lies in other eights or
// in the accumulator is not cut), so a block's sum is off by 7 * 2^-13 of the largest
// products of its eights at most (1.4 % of the half step that e4m3 values were rounded
// by). The instruction of 32 places does the same; values made 16 bits wide first would be
// exact, at half the rate. Sums of blocks are float.
__device__ __forceinline__ mm_f32x4 mm_mul8(mm_i32x8 x, mm_i32x8 y) {
  const mm_f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, zero, 0, 0, 0, 0, 0, 0);
}

// The sums of a wavefront's MI by NJ blocks (lane: row l % 16, columns 4 (l / 16) ..)
// written from (row, n) on, rows below `end`, columns below N.
template <int MI, int NJ, class O>
__device__ __forceinline__ void mm_write(const mm_f32x4 (&acc)[MI][NJ], O* out, int64_t row,
                                         int64_t end, int64_t n, int64_t N) {
  const int l = threadIdx.x % 16, q = threadIdx.x % WAVE / 16;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t r = row + i * 16 + l;
    if (r >= end) continue;
#pragma unroll
    for (int j = 0; j < NJ; j += 2) {
      const int64_t c = n + j * 16 + q * 8;
      O* to = out + r * N + c;
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = acc[i][j][k];
        v[k + 4] = acc[i][j + 1][k];
      }
      if (c + 8 <= N) {
        store_acc<O, float, 8>(to, v);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (c + k < N) to[k] = (O)v[k];
      }
    }
  }
}

template <int MI, int NJ>
__device__ __forceinline__ void mm_zero(mm_f32x4 (&acc)[MI][NJ]) {
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

template <class E, int BM_, int BN_, int WM_, int WN_, int ST_, bool ALONG_, bool DIRECT_>
struct MmConf {
  using Elem = E;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr bool ALONG = ALONG_;    // b's inner axis is contiguous
  static constexpr bool DIRECT = DIRECT_;  // from memory to LDS past the registers
  static constexpr int ST = ST_;
  static constexpr int THREADS = WM * WN * WAVE;
  static constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  static constexpr bool EIGHT = sizeof(E) == 1;
  static constexpr int SIZE = (int)sizeof(E);
  static constexpr int INNER = MM_STAGE / SIZE;  // inner places a stage
  using A = MmAlong<BM, THREADS, SIZE, false, DIRECT>;
  using B = std::conditional_t<ALONG, MmAlong<BN, THREADS, SIZE, true, DIRECT>,
                               MmAcross<BN, THREADS, DIRECT>>;
  static constexpr int SCALES = EIGHT ? (BM < WAVE ? WAVE : BM) * 4 : 0;
  static constexpr int STAGE_BYTES = A::BYTES + B::BYTES + SCALES;
  static constexpr int LOADS = A::LOADS + B::LOADS + (EIGHT ? 1 : 0);
  // workgroups on a compute unit, two at most (their LDS: 160 KB); one of eight
  // wavefronts that load 8-bit values through registers
  static constexpr int PER_CU =
      2 * ST * STAGE_BYTES <= 163840 && !(EIGHT && !DIRECT && THREADS > 256) ? 2 : 1;
  static constexpr int WAVES = PER_CU * THREADS / 256 > 0 ? PER_CU * THREADS / 256 : 1;
  static_assert(NJ % 2 == 0 && (DIRECT || ST == 2) && (ST - 2) * LOADS < 64, "");
  static_assert(!EIGHT || (ALONG && BM / WAVE <= WM * WN && 128 % (BN / WN) == 0), "");
};

struct MmArgs {
  const char* a;
  const char* b;
  const float* sa;  // 8 bits: [rows][blocks of K]
  const float* sb;  // [groups][blocks of K][blocks of N]
  void* out;
  const int64_t* seglen;
  int64_t rows;
  int groups, K, N;
  int out_dtype;  // 8 bits
  float* part;    // [splits][rows][N] with splits > 1
  int splits;     // parts of the inner axis, each a tile of its own
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::WAVES) expert_mm_kernel(MmArgs p) {
  using E = typename C::Elem;
  __shared__ __align__(256) char lds[C::ST * C::STAGE_BYTES];
  const uint32_t lds0 =
      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_char*)lds);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int l = threadIdx.x % 16, q = threadIdx.x % WAVE / 16;
  const int64_t row_bytes = (int64_t)p.K * C::SIZE;
  const uint32_t across = (uint32_t)((p.N + C::BN - 1) / C::BN);
  const int stages = (p.K + C::INNER - 1) / C::INNER;

  struct Tile {
    MmWalk<true> walk;
    MmOrder order;
    int group, part, stage0, stage1;
    uint32_t row, end, col;
    bool any;
  };
  auto seek = [&](Tile& t) {
    t.any = false;
    if (t.order.at >= t.order.end) return;
    uint32_t s, e, p0, p1, i, j;
    const uint32_t at = t.order.at / p.splits;
    t.part = (int)(t.order.at - at * p.splits);
    t.order.at += t.order.step;
    if (!t.walk.find(at / across, &t.group, &s, &e, &p0, &p1)) return;
    mm_band(at - p0 * across, p1 - p0, across, &i, &j);
    t.stage0 = (int)((int64_t)stages * t.part / p.splits);
    // the rest has no inner axis
    t.stage1 = t.group < p.groups ? (int)((int64_t)stages * (t.part + 1) / p.splits) : t.stage0;
    t.row = s + i * C::BM;
    t.end = e;
    t.col = j * C::BN;
    t.any = true;
  };
  Tile mine;  // what is multiplied
  mine.walk.init(p.seglen, p.groups, p.rows, C::BM);
  mine.order.init(mine.walk.total() * across * p.splits);
  Tile ahead = mine;  // what is loaded

  typename C::A A;
  typename C::B B;
  A.init((uint32_t)row_bytes);
  B.init(C::ALONG ? (uint32_t)row_bytes : (uint32_t)p.N * 2);
  [[maybe_unused]] mm_i32x4 scales;
  [[maybe_unused]] uint32_t scale_off = 0, scale_lds = 0;
  [[maybe_unused]] float scale_held = 0.0f;
  const int kb = (p.K + 127) / 128, nb = (p.N + 127) / 128;
  [[maybe_unused]] const int scale_row =
      wave % (C::SCALES / 256 + !C::EIGHT) * WAVE + (int)(threadIdx.x % WAVE);
  if constexpr (C::EIGHT) {
    scale_off = (uint32_t)scale_row * kb * 4;
    scale_lds = C::A::BYTES + C::B::BYTES + wave % (C::SCALES / 256) * 256;
  }
  int ahead_stage = 0;
  auto open = [&]() {  // the tile to load from
    do seek(ahead);
    while (ahead.any && ahead.stage0 == ahead.stage1);
    if (!ahead.any) return;
    const int rows = (int)(ahead.end - ahead.row);
    A.tile(p.a + ahead.row * row_bytes, rows);
    const char* block = p.b + ahead.group * (row_bytes * p.N);
    if constexpr (C::ALONG) {
      B.tile(block + ahead.col * row_bytes, p.N - (int)ahead.col);
    } else {
      B.tile(block + (int64_t)ahead.col * 2, p.K, (int64_t)(p.N - (int)ahead.col) * 2);
    }
    if constexpr (C::EIGHT) {
      const char* from = (const char*)(p.sa + (int64_t)ahead.row * kb);
      scales = mm_buffer(from, (int64_t)(rows < C::BM ? rows : C::BM) * kb * 4);
    }
    ahead_stage = ahead.stage0;
  };
  uint32_t fill = 0, use = 0;  // places in the ring
  auto issue = [&]() {
    if (!ahead.any) return;
    const uint32_t at = lds0 + fill * C::STAGE_BYTES;
    A.issue(at, ahead_stage);
    B.issue(at + C::A::BYTES, ahead_stage);
    if constexpr (C::EIGHT) {
      if constexpr (C::DIRECT) {
        mm_load4(scales, scale_off + ahead_stage * 4, at + scale_lds);
      } else {
        const int rows = (int)(ahead.end - ahead.row);
        scale_held = scale_row < (rows < C::BM ? rows : C::BM)
                         ? p.sa[(int64_t)(ahead.row + scale_row) * kb + ahead_stage] : 0.0f;
      }
    }
    if constexpr (C::DIRECT) {
      fill = fill + 1 == C::ST ? 0 : fill + 1;
      if (++ahead_stage == ahead.stage1) open();
    }
  };
  // through registers: what was issued before goes to LDS behind the products
  auto commit = [&]() {
    if constexpr (!C::DIRECT) {
      if (!ahead.any) return;
      const uint32_t at = lds0 + fill * C::STAGE_BYTES;
      A.commit(at);
      B.commit(at + C::A::BYTES);
      if constexpr (C::EIGHT)
        *(__attribute__((address_space(3))) float*)(lds_char*)(uintptr_t)(
            at + scale_lds + (threadIdx.x % WAVE) * 4) = scale_held;
      fill ^= 1;
      if (++ahead_stage == ahead.stage1) open();
    }
  };

  // what this lane reads, from a stage's start on
  uint32_t a_at[2], b_at[C::ALONG ? 4 : C::NJ / 2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int piece = C::EIGHT ? 2 * q + h : 4 * h + q;
    a_at[h] = (uint32_t)(wm * (C::BM / C::WM) * MM_STAGE) + C::A::read_at(piece);
    if constexpr (C::ALONG) {
      const uint32_t at = (uint32_t)C::A::BYTES + wn * (C::BN / C::WN) * MM_STAGE;
      b_at[h] = at + C::B::read_at(piece);
      // the second four of eight: four rows on, whose swizzle does not change
      b_at[h + 2] = b_at[h] + 4 * MM_STAGE;
    }
  }
  if constexpr (!C::ALONG)
#pragma unroll
    for (int j = 0; j < C::NJ / 2; ++j)
      b_at[j] = (uint32_t)C::A::BYTES +
                C::B::template read_at<true>(wn * (C::BN / C::WN / 32) + j);

  mm_f32x4 acc[C::MI][C::NJ];
  auto multiply = [&](uint32_t at, [[maybe_unused]] int stage) {
    if constexpr (C::EIGHT) {
      typedef const __attribute__((address_space(4))) float CF;
      const int n = (int)mine.col + wn * (C::BN / C::WN);
      const int c = n / 128 < nb ? n / 128 : nb - 1;
      const float sb = *(CF*)(p.sb + ((int64_t)mine.group * kb + stage) * nb + c);
      mm_i32x8 x[C::MI];
      float s[C::MI];
#pragma unroll
      for (int i = 0; i < C::MI; ++i) {
        const mm_i32x4 lo = mm_lds16(at + a_at[0] + i * 16 * MM_STAGE);
        const mm_i32x4 hi = mm_lds16(at + a_at[1] + i * 16 * MM_STAGE);
        x[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        s[i] = sb * mm_lds4(at + C::A::BYTES + C::B::BYTES +
                            (wm * (C::BM / C::WM) + i * 16 + l) * 4);
      }
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        const uint32_t more = j / 2 * 32 * MM_STAGE;
        const mm_i32x4 lo = mm_lds16(at + b_at[j % 2 * 2] + more);
        const mm_i32x4 hi = mm_lds16(at + b_at[j % 2 * 2 + 1] + more);
        const mm_i32x8 y = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int i = 0; i < C::MI; ++i) {
          const mm_f32x4 t = mm_mul8(y, x[i]);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            acc[i][j][k] = __builtin_fmaf(t[k], s[i], acc[i][j][k]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mm_i32x4 x[C::MI], y[C::NJ];
#pragma unroll
        for (int i = 0; i < C::MI; ++i) x[i] = mm_lds16(at + a_at[h] + i * 16 * MM_STAGE);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
          if constexpr (C::ALONG)
            y[j] = mm_lds16(at + b_at[h + j % 2 * 2] + j / 2 * 32 * MM_STAGE);
          else
            y[j] = mm_lds_turned(at + b_at[j / 2] + j % 2 * 8 + h * 32 * C::B::ROW, 4 * C::B::ROW);
        }
#pragma unroll
        for (int i = 0; i < C::MI; ++i)
#pragma unroll
          for (int j = 0; j < C::NJ; ++j) acc[i][j] = mm_mul(E{}, y[j], x[i], acc[i][j]);
      }
    }
  };

  open();
  if constexpr (C::DIRECT) {
    for (int i = 0; i < C::ST - 1; ++i) issue();
  } else {
    issue();
    commit();
  }
  for (seek(mine); mine.any; seek(mine)) {
    mm_zero(acc);
    for (int s = mine.stage0; s < mine.stage1; ++s) {
      // behind the last load fewer are outstanding than the ring holds
      if (C::ST > 2 && ahead.any) mm_wait<(C::ST - 2) * C::LOADS>();
      else mm_wait<0>();
      issue();
      multiply(lds0 + use * C::STAGE_BYTES, s);
      commit();
      use = use + 1 == C::ST ? 0 : use + 1;
    }
    const int64_t row = (int64_t)mine.row + wm * (C::BM / C::WM);
    const int64_t n = (int64_t)mine.col + wn * (C::BN / C::WN);
    if (p.splits > 1) {
      mm_write(acc, p.part + mine.part * (p.rows * p.N), row, mine.end, n, p.N);
    } else if constexpr (C::EIGHT) {
      if (p.out_dtype == DT_F32) mm_write(acc, (float*)p.out, row, mine.end, n, p.N);
      else if (p.out_dtype == DT_BF16) mm_write(acc, (bf16_t*)p.out, row, mine.end, n, p.N);
      else mm_write(acc, (f16_t*)p.out, row, mine.end, n, p.N);
    } else {
      mm_write(acc, (E*)p.out, row, mine.end, n, p.N);
    }
  }
}

// The parts of the inner axis added in order.
template <class O>
__global__ void __launch_bounds__(BLOCK) expert_mm_join_kernel(const float* part, O* out,
                                                               int64_t size, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * 4;
  if (i >= size) return;
  const int n = size - i < 4 ? (int)(size - i) : 4;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) {
    const float* from = part + s * size + i;
    if (n == 4) {
      float x[4];
      load_any<false>(from, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += x[k];
    } else {
      for (int k = 0; k < n; ++k) v[k] += from[k];
    }
  }
  if (n == 4) {
    store_acc<O, float, 4>(out + i, v);
  } else {
    for (int k = 0; k < n; ++k) out[i + k] = (O)v[k];
  }
}

// The gradient of b: out[g] = a[rows of g]^T grad[rows of g], [D1][D2] each, in tiles of
// BM of D1 by BN of D2, the inner axis along the rows. A group of more rows than a piece
// holds leaves one partial result a piece, which expert_mm_sum_kernel adds in order.
struct MmGradArgs {
  const char* a;     // [rows][D1]
  const char* grad;  // [rows][D2]
  void* out;
  float* part;  // [pieces][D1][D2]; null: every group is one piece
  const int64_t* seglen;
  int64_t rows;
  int groups, D1, D2;
  uint32_t piece;
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::WAVES) expert_mm_grad_kernel(MmGradArgs p) {
  using E = typename C::Elem;
  using A = MmAcross<C::BM, C::THREADS, C::DIRECT>;
  using B = MmAcross<C::BN, C::THREADS, C::DIRECT>;
  constexpr int BYTES = A::BYTES + B::BYTES, LOADS = A::LOADS + B::LOADS;
  __shared__ __align__(256) char lds[C::ST * BYTES];
  const uint32_t lds0 =
      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_char*)lds);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const uint32_t down = (uint32_t)((p.D1 + C::BM - 1) / C::BM);
  const uint32_t across = (uint32_t)((p.D2 + C::BN - 1) / C::BN);

  struct Tile {
    MmWalk<false> walk;
    MmOrder order;
    int group;
    uint32_t start, row, col, piece;  // first row of the piece; the tile's place
    int stages, rows;
    bool any, alone;
  };
  auto seek = [&](Tile& t) {
    t.any = false;
    if (t.order.at >= t.order.end) return;
    uint32_t s, e, p0, p1, i, j;
    const uint32_t at = t.order.at;
    t.order.at += t.order.step;
    t.piece = at / (down * across);
    if (!t.walk.find(t.piece, &t.group, &s, &e, &p0, &p1)) return;
    mm_band(at - t.piece * (down * across), down, across, &i, &j);
    t.start = s + (t.piece - p0) * p.piece;
    const uint32_t rows = e - t.start;
    t.rows = (int)(rows < p.piece ? rows : p.piece);
    t.stages = (t.rows + 63) / 64;
    t.row = i * C::BM;
    t.col = j * C::BN;
    t.alone = p1 - p0 == 1;
    t.any = true;
  };
  Tile mine;
  mine.walk.init(p.seglen, p.groups, p.rows, p.piece);
  mine.order.init(mine.walk.total() * (down * across));
  Tile ahead = mine;

  A la;
  B lb;
  la.init((uint32_t)p.D1 * 2);
  lb.init((uint32_t)p.D2 * 2);
  int ahead_stage = 0;
  auto open = [&]() {  // pieces without rows have nothing to load
    do seek(ahead);
    while (ahead.any && ahead.stages == 0);
    if (!ahead.any) return;
    la.tile(p.a + ((int64_t)ahead.start * p.D1 + ahead.row) * 2, ahead.rows,
            (int64_t)(p.D1 - (int)ahead.row) * 2);
    lb.tile(p.grad + ((int64_t)ahead.start * p.D2 + ahead.col) * 2, ahead.rows,
            (int64_t)(p.D2 - (int)ahead.col) * 2);
    ahead_stage = 0;
  };
  uint32_t fill = 0, use = 0;
  auto issue = [&]() {
    if (!ahead.any) return;
    const uint32_t at = lds0 + fill * BYTES;
    la.issue(at, ahead_stage);
    lb.issue(at + A::BYTES, ahead_stage);
    if constexpr (C::DIRECT) {
      fill = fill + 1 == C::ST ? 0 : fill + 1;
      if (++ahead_stage == ahead.stages) open();
    }
  };
  auto commit = [&]() {
    if constexpr (!C::DIRECT) {
      if (!ahead.any) return;
      const uint32_t at = lds0 + fill * BYTES;
      la.commit(at);
      lb.commit(at + A::BYTES);
      fill ^= 1;
      if (++ahead_stage == ahead.stages) open();
    }
  };

  uint32_t a_at[C::MI / 2], b_at[C::NJ / 2];
#pragma unroll
  for (int i = 0; i < C::MI / 2; ++i)
    a_at[i] = A::template read_at<false>(wm * (C::BM / C::WM / 32) + i);
#pragma unroll
  for (int j = 0; j < C::NJ / 2; ++j)
    b_at[j] = (uint32_t)A::BYTES + B::template read_at<true>(wn * (C::BN / C::WN / 32) + j);
  mm_f32x4 acc[C::MI][C::NJ];
  auto multiply = [&](uint32_t at) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mm_i32x4 x[C::MI], y[C::NJ];
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
        x[i] = mm_lds_turned(at + a_at[i / 2] + i % 2 * 32 + h * 32 * A::ROW, 4 * A::ROW);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j)
        y[j] = mm_lds_turned(at + b_at[j / 2] + j % 2 * 8 + h * 32 * B::ROW, 4 * B::ROW);
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) acc[i][j] = mm_mul(E{}, y[j], x[i], acc[i][j]);
    }
  };

  open();
  if constexpr (C::DIRECT) {
    for (int i = 0; i < C::ST - 1; ++i) issue();
  } else {
    issue();
    commit();
  }
  for (seek(mine); mine.any; seek(mine)) {
    mm_zero(acc);
    for (int s = 0; s < mine.stages; ++s) {
      if (C::ST > 2 && ahead.any) mm_wait<(C::ST - 2) * LOADS>();
      else mm_wait<0>();
      issue();
      multiply(lds0 + use * BYTES);
      commit();
      use = use + 1 == C::ST ? 0 : use + 1;
    }
    const int64_t row = (int64_t)mine.row + wm * (C::BM / C::WM);
    const int64_t n = (int64_t)mine.col + wn * (C::BN / C::WN);
    const int64_t size = (int64_t)p.D1 * p.D2;
    if (mine.alone)
      mm_write(acc, (E*)p.out + mine.group * size, row, p.D1, n, p.D2);
    else
      mm_write(acc, p.part + mine.piece * size, row, p.D1, n, p.D2);
  }
}

// Results of groups of several pieces: blockIdx.y a group, four values a thread.
template <class E>
__global__ void __launch_bounds__(BLOCK) expert_mm_sum_kernel(MmGradArgs p) {
  MmWalk<false> walk;
  walk.init(p.seglen, p.groups, p.rows, p.piece);
  const int g = blockIdx.y;
  while (g >= walk.base + WAVE) walk.next();
  const uint32_t p0 = (uint32_t)readlane_int((int)walk.first, g - walk.base);
  const uint32_t p1 = (uint32_t)readlane_int((int)walk.last, g - walk.base);
  if (p1 - p0 == 1) return;
  const int64_t size = (int64_t)p.D1 * p.D2;
  for (int64_t i = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * 4; i < size;
       i += (int64_t)gridDim.x * BLOCK * 4) {
    const int n = size - i < 4 ? (int)(size - i) : 4;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t c = p0; c < p1; ++c) {
      const float* from = p.part + c * size + i;
      if (n == 4) {
        float x[4];
        load_any<false>(from, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += x[k];
      } else {
        for (int k = 0; k < n; ++k) v[k] += from[k];
      }
    }
    E* to = (E*)p.out + g * size + i;
    for (int k = 0; k < n; ++k) to[k] = (E)v[k];
  }
}

template <class C>
hipError_t run_expert_mm_grad(const MmGradArgs& p, int64_t most_tiles, hipStream_t s) {
  const int64_t full = 256 * C::PER_CU;
  const int64_t grid = most_tiles < full ? (most_tiles + 7) / 8 * 8 : full;
  expert_mm_grad_kernel<C><<<grid, C::THREADS, 0, s>>>(p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.part) return e;
  const int64_t blocks = ((int64_t)p.D1 * p.D2 + BLOCK * 4 - 1) / (BLOCK * 4);
  expert_mm_sum_kernel<typename C::Elem>
      <<<dim3((unsigned)(blocks < 1024 ? blocks : 1024), p.groups), BLOCK, 0, s>>>(p);
  return hipGetLastError();
}

template <class O>
hipError_t run_expert_mm_join(const MmArgs& p, hipStream_t s) {
  const int64_t size = p.rows * p.N, grid = (size + BLOCK * 4 - 1) / (BLOCK * 4);
  expert_mm_join_kernel<O><<<grid, BLOCK, 0, s>>>(p.part, (O*)p.out, size, p.splits);
  return hipGetLastError();
}

template <class C>
hipError_t run_expert_mm(const MmArgs& p, int64_t most_tiles, hipStream_t s) {
  const int64_t full = 256 * C::PER_CU;
  const int64_t grid = most_tiles < full ? (most_tiles + 7) / 8 * 8 : full;
  expert_mm_kernel<C><<<grid, C::THREADS, 0, s>>>(p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  using E = typename C::Elem;
  if constexpr (C::EIGHT) {
    if (p.out_dtype == DT_F32) return run_expert_mm_join<float>(p, s);
    if (p.out_dtype == DT_BF16) return run_expert_mm_join<bf16_t>(p, s);
    return run_expert_mm_join<f16_t>(p, s);
  } else {
    return run_expert_mm_join<E>(p, s);
  }
}

// The shapes of mm_shapes (expert_mm_plan.hip).
template <class E, bool ALONG>
hipError_t run_expert_mm_shape(const ExpertMmParams& q) {
  MmArgs p{};
  p.a = (const char*)q.a;
  p.b = (const char*)q.b;
  p.sa = q.a_scale;
  p.sb = q.b_scale;
  p.out = q.out;
  p.seglen = q.seglen;
  p.rows = q.rows;
  p.groups = (int)q.groups;
  p.K = (int)q.inner;
  p.N = (int)q.cols;
  p.out_dtype = q.out_dtype;
  p.part = (float*)q.workspace;
  p.splits = q.plan.splits;
  const int64_t tiles = q.plan.tiles;
  hipStream_t s = q.stream;
  switch (q.plan.shape) {
    case 0: return run_expert_mm<MmConf<E, 64, 128, 1, 4, 3, ALONG, true>>(p, tiles, s);
    case 1: return run_expert_mm<MmConf<E, 128, 128, 2, 2, 2, ALONG, true>>(p, tiles, s);
    case 2: return run_expert_mm<MmConf<E, 256, 256, 2, 4, 2, ALONG, true>>(p, tiles, s);
    case 3: return run_expert_mm<MmConf<E, 64, 128, 1, 4, 2, ALONG, false>>(p, tiles, s);
    default:
      // eight wavefronts where four would hold more values than they have registers
      return run_expert_mm<MmConf<E, 128, 128, 2, sizeof(E) == 1 ? 4 : 2, 2, ALONG, false>>(
          p, tiles, s);
  }
}

template <class E>
hipError_t run_expert_mm_grad_shape(const ExpertMmParams& q) {
  MmGradArgs p{};
  p.a = (const char*)q.a;
  p.grad = (const char*)q.b;
  p.out = q.out;
  p.part = (float*)q.workspace;
  p.seglen = q.seglen;
  p.rows = q.rows;
  p.groups = (int)q.groups;
  p.D1 = (int)q.inner;
  p.D2 = (int)q.cols;
  p.piece = (uint32_t)q.plan.piece;
  const int64_t tiles = q.plan.tiles;
  hipStream_t s = q.stream;
  switch (q.plan.shape) {
    case 1: return run_expert_mm_grad<MmConf<E, 128, 128, 2, 2, 2, false, true>>(p, tiles, s);
    case 2: return run_expert_mm_grad<MmConf<E, 256, 256, 2, 4, 2, false, true>>(p, tiles, s);
    default: return run_expert_mm_grad<MmConf<E, 128, 128, 2, 2, 2, false, false>>(p, tiles, s);
  }
}

}  // namespace mdgl
