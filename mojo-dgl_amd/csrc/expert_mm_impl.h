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
// of 32 bytes lie at piece ^ swizzle(row), so that the eight rows that 32 lanes read use
// all banks.
//
// The product is formed transposed (b's values as the first operand), which leaves a
// lane with four neighbouring columns of one row; an exchange between lanes makes them
// eight: results leave in stores of 16 bytes.
//
// Past the edges: rows past the tile's group and inner places past the end are read as
// zeros by the buffer's own bounds check (a lane past the inner end is given an offset
// behind the buffer), so no stage has a case of its own. The loads take any alignment. Where
// a row may end inside a piece of 16 bytes, or an operand inside four of them, the tile's
// last stage is mended in LDS before it is read (kernels of their own: !WHOLE).
//
// Tiles are counted on the GPU from the experts' lengths, which the host need not know:
// every wavefront walks them 64 experts at a time. A tile index in the order of the
// experts, each in bands of 8 column tiles; an XCD takes one contiguous run of tiles,
// so that the rows and blocks its workgroups share lie in its own L2. Rows behind the
// last expert's form a group without an inner axis: they are written as zeros.
//
// Measured: 8,192 rows by 8,192 by 8,192 in 824 us (bfloat16, b's inner axis contiguous; 808
// the other way; 839 the gradient of b), where the matrix cores are busy for 55 % of the
// cycles, and in 476 us in 8 bits (normal values; of others up to 528, by what they draw).
// 65,536 rows of 2,048 to 1,536 through 64 experts: 425 us forward, 450 and 450 the
// gradients. There loads that came from L2 alone would save 11 to
// 19 %, no stores 6 to 16 %: the tiles of a round end together, and their results' burst delays
// the loads behind it. Few rows are bound by reading the experts called: 64 of them by 8
// rows each in 76 us (5.3 TB/s).
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
constexpr uint32_t MM_PAST = 0x80000000u;  // this and more: an offset behind every buffer

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
  uint32_t end, last;  // a lane's group: where its rows and its pieces end

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
    int lane = threadIdx.x % WAVE;
    asm volatile("" : "+v"(lane));  // its address is formed here, not held all along
    const int g = base + lane;
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
    const uint32_t start = sum - len < rows ? sum - len : rows;
    uint32_t pieces = (end - start) / size + ((end - start) % size != 0);
    if (!REST && g < groups && pieces == 0) pieces = 1;
    last = piece_before + mm_scan(pieces);
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
    const int lane = __builtin_ctzll(__ballot(piece < last));
    *group = base + lane;
    bounds(lane, s, e, p0, p1);
    return true;
  }
  __device__ __forceinline__ void bounds(int lane, uint32_t* s, uint32_t* e, uint32_t* p0,
                                         uint32_t* p1) const {
    *s = lane ? (uint32_t)readlane_int((int)end, lane - 1) : rows_before;
    *e = (uint32_t)readlane_int((int)end, lane);
    *p0 = lane ? (uint32_t)readlane_int((int)last, lane - 1) : piece_before;
    *p1 = (uint32_t)readlane_int((int)last, lane);
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
// counter, which the compiler does not do for it. Nor does it keep the distances that the
// machine asks for in front of it: one wait state behind m0, five behind a vector
// instruction that wrote a scalar register of `buf` (readlanes, of registers that the
// compiler keeps in lanes, too). The move and the s_nop are these five.
__device__ __forceinline__ void mm_load16(mm_i32x4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(buf), "s"(lds)
               : "m0");
}
__device__ __forceinline__ void mm_load4(mm_i32x4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dword %0, %1, 0 offen lds"
               :
               : "v"(off), "s"(buf), "s"(lds)
               : "m0");
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
template <int ROWS, int THREADS, int SIZE, bool WHOLE>
struct MmAlong {
  static constexpr int BYTES = ROWS * MM_STAGE;
  static constexpr int PIECES = ROWS * 8;
  static constexpr int LOADS = PIECES < THREADS ? 1 : PIECES / THREADS;
  static constexpr int STEP = THREADS / 8;  // rows a load of the workgroup
  mm_i32x4 buf;
  uint32_t off, lds;  // this lane's source; this wavefront's place
  uint32_t stride;    // bytes of a row
  int col;            // bytes to its place in a row
  uint32_t from;      // of the stage being loaded: this lane's source
  const char* lost;   // the last row's end, if the row's last bytes are not read
  int live;           // rows

  // 16 lanes are served at a time: two neighbouring q (read_at) of 8 rows, two rows to all
  // banks. In 16 bits they read pieces q and q + 1, in 8 bits 2 q and 2 q + 2.
  __device__ static __forceinline__ int swizzle(int r) {
    return SIZE == 1 ? (r >> 1 & 1) | (r & 4) : r & 7;
  }
  __device__ __forceinline__ void init(uint32_t row_bytes) {
    // with fewer pieces than threads some wavefronts load the same ones again
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE) % (PIECES / WAVE);
    const int piece = wave * WAVE + (int)(threadIdx.x % WAVE);
    const int row = piece / 8;
    col = ((piece & 7) ^ swizzle(row)) * 16;
    stride = row_bytes;
    off = (uint32_t)row * stride + (uint32_t)col;
    lds = (uint32_t)wave * (WAVE * 16);
  }
  // `rows` rows from `at` on, where the operand has `left` bytes.
  __device__ __forceinline__ void tile(const char* at, int rows, int64_t left) {
    live = rows < ROWS ? rows : ROWS;
    int64_t bytes = (int64_t)live * stride;
    if constexpr (!WHOLE) {
      // the bounds check is by four bytes: those that begin in the last row are wanted
      lost = nullptr;
      if (left >= bytes + 3) {
        bytes += 3;
      } else if (stride % 4) {
        lost = at + bytes;
      }
    }
    buf = mm_buffer(at, bytes);
  }
  // No tile: its loads give zeros. A workgroup may never have one, so nothing is left from
  // the tile before.
  __device__ __forceinline__ void none() { buf = mm_buffer(nullptr, 0); }
  __device__ __forceinline__ void begin(uint32_t stage) {
    from = stage * MM_STAGE + (uint32_t)col < stride ? off + stage * MM_STAGE : MM_PAST;
  }
  __device__ __forceinline__ void load(uint32_t at, int i) {
    mm_load16(buf, from + i * (STEP * stride), at + lds + i * (THREADS * 16));
  }
  // The last stage, where a row's last piece holds what follows in memory: zeros in its
  // place (not left to the other operand's zeros: what follows may be infinite).
  __device__ __forceinline__ void mend(uint32_t at) {
    const int end = (int)(stride % MM_STAGE), word = end % 16 / 4, more = end % 4;
    if (end % 16 == 0) return;
    int r = threadIdx.x;
    asm volatile("" : "+v"(r));  // its places are formed here, not held all along
    for (; r < ROWS; r += THREADS) {
      auto* piece = (__attribute__((address_space(3))) mm_i32x4*)(lds_char*)(uintptr_t)(
          at + r * MM_STAGE + ((end / 16 ^ swizzle(r)) * 16));
      mm_i32x4 v = *piece;
      uint32_t last = 0;
      // (rows of one byte: the last three end inside the operand's last four)
      const int behind = (live - 1 - r) * (int)stride;
      if (lost && behind >= 0 && behind + more < 4)
        for (int i = 0; i < more; ++i) last |= (uint32_t)(uint8_t)lost[i - more - behind] << 8 * i;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k == word) v[k] = (int)(((uint32_t)v[k] & ((1u << 8 * more) - 1)) | last);
        if (k > word) v[k] = 0;
      }
      *piece = v;
    }
  }
  // Where this lane reads piece `first` of its row of a block of 16; the pieces
  // 4 (of 16 bits) and 1 (of 8) behind it lie at the place xor 64 and 16, as stages start on
  // multiples of 256.
  __device__ static __forceinline__ uint32_t read_at(int first) {
    const int r = threadIdx.x % 16;
    return (uint32_t)(r * MM_STAGE + ((first ^ swizzle(r)) * 16));
  }
};

// An operand whose other axis is contiguous (16 bits): 64 inner places of COLS columns.
template <int COLS, int THREADS, bool WHOLE>
struct MmAcross {
  static constexpr int BYTES = COLS * MM_STAGE;
  static constexpr int ROW = COLS * 2;  // bytes
  static constexpr int PER = COLS / 8;  // pieces a row
  static constexpr int LOADS = 64 * PER / THREADS;
  static constexpr int STEP = THREADS / PER;
  static_assert(STEP % 16 == 0 && COLS >= 128, "");
  mm_i32x4 buf;
  const char* p;
  uint32_t off, lds, stride;
  int64_t bytes;  // to be read, from the tile's first on
  const char* lost;       // the operand's end, if its last value is not read
  uint32_t lost_at;       // that value's place in the stage

  __device__ static __forceinline__ int swizzle(int r) { return (r & 3) | (r >> 1 & 4); }
  // Piece `at` of row r lies at this place of it, and the other way round.
  __device__ static __forceinline__ int placed(int r, int at) {
    return ((at >> 1) ^ swizzle(r)) * 2 + (at & 1);
  }
  __device__ __forceinline__ void init(uint32_t row_bytes) {
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
    const int piece = wave * WAVE + (int)(threadIdx.x % WAVE);
    const int row = piece / PER;
    stride = row_bytes;
    off = (uint32_t)row * stride + (uint32_t)placed(row, piece % PER) * 16;
    lds = (uint32_t)wave * (WAVE * 16);
  }
  // `n` inner places from `at` on, `width` bytes to the end of a row; the operand has `left`
  // bytes there.
  __device__ __forceinline__ void tile(const char* at, int64_t n, int64_t width, int64_t left) {
    p = at;
    // columns past the width hold what follows in memory: they meet only results that are
    // not written
    bytes = (n - 1) * stride + width;
    if constexpr (!WHOLE) {  // as in MmAlong
      lost = nullptr;
      if (left >= bytes + 3) {
        bytes += 3;
      } else if (width % 4 && width <= ROW) {
        const int r = (int)(n - 1) % 64, c = (int)width - 2;
        lost = at + bytes;
        lost_at = (uint32_t)(r * ROW + placed(r, c / 16) * 16 + c % 16);
      }
    }
  }
  __device__ __forceinline__ void none() {
    p = nullptr;
    bytes = 0;
  }
  __device__ __forceinline__ void begin(uint32_t stage) {
    const int64_t first = (int64_t)stage * 64;
    buf = mm_buffer(p + first * stride, bytes - first * stride);
    asm volatile("" : "+v"(off));  // the loads' offsets are formed anew, not held all along
  }
  __device__ __forceinline__ void load(uint32_t at, int i) {
    mm_load16(buf, off + i * (STEP * stride), at + lds + i * (THREADS * 16));
  }
  __device__ __forceinline__ void mend(uint32_t at) {
    if (lost && threadIdx.x == 0)
      *(__attribute__((address_space(3))) uint16_t*)(lds_char*)(uintptr_t)(at + lost_at) =
          *reinterpret_cast<const uint16_t*>(lost - 2);
  }
  // Where this lane reads block `unit` of 16 columns, inner places 8 q + l / 4; block
  // unit + n, n below the power of two that divides `unit`, lies at the place xor 32 n.
  __device__ static __forceinline__ uint32_t read_at(int unit) {
    const int l = threadIdx.x % 16, q = threadIdx.x % WAVE / 16, r = 8 * q + l / 4;
    return (uint32_t)(r * ROW + (unit ^ swizzle(r)) * 32 + (l % 4) * 8);
  }
};

// ---------------------------------------------------------------- operands and products

// `more` is a constant: as a pointer's offset it goes into the instruction.
__device__ __forceinline__ mm_i32x4 mm_lds16(uint32_t at, int more) {
  return *(__attribute__((address_space(3))) mm_i32x4*)((lds_char*)(uintptr_t)at + more);
}
__device__ __forceinline__ float mm_lds4(uint32_t at, int more) {
  return *(__attribute__((address_space(3))) float*)((lds_char*)(uintptr_t)at + more);
}
// Eight inner places of this lane's column: two transposing loads, four rows apart.
__device__ __forceinline__ mm_i32x4 mm_lds_turned(uint32_t at, int more, int four_rows) {
  typedef __attribute__((address_space(3))) mm_i16x4 L;
  lds_char* p = (lds_char*)(uintptr_t)at + more;
  const mm_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)p);
  const mm_i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(p + four_rows));
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
// written from (row, n) on, rows below `end`, columns below N. Two blocks of columns
// exchange fours between neighbouring rows of 16 lanes, which leaves a lane with eight
// columns in a row.
template <int MI, int NJ, class O>
__device__ __forceinline__ void mm_write(const mm_f32x4 (&acc)[MI][NJ], O* out, int64_t row,
                                         int64_t end, int64_t n, int64_t N) {
  const int l = threadIdx.x % 16, q = threadIdx.x % WAVE / 16;
  const int64_t c = n + (q & 1) * 16 + (q >> 1) * 8;
  O* to = out + (row + l) * N + c;
  const int rows = (int)(end - row < MI * 16 ? end - row : MI * 16);
  const int cols = (int)(N - c < NJ * 16 ? N - c : NJ * 16);
#pragma unroll
  for (int i = 0; i < MI; ++i) {
#pragma unroll
    for (int j = 0; j < NJ; j += 2) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const auto both = __builtin_amdgcn_permlane16_swap(
            __float_as_uint(acc[i][j][k]), __float_as_uint(acc[i][j + 1][k]), false, false);
        v[k] = __uint_as_float(both[0]);
        v[k + 4] = __uint_as_float(both[1]);
      }
      if (l + i * 16 >= rows) continue;
      if (j * 16 + 8 <= cols) {
        store_acc<O, float, 8>(to + j * 16, v);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (j * 16 + k < cols) to[j * 16 + k] = (O)v[k];
      }
    }
    to += 16 * N;
    // one row block's values and addresses at a time: the registers are full
    __builtin_amdgcn_sched_barrier(0);
  }
}

template <int MI, int NJ>
__device__ __forceinline__ void mm_zero(mm_f32x4 (&acc)[MI][NJ]) {
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// What a wavefront multiplies of half a stage in 16 bits, and its products.
template <int MI, int NJ>
struct MmHalf {
  mm_i32x4 x[MI], y[NJ];
};
// Among them, in this order: read(0 .. MI + NJ - 1), the next half from LDS, over the first
// three quarters, and load(0 .. LOADS - 1), a stage from memory, over all. The memory
// pipeline takes a load to LDS every 16 cycles and LDS a read every 4, and a wavefront
// that issues its own one behind the other, as all do behind a barrier, multiplies nothing
// meanwhile; left to itself the compiler puts reads right in front of the wait for them.
template <class E, int LOADS, int MI, int NJ, class Read, class Load>
__device__ __forceinline__ void mm_half(const MmHalf<MI, NJ>& f, mm_f32x4 (&acc)[MI][NJ],
                                        Read read, Load load) {
  constexpr int N = MI * NJ, READS = MI + NJ;
#pragma unroll
  for (int m = 0; m < N; ++m) {
#pragma unroll
    for (int k = 0; k < READS; ++k)
      if (k * N * 3 / 4 / READS == m) read(k);
#pragma unroll
    for (int k = 0; k < LOADS; ++k)
      if (k * N / (LOADS ? LOADS : 1) == m) load(k);
    __builtin_amdgcn_sched_barrier(0);
    acc[m / NJ][m % NJ] = mm_mul(E{}, f.y[m % NJ], f.x[m / NJ], acc[m / NJ][m % NJ]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// What a wavefront has of a stage in 8 bits: values, the rows' scales and its columns'.
template <int MI, int NJ>
struct MmHalf8 {
  static constexpr int W = 4;  // row blocks
  mm_i32x8 x[W], y[NJ];
  float s[W], sb;
};

// The ring of stages in LDS. While one half of a stage is multiplied the next half is
// read from LDS: the second half of the stage, then the first of the next one. Between
// the two the wavefronts meet, once a stage: the next stage is there, and nobody reads
// the one whose second half all have in registers, so its place is filled again.
// Behind the last stage of the last tile it goes on with loads of nothing, so that as
// many are outstanding at every wait. `Loader`: begin(), load(place, i) for its LOADS loads,
// next() to the stage behind, mend(place) of the newest one when it is there.
template <int ST, int BYTES, class Loader>
struct MmRing {
  static_assert(Loader::WHOLE || ST == 2, "");  // what is read next is the newest
  Loader& loader;
  uint32_t base;
  uint32_t use = 0;     // the place of the stage
  bool stored = false;  // STORES stores are newer than all loads

  // All but the `N` newest loads are there, and all LDS reads; all wavefronts are here. The
  // stores of a tile's results need not have ended.
  template <int N, int STORES>
  __device__ __forceinline__ void wait() {
    if (stored) mm_wait<N + STORES>();
    else mm_wait<N>();
    stored = false;
  }
  template <class Read>
  __device__ __forceinline__ void start(Read first) {
#pragma unroll
    for (int i = 0; i < ST; ++i) {
      if (i) loader.next();
      loader.begin();
#pragma unroll
      for (int k = 0; k < Loader::LOADS; ++k) loader.load(base + i * BYTES, k);
      if (!Loader::WHOLE && i == 0) {
        mm_wait<0>();
        loader.mend(base);
      }
    }
    if (Loader::WHOLE) mm_wait<(ST - 1) * Loader::LOADS>();
    first(base);
  }
  // The stage at `place` is there for all, and the loads of the one behind the newest begin.
  template <int STORES>
  __device__ __forceinline__ void turn(uint32_t place) {
    if constexpr (Loader::WHOLE) {
      loader.next();
      loader.begin();
      wait<(ST - 2) * Loader::LOADS, STORES>();
    } else {
      wait<0, STORES>();
      loader.mend(place);
      loader.next();
      loader.begin();
    }
  }
  // A stage in 16 bits. read(half, place, h, k): part k of half h.
  template <class E, int MI, int NJ, class Read>
  __device__ __forceinline__ void step(E, MmHalf<MI, NJ>& f0, MmHalf<MI, NJ>& f1,
                                       mm_f32x4 (&acc)[MI][NJ], Read read) {
    const uint32_t at = base + use * BYTES;
    use = use + 1 == ST ? 0 : use + 1;
    const uint32_t next = base + use * BYTES;
    mm_half<E, 0>(f0, acc, [&](int k) { read(f1, at, 1, k); }, [](int) {});
    turn<MI * NJ / 2>(next);
    mm_half<E, Loader::LOADS>(f1, acc, [&](int k) { read(f0, next, 0, k); },
                              [&](int k) { loader.load(at, k); });
  }
  // A stage in 8 bits, row block by row block: at most four of them are in registers, and
  // a block's place takes the fourth behind it, of this stage or the next; y takes the
  // next stage's values behind its last use. The wavefronts meet behind block MEET, when
  // all of the stage is in registers. A product is scaled and added while the LAG behind it
  // are formed: with one, every second sum waited for its product (8,192 rows by 8,192 by
  // 8,192: 548 us, with two 528).
  template <int MI, int NJ, class ReadX, class ReadY>
  __device__ __forceinline__ void step8(MmHalf8<MI, NJ>& f, mm_f32x4 (&acc)[MI][NJ],
                                        ReadX read_x, ReadY read_y) {
    constexpr int W = MmHalf8<MI, NJ>::W, MEET = MI == 8 ? 4 : 1, N = (MI - 1 - MEET) * NJ;
    static_assert(MI == 8 || MI == 4, "");
    const uint32_t at = base + use * BYTES;
    use = use + 1 == ST ? 0 : use + 1;
    const uint32_t next = base + use * BYTES;
    constexpr int LAG = 2;
    mm_f32x4 before[LAG];
    float scale[LAG];
    auto add = [&](int m) {  // the stage's product m
      mm_f32x4& to = acc[m / NJ][m % NJ];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        to[k] = __builtin_fmaf(before[m % LAG][k], scale[m / NJ % LAG], to[k]);
      // here and not behind the stage, where the compiler would move all of them
      asm volatile("" : "+v"(to));
      __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      scale[i % LAG] = f.sb * f.s[i % W];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int m = (i - 1 - MEET) * NJ + j, n = i * NJ + j;
#pragma unroll
        for (int k = 0; k < Loader::LOADS; ++k)
          if (m >= 0 && k * N / Loader::LOADS == m) loader.load(at, k);
        __builtin_amdgcn_sched_barrier(0);
        const mm_f32x4 t = mm_mul8(f.y[j], f.x[i % W]);
        __builtin_amdgcn_sched_barrier(0);
        if (n >= LAG) add(n - LAG);
        before[n % LAG] = t;
        if (i == MI - 1) read_y(next, j);
      }
      if (i + W < MI) read_x(at, i + W);
      if (i == MEET) {
        turn<MI * NJ / 2>(next);
#pragma unroll
        for (int r = 0; r <= MEET; ++r)
          if (r + W >= MI) read_x(next, r + W - MI);
      } else if (i > MEET) {
        read_x(next, i + W - MI);
      }
    }
#pragma unroll
    for (int n = MI * NJ - LAG; n < MI * NJ; ++n) add(n);
  }
  // Where the stage that is multiplied next lies.
  __device__ __forceinline__ uint32_t place() const { return base + use * BYTES; }
  // Nothing is left on its way to LDS.
  __device__ __forceinline__ void finish() const { mm_wait<0>(); }
};

template <class E, int BM_, int BN_, int WM_, int WN_, int ST_, bool ALONG_, bool WHOLE_>
struct MmConf {
  using Elem = E;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr bool ALONG = ALONG_;    // b's inner axis is contiguous
  static constexpr bool WHOLE = WHOLE_;  // nothing is to be mended
  static constexpr int ST = ST_;
  static constexpr int THREADS = WM * WN * WAVE;
  static constexpr int MI = BM / WM / 16, NJ = BN / WN / 16;
  static constexpr bool EIGHT = sizeof(E) == 1;
  static constexpr int SIZE = (int)sizeof(E);
  static constexpr int INNER = MM_STAGE / SIZE;  // inner places a stage
  using A = MmAlong<BM, THREADS, SIZE, WHOLE>;
  using B =
      std::conditional_t<ALONG, MmAlong<BN, THREADS, SIZE, WHOLE>, MmAcross<BN, THREADS, WHOLE>>;
  // the rows' scales, then those of the tile's blocks of 128 columns
  static constexpr int SCALES = EIGHT ? BM * 4 : 0;
  static constexpr int STAGE_BYTES = A::BYTES + B::BYTES + SCALES + (EIGHT ? 256 : 0);
  static constexpr int LOADS = A::LOADS + B::LOADS + (EIGHT ? 1 : 0);
  // workgroups on a compute unit, two at most (their LDS: 160 KB)
  static constexpr int PER_CU = 2 * ST * STAGE_BYTES <= 163840 ? 2 : 1;
  static constexpr int WAVES = PER_CU * THREADS / 256 > 0 ? PER_CU * THREADS / 256 : 1;
  static_assert(NJ % 2 == 0 && (ST - 2) * LOADS + MI * NJ / 2 < 64, "");
  static_assert(!EIGHT || (ALONG && BM / WAVE < WM * WN && 128 % (BN / WN) == 0 && BN % 128 == 0),
                "");
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

// A tile of results: rows [row, end) of its group (BM at most), columns from `col` on,
// stages [stage0, stage1) of the inner axis.
template <class C>
struct MmTile {
  MmWalk<true> walk;
  MmOrder order;
  int group, part, stage0, stage1;
  uint32_t row, end, col;
  bool any;

  __device__ __forceinline__ void init(const MmArgs& p) {
    group = part = stage0 = stage1 = 0;
    row = end = col = 0;
    any = false;
    walk.init(p.seglen, p.groups, p.rows, C::BM);
    order.init(walk.total() * across(p) * p.splits);
  }
  __device__ static __forceinline__ uint32_t across(const MmArgs& p) {
    return (uint32_t)((p.N + C::BN - 1) / C::BN);
  }
  __device__ __forceinline__ void seek(const MmArgs& p) {
    any = false;
    if (order.at >= order.end) return;
    uint32_t s = 0, p0 = 0, p1 = 0, i, j;
    const uint32_t at = order.at / p.splits, wide = across(p);
    part = (int)(order.at - at * p.splits);
    order.at += order.step;
    if (!walk.find(at / wide, &group, &s, &end, &p0, &p1)) return;
    mm_band(at - p0 * wide, p1 - p0, wide, &i, &j);
    const int stages = (p.K + C::INNER - 1) / C::INNER;
    stage0 = (int)((int64_t)stages * part / p.splits);
    // the rest has no inner axis
    stage1 = group < p.groups ? (int)((int64_t)stages * (part + 1) / p.splits) : stage0;
    row = s + i * C::BM;
    col = j * C::BN;
    any = true;
  }
};

// The stages of a workgroup's tiles, one after the other, on their way to LDS.
template <class C>
struct MmSource {
  static constexpr int LOADS = C::LOADS;
  static constexpr bool WHOLE = C::WHOLE;
  const MmArgs& p;
  MmTile<C> tile;
  typename C::A A;
  typename C::B B;
  int stage;
  int64_t row_bytes;
  // 8 bits: the first wavefronts load the rows' scales, one a lane, the others the columns'
  mm_i32x4 scales;
  uint32_t scale_off, scale_step, scale_lds;
  int kb, nb;  // blocks of K and N
  bool of_rows;

  __device__ __forceinline__ void init(const MmTile<C>& first) {
    tile = first;
    row_bytes = (int64_t)p.K * C::SIZE;
    A.init((uint32_t)row_bytes);
    B.init(C::ALONG ? (uint32_t)row_bytes : (uint32_t)p.N * 2);
    if constexpr (C::EIGHT) {
      const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
      const int lane = (int)(threadIdx.x % WAVE);
      of_rows = wave < C::BM / WAVE;
      kb = (p.K + 127) / 128;
      nb = (p.N + 127) / 128;
      scale_off = of_rows ? (uint32_t)(threadIdx.x * kb * 4)
                          : lane < C::BN / 128 ? (uint32_t)lane * 4 : MM_PAST;
      scale_step = of_rows ? 4 : nb * 4;
      scale_lds = C::A::BYTES + C::B::BYTES + (of_rows ? wave * 256 : C::SCALES);
    }
    open();
  }
  __device__ __forceinline__ void open() {
    do tile.seek(p);
    while (tile.any && tile.stage0 == tile.stage1);
    stage = 0;
    if (!tile.any) {
      A.none();
      B.none();
      if constexpr (C::EIGHT) scales = mm_buffer(nullptr, 0);
      return;
    }
    stage = tile.stage0;
    const int rows = (int)(tile.end - tile.row);
    A.tile(p.a + tile.row * row_bytes, rows, (p.rows - tile.row) * row_bytes);
    const char* block = p.b + tile.group * (row_bytes * p.N);
    const int64_t left = (p.groups - tile.group) * (row_bytes * p.N);
    const int64_t col = tile.col;
    if constexpr (C::ALONG)
      B.tile(block + col * row_bytes, p.N - (int)col, left - col * row_bytes);
    else
      B.tile(block + col * 2, p.K, (p.N - (int)col) * (int64_t)2, left - col * 2);
    if constexpr (C::EIGHT) {
      const int64_t c = tile.col / 128, block = (int64_t)kb * nb;
      const float* from = of_rows ? p.sa + (int64_t)tile.row * kb : p.sb + tile.group * block + c;
      scales = mm_buffer((const char*)from,
                         (of_rows ? (int64_t)(rows < C::BM ? rows : C::BM) * kb : block - c) * 4);
    }
  }
  __device__ __forceinline__ void begin() {
    A.begin(stage);
    B.begin(stage);
  }
  __device__ __forceinline__ void load(uint32_t at, int i) {
    if (i < C::A::LOADS) {
      A.load(at, i);
    } else if (i < C::A::LOADS + C::B::LOADS) {
      B.load(at + C::A::BYTES, i - C::A::LOADS);
    } else if constexpr (C::EIGHT) {
      mm_load4(scales, scale_off + stage * scale_step, at + scale_lds);
    }
  }
  __device__ __forceinline__ void next() {
    if (tile.any && ++stage == tile.stage1) open();
  }
  __device__ __forceinline__ void mend(uint32_t at) {
    if (!tile.any || (stage + 1) * C::INNER < p.K) return;
    A.mend(at);
    B.mend(at + C::A::BYTES);
    mm_wait<63>();
  }
};

// 32 bytes of row `i` of `rows` from place k on, zeros past the end of it or of the rows.
__device__ __forceinline__ mm_i32x8 mm_bytes(const char* p, int64_t i, int64_t rows, int K, int k) {
  mm_i32x8 v;
#pragma unroll
  for (int w = 0; w < 8; ++w, k += 4) {
    uint32_t word = 0;
    if (i < rows) {
      const char* at = p + i * K + k;
      if (k + 4 <= K) {
        __builtin_memcpy(&word, at, 4);
      } else {
        for (int b = 0; b < K - k; ++b) word |= (uint32_t)(uint8_t)at[b] << 8 * b;
      }
    }
    v[w] = (int)word;
  }
  return v;
}

// Two finite scales whose product is not: both are above 1, and one is 2^64 at least.
__device__ __forceinline__ bool mm_apart(float a, float b) {
  return __builtin_isinf(a * b) && !__builtin_isinf(a) && !__builtin_isinf(b);
}
// A wavefront's part of a tile that has such, block of 16 by 16 after block, straight from
// memory: there a block's sum takes one scale after the other, so that 0 stays 0 and what is
// in float's range stays. No path for speed: 10,001 rows by 4,096 by 8,192, all of them such,
// take 20 ms (weights' scales above 1 without such products 373 us, others 318).
template <class C>
__device__ __forceinline__ void mm_write_apart(const MmArgs& p, const MmTile<C>& t, int64_t row0,
                                               int64_t n0) {
  int lane = threadIdx.x % WAVE;
  asm volatile("" : "+v"(lane));  // nothing of this is formed in front of the tiles
  const int l = lane % 16, q = lane / 16;
  const int kb = (p.K + 127) / 128, nb = (p.N + 127) / 128;
  const char* b = p.b + t.group * ((int64_t)p.K * p.N);
  const float* sb = p.sb + t.group * ((int64_t)kb * nb) + n0 / 128;
  if (n0 >= p.N) return;  // none of the wavefront's columns are there
#pragma unroll 1
  for (int block = 0; block < C::MI * C::NJ; ++block) {
    const int64_t r = row0 + block / C::NJ * 16 + l, n = n0 + block % C::NJ * 16;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    for (int s = t.stage0; s < t.stage1; ++s) {
      const mm_i32x8 x = mm_bytes(p.a, r, t.end, p.K, s * 128 + q * 32);
      const mm_i32x8 y = mm_bytes(b, n + l, p.N, p.K, s * 128 + q * 32);
      const mm_f32x4 sum = mm_mul8(y, x);
      const float sr = r < t.end ? p.sa[r * kb + s] : 0.0f, sc = sb[s * nb];
      const bool apart = mm_apart(sr, sc);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = __builtin_fmaf(apart ? sum[k] * sr : sum[k], apart ? sc : sr * sc, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t c = n + 4 * q + k, at = r * p.N + c;
      if (r >= t.end || c >= p.N) continue;
      if (p.splits > 1) p.part[t.part * (p.rows * p.N) + at] = v[k];
      else if (p.out_dtype == DT_F32) ((float*)p.out)[at] = v[k];
      else if (p.out_dtype == DT_BF16) ((bf16_t*)p.out)[at] = (bf16_t)v[k];
      else ((f16_t*)p.out)[at] = (f16_t)v[k];
    }
  }
}

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::WAVES) expert_mm_kernel(MmArgs p) {
  using E = typename C::Elem;
  __shared__ __align__(256) char lds[C::ST * C::STAGE_BYTES];
  const uint32_t lds0 =
      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_char*)lds);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int q = threadIdx.x % WAVE / 16;

  // what this lane reads, from a stage's start on
  const uint32_t a_at = (uint32_t)(wm * (C::BM / C::WM) * MM_STAGE) +
                        C::A::read_at(C::EIGHT ? 2 * q : q);
  uint32_t b_at = C::A::BYTES;
  if constexpr (C::ALONG)
    b_at += wn * (C::BN / C::WN) * MM_STAGE + C::B::read_at(C::EIGHT ? 2 * q : q);
  else
    b_at += C::B::read_at(wn * C::NJ);

  MmTile<C> mine;  // what is multiplied
  mine.init(p);
  MmSource<C> source{p};  // what is loaded
  source.init(mine);
  MmRing<C::ST, C::STAGE_BYTES, MmSource<C>> ring{source, lds0};
  mm_f32x4 acc[C::MI][C::NJ];
  auto write = [&]() {
    const int64_t row = (int64_t)mine.row + wm * (C::BM / C::WM);
    const int64_t n = (int64_t)mine.col + wn * (C::BN / C::WN);
    // a whole tile of 16 bits is one store for every two blocks
    ring.stored = p.splits == 1 && (!C::EIGHT || p.out_dtype != DT_F32) &&
                  row + C::MI * 16 <= mine.end && n + C::NJ * 16 <= p.N;
    if (p.splits > 1) {
      mm_write(acc, p.part + mine.part * (p.rows * p.N), row, mine.end, n, p.N);
    } else if constexpr (C::EIGHT) {
      if (p.out_dtype == DT_F32) mm_write(acc, (float*)p.out, row, mine.end, n, p.N);
      else if (p.out_dtype == DT_BF16) mm_write(acc, (bf16_t*)p.out, row, mine.end, n, p.N);
      else mm_write(acc, (f16_t*)p.out, row, mine.end, n, p.N);
    } else {
      mm_write(acc, (E*)p.out, row, mine.end, n, p.N);
    }
  };
  if constexpr (C::EIGHT) {
    MmHalf8<C::MI, C::NJ> f;
    const uint32_t s_at = (uint32_t)C::A::BYTES + C::B::BYTES +
                          (wm * (C::BM / C::WM) + threadIdx.x % 16) * 4;
    const uint32_t sb_at = (uint32_t)C::A::BYTES + C::B::BYTES + C::SCALES +
                           wn * (C::BN / C::WN) / 128 * 4;
    auto read_x = [&](uint32_t at, int i) {
      const mm_i32x4 lo = mm_lds16(at + a_at, i * 16 * MM_STAGE);
      const mm_i32x4 hi = mm_lds16((at + a_at) ^ 16, i * 16 * MM_STAGE);
      f.x[i % f.W] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      f.s[i % f.W] = mm_lds4(at + s_at, i * 16 * 4);
    };
    auto read_y = [&](uint32_t at, int j) {
      const mm_i32x4 lo = mm_lds16(at + b_at, j * 16 * MM_STAGE);
      const mm_i32x4 hi = mm_lds16((at + b_at) ^ 16, j * 16 * MM_STAGE);
      f.y[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      if (j == 0) f.sb = mm_lds4(at + sb_at, 0);
    };
    ring.start([&](uint32_t at) {
#pragma unroll
      for (int i = 0; i < f.W; ++i) read_x(at, i);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) read_y(at, j);
    });
    for (mine.seek(p); mine.any; mine.seek(p)) {
      mm_zero(acc);
      bool apart = false;
      for (int k = mine.stage0; k < mine.stage1; ++k) {
        // one scale for the wavefront's columns; only one above 1 (of weights above 448) can
        // have an infinite product, and others cost this comparison (10,001 rows by 4,096
        // by 8,192: 335 us without it, 338 with it; 348 with the scales' powers of two in
        // the matrix instruction)
        const float sb = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(f.sb)));
        if (__builtin_expect(__builtin_fabsf(sb) > 1.0f, 0)) {
          const uint32_t rows = ring.place() + C::A::BYTES + C::B::BYTES +
                                (wm * (C::BM / C::WM) + threadIdx.x % WAVE) * 4;
          bool any = false;
#pragma unroll
          for (int i = 0; i < C::MI * 16 / WAVE; ++i) any |= mm_apart(mm_lds4(rows, i * 256), sb);
          apart |= __builtin_amdgcn_readfirstlane(__any(any)) != 0;
        }
        ring.step8(f, acc, read_x, read_y);
      }
      if (__builtin_expect(apart, 0)) {
        mm_write_apart(p, mine, (int64_t)mine.row + wm * (C::BM / C::WM),
                       (int64_t)mine.col + wn * (C::BN / C::WN));
        ring.stored = false;
        continue;
      }
      write();
    }
  } else {
    // half a stage: 32 inner places
    using Half = MmHalf<C::MI, C::NJ>;
    Half f0, f1;
    auto read = [&](Half& f, uint32_t at, int h, int k) {
      const int j = k - C::MI;
      if (j < 0)
        f.x[k] = mm_lds16((at + a_at) ^ h * 64, k * 16 * MM_STAGE);
      else if constexpr (C::ALONG)
        f.y[j] = mm_lds16((at + b_at) ^ h * 64, j * 16 * MM_STAGE);
      else
        f.y[j] = mm_lds_turned((at + b_at) ^ j * 32, h * 32 * C::B::ROW, 4 * C::B::ROW);
    };
    ring.start([&](uint32_t at) {
#pragma unroll
      for (int k = 0; k < C::MI + C::NJ; ++k) read(f0, at, 0, k);
    });
    for (mine.seek(p); mine.any; mine.seek(p)) {
      mm_zero(acc);
      for (int s = mine.stage0; s < mine.stage1; ++s)
        ring.step(E{}, f0, f1, acc, read);
      write();
    }
  }
  ring.finish();
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
struct MmGradTile {
  MmWalk<false> walk;
  MmOrder order;
  int group, stages, rows;
  uint32_t start, row, col, piece;  // first row of the piece; the tile's place
  bool any, alone;

  __device__ static __forceinline__ uint32_t down(const MmGradArgs& p) {
    return (uint32_t)((p.D1 + C::BM - 1) / C::BM);
  }
  __device__ static __forceinline__ uint32_t across(const MmGradArgs& p) {
    return (uint32_t)((p.D2 + C::BN - 1) / C::BN);
  }
  __device__ __forceinline__ void init(const MmGradArgs& p) {
    group = stages = rows = 0;
    start = row = col = piece = 0;
    any = alone = false;
    walk.init(p.seglen, p.groups, p.rows, p.piece);
    order.init(walk.total() * (down(p) * across(p)));
  }
  __device__ __forceinline__ void seek(const MmGradArgs& p) {
    any = false;
    if (order.at >= order.end) return;
    uint32_t s = 0, e = 0, p0 = 0, p1 = 0, i, j;
    const uint32_t at = order.at, tiles = down(p) * across(p);
    order.at += order.step;
    piece = at / tiles;
    if (!walk.find(piece, &group, &s, &e, &p0, &p1)) return;
    mm_band(at - piece * tiles, down(p), across(p), &i, &j);
    start = s + (piece - p0) * p.piece;
    rows = (int)(e - start < p.piece ? e - start : p.piece);
    stages = (rows + 63) / 64;
    row = i * C::BM;
    col = j * C::BN;
    alone = p1 - p0 == 1;
    any = true;
  }
};

template <class C>
struct MmGradSource {
  using A = MmAcross<C::BM, C::THREADS, C::WHOLE>;
  using B = MmAcross<C::BN, C::THREADS, C::WHOLE>;
  static constexpr bool WHOLE = C::WHOLE;
  static constexpr int LOADS = A::LOADS + B::LOADS, BYTES = A::BYTES + B::BYTES;
  const MmGradArgs& p;
  MmGradTile<C> tile;
  A a;
  B b;
  int stage;

  __device__ __forceinline__ void init(const MmGradTile<C>& first) {
    tile = first;
    a.init((uint32_t)p.D1 * 2);
    b.init((uint32_t)p.D2 * 2);
    open();
  }
  __device__ __forceinline__ void open() {  // pieces without rows have nothing to load
    do tile.seek(p);
    while (tile.any && tile.stages == 0);
    stage = 0;
    if (!tile.any) {
      a.none();
      b.none();
      return;
    }
    const int64_t rows = p.rows - tile.start;
    a.tile(p.a + ((int64_t)tile.start * p.D1 + tile.row) * 2, tile.rows,
           (int64_t)(p.D1 - (int)tile.row) * 2, (rows * p.D1 - tile.row) * 2);
    b.tile(p.grad + ((int64_t)tile.start * p.D2 + tile.col) * 2, tile.rows,
           (int64_t)(p.D2 - (int)tile.col) * 2, (rows * p.D2 - tile.col) * 2);
  }
  __device__ __forceinline__ void begin() {
    a.begin(stage);
    b.begin(stage);
  }
  __device__ __forceinline__ void load(uint32_t at, int i) {
    if (i < A::LOADS) a.load(at, i);
    else b.load(at + A::BYTES, i - A::LOADS);
  }
  __device__ __forceinline__ void next() {
    if (tile.any && ++stage == tile.stages) open();
  }
  __device__ __forceinline__ void mend(uint32_t at) {
    if (!tile.any || stage + 1 < tile.stages) return;
    a.mend(at);
    b.mend(at + A::BYTES);
    mm_wait<63>();
  }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::WAVES) expert_mm_grad_kernel(MmGradArgs p) {
  using E = typename C::Elem;
  using S = MmGradSource<C>;
  __shared__ __align__(256) char lds[C::ST * S::BYTES];
  const uint32_t lds0 =
      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_char*)lds);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const uint32_t a_at = S::A::read_at(wm * C::MI);
  const uint32_t b_at = (uint32_t)S::A::BYTES + S::B::read_at(wn * C::NJ);
  using Half = MmHalf<C::MI, C::NJ>;
  Half f0, f1;
  auto read = [&](Half& f, uint32_t at, int h, int k) {
    const int j = k - C::MI;
    if (j < 0)
      f.x[k] = mm_lds_turned((at + a_at) ^ k * 32, h * 32 * S::A::ROW, 4 * S::A::ROW);
    else
      f.y[j] = mm_lds_turned((at + b_at) ^ j * 32, h * 32 * S::B::ROW, 4 * S::B::ROW);
  };

  MmGradTile<C> mine;
  mine.init(p);
  S source{p};
  source.init(mine);
  MmRing<C::ST, S::BYTES, S> ring{source, lds0};
  mm_f32x4 acc[C::MI][C::NJ];
  ring.start([&](uint32_t at) {
#pragma unroll
    for (int k = 0; k < C::MI + C::NJ; ++k) read(f0, at, 0, k);
  });
  for (mine.seek(p); mine.any; mine.seek(p)) {
    mm_zero(acc);
    for (int s = 0; s < mine.stages; ++s) ring.step(E{}, f0, f1, acc, read);
    const int64_t row = (int64_t)mine.row + wm * (C::BM / C::WM);
    const int64_t n = (int64_t)mine.col + wn * (C::BN / C::WN);
    const int64_t size = (int64_t)p.D1 * p.D2;
    if (mine.alone)
      mm_write(acc, (E*)p.out + mine.group * size, row, p.D1, n, p.D2);
    else
      mm_write(acc, p.part + mine.piece * size, row, p.D1, n, p.D2);
  }
  ring.finish();
}

// Results of groups of several pieces: blockIdx.y a group, four values a thread.
template <class E>
__global__ void __launch_bounds__(BLOCK) expert_mm_sum_kernel(MmGradArgs p) {
  MmWalk<false> walk;
  walk.init(p.seglen, p.groups, p.rows, p.piece);
  const int g = blockIdx.y;
  while (g >= walk.base + WAVE) walk.next();
  uint32_t s, e, p0, p1;
  walk.bounds(g - walk.base, &s, &e, &p0, &p1);
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

// The shapes as expert_mm_plan.hip lists them.
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
    case 4: return run_expert_mm<MmConf<E, 128, 128, 2, 2, 2, ALONG, false>>(p, tiles, s);
    default: return run_expert_mm<MmConf<E, 256, 256, 2, 4, 2, ALONG, false>>(p, tiles, s);
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
    case 4: return run_expert_mm_grad<MmConf<E, 128, 128, 2, 2, 2, false, false>>(p, tiles, s);
    default: return run_expert_mm_grad<MmConf<E, 256, 256, 2, 4, 2, false, false>>(p, tiles, s);
  }
}

}  // namespace mdgl
