// The shape of a product's tiles.
#include "mdgl_kernels.h"

namespace mdgl {

namespace {

struct Shape {
  int bm, bn;
  bool whole;
  int slots;       // tiles at a time on the card
  float stage[2];  // us a stage of a tile with all slots taken: 16 bits, 8 bits
};

// us a stage from products of 8,192 rows by 8,192 by 8,192: 842, 1,120 and 1,290 TFLOP/s in
// 16 bits and 1,250, 1,760 and 2,000 in 8; of 8,191 by 8,191: 498, 680 and 980, and 824,
// 1,038 and 1,530. At 8 to 1,024 rows of 2,048 to 1,536 for each of 64 experts the choice is
// the fastest of the three or within 11 % of it (16 bits, 192 rows: 151 and 136 us).
constexpr Shape shapes[] = {{64, 128, true, 512, {0.64f, 0.86f}},
                            {128, 128, true, 512, {0.96f, 1.22f}},
                            {256, 256, true, 256, {1.67f, 2.15f}},
                            {64, 128, false, 512, {1.08f, 1.30f}},
                            {128, 128, false, 512, {1.58f, 2.07f}},
                            {256, 256, false, 256, {2.19f, 2.81f}}};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

// A tile that has the card to itself takes about half the time of one of a full card, hence
// the 0.5. The inner axis goes in parts where the tiles leave compute units without work: a
// part's sums in float are written and read again (0.75 us a MB) by another launch (2.5 us).
// 64 rows of 4,096 to 4,096 in bfloat16: 24.9 us whole, 17.9, 14.1 and 15.1 in 2, 4 and 8
// parts (by the formula 23.8, 17.7, 14.3 and 15.2). 32 rows through 16 experts of 2,048
// to 2,048, which is bound by reading the experts: 21.2 us whole, 23.3 in 2 parts.
ExpertMmPlan expert_mm_plan(int64_t rows, int64_t groups, int64_t inner, int64_t cols, int size,
                            bool whole) {
  ExpertMmPlan best{-1, 1, 0, 0, 0};
  const int64_t stages = up(inner * size, 128);
  const int64_t called = groups < rows ? groups : rows;
  const double read = (double)called * (double)inner * (double)cols * size / 5e6;  // us
  double least = 0;
  for (int i = 0; i < 6; ++i) {
    const Shape& s = shapes[i];
    if (s.whole != whole) continue;
    const int64_t across = up(cols, s.bn);
    // half a tile of each expert's rows is empty on average
    const double want = (double)rows / s.bm + 0.5 * (double)called;
    const double tiles = (want > (double)called ? want : (double)called) * (double)across;
    for (int parts = 1; parts == 1 || (parts <= 8 && stages >= 8 * parts); parts *= 2) {
      const double most = ((double)rows / s.bm + (double)groups + 2) * (double)across * parts;
      if (most >= 0x1p31) break;
      const int64_t bytes = parts > 1 ? parts * rows * cols * 4 : 0;
      double us = (tiles * parts / s.slots + 0.5) * ((double)stages / parts + 2) *
                  s.stage[size == 1];
      if (us < read) us = read;
      if (parts > 1) us += 2.5 + (double)bytes * 0.75e-6;
      if (best.shape >= 0 && us >= least) continue;
      least = us;
      best = {i, parts, 0, (int64_t)most, bytes};
    }
  }
  return best;
}

ExpertMmPlan expert_mm_grad_plan(int64_t rows, int64_t groups, int64_t d1, int64_t d2,
                                 bool whole) {
  const auto tiles_of = [&](int b) { return up(d1, b) * up(d2, b); };
  // tiles of 256 run at 1.27 times the rate of those of 128 (8,192 rows of 8,192 and 8,192:
  // 1,275 and 1,005 TFLOP/s; of 8,191 1,038 and 754), and leave more of them empty
  const bool big = tiles_of(256) * groups >= 256 &&
                   (double)tiles_of(256) * 4 < 1.27 * (double)tiles_of(128);
  const int64_t tiles = tiles_of(big ? 256 : 128), slots = big ? 256 : 512;
  // without rows, too, a piece has a size: the groups' pieces are counted by it
  ExpertMmPlan p{(big ? 2 : 1) + (whole ? 0 : 3), 1, rows > 0 ? rows : 1, 0, 0};
  int64_t pieces = groups;
  if (tiles * groups < slots) {
    // few tiles: long groups in pieces that fill the card once, of 512 rows at least; half a
    // piece of each group is its rest. (24 groups of 1,125 rows on average, 602 by 301: pieces
    // of 1,408 rows 35 us with their sums, of 896, which leave the card half empty the second
    // time, 46, whole groups 44.)
    const double count = (double)slots / (double)tiles - 0.5 * (double)groups;
    int64_t piece = up((int64_t)((double)rows / count) + 1, 64) * 64;
    if (piece < 512) piece = 512;
    if (piece < rows) {
      p.piece = piece;
      pieces = rows / piece + groups;
      p.bytes = pieces * d1 * d2 * 4;
    }
  }
  const double most = (double)pieces * (double)tiles;
  p.tiles = (int64_t)most;
  if (most >= 0x1p31) p.shape = -1;
  return p;
}

}  // namespace mdgl
