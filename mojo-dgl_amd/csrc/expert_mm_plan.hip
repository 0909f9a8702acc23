// The shape of a product's tiles.
#include "mdgl_kernels.h"

namespace mdgl {

namespace {

struct Shape {
  int bm, bn;
  bool direct;
  int slots[2];    // tiles at a time on the card: 16 bits, 8 bits
  float stage[2];  // us a stage of a tile with all slots taken
};

// us a stage from products of 8,192 rows by 8,192 by 8,192: 810, 1,090 and 1,330 TFLOP/s in
// 16 bits, 1,000, 1,650 and 1,900 in 8 bits; through registers 450 and 580.
constexpr Shape shapes[] = {{64, 128, true, {512, 512}, {0.66f, 1.07f}},
                            {128, 128, true, {512, 512}, {0.98f, 1.30f}},
                            {256, 256, true, {256, 256}, {1.61f, 2.26f}},
                            {64, 128, false, {512, 512}, {1.2f, 1.4f}},
                            {128, 128, false, {512, 256}, {1.85f, 1.0f}}};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

ExpertMmPlan expert_mm_plan(int64_t rows, int64_t groups, int64_t inner, int64_t cols, int size,
                            bool direct) {
  ExpertMmPlan best{-1, 1, 0, 0, 0};
  const int64_t stages = up(inner * size, 128);
  const int64_t called = groups < rows ? groups : rows;
  double least = 0;
  for (int i = 0; i < 5; ++i) {
    const Shape& s = shapes[i];
    if (s.direct != direct) continue;
    const int64_t across = up(cols, s.bn);
    const double most = ((double)rows / s.bm + (double)groups + 2) * (double)across;
    if (most >= 0x1p31) continue;
    // half a tile of each expert's rows is empty on average
    const double want = (double)rows / s.bm + 0.5 * (double)called;
    const double tiles = (want > (double)called ? want : (double)called) * (double)across;
    const double us = (tiles / s.slots[size == 1] + 0.5) * (double)(stages + 2) * s.stage[size == 1];
    if (best.shape >= 0 && us >= least) continue;
    least = us;
    best = {i, 1, 0, (int64_t)most, 0};
  }
  return best;
}

ExpertMmPlan expert_mm_grad_plan(int64_t rows, int64_t groups, int64_t d1, int64_t d2,
                                 bool direct) {
  const auto tiles_of = [&](int b) { return up(d1, b) * up(d2, b); };
  // tiles of 256 run at 1.15 times the rate of those of 128, and leave more of them empty
  const bool big = direct && tiles_of(256) * groups >= 256 &&
                   (double)tiles_of(256) * 4 < 1.15 * (double)tiles_of(128);
  const int64_t tiles = tiles_of(big ? 256 : 128), slots = big ? 256 : 512;
  // without rows, too, a piece has a size: the groups' pieces are counted by it
  ExpertMmPlan p{big ? 2 : direct ? 1 : 4, 1, rows > 0 ? rows : 1, 0, 0};
  int64_t pieces = groups;
  if (tiles * groups < slots) {
    // few tiles: long groups in pieces that fill the card, of 512 rows at least
    const int64_t want = up(slots, tiles);
    int64_t piece = up(up(rows, want), 64) * 64;
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
