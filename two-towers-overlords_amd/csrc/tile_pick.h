// Host rules of the matrix-product tiles (mfma_tile.h): which tile shape a product takes, and which parts of a row its waves
// leave.  Plain C++.  Internal to the library.
#pragma once
#include "../../include/tt_hotpath.h"

namespace ttm {

// Edge of the output tile, 64, 128 or 256, for a product of M x N outputs in `splits` parts: the least estimated time, in units
// of a compute unit's work (`cost`).  A round of tiles takes as long as the tiles that share a compute unit; `rate` is what a tile
// shape reaches of the best one's on full rounds: bf16 8192 cubed 460 / 998 / 1120 TFLOP/s, float 16384 x 4096 x 1024 120 / 131;
// float has no registers for the largest.  A tile alone on a compute unit takes (1 + kAlone / 2) / 2 of two (float 2048 x 2048 x
// 384, 256 tiles of 128 against 1024 of 64: both passes of the loss 171 -> 161 us; 0.4 to 1 choose alike).
// `three`: 192 stands for 256 x 192 (dx and dw of 8192 x 30522 logits, 384 wide, bf16: 352 + 278 -> 201 + 207 us).
constexpr double kAlone = 0.68;
inline int pick_tile(long long M, long long N, long long splits, int dtype, bool three = false, double* cost = nullptr) {
  static const struct { int edge, m, n, share; float rate16, rate32; } kinds[] = {
      {64, 64, 64, 4, 0.42f, 0.92f}, {128, 128, 128, 2, 0.9f, 1.f}, {192, 256, 192, 1, 0.95f, 0.f}, {256, 256, 256, 1, 1.f, 0.f}};
  int best = 64;
  double least = 1e300;
  for (const auto& k : kinds) {
    if ((dtype == TT_F32 && k.rate32 == 0.f) || (k.edge == 192 && !three)) continue;
    const long long tiles = ((M + k.m - 1) / k.m) * ((N + k.n - 1) / k.n) * splits;
    const double rounds = (double)((tiles + 256 * k.share - 1) / (256 * k.share));
    // the last round's compute units share their tiles only as far as there are any; fewer workgroups hide less of their waits
    const long long last = tiles - (long long)(rounds - 1) * 256 * k.share;
    const double n = (double)((last + 255) / 256), share = rounds - 1 + (n + kAlone * (1. - n / k.share)) / k.share;
    const double t = share * k.share * k.m * k.n / (dtype == TT_F32 ? k.rate32 : k.rate16);
    if (t < least) {
      least = t;
      best = k.edge;
    }
  }
  if (cost) *cost = least;
  return best;
}

// Parts of a row that the waves of a product with tiles of `edge` leave where each owns edge / 2 columns (WN = 2) and only those
// that start before `columns`, a multiple of 128, write theirs: the last tile may reach further than the columns, its second
// wave then writes nothing.
inline int row_parts(int edge, int gn, long long columns) {
  const long long inside = columns / (edge / 2), all = 2LL * gn;
  return (int)(inside < all ? inside : all);
}

}  // namespace ttm
