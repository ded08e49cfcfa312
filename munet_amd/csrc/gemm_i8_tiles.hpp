// Which kernel and block tile a product of 8-bit integers takes, by its sizes.
// Host arithmetic only (tests/cxx/gemm_i8_tiles_check.cpp).
#pragma once

#include <algorithm>
#include <cstdint>

namespace mh {

// Codes: 1 to 9 rows in whole 16-byte blocks, 0 and 10 rows from anywhere
// (gemm_i8.hip), 100 and 101 few rows from anywhere (gemm_i8_few.hip).
//
// A tile's time over n = its tiles in the product: launch + the longer of
// rounds(n) (first + k K / 1024) us and the bytes: operands and results (16 bits) at
// `hbm` TB/s, what the workgroups read at `near` TB/s.  A round is per_cu workgroups
// on each of 256 CUs; a last partial one takes `half` of that up to one workgroup
// per CU, and from there that and `over` of the rest, to 1 (per_cu 1: `half` to 1).
// Fitted to products of M 1 to 8192 by 18 and 8 N x K (of 768 x 768 to 32000 x 768 and
// 12800 x 4096; bf16 results, weights not in L2), those near the fastest weighing
// most: 3 to 7% rms per tile (few unaligned rows 11%); the tile of least predicted
// time takes 1.7% longer than the fastest on average, 33% at worst (unaligned 0.6
// and 11%).
struct I8Tile {
  int code, bm, bn, per_cu;
  double half, over, first, k, launch, hbm, near;
};
constexpr I8Tile kI8Tiles[] = {
    {1, 256, 256, 1, 0.74, 0.00, 8.90, 12.00, 1.48, 4.20, 11.7},
    {2, 256, 128, 1, 0.63, 0.00, 5.35, 6.63, 2.58, 3.01, 29.9},
    {3, 128, 128, 1, 0.75, 0.00, 4.17, 4.10, 1.51, 3.97, 22.3},
    {4, 128, 64, 1, 0.77, 0.00, 2.98, 2.62, 1.65, 4.36, 25.9},
    {5, 64, 64, 2, 0.60, 1.00, 2.88, 2.73, 1.88, 5.11, 25.8},
    {6, 64, 64, 3, 0.59, 0.47, 3.51, 3.47, 1.23, 4.37, 23.9},
    {7, 64, 32, 2, 0.58, 1.00, 2.04, 2.33, 1.91, 6.25, 24.7},
    {8, 32, 32, 2, 0.61, 1.00, 2.13, 1.75, 1.61, 5.78, 31.9},
    {9, 64, 128, 2, 0.68, 1.00, 4.22, 4.11, 0.73, 4.14, 21.1},
    {100, 16, 16, 5, 0.22, 0.19, 0.68, 3.52, 2.30, 7.95, 12.3},
    {101, 16, 32, 2, 0.50, 0.77, 0.80, 2.65, 2.04, 8.37, 11.4},
};
constexpr I8Tile kI8AnyTiles[] = {
    {0, 64, 64, 5, 0.40, 0.00, 5.71, 12.58, 2.80, 3.03, 14.0},
    {10, 128, 128, 2, 0.70, 0.87, 12.63, 11.09, 0.63, 7.47, 14.9},
    {100, 16, 16, 5, 0.22, 0.17, 0.00, 4.51, 2.58, 8.20, 11.3},
    {101, 16, 32, 2, 0.65, 1.00, 2.48, 2.43, 1.08, 7.04, 7.8},
};
// Rows that the kernels of few rows take at most.
constexpr int kI8FewRows = 256;

// Workgroups of a launch; a product's 64 x 64 tiles are no more.
constexpr int64_t kI8MaxTiles = 1 << 22;

inline double i8_tile_time(const I8Tile &t, int64_t M, int64_t N, int64_t K) {
  const int64_t tm = (M + t.bm - 1) / t.bm, tn = (N + t.bn - 1) / t.bn, n = tm * tn, round = 256 * t.per_cu, rem = n % round;
  double rounds = double(n / round);
  if (rem && t.per_cu == 1) rounds += t.half + (1 - t.half) * double(rem) / 256;
  else if (rem <= 256) rounds += rem ? t.half : 0;
  else rounds += t.half + (1 - t.half) * (t.over + (1 - t.over) * double(rem - 256) / double(round - 256));
  const double bytes = (double(M) * K + double(N) * K + 2. * M * N) / (t.hbm * 1e6);
  const double reads = (double(tn) * M + double(tm) * N) * K / (t.near * 1e6);
  return t.launch + std::max(bytes + reads, rounds * (t.first + t.k * K / 1024));
}

// blocks: the operands' rows lie in whole 16-byte blocks.
inline int i8_tile(bool blocks, int64_t M, int64_t N, int64_t K) {
  int best = 0;
  double best_t = 1e300;
  auto look = [&](const I8Tile &t) {
    if (t.code >= 100 && M > kI8FewRows) return;
    if (((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn) > kI8MaxTiles) return;
    const double us = i8_tile_time(t, M, N, K);
    if (us < best_t) {
      best_t = us;
      best = t.code;
    }
  };
  if (blocks)
    for (const I8Tile &t : kI8Tiles) look(t);
  else
    for (const I8Tile &t : kI8AnyTiles) look(t);
  return best;
}

}  // namespace mh
