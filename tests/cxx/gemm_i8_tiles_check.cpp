// The choice of kernel and tile of the 8-bit integer products: every size gets one that
// its operands allow and that a launch holds.
#include <cstdio>

#include "gemm_i8_tiles.hpp"

using namespace mh;

int main() {
  const int64_t sizes[] = {1, 2, 7, 15, 16, 17, 31, 33, 64, 65, 100, 127, 128, 255, 256, 257, 511, 768, 1000, 2304, 4096, 8191, 8192, 16384, 40000,
                           131071, 1 << 20, (1 << 24) - 3, 1 << 28, 0x7fffffff};
  long seen[128] = {};
  for (int64_t M : sizes)
    for (int64_t N : sizes) {
      if (((M + 63) / 64) * ((N + 63) / 64) > kI8MaxTiles) continue;  // (refused)
      for (int64_t K : {int64_t(1), int64_t(16), int64_t(100), int64_t(768), int64_t(4096), int64_t(16384), int64_t(131071)})
        for (int b = 0; b < 2; ++b) {
          const int c = i8_tile(b, M, N, K);
          const bool few = c == 100 || c == 101, any = c == 0 || c == 10, whole = c >= 1 && c <= 9;
          if (!few && !any && !whole) return std::printf("code %d\n", c), 1;
          if (whole && !b) return std::printf("blocks for rows that are none: %d\n", c), 1;
          if (few && M > kI8FewRows) return std::printf("few rows: %ld\n", long(M)), 1;
          int64_t bm = 64, bn = 64;
          for (const I8Tile &t : kI8Tiles)
            if (t.code == c) bm = t.bm, bn = t.bn;
          for (const I8Tile &t : kI8AnyTiles)
            if (t.code == c) bm = t.bm, bn = t.bn;
          if (((M + bm - 1) / bm) * ((N + bn - 1) / bn) > kI8MaxTiles) return std::printf("tiles of %d\n", c), 1;
          ++seen[c];
        }
    }
  // each kernel is some size's choice
  for (const I8Tile &t : kI8Tiles)
    if (!seen[t.code]) return std::printf("%d is never chosen\n", t.code), 1;
  for (const I8Tile &t : kI8AnyTiles)
    if (!seen[t.code]) return std::printf("%d is never chosen\n", t.code), 1;
  // a partial round is no dearer than a whole one, and more rows no cheaper
  for (const I8Tile &t : kI8Tiles)
    for (int64_t M = 1; M < 20000; M += 61)
      if (i8_tile_time(t, M + 61, 4096, 4096) < 0.999 * i8_tile_time(t, M, 4096, 4096)) return std::printf("%d at %ld\n", t.code, long(M)), 1;
  std::puts("ok");
  return 0;
}
