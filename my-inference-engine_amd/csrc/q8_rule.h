// Which kernel computes a product in 8 bits, and in what tiles.  No device code: tests ask it on the CPU.
#pragma once

#include <stdint.h>
#ifdef Q8_TUNE
#include <cstdlib>
#endif

namespace mi_fa2 {

constexpr int kQ8RowsMax = 64;    // rows that the few-row kernel takes
constexpr int kQ8KeepK = 2048;    // (padded) in features whose rows it keeps in registers
constexpr int kQ8FusedMax = 16;   // rows that it brings to 8 bits itself, of at most kQ8KeepK
constexpr int kQ8FloatMax = 4, kQ8FloatK = 12288;   // fp32 rows that it does, and their most features

enum Q8Kernel { kQ8FewRows = 0, kQ8Tile32 = 1, kQ8Tile64 = 2, kQ8Gemm64 = 3, kQ8Gemm128 = 4 };

struct Q8Plan {
  int32_t kernel;   // Q8Kernel
  int32_t tiles;    // work-groups
};

// The tile kernel (32 or 64 tokens by 64 features, K split over the work-group's waves, straight from
// memory) hides the most latency but reads x and W once for every tile that needs them: it is taken while
// its tiles are no more than the 256 CUs.  Behind that the products that share operands through LDS:
// 64 x 64 tiles until there are enough of 128 x 128 for every CU.  Measured (us, 32 x 64 / 64 x 64 straight from
// memory, 64 x 64 / 128 x 128 through LDS):
//   tokens x features x K: 96 x 1536 x 8960 12.1 16.9 22.5 39;  512 x 1536 x 8960 22.3 18.3 22.9 41;
//   1024 x 1536 x 8960 37.0 35.4 26.9 42;  256 x 2048 x 1536 5.2 6.3 6.4 11;  400 x 2048 x 1536 7.3 6.6 6.6 11;
//   1024 x 2048 x 1536 13.6 13.1 8.5 12;  4096 x 2048 x 1536 - - 25.7 20.0;  150 x 17920 x 1536 19.4 23.6 13.6
//   14.8;  512 x 17920 x 1536 48 51 28.2 25.2
inline Q8Plan q8_plan(int32_t rows, int32_t panels, int32_t kp) {
  constexpr int64_t kCus = 256;
  (void)kp;
  const auto tiles = [&](int tm, int np) {
    return (int64_t)((rows + tm - 1) / tm) * ((panels + np - 1) / np);
  };
#ifdef Q8_TUNE
  if (getenv("Q8_NP") && (rows > 64 || atoi(getenv("Q8_NP")))) {
    const int np = atoi(getenv("Q8_NP"));
    if (np == 1) return {kQ8Tile32, (int32_t)tiles(32, 4)};
    if (np == 2) return {kQ8Tile64, (int32_t)tiles(64, 4)};
    if (np == 4) return {kQ8Gemm64, (int32_t)tiles(64, 4)};
    if (np == 8) return {kQ8Gemm128, (int32_t)tiles(128, 8)};
  }
#endif
  if (rows <= kQ8RowsMax) return {kQ8FewRows, 0};
  if (tiles(32, 4) <= kCus) return {kQ8Tile32, (int32_t)tiles(32, 4)};
  if (tiles(64, 4) <= kCus) return {kQ8Tile64, (int32_t)tiles(64, 4)};
  if (tiles(128, 8) < kCus) return {kQ8Gemm64, (int32_t)tiles(64, 4)};
  return {kQ8Gemm128, (int32_t)tiles(128, 8)};
}

}  // namespace mi_fa2
