// Which kernel computes a product in 8 bits, and in what tiles.  No device code: tests ask it on the CPU.
#pragma once

#include <stddef.h>
#include <stdint.h>
#ifdef Q8_TUNE
#include <cstdlib>
#endif

namespace mi_fa2 {

constexpr int kQ8RowsMax = 64;    // rows that the few-row kernel takes
constexpr int kQ8KeepK = 2048;    // (padded) in features whose rows it keeps in registers
constexpr int kQ8FusedMax = 16;   // rows that it brings to 8 bits itself, of at most kQ8KeepK

struct Q8Plan {
  int32_t np;       // panels of W a tile, 0: the few-row kernel
  int32_t tm;       // tokens a tile
  int32_t tiles;
  int32_t splits;   // work-groups that share a tile's K
  size_t part;      // bytes of their sums (4 for each number of every tile and share), 0 for one
  size_t count;     // bytes of their arrival counts
};

inline Q8Plan q8_plan(int32_t rows, int32_t panels, int32_t kp) {
  Q8Plan p{};
  p.splits = 1;
  if (rows <= kQ8RowsMax) return p;
  const int steps = kp / 64;
  p.np = 16;
  p.tm = 128;
#ifdef Q8_TUNE
  if (const char* e = getenv("Q8_NP")) { p.np = atoi(e); p.tm = p.np == 4 ? 64 : 128; }
  if (const char* e = getenv("Q8_SPLITS")) p.splits = atoi(e) < steps ? atoi(e) : steps;
#endif
  (void)steps;
  const int64_t tiles = (int64_t)((rows + p.tm - 1) / p.tm) * ((panels + p.np - 1) / p.np);
  p.tiles = (int32_t)tiles;
  if (p.splits > 1) {
    p.part = (size_t)tiles * p.splits * p.np * 16 * p.tm * 4;
    p.count = (size_t)tiles * 4;
  }
  return p;
}

}  // namespace mi_fa2
