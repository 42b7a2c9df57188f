// Which kernel computes a product in 8 bits, and in what tiles.  No device code: tests ask it on the CPU.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace mi_fa2 {

constexpr int kQ8RowsMax = 64;    // rows that the few-row kernel takes
constexpr int kQ8KeepK = 2048;    // (padded) in features whose rows it keeps in registers
constexpr int kQ8FusedMax = 16;   // rows that it brings to 8 bits itself, of at most kQ8KeepK
constexpr int kQ8FloatMax = 4, kQ8FloatK = 12288;   // fp32 rows that it does, and their most features

// What a product's rows are (and what is brought to 8 bits): 16-bit rows, the same normalised, fp32 rows, rows in 8 bits.
enum Q8Source { kQ8Plain = 0, kQ8Norm = 1, kQ8Float = 2, kQ8Rows = 3 };

// (tokens by features)
enum Q8Kernel {
  kQ8FewRows, kQ8Tile32x32, kQ8Tile32x64, kQ8Tile64x64, kQ8Gemm64, kQ8Gemm128, kQ8Gemm128x192, kQ8Gemm192x128,
  kQ8Gemm128x256, kQ8Gemm192x192, kQ8Gemm256x256
};

// How the few-row kernel takes more panels than there are CUs, where x stays in registers (q8_pad(K) <= kQ8KeepK, 16
// rows at most): panels between two barriers, and work-groups a CU.  More panels put more loads in flight and
// share a barrier; a second work-group computes while the first waits, until registers (K past 1536) or an
// uneven last round cost more.  Measured with the norm, weights from memory (us; panels x work-groups a CU):
//   tokens x features x K        1 x 1    1 x 2    2 x 1    2 x 2    4 x 1
//   16 x 6720 x 1536             6.63     7.35     6.37     6.24     6.86
//   1 x 9728 x 896               5.53     5.01     4.87     5.35     4.60
//   16 x 14400 x 1536            9.52     8.42     8.22     8.62     8.06
//   1 x 17920 x 1536             9.02     7.85     7.90     7.42     8.36
//   16 x 17920 x 1536            10.6     8.95     9.39     8.81     9.59
//   16 x 28672 x 1536            13.1     11.4     11.3     10.0     10.9
//   16 x 28672 x 896             11.5     9.53     9.55     8.41     8.28
//   16 x 22016 x 2048            13.5     11.9     11.8     13.7     12.3
//   1 x 96000 x 1536             34.5     25.9     25.2     24.6     23.9
// (Over 45 sizes by 1, 4 and 16 tokens 0.5% behind the best of each, 1 x 1 always 18%.)
struct Q8RowsShape {
  int32_t panels, per_cu;
};
inline Q8RowsShape q8_rows_shape(int32_t panels, int32_t kp, int32_t cus) {
  if (panels <= cus) return {1, 1};
  if (panels <= 2 * cus || kp > 1536) return {2, 1};
  if (kp > 1024 && panels > 4 * cus && panels <= 8 * cus) return {2, 2};
  return {4, 1};
}

// The variant of the few-row kernel.
struct Q8RowsChoice {
  int32_t mt;      // tokens by 16
  int32_t panels;  // a tile's, or half: one panel's halves
  int32_t half;
  int32_t keep;    // x stays in registers
  int32_t steps;   // of K that a wave takes at a time (keep: all of its share)
  int32_t grid;
};
inline Q8RowsChoice q8_rows_choice(int32_t rows, int32_t panels, int32_t kp, int32_t cus, Q8Source source, bool gated) {
  const bool keep = source != kQ8Float && kp <= kQ8KeepK;
  Q8RowsChoice c{rows > 32 ? 4 : rows > 16 ? 2 : 1, 1, 0, keep, 0, std::min(panels, cus)};
  // (from 17 rows on a panel at a time; two work-groups a CU: 64 x 6400 x 2048 5.7 -> 6.7 us, 64 x 8192 x 1536 4.8 ->
  // 5.2)
  if (c.mt == 1) {
    if (!gated && !keep && 2 * panels <= cus) {
      // few panels of many features: half a panel a work-group (1536 x 8960 by one token 6.4 -> 5.8 us)
      c.half = 1;
      c.grid = 2 * panels;
    } else if (keep && (source != kQ8Rows || kp <= 1536)) {   // (else 16 rows in 8 bits x 6400 x 2048 3.5 -> 4.3 us)
      const Q8RowsShape shape = q8_rows_shape(panels, kp, cus);
      c.panels = shape.panels;
      c.grid = std::min((panels + shape.panels - 1) / shape.panels, shape.per_cu * cus);
    } else if (!keep && source != kQ8Float && panels >= 16 * cus) {   // (16 x 100000 x 4096 94 -> 85 us; one token 78
      c.panels = 4;                                                   // and 79)
    }
  }
  // Where x does not stay: one token's half tiles of 1536 x 8960 take all 18 steps of a wave at once (the feed-forward
  // block 17.1 -> 15.4 us); with rows in 8 bits beside them 9 (6.0 us, 18: 7.1).  Past 9,216 features, where a wave
  // has more than 18, nothing shows of it: blocks of 1536 x 8192, 9216, 9472, 10240, 12288 13.8, 14.9, 15.6, 16.6,
  // 17.9 us (weights from memory; 12416, in a launch more, 22.8).
  c.steps = keep ? std::max(2, (kp + 511) / 512) : source == kQ8Float && c.half ? 18 : c.mt == 1 ? 9 : 6;
  return c;
}

struct Q8Plan {
  int32_t kernel;   // Q8Kernel
  int32_t tiles;    // work-groups
};

// Three families.  The few-row kernel streams W once past 16 to 64 tokens.  The tile kernel (32 or 64 tokens by 32
// or 64 features, K split over the work-group's waves, operands straight from memory) hides the most latency,
// but reads x and W again for every tile that needs them: it is taken while its tiles are no more than the 256
// CUs.  Behind both, the products that share operands through LDS: 64 x 64 tiles until there are enough of
// 128 x 128 for every CU, then the tile below.  Measured (us; few-row, 32 x 32, 32 x 64, 64 x 64 in LDS, 128 x 128 in LDS):
//   tokens x features x K        few    32x32  32x64  64L    128L
//   17 x 2048 x 1536             3.5    4.8    5.2    6.0    9.7
//   32 x 1536 x 8960             7.9    10.0   12.5   22.1   38.4
//   32 x 6144 x 4096             9.8    7.9    8.9    12.0   20.3
//   32 x 14336 x 4096            15.8   13.1   12.6   13.2   20.8
//   64 x 6144 x 2048             7.1    7.8    7.6    8.2    12.8
//   64 x 9728 x 896              7.1    8.8    7.8    5.3    8.1
//   64 x 17920 x 1536            9.7    14.2   11.8   8.8    12.0
//   64 x 151936 x 1536           67     102    78     55     49
//   64 x 1536 x 8960             11.3   10.0   12.4   22.2   38.9
//   150 x 896 x 4864             -      7.7    9.3    13.8   26.6
//   256 x 1536 x 8960            -      16.7   13.1   22.6   45.3
//   512 x 17920 x 1536           -      -      48     28.2   25.2
// (512 x 1536 x 8960: 64 x 64 straight from memory 18.3, through LDS 22.9; 400 x 2048 x 1536 6.6 both.)
//
// Of the large tiles the one whose work for the CU with the most tiles is least: rounds of 256 tiles, times the tile's
// area, times 0.9 at one and a half times 128 x 128, 0.84 at twice and 0.81 at four times, which read each operand for
// more products; a single round of work-groups of four waves counts 1.2 times, with nothing beside them to hide their
// waits.  Over 22 shapes from 512 x 17920 x 1536 to 8192^3 that is 0.3% behind the best of the first five, 128 x 128
// always 6.8%:
//   tokens x features x K        128x128  128x192  192x128  128x256  192x192  256x256
//   512 x 17920 x 1536           20.7     20.5     19.4     23.9     27.7
//   2048 x 17920 x 1536          62.0     60.8     65.9     62.9     67.3
//   4096 x 17920 x 1536          120      118      124      112      119      128
//   4096 x 2048 x 1536           16.1     20.3     18.2     18.2     21.0
//   4001 x 1536 x 8960           58.5     52.9     52.8     55.6     57.9
//   16384 x 1536 x 8960          211      199      230      187      192      201
//   1024 x 6144 x 4096           29.4     27.1     36.0     29.4     31.5
//   6001 x 6144 x 4096           142      137      137      139      130      156
//   1000 x 14336 x 4096          62.3     65.3     63.6     55.9     59.8     53.6
//   4096 x 4096 x 4096           65.9     67.8     67.2     61.0     66.7     60.4
//   4096 x 4096 x 14336          223      -        -        194      206      184
//   8192 x 8192 x 8192           483      473      460      441      458      426
// The gated product likewise, a block's three launches (tokens x hidden x inner size):
//   4001 x 1536 x 8960           243      237      228      227      219
//   1024 x 1536 x 8960           76.9     75.8     80.5     79.2     81.1
//   2048 x 4096 x 14336          399      395      392      374      382
inline Q8Plan q8_plan(int32_t rows, int32_t panels, int32_t kp) {
  constexpr int64_t kCus = 256;
  const auto plan = [&](Q8Kernel kernel, int tm, int np) {
    return Q8Plan{kernel, (int32_t)((int64_t)((rows + tm - 1) / tm) * ((panels + np - 1) / np))};
  };
  const Q8Plan t32x32 = plan(kQ8Tile32x32, 32, 2), t32x64 = plan(kQ8Tile32x64, 32, 4),
               t64x64 = plan(kQ8Tile64x64, 64, 4), g64 = plan(kQ8Gemm64, 64, 4),
               g128 = plan(kQ8Gemm128, 128, 8);
  const bool keep = kp <= kQ8KeepK;
  if (rows <= 16) return {kQ8FewRows, 0};
  if (rows <= kQ8RowsMax && (keep ? panels <= 512 : rows <= 32 && panels < 256)) return {kQ8FewRows, 0};
  if (rows > kQ8RowsMax || !keep) {
    if (t32x32.tiles <= kCus) return t32x32;
    if (t32x64.tiles <= kCus) return t32x64;
    if (t64x64.tiles <= kCus && !keep) return t64x64;
  }
  if (g128.tiles < kCus) return g64;
  Q8Plan best = g128;
  int64_t least = INT64_MAX;
  const auto consider = [&](Q8Kernel kernel, int tm, int np, int weight) {
    const Q8Plan t = plan(kernel, tm, np);
    const int64_t rounds = (t.tiles + kCus - 1) / kCus;
    const bool alone = rounds == 1 && kernel != kQ8Gemm256x256;
    const int64_t cost = rounds * weight * (alone ? 6 : 5);
    if (cost < least) least = cost, best = t;
  };
  consider(kQ8Gemm128, 128, 8, 100);
  consider(kQ8Gemm192x128, 192, 8, 135);
  consider(kQ8Gemm128x192, 128, 12, 135);
  consider(kQ8Gemm192x192, 192, 12, 189);
  consider(kQ8Gemm128x256, 128, 16, 168);
  consider(kQ8Gemm256x256, 256, 16, 325);
  return best;
}

}  // namespace mi_fa2
