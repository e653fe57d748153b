// Which launches of the grouped FP8 products (persistent_capi.hip, product_capi.hip) take the mid-tile kernel.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "mid_gemm.h"
#include "persistent_kernel.h"
#include "persistent_wide.h"

namespace ggemm {
namespace host {

inline int64_t mid_tiles(int rows, int G, int N, int64_t M_total) {
  return (M_total / rows + (G < M_total ? G : M_total)) * ((N + 127) / 128);
}

// The second look at a launch of more than four groups that the estimate of mid_preferred gives to 128-row
// tiles: both sides in whole rounds, for rows spread evenly over the groups and for any (half a row tile more
// for each group), and the mean of the two. Of 1553 drawn launches on 128 rows (1 to 64 groups, 1 to 60000 rows,
// features 64 to 5760, even, exponential and Zipf lengths) 35 were more than 3 % slower than before there were mid
// tiles, 16 more than 10 %: 13 groups, 5788 rows, N = K = 2880 75 us, 51 on the wide tiles; 15, 7007, N = 2560, K
// = 5760 112, 85. With this rule 27 and 9 are, and 7 lose a gain of 20 % or more. For up to four groups it lost
// as often as it gained.
// extra: us that a large tile's epilogue takes with nothing beside it; tn: the large tiles' columns.
inline bool rows128_faster(int N, double M, double g, double stages, double mem, bool wide, int tn, int cus, double extra) {
  constexpr int kRun = ggemm::mid::kXcdRun;
  double mid = 0, big = 0;
  for (const bool even : {true, false}) {
    auto tiles = [&](double h, double w) {
      return (even ? g * std::ceil(M / g / h) : std::max(1.0, M / h + g / 2)) * std::ceil(N / w);
    };
    const double t = tiles(128, 128), all = ggemm::kXcds * kRun, runs = std::floor(t / all);
    // half rounds of two workgroups on every CU of the XCD that takes most tiles (tile_of_block)
    const double most = kRun * runs + std::min<double>(kRun, t - runs * all);
    const double half = std::ceil(most * ggemm::kXcds / cus);
    mid += 6.6 + (0.976 * half / 2 - 0.28) * (stages + 2) + 0.33 * mem;
    const double r = std::ceil(tiles(wide ? ggemm::pw::kTM : ggemm::kTileM, tn) / cus);
    big += wide        ? 2.6 + r * (1.19 * stages + 6.1) + 0.32 * mem
           : tn == 320 ? 2.0 + r * (1.12 * stages + 6.8) + 0.29 * mem
                       : 4.6 + r * (1.27 * stages + 5.0) + 0.43 * mem;
    big += r * extra;
  }
  return mid < 1.05 * big;
}

// The mid-tile kernel's row-tile height (64 or 128) where it is the faster one, else 0: the estimated
// microseconds of each kernel compared. The lengths of the groups are on the device; M_total rows over
// G groups are taken to make max(g, M_total / height + g / 2) row tiles, g the groups that can have a
// row. Per 128-byte K stage and tile: 1.85 us (wide) or 1.75 us (512-thread) for the persistent kernels,
// their tiles one to a CU in whole rounds; 0.69 / 1.06 us for the mid tiles of 64 / 128 rows with two
// workgroups on every CU (0.41 / 0.64 with few), and they feel the memory's time too; 4 us around
// either. Measured (us, the better of 512-thread and wide kernel -> the choice): N = 5760, K = 2880, G =
// 32: 256 rows 149 -> 95 (64), 3072 rows 148 -> 118 (128), 6144 rows 162, mid 182 (stays); N = K = 2880,
// G = 4: 512 rows 38 -> 14, 8192 rows 83 -> 75, 16384 rows 132, mid 153 (stays); N = 2048, K = 1424, G =
// 7: 512 rows 25 -> 9, 5003 rows 28, mid 31 (stays); N = 512, K = 1024, G = 8: 100000 rows 92 -> 77.
// Products with an epilogue give more: extra, as above, how far below the 128-row tiles' estimate that of 64 rows has to be
// (product_launch.h), and whether z is kept in 8 bits, with which the 512-thread kernel's tiles are 384 wide (persistent_entry).
inline int mid_preferred(int G, int N, int K, int scm, int64_t M_total, bool wide, int cus, double extra = 0,
                         double below = 0.97, bool kept8 = false) {
  if (G > ggemm::mid::kMaxGroups || M_total <= 0 || mid_tiles(64, G, N, M_total) > (1 << 22)) return 0;
  if ((int64_t)scm * 2 * 64 >= (int64_t)ggemm::nt::kOob) return 0;   // a wave's rows of C: 32-bit offsets
  const double M = (double)M_total, g = G < M ? G : M;
  const double stages = (K + 127) / 128 + 2;                          // two more for the tile's ends
  const double mem = (M * K + g * N * K + 2 * M * N) / 5.1e6;
  auto tiles = [&](double h, double w) { return std::max(g, M / h + g / 2) * std::ceil(N / w); };
  const int tn = !wide && (kept8 || ggemm::wide_tiles(N, false)) ? 384 : 320;
  double big;
  if (wide) {
    big = 4 + std::ceil(tiles(256, tn) / cus) * (stages * 1.85 + extra);
  } else {
    big = 4 + std::ceil(tiles(192, tn) / cus) * (stages * (tn == 384 ? 1.75 : 1.58) + extra) + 0.2 * mem;
  }
  const double f64 = tiles(64, 128) / (2 * cus), f128 = tiles(128, 128) / (2 * cus);
  const double c64 = 4 + std::max(1.0, f64) * stages * (0.41 + 0.28 * std::min(1.0, f64)) + 0.3 * mem;
  const double c128 = 4 + std::max(1.0, f128) * stages * (0.64 + 0.42 * std::min(1.0, f128)) + 0.3 * mem;
  if (std::min(c64, c128) >= 0.92 * big) return 0;   // near the line the estimate is a few per cent off
  if (c64 < below * c128) return 64;
  return g <= 4 || rows128_faster(N, M, g, (K + 127) / 128, mem, wide, tn, cus, extra) ? 128 : 0;
}

}  // namespace host
}  // namespace ggemm
