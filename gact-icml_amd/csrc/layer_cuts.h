// How the layers' products are cut into tiles and parts: the host's choice alone, in a file of its own so that tests can ask for it.
#pragma once
#include <stdint.h>

#include <initializer_list>

#include "gact_hip.h"

namespace {

constexpr int kComputeUnits = 256;
inline int size_of(int dtype) { return dtype == GACT_F32 ? 4 : 2; }

// workgroups of a tile whose LDS (two steps of both operands, and up to 14 KB beside them) a compute unit holds
constexpr int slots_per_cu(int bm, int bn) { return bm + bn <= 128 ? 4 : bm + bn <= 256 ? 2 : 1; }

// How a product is cut: the side of its tiles, and parts of its depth whose sums are added up afterwards.  Of the cuts there are the one with the
// least estimated time is taken.  A step of a tile takes as long as one workgroup alone on a compute unit needs for it, or as the unit's share of
// all workgroups needs; parts cost a launch and the traffic of their sums.  us per step of 128 bytes, alone / shared, from timings of
// 19 products of 76 million to 17 billion multiplications, each in all of its cuts, both types, forward and with codes (whole, rows x inner x outer):
//   halves  1024x1024x1024   in tiles of 64  8.5   of 128 10.8   of 256 23.7, in two parts of 64 14.6
//           1024x1024x4096                  16.5          12.7          24.6
//           4096x1024x4096                  61.3          37.1          33.3
//           512x4096x1024                   34.5          42.9          72.1, in 2 / 4 / 8 parts of 64 18.1 / 17.7 / 22.8
//           8192x512x512, dW                88            118           196, in 8 parts of 64 23.8
//   floats  1024x1024x1024                  22.7          67.5
//           4096x1024x4096                 264           249
//           512x4096x1024                   78           253, in 4 parts of 64 42.8
// Over the 113 of them that leave a choice the estimate's cut takes 1.2 % longer than the best one.
struct Rate {
  float alone, shared;
};
constexpr Rate kRates[2][2][3] = {      // [codes][halves, floats][64, 128, 256]
    {{{0.33f, 0.23f}, {0.5f, 0.53f}, {1.3f, 1.75f}}, {{0.6f, 0.52f}, {2.0f, 1.95f}}},
    {{{0.6f, 0.33f}, {0.95f, 0.65f}, {1.85f, 2.15f}}, {{0.9f, 0.62f}, {2.3f, 2.1f}}}};
struct Cut {
  int side, parts;
  int64_t per_part;
};
inline Cut cut_of(int dtype, bool coded, int64_t rows, int64_t cols, int64_t depth, int largest, int largest_in_parts) {
  const int64_t step = 128 / size_of(dtype), steps = (depth + step - 1) / step;
  Cut cut = {64, 1, steps * step};
  float least = __builtin_inff();
  for (int n = 0; n < (dtype == GACT_F32 ? 2 : 3); n++) {
    const int side = 64 << n;
    if (side > largest) break;
    const int64_t tiles = ((rows + side - 1) / side) * ((cols + side - 1) / side), slots = kComputeUnits * slots_per_cu(side, side);
    const Rate rate = kRates[coded][dtype == GACT_F32][n];
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (parts > 1 && (parts * 4 > steps || side > largest_in_parts)) break;
      const int64_t per = (steps + parts - 1) / parts, made = (steps + per - 1) / per, work = tiles * made;
      const float alone = rate.alone * (float)((work + slots - 1) / slots);
      const float shared = rate.shared * (float)((work + kComputeUnits - 1) / kComputeUnits);
      const float sums = made == 1 ? 0.0f : 3.0f + (float)(rows * cols) * (float)(8 * made + size_of(dtype)) * 0.25e-6f;
      const float us = (float)per * (alone > shared ? alone : shared) + sums;
      if (us < least) {
        least = us;
        cut = {side, (int)made, per * step};
      }
      if (work >= slots) break;      // more parts only add to the sums
    }
  }
  return cut;
}

// How a forward product is run (times in us, halves / floats, rows x inner x outer).
//  few       rows go to the kernel that reads the weights once and the activations once per 16 columns: up to 16 rows (16x1024x4096 5.2 / 8.1, as
//            tiles 9.9 / 14.4; 16x8192x8192 41.8 / 79, as tiles 38.9 / 82), more where those reads, from the caches, come to no
//            more than 64 MiB (64x1024x4096 7.9 / 16.7, as tiles 10.9 / 16.0; 64x4096x4096 23.3 / 52, as tiles 17.5 / 29.8), and
//            operands of unaligned rows.  In parts of at least 2048 bytes of a row where the strips of columns leave half the compute units
//            idle: 24x4096x1024 11.8 / 27.1 whole, 8.6 / 12.8 in parts
//  finished  by finish_kernel: parts; and the pre-activation's codes, where the tiles that hold whole groups of columns are too few.  Halves: fewer
//            than half the compute units (1024x1024x4096, at half, 25.0 in such tiles, 27.6 finished; 512x1024x4096 23.9 and 21.6; 2048x1024x4096
//            27.3 and 44.6).  Floats, whose tiles are bound by the matrix pipe alone: fewer than the compute units (1024x1024x4096 138 and 80;
//            2048x1024x4096, at all of them, 139 and 150)
struct Forward {
  bool few, finished;
  Cut cut;      // few: parts alone.  Of codes that are not finished: nothing
};
inline Forward forward_of(int dtype, int64_t rows, int64_t inner, int64_t outer, bool codes, bool whole) {
  const int64_t strips = (outer + 15) / 16;
  const bool cached = (rows + 15) / 16 * 16 * strips * inner * size_of(dtype) <= ((int64_t)64 << 20);
  Forward f = {rows <= 16 || (rows <= GACT_LINEAR_FEW_ROWS && (cached || !whole)), codes, {0, 1, inner}};
  if (f.few) {
    const int64_t step = 128 / size_of(dtype), steps = (inner + step - 1) / step;
    int64_t parts = strips <= kComputeUnits / 2 ? kComputeUnits / strips : 1;
    if (parts > steps / 16) parts = steps / 16;
    if (parts > 1) {
      const int64_t per = (steps + parts - 1) / parts;
      f.cut = {0, (int)((steps + per - 1) / per), per * step};
    }
  } else {
    const int64_t tiles = ((rows + 127) / 128) * ((outer + 255) / 256);
    if (codes && tiles >= (dtype == GACT_F32 ? kComputeUnits : kComputeUnits / 2)) f.finished = false;
    f.cut = cut_of(dtype, false, rows, outer, inner, codes ? 64 : 256, 64);
  }
  if (!codes) f.finished = f.cut.parts > 1;
  return f;
}

// Rows of a forward product's tiles that hold the pre-activation's codes, 256 columns wide.  The larger ones where they fill the card (16384x1024x4096
// halves 165, the others 205)
inline int coded_rows_of(bool floats, int64_t rows, int64_t outer) {
  return !floats && ((rows + 255) / 256) * ((outer + 255) / 256) >= kComputeUnits ? 256 : 128;
}

}  // namespace
