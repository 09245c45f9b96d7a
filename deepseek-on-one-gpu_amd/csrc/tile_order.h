// Order of the GEMM tiles over workgroups and XCDs.
//
// Workgroup i runs on XCD i % 8.  xcd_run gives each XCD a contiguous run of the tiles;
// tile_coords orders them in panels of `panel` column tiles, row tiles within a panel, so
// that the tiles an XCD holds at a time share their operands through its L2: of 64 tiles
// panels of 8 read 8 + 8 operands.  Where the row tiles are fewer than a panel's columns
// they come together for each column tile (the weights are then the larger operand).
// `panel` is 8 for the largest tiles; callers with smaller row tiles pass fewer, so that the
// weight rows of a panel stay about as many as the activation rows read beside them.
#pragma once

#include "amla_common.h"

namespace amla {

// Column tiles a panel holds (the row tiles of a panel come one after another).
constexpr int TL_PANEL = 8;

AMLA_DEV void tile_coords(int t, int n_tiles, int m_tiles, int &nt, int &mt, int panel = TL_PANEL) {
  if (m_tiles <= panel) {
    nt = t / m_tiles;
    mt = t - nt * m_tiles;
    return;
  }
  const int per = panel * m_tiles, p = t / per, r = t - p * per;
  const int width = min(panel, n_tiles - p * panel);
  mt = r / width;
  nt = p * panel + r - mt * width;
}
// logical index of workgroup i of n (or -1): a contiguous run per XCD
AMLA_DEV int xcd_run(int i, int n) {
  const int run = (n + 7) >> 3, l = (i & 7) * run + (i >> 3);
  return (i >> 3) < run && l < n ? l : -1;
}

}  // namespace amla
