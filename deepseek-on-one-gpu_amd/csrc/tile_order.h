// Order of the GEMM tiles over workgroups and XCDs.
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
