// Order of the GEMM tiles over workgroups and XCDs.
#pragma once

#include "amla_common.h"

namespace amla {

// Column tiles a panel holds (the row tiles of a panel come one after another).
constexpr int TL_PANEL = 8;

AMLA_DEV void tile_coords(int t, int n_tiles, int m_tiles, int &nt, int &mt) {
  if (m_tiles <= TL_PANEL) {
    nt = t / m_tiles;
    mt = t - nt * m_tiles;
    return;
  }
  const int per = TL_PANEL * m_tiles, p = t / per, r = t - p * per;
  const int width = min(TL_PANEL, n_tiles - p * TL_PANEL);
  mt = r / width;
  nt = p * TL_PANEL + r - mt * width;
}
// logical index of workgroup i of n (or -1): a contiguous run per XCD
AMLA_DEV int xcd_run(int i, int n) {
  const int run = (n + 7) >> 3, l = (i & 7) * run + (i >> 3);
  return (i >> 3) < run && l < n ? l : -1;
}

}  // namespace amla
