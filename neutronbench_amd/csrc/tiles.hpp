// Which tile of a product a block takes.
#pragma once

#include "common.hpp"

namespace nts {

// Blocks are handed to the eight chiplets, each with an L2 of its own, in turn.  Where there are kXcdTiles tiles of rows or more, a
// chiplet takes `group` of them at a time, every column of tiles for all of the group before the next: blocks that run together share
// rows and columns.  With fewer, tiles in turn fill the chip more evenly.  4-bit product of 232,965 rows of 602 by 256: 79.5 -> 65.5
// us, its rows' gradient of 169,343 by 640 by 640: 607 -> 489.
constexpr uint32_t kXcdTiles = 64;
#if defined(__HIPCC__)
__device__ __forceinline__ void tile_of(uint32_t tiles_n, bool by_xcd, uint32_t group, uint32_t *tm, uint32_t *tn) {
  if (by_xcd) {
    const uint32_t x = blockIdx.x / 8u, of = group * tiles_n, within = x % of;
    *tm = (x / of * group + within % group) * 8u + blockIdx.x % 8u;
    *tn = within / group;
  } else {
    *tm = blockIdx.x / tiles_n;
    *tn = blockIdx.x % tiles_n;
  }
}
#endif
inline uint32_t tile_blocks(uint32_t tiles_m, uint32_t tiles_n, uint32_t group) {
  return (tiles_m >= kXcdTiles ? ceil_div(tiles_m, 8 * group) * 8u * group : tiles_m) * tiles_n;
}

}  // namespace nts
