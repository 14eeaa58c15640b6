// Pieces that the tiled products share (gfx950): tile order and the waits of their
// direct-to-LDS loads (load_lds16_base).
#pragma once

#include "tmhd_internal.h"

namespace tmhd {

// Workgroup b of G as a logical id: consecutive ids run on one XCD (workgroups
// are dealt to the 8 XCDs in turn), whose L2 then holds their shared panels.
__device__ __forceinline__ int xcd_logical_id(int b, int G) {
  const int xcd = b & 7, pos = b >> 3, per = G >> 3, rem = G & 7;
  return xcd < rem ? xcd * (per + 1) + pos : rem * (per + 1) + (xcd - rem) * per + pos;
}

// Tile (tm, tn) of logical tile L: 4 row tiles share each column sweep (L2
// reuse).  Measured on the 12,252-row INT8 projections: 4 beats 2, 6, 8, 16 and 48
// (about 3% against 8 on 5,120 x 13,824, 1.4% on the 5,376 x 28,672 FC1).
__device__ __forceinline__ void grouped_tile(int L, int tm_count, int tn_count, int &tm, int &tn) {
  constexpr int GROUP = 4;
  const int per_group = GROUP * tn_count;
  const int first_tm = (L / per_group) * GROUP;
  const int gsize = min(tm_count - first_tm, GROUP);
  tm = first_tm + (L % per_group) % gsize;
  tn = (L % per_group) / gsize;
}

// s_waitcnt immediate that leaves n vector-memory operations in flight (and waits for nothing else)
constexpr int vmcnt_imm(int n) { return 0x0f70 | (n & 15) | ((n >> 4) << 14); }

}  // namespace tmhd
