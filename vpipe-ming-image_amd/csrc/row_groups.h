// Where a block's rows are in a ragged plan: offsets[0..E] ascending, group e
// the rows [offsets[e], offsets[e + 1]). The sizes are known on the device
// alone, so every wave finds its block's group itself: each lane sums up E / 64
// groups, a scan over the wave and a ballot name the lane, the lane the group. It is a
// chain of latencies before a block's first load: with the scan in registers (not through
// LDS) and, up to 64 groups, the ends from the lane that has them (not loaded again), 8 x 8
// places of [64][2048, 2048] dense and gated took 54.4 us where it was 58.4.
#pragma once

#include "common.h"

namespace ming {

struct RowGroup {
  int e;       // -1: none for this block
  int p0;      // first row
  int rows;
  int index;   // the block's index inside the group
};

// The sums over lanes 0 .. lane: inside rows of 16 by shifts, then over the rows by their
// last lanes.
__device__ __forceinline__ int scan_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row_bcast:15, rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // row_bcast:31, rows 2, 3
  return v;
}

// The group of unit pick(total) where group e has units(rows of e) consecutive
// ones; none where pick says -1. Offsets are kept inside [0, n] and a group that
// ends before it begins is empty, so a plan that is not one can name wrong rows
// but none outside.
template <class Units, class Pick>
__device__ __forceinline__ RowGroup find_group(const int32_t* __restrict__ offsets, int E, int n,
                                               Units&& units, Pick&& pick) {
  const int lane = (int)threadIdx.x & 63;
  const int per = (E + 63) / 64;
  const int e0 = lane * per;
  auto at = [&](int e) {
    const int v = offsets[e < E ? e : E];
    return v < 0 ? 0 : v < n ? v : n;
  };
  auto count = [&](int lo, int hi) { return hi > lo ? units(hi - lo) : 0; };
  const int lo0 = at(e0), hi0 = at(e0 + 1);
  int sum = count(lo0, hi0), lo = hi0;
  for (int j = 1; j < per; ++j) {
    const int hi = at(e0 + j + 1);
    sum += count(lo, hi);
    lo = hi;
  }
  // A launch holds fewer units than 2^24 and no group of a plan more; the lanes of
  // what is no plan are cut so that their total stays an int.
  sum = sum < (1 << 25) - 1 ? sum : (1 << 25) - 1;
  const int run = scan_sum(sum);
  RowGroup g = {-1, 0, 0, 0};
  const int b = pick(__builtin_amdgcn_readlane(run, 63));
  const uint64_t past = __ballot(run > b);
  if (b < 0 || !past) return g;
  const int w = __builtin_ctzll(past);     // the lane whose groups hold the block
  int left = b - (__builtin_amdgcn_readlane(run, w) - __builtin_amdgcn_readlane(sum, w));
  if (per == 1) {                          // the lane has its one group's ends
    const int p0 = __builtin_amdgcn_readlane(lo0, w);
    return {w, p0, __builtin_amdgcn_readlane(hi0, w) - p0, left};
  }
  int e = w * per;
  lo = at(e);                              // wave-uniform from here on
  for (int j = 0; j < per; ++j, ++e) {
    const int hi = at(e + 1);
    const int u = count(lo, hi);
    if (left < u) {
      g.e = __builtin_amdgcn_readfirstlane(e);
      g.p0 = __builtin_amdgcn_readfirstlane(lo);
      g.rows = __builtin_amdgcn_readfirstlane(hi - lo);
      g.index = __builtin_amdgcn_readfirstlane(left);
      return g;
    }
    left -= u;
    lo = hi;
  }
  return g;
}

// Tile tm of a group of `rows` that takes `tiles` of them, in units of U rows spread
// over the tiles as evenly as they go: heights differ by a unit at most, so no block
// is left with the sliver of a group, whose stages cost nearly a full tile's.
struct RowTile {
  int first, rows;
};
template <int U>
__device__ __forceinline__ RowTile row_tile(int rows, int tiles, int tm) {
  const int units = (rows + U - 1) / U, each = units / tiles, more = units - each * tiles;
  const int first = U * (each * tm + (tm < more ? tm : more));
  const int h = U * (each + (tm < more ? 1 : 0));
  return {first, rows - first < h ? rows - first : h};
}

}  // namespace ming
