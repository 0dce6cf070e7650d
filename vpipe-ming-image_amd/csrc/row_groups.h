// Where a block's rows are in a ragged plan: offsets[0..E] ascending, group e
// the rows [offsets[e], offsets[e + 1]). The sizes are known on the device
// alone, so every wave finds its block's group itself: each lane sums up E / 64
// groups, a scan over the wave and a ballot name the lane, the lane the group.
#pragma once

#include "common.h"

namespace ming {

struct RowGroup {
  int e;       // -1: none for this block
  int p0;      // first row
  int rows;
  int index;   // the block's index inside the group
};

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
  int sum = 0, lo = at(e0);
  for (int j = 0; j < per; ++j) {
    const int hi = at(e0 + j + 1);
    sum += count(lo, hi);
    lo = hi;
  }
  // A launch holds fewer units than 2^24 and no group of a plan more; the lanes of
  // what is no plan are cut so that their total stays an int.
  sum = sum < (1 << 25) - 1 ? sum : (1 << 25) - 1;
  int run = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(run, o, 64);
    if (lane >= o) run += v;
  }
  RowGroup g = {-1, 0, 0, 0};
  const int b = pick(__builtin_amdgcn_readlane(run, 63));
  const uint64_t past = __ballot(run > b);
  if (b < 0 || !past) return g;
  const int w = __builtin_ctzll(past);     // the lane whose groups hold the block
  int left = b - (__builtin_amdgcn_readlane(run, w) - __builtin_amdgcn_readlane(sum, w));
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
