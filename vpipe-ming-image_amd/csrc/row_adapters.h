// What a row's own adapter adds to its outputs, for epilogues over few rows, where
// the up-projection is too small for tiles.
#pragma once

#include "common.h"
#include "kernels.h"

namespace ming {

// r[v] += T[m] . B_a[n + v] for NV consecutive columns: f32 sums of their own, ranks
// in order. A row without an adapter is left as it is.
template <int NV>
__device__ __forceinline__ void add_row_adapter(const RowAdapters& ra, int m, int n,
                                                float (&r)[NV]) {
  const int a = ra.rid[m];
  if (a < 0) return;
  const int r8 = ra.table[a].r8;
  const uint16_t* const t = ra.t + (long long)m * ra.ldt;
  const uint16_t* const b = ra.table[a].B + (long long)n * r8;
  float s[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) s[v] = 0.0f;
  for (int k = 0; k < r8; k += 8) {
    const uint4 tv = *reinterpret_cast<const uint4*>(t + k);
    const uint32_t* const tp = &tv.x;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const uint4 bv = *reinterpret_cast<const uint4*>(b + (long long)v * r8 + k);
      const uint32_t* const bp = &bv.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[v] = fmaf(bf16_lo(tp[i]), bf16_lo(bp[i]), s[v]);
        s[v] = fmaf(bf16_hi(tp[i]), bf16_hi(bp[i]), s[v]);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) r[v] += s[v];
}

}  // namespace ming
