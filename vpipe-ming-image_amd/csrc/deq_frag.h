// Codes of the fast resident layout to fp16 MFMA fragments (qproj_fast.hip says
// how the layout is built), and where a code tile's chunks lie in LDS.
//
// A weight, code * scale + bias, is rounded here once to fp16, at most 2^-11 of it: the
// matrix operand's type, three bits more than the output keeps. Against weights in f32
// sums move by 2e-4 (w8) and 4e-5 (w4, where code * scale has four bits less) of
// themselves: bf16 outputs then differ by 9e-4 and 3e-4 in the 2-norm, where a value
// falls to the other side, and their error against 64 bits stays at 1.7e-3, bf16's own.
#pragma once

#include "common.h"

namespace ming {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// 8 codes (one w4 word) -> 8 fp16 dequantized values. The word's nibbles
// are ordered {k0,k4,k1,k5,k2,k6,k3,k7}, so lo = w & 0x0F0F0F0F holds
// k0..k3 one per byte and hi = (w >> 4) & 0x0F0F0F0F holds k4..k7; one
// v_perm per pair then lays a code under the 0x64 magic byte.
__device__ __forceinline__ uint4 deq_w4(uint32_t w, half2v s2, half2v b2) {
  const half2v k1024 = {(_Float16)1024.0f, (_Float16)1024.0f};
  const uint32_t lo = w & 0x0F0F0F0Fu;
  const uint32_t hi = (w >> 4) & 0x0F0F0F0Fu;
  uint32_t v[4];
  v[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x05010400u);
  v[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x05030402u);
  v[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x05010400u);
  v[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x05030402u);
  uint4 o;
  uint32_t* op = &o.x;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const half2v c = __builtin_bit_cast(half2v, v[p]) - k1024;
    op[p] = __builtin_bit_cast(uint32_t, c * s2 + b2);
  }
  return o;
}

// 8 codes (two w8 words, bytes in k order) -> 8 fp16.
__device__ __forceinline__ uint4 deq_w8(uint32_t w0, uint32_t w1, half2v s2,
                                        half2v b2) {
  const half2v k1024 = {(_Float16)1024.0f, (_Float16)1024.0f};
  uint32_t v[4];
  v[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x05010400u);
  v[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x05030402u);
  v[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x05010400u);
  v[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x05030402u);
  uint4 o;
  uint32_t* op = &o.x;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const half2v c = __builtin_bit_cast(half2v, v[p]) - k1024;
    op[p] = __builtin_bit_cast(uint32_t, c * s2 + b2);
  }
  return o;
}

// Code-chunk swizzle inside a row group: chunk h of row n sits at
// n*CPR + (h ^ sw(n)), so the 16 rows a fragment read serves per LDS cycle
// land on distinct banks (rows are 32 B (w4) / 64 B (w8) apart).
template <int CPR>
__device__ __forceinline__ int wswz(int n) {
  return CPR == 2 ? ((n >> 3) & 1) : ((n >> 2) & 3);
}
template <int CPR>
__device__ __forceinline__ int wchunk(int n, int h) {
  return n * CPR + (h ^ wswz<CPR>(n));
}

}  // namespace ming
