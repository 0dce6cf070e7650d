// The down-projection T = x . A^T of every row's own adapter.
#pragma once

#include "common.h"
#include "kernels.h"

namespace ming {

// T[m] = strength * fold * (x[m] . A_a^T), a = ids[m], f32 sums rounded once to bf16: T
// is a matrix operand beside B, and a request gets what ming_lin's own adapters give it,
// whose T is bf16 too. Outputs of rows whose adapters add a third as much as the weight
// move by 3e-4 before their own rounding, their error against 64 bits stays at 1.7e-3.
// A block takes 16 or 32 rows; the adapters among them (in any order) are found with
// ballots, and each adapter's 16-rank chunks are v_mfma_f32_16x16x32_bf16 tiles over
// all the rows, of which only that adapter's are stored: requests' rows lie together,
// so a block has one or two adapters, and where every row has its own the time is
// that of reading their A. K is shared out over the eight waves by 64-groups, the
// sums meet in LDS and are added in wave order (no atomics). A is resident in the
// operand's own order (launch_repack_adapter): a wave's load is one run of 1 KB, of
// which lanes past the rank take no part.
//
// Two forms. Few rows (row_xa_block; also beside a split projection's own blocks,
// which need T in their sum alone): 16 rows, a chunk a block and turn, operands
// straight from memory, all of a chunk's at once and under the chunk before it;
// `ny` blocks share out the chunks. Bound by three memory latencies in a row (ids,
// table, A) and, where every row brings its own adapter, by a chunk's bytes at a CU's
// rate (4.8 us at 4 rows of [3840], 8.7 at 37, as many adapters). Many rows
// (row_xa_many_kernel): x passes through LDS in whole 1 KB row pieces, read from memory
// once for two (or four) chunks and for the fp16 copy of x that a quantized projection
// multiplies. Bound by HBM, x once and its copy once ([8704, 3840] with the copy: 38 to
// 45 us, 79 with x from memory a lane's 16 bytes at a time).

__device__ __forceinline__ uint4 to_f16(const uint4& v, uint32_t& seen) {
  seen = range_track4(seen, v);
  uint4 f;
  f.x = bf16x2_to_f16x2(v.x);
  f.y = bf16x2_to_f16x2(v.y);
  f.z = bf16x2_to_f16x2(v.z);
  f.w = bf16x2_to_f16x2(v.w);
  return f;
}

// The adapter of row m with its entry and the factor of its T; id -1 for none.
struct RowOf {
  int id;
  float coef;
  AdapterEntry e;
};
__device__ __forceinline__ RowOf resolve(const RowXaArgs& a, int m) {
  RowOf r = {-1, 0.0f, {}};
  if (m >= a.M) return r;
  const int id = a.ids[m];
  const float s = a.scale ? a.scale[m] : 1.0f;
  if (id < 0 || id >= a.cap || s == 0.0f) return r;
  r.e = a.table[id];
  if (r.e.r8 == 0) return r;
  r.id = id;
  r.coef = s * r.e.fold;
  return r;
}

// The 16-rank chunks of a block's rows in order: `visit(adapter, r8, A, first
// rank)`, all wave-uniform, out of what the lanes hold (a table read an adapter would
// be one memory latency each). T's columns past the rank, up to whole 32, are zeros:
// `zero(adapter, r8, first rank)` for a chunk that lies there.
template <class F, class Z>
__device__ __forceinline__ void each_chunk(const RowOf& row, F&& visit, Z&& zero) {
  uint64_t left = __ballot(row.id >= 0);
  const uint64_t p = (uint64_t)(uintptr_t)row.e.A;
  while (left) {
    const int w = __builtin_ctzll(left);
    const int cur = __builtin_amdgcn_readlane(row.id, w);
    left &= ~__ballot(row.id == cur);
    const int r8 = __builtin_amdgcn_readlane(row.e.r8, w);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)p, w);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), w);
    const uint4* const A = reinterpret_cast<const uint4*>((uintptr_t)(hi << 32 | lo));
    for (int ch = 0; ch < r8; ch += 16) visit(cur, r8, A, ch);
    if ((r8 + 15 & ~15) & 16) zero(cur, r8, r8 + 15 & ~15);
  }
}

// T's columns ch + 4g .. + 3 of row m from four sums.
__device__ __forceinline__ void store_t(const RowXaArgs& a, int m, float coef, int r8, int r0,
                                        const floatx4_t& v) {
  uint2 o = make_uint2(0, 0);
  if (r0 < r8) {                             // r8 is a multiple of 8, r0 of 4
    o.x = pack_bf16x2_rne(coef * v[0], coef * v[1]);
    o.y = pack_bf16x2_rne(coef * v[2], coef * v[3]);
  }
  *reinterpret_cast<uint2*>(a.t + (long long)m * a.ldt + r0) = o;
}

// Where a lane reads a chunk's operand (16-byte units of the resident order, half h
// of 64-group kt at + 64 (2 kt + h)). Lanes past the rank read the last one's, which
// costs no memory; store_t writes zeros for them.
__device__ __forceinline__ const uint4* chunk_lane(const uint4* A, int r8, int K, int ch, int lane) {
  const int c = lane & 15, last = r8 - 1 - ch;
  return A + (long long)(ch / 16) * (K / 32) * 64 + (lane & 48) + (c < last ? c : last);
}

__device__ __forceinline__ floatx4_t mfma_rows(const uint4& w, const uint4& x, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w),
                                                 __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
}

// Block (bx, by) of ny over 16 rows, XW waves.
template <int XW>
__device__ __forceinline__ void row_xa_block(const RowXaArgs& a, int bx, int by, int ny,
                                             floatx4_t (*red)[64]) {
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int m0 = bx * 16, m = m0 + c;
  const int KT = a.K / 64;
  constexpr int U = 8;                       // 64-groups of a wave at once
  const uint16_t* const xr = a.x + (long long)(m < a.M ? m : a.M - 1) * a.ldx + 8 * g;
  uint4 xv[U][2];
  auto load_x = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kt = k0 + XW * u < KT ? k0 + XW * u : KT - 1;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        xv[u][h] = *reinterpret_cast<const uint4*>(xr + 64 * kt + 32 * h);
    }
  };
  const bool whole = KT <= XW * U;           // x fits the registers
  if (whole) load_x(wave);                   // (while the adapters are looked up)
  const RowOf row = resolve(a, m);           // the wave's quarters hold the same rows
  if (by == 0 && wave == 0 && lane < 16 && m < a.M) a.rid[m] = row.id;
  if (a.xh) {
    // the fp16 copy of the block's rows, grid y sharing out the columns
    const int k8 = a.K / 8, c0 = k8 * by / ny;
    const int c1 = k8 * (by + 1) / ny;
    uint32_t seen = 0;
    for (int r = wave; r < 16 && m0 + r < a.M; r += XW)
      for (int k = c0 + lane; k < c1; k += 64) {
        const uint4 v = *reinterpret_cast<const uint4*>(a.x + (long long)(m0 + r) * a.ldx + 8 * k);
        *reinterpret_cast<uint4*>(a.xh + (long long)(m0 + r) * a.K + 8 * k) = to_f16(v, seen);
      }
    range_report(a.range, seen);
  }
  struct Held {
    int id, r8, ch;
  };
  auto load_a = [&](uint4 (&av)[U][2], const uint4* ar, int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kt = k0 + XW * u < KT ? k0 + XW * u : KT - 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) av[u][h] = ar[64 * (2 * kt + h)];
    }
  };
  auto sums = [&](const uint4 (&av)[U][2], int k0, floatx4_t& acc) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + XW * u < KT) {
#pragma unroll
        for (int h = 0; h < 2; ++h) acc = mfma_rows(av[u][h], xv[u][h], acc);
      }
  };
  // barriers for LDS alone: the next chunk's operands stay in flight over them
  auto join = [&](const floatx4_t& acc, const Held& q) {
    red[wave][lane] = acc;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (wave == 0) {
      floatx4_t v = red[0][lane];
#pragma unroll
      for (int w = 1; w < XW; ++w) v += red[w][lane];
      if (row.id == q.id) store_t(a, m, row.coef, q.r8, q.ch + 4 * g, v);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  auto finish = [&](const uint4 (&av)[U][2], const Held& q) {
    floatx4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    sums(av, wave, acc);
    join(acc, q);
  };
  // T's columns past the rank, up to whole 32
  const int r16 = (row.e.r8 + 15) & ~15;
  if (by == 0 && wave == 0 && row.id >= 0 && (r16 & 16))
    store_t(a, m, 0.0f, row.e.r8, r16 + 4 * g, floatx4_t{0.0f, 0.0f, 0.0f, 0.0f});
  // this block's next chunk and where its operand lies
  uint64_t left = __ballot(row.id >= 0);
  const uint64_t p = (uint64_t)(uintptr_t)row.e.A;
  int skip = by, at = 0;                     // chunks of other blocks, then this adapter's
  auto next = [&](Held& q, const uint4*& ar) {
    while (left) {
      const int w = __builtin_ctzll(left);
      q.id = __builtin_amdgcn_readlane(row.id, w);
      q.r8 = __builtin_amdgcn_readlane(row.e.r8, w);
      const int n = (q.r8 + 15) / 16;
      if (at + skip >= n) {
        skip -= n - at;
        at = 0;
        left &= ~__ballot(row.id == q.id);
        continue;
      }
      q.ch = 16 * (at + skip);
      at += skip + 1;
      skip = ny - 1;
      const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)p, w);
      const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), w);
      ar = chunk_lane(reinterpret_cast<const uint4*>((uintptr_t)(hi << 32 | lo)), q.r8, a.K, q.ch,
                      lane);
      return true;
    }
    return false;
  };
  uint4 a0[U][2];
  Held q0, q1;
  const uint4* ar;
  if (!whole) {
    while (next(q0, ar)) {
      floatx4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int k0 = wave; k0 < KT; k0 += XW * U) {
        load_a(a0, ar, k0);
        load_x(k0);
        sums(a0, k0, acc);
      }
      join(acc, q0);
    }
    return;
  }
  // a chunk's operands in flight over the one before it
  if (!next(q0, ar)) return;
  load_a(a0, ar, wave);
  uint4 a1[U][2];
  while (true) {
    const bool more = next(q1, ar);
    if (more) load_a(a1, ar, wave);
    finish(a0, q0);
    if (!more) return;
    const bool again = next(q0, ar);
    if (again) load_a(a0, ar, wave);
    finish(a1, q1);
    if (!again) return;
  }
}

}  // namespace ming
