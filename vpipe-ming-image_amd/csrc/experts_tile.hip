// The experts' products over many rows, dense bf16 weights: y[p] = x[row(p)] .
// W_e^T for the places p of every expert's group, plain or SwiGLU-gated.
//
// MFMA-bound. A block is a tile of 64*RF places of one expert x 256 rows of its
// weights: 8 wave64s in 2 x 4, each 32*RF places x 64 weight rows (2 x RF tiles
// of v_mfma_f32_32x32x16_bf16). Gated, a wave's 64 weight rows are 32 of the gate
// and the same 32 of the up projection, so both halves of an output are in one
// lane's registers and the SwiGLU costs no exchange: 128 columns a tile. The
// rows of x are gathered by the DMA itself, whose lanes each carry an address
// of their own. K runs in stages of 64 through an LDS ring filled by direct
// global->LDS DMA, one barrier a stage before its last k16 step; three stages
// where they fit (RF <= 2), else five 32 KB slots taken by x and W tiles in
// turn, so that x runs three stages ahead and W two.
//
// The grid is an upper bound (the groups' sizes are on the device): a block
// finds its tile by find_group, the rest leave. An XCD takes a contiguous range
// of tiles, an expert's columns outermost, so its L2 holds the weights in use.
// [64][2048, 2048] gated: 32768 places in groups of 512, 234 us (1177 TFLOP/s); 34816
// in uneven ones 294 to 308, by the card (matrix pipes 53% busy, 1.0 GB past the L2s).
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "lds_ring.h"
#include "row_groups.h"

namespace ming {
namespace {

constexpr int TBN = 256, TBK = 64, NW = 8;

// One tile: places p0 .. p0 + rows - 1 of expert e, output columns from n0.
template <int RF, bool GATED>
__device__ __forceinline__ void experts_tile(const ExpertsArgs& a, uint4* const ring, int e, int p0,
                                             int rows, int n0) {
  constexpr int BMT = 64 * RF;
  constexpr int XD = 8 * RF / NW, WD = 32 / NW;    // DMAs per wave per stage
  constexpr int JF = 2;                            // weight fragments per wave
  constexpr bool FIVE = RF >= 3;
  constexpr int XCH = BMT * 8, WCH = TBN * 8;      // 16-B chunks of the tiles
  constexpr int PERIOD = FIVE ? 5 : 3;
  auto xslot = [&](int ph) -> const uint4* {
    return FIVE ? ring + ((2 * ph) % 5) * WCH : ring + (ph % 3) * (XCH + WCH);
  };
  auto wslot = [&](int ph) -> const uint4* {
    return FIVE ? ring + ((2 * ph + 1) % 5) * WCH : ring + (ph % 3) * (XCH + WCH) + XCH;
  };
  constexpr int WAHEAD = FIVE ? 2 : 3;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 31, fk = lane >> 5;
  const int wm = wave & 1, wn = wave >> 1;

  const uint16_t* const w16 = a.w16 + (long long)e * a.NW * a.K;
  const int KT = a.K / TBK;

  // LDS chunk p of a tile holds row p >> 3, logical chunk (p & 7) ^ swizzle.
  auto chunk_of = [&](int p) { return (p & 7) ^ (((p >> 3) >> 1) & 7); };
  uint32_t xoff[XD], woff[WD];
#pragma unroll
  for (int i = 0; i < XD; ++i) {
    const int p = 64 * (XD * wave + i) + lane;
    const int r = (p >> 3) < rows ? (p >> 3) : rows - 1;
    int src = p0 + r;
    if (a.order) src = a.order[src] / a.fan;
    src = src < 0 ? 0 : src < a.x_rows ? src : a.x_rows - 1;
    xoff[i] = (uint32_t)(((long long)src * a.ldx + 8 * chunk_of(p)) * 2);
  }
#pragma unroll
  for (int i = 0; i < WD; ++i) {
    const int p = 64 * (WD * wave + i) + lane;
    const int r = p >> 3;
    int n = GATED ? n0 + 32 * (r >> 6) + (r & 31) : n0 + r;
    n = n < a.N ? n : a.N - 1;
    if (GATED && (r & 32)) n += a.N;
    woff[i] = (uint32_t)((n * 64 + 8 * chunk_of(p)) * 2);
  }

  floatx16_t acc[JF][RF];
#pragma unroll
  for (int j = 0; j < JF; ++j)
#pragma unroll
    for (int i = 0; i < RF; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.0f;

  uint4 wa[JF], xb[RF];
  auto read_frags = [&](const uint4* X, const uint4* W, int kk, uint4 (&av)[JF],
                        uint4 (&bv)[RF]) {
    const int c = 2 * kk + fk;
#pragma unroll
    for (int j = 0; j < JF; ++j) av[j] = W[swz8(32 * JF * wn + 32 * j + fr, c)];
#pragma unroll
    for (int i = 0; i < RF; ++i) bv[i] = X[swz8(32 * RF * wm + 32 * i + fr, c)];
  };
  // Past the last stage the DMA re-reads it into a tile nothing reads, so every
  // stage issues and waits alike.
  auto issue_w = [&](int t, const uint4* S) {
    const void* base = w16 + (long long)(t < KT ? t : KT - 1) * a.NW * TBK;
#pragma unroll
    for (int i = 0; i < WD; ++i) dma16_sb(base, woff[i], lds_addr(S + 64 * (WD * wave + i)));
  };
  auto issue_x = [&](int t, const uint4* S, int h) {
    const void* base = a.x + (long long)(t < KT ? t : KT - 1) * TBK;
#pragma unroll
    for (int i = h ? XD / 2 : 0; i < (h ? XD : XD / 2); ++i)
      dma16_sb(base, xoff[i], lds_addr(S + 64 * (XD * wave + i)));
  };
  auto body = [&](auto ph, int t) {
    constexpr int PH = decltype(ph)::value;
    const uint4 *const X = xslot(PH), *const W = wslot(PH);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint4 an[JF], bn[RF];
      if (kk < 2) issue_x(t + 2, xslot((PH + 2) % PERIOD), kk);   // freed by stage t - 1
      if (kk == 3) issue_w(t + WAHEAD, wslot((PH + WAHEAD) % PERIOD));
      if (kk < 3) {
        read_frags(X, W, kk + 1, an, bn);
      } else {
        read_frags(xslot((PH + 1) % PERIOD), wslot((PH + 1) % PERIOD), 0, an, bn);
      }
#pragma unroll
      for (int i = 0; i < RF; ++i)
#pragma unroll
        for (int j = 0; j < JF; ++j)
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8_t, wa[j]), __builtin_bit_cast(bf16x8_t, xb[i]),
              acc[j][i], 0, 0, 0);
      constexpr int DPM = JF * RF >= JF + RF ? 1 : 2;
#pragma unroll
      for (int g = 0; g < (JF + RF + DPM - 1) / DPM; ++g) {
        __builtin_amdgcn_sched_group_barrier(0x100, DPM, 0);   // DS read
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);     // MFMA
      }
      __builtin_amdgcn_sched_barrier(0);
      if (kk == 2) {
        // stage t + 1 landed; newer: x of stage t + 2 (and W, three stages)
        ring_wait<XD + (FIVE ? 0 : WD)>();
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < JF; ++j) wa[j] = an[j];
#pragma unroll
      for (int i = 0; i < RF; ++i) xb[i] = bn[i];
    }
  };
  const std::integral_constant<int, 0> ph0{};
  const std::integral_constant<int, 1> ph1{};
  const std::integral_constant<int, 2> ph2{};
  issue_w(0, wslot(0));
  issue_x(0, xslot(0), 0);
  issue_x(0, xslot(0), 1);
  issue_x(1, xslot(1), 0);
  issue_x(1, xslot(1), 1);
  issue_w(1, wslot(1));
  if constexpr (!FIVE) issue_w(2, wslot(2));
  // stage 0 landed; newer: stage 1 (and W of stage 2)
  ring_wait<XD + (FIVE ? WD : 2 * WD)>();
  read_frags(xslot(0), wslot(0), 0, wa, xb);
  int t = 0;
  for (; t + PERIOD <= KT; t += PERIOD) {
    body(ph0, t);
    body(ph1, t + 1);
    body(ph2, t + 2);
    if constexpr (FIVE) {
      body(std::integral_constant<int, 3>{}, t + 3);
      body(std::integral_constant<int, 4>{}, t + 4);
    }
  }
  if (KT - t >= 1) body(ph0, t);
  if (KT - t >= 2) body(ph1, t + 1);
  if constexpr (FIVE) {
    if (KT - t >= 3) body(ph2, t + 2);
    if (KT - t >= 4) body(std::integral_constant<int, 3>{}, t + 3);
  }
  ring_wait<0>();                          // drained; LDS free

  // Epilogue through LDS, each wave in a region of its own (its LDS accesses
  // complete in order: no barrier): whole row segments leave, 64 columns a row
  // plain and 32 gated, chunks swizzled so that both ways are conflict-free.
  constexpr int RROWS = 32 * RF;
  constexpr int CH = GATED ? 4 : 8;        // 16-B chunks of a row segment
  uint4* const E = ring + (RROWS * CH) * wave;
  uint2* const E2 = reinterpret_cast<uint2*>(E);
  auto swz = [&](int ml, int c) { return GATED ? swz4(ml, c) : swz8(ml, c); };
  // the lane anew, so that nothing of it stays in a register across the loop
  // (the 256-row tile has none to spare)
  int el;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(el));
  const int er = el & 31, ek = el >> 5;
#pragma unroll
  for (int j = 0; j < (GATED ? 1 : 2); ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < RF; ++i) {
        const int ml = 32 * i + er;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = acc[j][i][4 * q + k];
          if constexpr (GATED) v[k] = silu_f(v[k]) * acc[1][i][4 * q + k];
        }
        uint2 o;
        o.x = pack_bf16x2_rne(v[0], v[1]);
        o.y = pack_bf16x2_rne(v[2], v[3]);
        E2[2 * swz(ml, 4 * j + q) + ek] = o;
      }
  constexpr int LR = 64 / CH;              // rows a store instruction covers
  const int cl = el % CH;
  const int n = n0 + 8 * CH * wn + 8 * cl;
#pragma unroll
  for (int r = 0; r < RROWS / LR; ++r) {
    const int ml = LR * r + el / CH;
    const uint4 v = E[swz(ml, cl)];
    const int row = RROWS * wm + ml;
    if (row < rows && n < a.N)
      *reinterpret_cast<uint4*>(a.y + (long long)(p0 + row) * a.ldy + n) = v;
  }
}

// Groups of more than 64 * MAX places are cut into the fewest tiles that hold them.
template <int MAX, bool GATED>
__global__ __launch_bounds__(64 * NW, 1) void experts_tile_kernel(const ExpertsArgs a) {
  constexpr int CUT = 64 * MAX;
  constexpr int BNT = GATED ? TBN / 2 : TBN;       // output columns of a tile
  __shared__ uint4 ring[MAX >= 3 ? 5 * TBN * 8 : 3 * (CUT + TBN) * 8];
  const int tiles_n = (a.N + BNT - 1) / BNT;
  const RowGroup rg = find_group(
      a.offsets, a.E, a.n, [&](int rows) { return (rows + CUT - 1) / CUT * tiles_n; },
      [&](int total) {
        const int b = (int)blockIdx.x, q = total / 8, rem = total % 8, xcd = b % 8;
        return b < total ? xcd * q + (xcd < rem ? xcd : rem) + b / 8 : -1;
      });
  if (rg.e < 0) return;
  const int tiles_m = (rg.rows + CUT - 1) / CUT;
  const int tn = rg.index / tiles_m, tm = rg.index - tn * tiles_m;
  const RowTile rt = row_tile<64>(rg.rows, tiles_m, tm);
  const int p0 = rg.p0 + rt.first, rows = rt.rows, n0 = tn * BNT;
  if constexpr (MAX >= 4)
    if (rows > 192) return experts_tile<4, GATED>(a, ring, rg.e, p0, rows, n0);
  if constexpr (MAX >= 3)
    if (rows > 128) return experts_tile<3, GATED>(a, ring, rg.e, p0, rows, n0);
  if (rows > 64)
    experts_tile<2, GATED>(a, ring, rg.e, p0, rows, n0);
  else
    experts_tile<1, GATED>(a, ring, rg.e, p0, rows, n0);
}

template <int MAX>
void launch_max(bool gated, const ExpertsArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)experts_tiles(16, gated, MAX, a.n, a.E, a.N));
  if (gated)
    hipLaunchKernelGGL((experts_tile_kernel<MAX, true>), grid, dim3(64 * NW), 0, s, a);
  else
    hipLaunchKernelGGL((experts_tile_kernel<MAX, false>), grid, dim3(64 * NW), 0, s, a);
}

}  // namespace

hipError_t launch_experts_tile(bool gated, const ExpertsArgs& a, int max, hipStream_t s) {
  if (a.n <= 0 || a.N <= 0) return hipSuccess;
  if (a.K % 64 || a.N % 8 || a.NW != a.N * (gated ? 2 : 1) || a.E < 1 || a.fan < 1 ||
      a.x_rows < 1 || a.ldy % 8)
    return hipErrorInvalidValue;
  switch (max) {
    case 2: launch_max<2>(gated, a, s); break;
    case 4: launch_max<4>(gated, a, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t validate_experts_tile_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {reinterpret_cast<const void*>(&experts_tile_kernel<2, false>),
                       reinterpret_cast<const void*>(&experts_tile_kernel<4, false>),
                       reinterpret_cast<const void*>(&experts_tile_kernel<2, true>),
                       reinterpret_cast<const void*>(&experts_tile_kernel<4, true>)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
