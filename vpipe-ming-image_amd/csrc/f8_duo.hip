// The 8-bit products of some hundred rows: 64 x 128 tiles whose two halves of four
// waves take the blocks of K in turn, so that a tile is done in half the steps where
// there are too few tiles to fill the chip (plain projections; f8_tile.hip has the rest).
//
// Bound by a stage's latencies: barrier, LDS reads and the DMAs' issue, not by the matrix
// cores. A stage is two blocks of K, one a half, through an LDS ring filled by direct
// global->LDS DMA; a wave takes 32 rows x 64 columns of its half's block, its next
// operands read from LDS under this stage's matrix instructions, one barrier a stage.
// The halves' f32 sums meet in LDS at the end. Where even that leaves most CUs idle over a
// long K, slices of K go to workgroups of their own and meet in f32 in memory.
//
// Measured out of cold caches: 203 x [2560, 10240] 17.8 us in slices (28.3 in one; the
// few-row kernel 28, tiles of 64 rows 43.6), 13.5 x [3840, 3840], 1024 rows 22.3 (1350
// TFLOP/s). A stage of two blocks is 0.53 us a workgroup out of L2, 0.7 out of memory, after
// a start of 3.2 that fills the ring at 107 GB/s a CU; with the weights' scales by DMA that
// start is 2.7, and the first stage lands as much later.
#include <type_traits>

#include "common.h"
#include "f8.h"
#include "kernels.h"
#include "lds_ring.h"

namespace ming {
namespace {

constexpr int DBN = 128, NW = 8;

constexpr int BM = 64, NST = 3, MF = 2, NF = 4;
constexpr int kX = BM * 8, kW = DBN * 8, kS = BM / 4;            // 16-byte units
constexpr int kHalf = kX + kW + kS, kStage = 2 * kHalf;
constexpr int XD = 2, WD = 4, kDma = XD + WD + 1;                 // DMAs a wave and stage

template <bool SPLIT>
__global__ __launch_bounds__(64 * NW, 1) void f8_duo_kernel(const F8Args a, int slices) {
  __shared__ uint4 ring[NST * kStage + kF8TileBlocks / 4 + 1];
  float* const wsc = reinterpret_cast<float*>(ring + NST * kStage);

  const int tid = (int)threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = wave >> 2, gw = wave & 3, wm = gw & 1, wn = gw >> 1;

  const int tiles_m = (a.n + BM - 1) / BM;
  const int tiles = tiles_m * (a.NR / DBN), slice = SPLIT ? (int)blockIdx.x / tiles : 0;
  int tm, tn;
  tile_of_block((int)blockIdx.x - slice * tiles, tiles_m, a.NR / DBN, &tm, &tn);
  const int p0 = BM * tm, rows = a.n - p0 < BM ? a.n - p0 : BM;
  // blocks kb0 .. KB - 1 of K
  const int kb0 = SPLIT ? (int)((long long)a.KB * slice / slices) : 0;
  const int KB = SPLIT ? (int)((long long)a.KB * (slice + 1) / slices) : a.KB;
  const int stages = (KB - kb0 + 1) / 2;

  auto source = [&](int r) { return r < rows ? r : rows - 1; };
  auto chunk_of = [&](int p) { return (p & 7) ^ ((p >> 4) & 7); };
  uint32_t xrow[XD];
#pragma unroll
  for (int i = 0; i < XD; ++i)
    xrow[i] = (uint32_t)(source((64 * (XD * gw + i) + lane) >> 3) * (long long)a.ldx);
  // a lane's MF rows of a wave's 16 MF lie side by side: dword c * MF + i is row 16 i + c
  const int si = lane % (16 * MF);
  const uint32_t soff = 2u * (uint32_t)source(lane - si + 16 * (si % MF) + si / MF);
  // chunks of the last block
  const int klast = KB == a.KB ? (a.K - 128 * (KB - 1)) / 16 : 8;

  // The DMAs of the half's next block, one at a time. Past the last block it is read again:
  // an odd count's last stage multiplies it by a scale of 0 in the second half, and the
  // slots behind are not multiplied.
  int kb = kb0 + half < KB ? kb0 + half : KB - 1;
  const uint8_t* xnext = a.x + (long long)p0 * a.ldx + kb * 128ll;
  const uint8_t* wnext = a.w + ((long long)kb * a.NR + (long long)tn * DBN) * 128 + gw * 4096;
  const uint16_t* snext = a.xs + p0 + kb * a.ldxs;
  auto issue = [&](int q, const uint4* S) {
    if (q < XD) {
      // past K the weights are zeros: any chunk of x's own block will do
      const int ch = chunk_of(64 * (XD * gw + q) + lane), cut = kb == KB - 1 ? klast : 8;
      dma16_sb(xnext, xrow[q] + (ch < cut ? 16 * ch : 0), lds_addr(S + 64 * (XD * gw + q)));
    } else if (q < XD + WD) {
      const uint32_t to = lds_addr(S + kX + 256 * gw), off = (uint32_t)(16 * lane);
      switch (q - XD) {
        case 0: dma16_off<0>(wnext, off, to); break;
        case 1: dma16_off<1024>(wnext, off, to); break;
        case 2: dma16_off<2048>(wnext, off, to); break;
        default: dma16_off<3 * 1024>(wnext, off, to); break;
      }
    } else {
      dma2_sb(snext, soff, lds_addr(S + kX + kW));
      const int next = kb + 2 < KB ? kb + 2 : KB - 1, by = next - kb;
      kb = next;
      xnext += by * 128;
      wnext += by * (a.NR * 128ll);
      snext += by * a.ldxs;
    }
  };

  for (int k = tid; k < 2 * stages; k += 64 * NW)
    wsc[k] = kb0 + k < KB ? a.ws[(long long)(kb0 + k) * a.NB + tn] : 0.0f;

  floatx4_t acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};

  const int fx = (32 * wm + c) * 8 + (g ^ (c >> 1)), fw = 512 * wn + lane;
  struct Operands {
    F8Frag w[NF], x[MF];
    uint32_t sx[MF];
    float sw;
  };
  auto read = [&](const uint4* S, int t, Operands& o) {
#pragma unroll
    for (int j = 0; j < NF; ++j)
      o.w[j] = F8Frag{S[kX + fw + 128 * j], S[kX + fw + 128 * j + 64]};
#pragma unroll
    for (int i = 0; i < MF; ++i) o.x[i] = F8Frag{S[fx + 128 * i], S[(fx ^ 4) + 128 * i]};
    const uint32_t* p =
        reinterpret_cast<const uint32_t*>(S + kX + kW) + 16 * MF * wm + MF * c;
#pragma unroll
    for (int i = 0; i < MF; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + i);
      o.sx[i] = v.x;
      o.sx[i + 1] = v.y;
    }
    o.sw = wsc[2 * t + half];
  };
  const uint4* const base = ring + half * kHalf;
  Operands cur, nxt;
  // Stage t's slot is free after the barrier (its operands are in registers), and stage
  // t + 1 has landed.
  auto body = [&](auto ph, int t, Operands& now, Operands& then) {
    constexpr int PH = decltype(ph)::value;
    const uint4 *const S = base + PH * kStage, *const Sn = base + (PH + 1) % NST * kStage;
    ring_wait<(NST - 2) * kDma>();
    __builtin_amdgcn_sched_barrier(0);
    read(Sn, t + 1 < stages ? t + 1 : t, then);
    float s[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
      // (not a product by the 0 of a block behind the last: x's scale may be inf)
      s[i] = kb0 + 2 * t + half < KB ? __uint_as_float(now.sx[i] << 16) * now.sw : 0.0f;
    floatx4_t dp[NF];
    constexpr int kEach = (kDma + MF - 1) / MF;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
      for (int q = i * kEach; q < (i + 1) * kEach && q < kDma; ++q) issue(q, S);
      floatx4_t d[NF];
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        d[j] = f8_mfma(now.w[j], now.x[i]);
        if (i > 0) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][i - 1][r] = fmaf(dp[j][r], s[i - 1], acc[j][i - 1][r]);
        }
      }
#pragma unroll
      for (int j = 0; j < NF; ++j) dp[j] = d[j];
    }
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[j][MF - 1][r] = fmaf(dp[j][r], s[MF - 1], acc[j][MF - 1][r]);
    __builtin_amdgcn_sched_barrier(0);
  };

#pragma unroll
  for (int t = 0; t < NST; ++t)
#pragma unroll
    for (int q = 0; q < kDma; ++q) issue(q, base + t * kStage);
  ring_wait<(NST - 1) * kDma>();           // stage 0 landed, the scales written
  read(base, 0, cur);
  const std::integral_constant<int, 0> p0c{};
  const std::integral_constant<int, 1> p1c{};
  const std::integral_constant<int, 2> p2c{};
  int t = 0;
  for (; t + 6 <= stages; t += 6) {
    body(p0c, t, cur, nxt);
    body(p1c, t + 1, nxt, cur);
    body(p2c, t + 2, cur, nxt);
    body(p0c, t + 3, nxt, cur);
    body(p1c, t + 4, cur, nxt);
    body(p2c, t + 5, nxt, cur);
  }
  if (stages - t >= 1) body(p0c, t, cur, nxt);
  if (stages - t >= 2) body(p1c, t + 1, nxt, cur);
  if (stages - t >= 3) body(p2c, t + 2, cur, nxt);
  if (stages - t >= 4) body(p0c, t + 3, nxt, cur);
  if (stages - t >= 5) body(p1c, t + 4, cur, nxt);
  ring_wait<0>();                          // drained; LDS free

  // the second half's sums to the first, then its rows through LDS in whole pieces
  floatx4_t* const meet = reinterpret_cast<floatx4_t*>(ring) + gw * (NF * MF * 64) + lane;
  if (half == 1) {
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int i = 0; i < MF; ++i) meet[(j * MF + i) * 64] = acc[j][i];
  }
  __syncthreads();
  if (half == 1) return;
  if constexpr (SPLIT) {
    // whole tiles in the accumulators' order, 1 KB a store
    floatx4_t* const out =
        reinterpret_cast<floatx4_t*>(a.part) +
        (((long long)slice * tiles_m + tm) * (a.NR / DBN) + tn) * (BM * DBN / 4) +
        gw * (NF * MF * 64) + lane;
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int i = 0; i < MF; ++i)
        out[(j * MF + i) * 64] = acc[j][i] + meet[(j * MF + i) * 64];
    return;
  }
  uint4* const E = ring + 4 * NF * MF * 64 + 32 * 8 * gw;
  uint2* const E2 = reinterpret_cast<uint2*>(E);
  const int nb = DBN * tn + 64 * wn;
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    floatx4_t b = {0.0f, 0.0f, 0.0f, 0.0f};
    const int n = nb + 16 * j + 4 * g;
    if (a.bias && n < a.N) {
      const uint2 v = *reinterpret_cast<const uint2*>(a.bias + n);
      b = floatx4_t{bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y)};
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int row = 16 * i + c;
      const floatx4_t v = acc[j][i] + meet[(j * MF + i) * 64] + b;
      E2[(row * 8 + ((2 * j + (g >> 1)) ^ ((row >> 1) & 7))) * 2 + (g & 1)] =
          make_uint2(pack_bf16x2_rne(v[0], v[1]), pack_bf16x2_rne(v[2], v[3]));
    }
  }
  const int cl = lane & 7, n = nb + 8 * cl;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int ml = 8 * k + (lane >> 3), row = 32 * wm + ml;
    const uint4 v = E[ml * 8 + (cl ^ ((ml >> 1) & 7))];
    if (row < rows && n < a.N)
      *reinterpret_cast<uint4*>(a.y + (long long)(p0 + row) * a.ldy + n) = v;
  }
}

// The slices' sums in their order, and the results: a workgroup a tile's two row
// fragments of f8_duo_kernel's four waves. 3.1 to 4.2 us at 203 x 2560 (three slices).
__global__ __launch_bounds__(256) void f8_join_kernel(const F8Args a, int slices) {
  const int lane = (int)threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int gw = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tiles_m = (a.n + BM - 1) / BM, tiles_n = a.NR / DBN;
  const int tile = (int)blockIdx.x / NF, j = (int)blockIdx.x - tile * NF, tn = tile % tiles_n;
  const int n = DBN * tn + 64 * (gw >> 1) + 16 * j + 4 * g;
  const long long plane = (long long)tiles_m * tiles_n * (BM * DBN / 4);
  const floatx4_t* p = reinterpret_cast<const floatx4_t*>(a.part) +
                       (long long)tile * (BM * DBN / 4) + (gw * NF + j) * (MF * 64) + lane;
  floatx4_t v[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) v[i] = p[64 * i];
  for (int s = 1; s < slices; ++s) {
    p += plane;
#pragma unroll
    for (int i = 0; i < MF; ++i) v[i] += p[64 * i];
  }
  if (n >= a.N) return;
  floatx4_t b = {0.0f, 0.0f, 0.0f, 0.0f};
  if (a.bias) {
    const uint2 u = *reinterpret_cast<const uint2*>(a.bias + n);
    b = floatx4_t{bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)};
  }
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int row = BM * (tile / tiles_n) + 32 * (gw & 1) + 16 * i + c;
    if (row >= a.n) continue;
    v[i] += b;
    *reinterpret_cast<uint2*>(a.y + (long long)row * a.ldy + n) =
        make_uint2(pack_bf16x2_rne(v[i][0], v[i][1]), pack_bf16x2_rne(v[i][2], v[i][3]));
  }
}

}  // namespace

hipError_t launch_f8_duo(const F8Args& a, int slices, hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  if (a.N <= 0 || a.N % 8 || a.K % 16 || a.KB > kF8TileBlocks || a.E != 1 || a.NR % DBN ||
      slices < 1 || slices > a.KB || (slices > 1 && !a.part))
    return hipErrorInvalidValue;
  const unsigned tiles = (unsigned)f8_duo_blocks(a.n, a.NR);
  if (slices == 1) {
    hipLaunchKernelGGL((f8_duo_kernel<false>), dim3(tiles), dim3(64 * NW), 0, s, a, 1);
  } else {
    hipLaunchKernelGGL((f8_duo_kernel<true>), dim3(tiles * (unsigned)slices), dim3(64 * NW), 0, s, a,
                       slices);
    hipLaunchKernelGGL(f8_join_kernel, dim3(tiles * NF), dim3(256), 0, s, a, slices);
  }
  return hipGetLastError();
}

hipError_t validate_f8_duo_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {reinterpret_cast<const void*>(&f8_duo_kernel<false>),
                       reinterpret_cast<const void*>(&f8_duo_kernel<true>),
                       reinterpret_cast<const void*>(&f8_join_kernel)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
