// The experts' products over many rows, w4 and w8 stacks: y[p] = x[row(p)] .
// W_e^T for the places p of every expert's group, plain or SwiGLU-gated, x as
// fp16 carrying bf16 values (exact inside fp16's range; rows that it cannot hold are
// marked, and reported by the tiles whose places name them) and every scale and bias
// exact in fp16.
//
// MFMA-bound over many rows an expert, HBM-bound (the weights, once) over few. A
// block is a tile of up to 256 places of one expert x 256 rows of its weights, 4
// wave64s that split the weights' rows, 64 each, so each weight is
// dequantized once: raw codes come to LDS by DMA beside the x tile and become
// fp16 fragments with packed-fp16 arithmetic in the step before their MFMAs
// (v_mfma_f32_32x32x16_f16). Gated, a wave's 64 rows are 32 of the gate and the
// same 32 of the up projection: both halves of an output are in one lane's
// registers. The rows of x are gathered by the DMA, whose lanes each carry an
// address of their own. Three LDS stages of 64 of K, one barrier a stage.
//
// The grid is an upper bound (the groups' sizes are on the device): a block
// finds its tile by find_group, the rest leave. Groups are cut every 64 to 256
// places; what is left of one runs at the height it needs. The lower cuts leave LDS
// and registers for two or three blocks a CU, which hide each other's barriers and
// starts and keep more of the weights in flight: experts_cut says which cut.
// [128][1024, 2048] w4 gated, 16384 places in uneven groups 85 to 95 us, by the card, groups
// of 128 61 to 65; [60][2048, 1024] w8, 1218 places 25.2, its weights at 5.6 TB/s.
#include "common.h"
#include "deq_frag.h"
#include "kernels.h"
#include "lds_ring.h"
#include "row_groups.h"

namespace ming {
namespace {

constexpr int QBN = 256, QBK = 64, NW = 4, JT = 2;

// The row of x at a place, inside x whatever the order says.
__device__ __forceinline__ int source_row(const ExpertsArgs& a, int place) {
  const int src = a.order ? a.order[place] / a.fan : place;
  return src < 0 ? 0 : src < a.x_rows ? src : a.x_rows - 1;
}

// One tile: places p0 .. p0 + rows - 1 of expert e, output columns from n0;
// st0..st2 the ring's stages.
template <int BITS, bool GATED, int RF, int PP>
__device__ __forceinline__ void experts_qtile(const ExpertsArgs& a, uint4* const st0,
                                              uint4* const st1, uint4* const st2, int e, int p0,
                                              int rows, int n0) {
  constexpr int WCH = BITS == 4 ? 512 : 1024;    // 16-B code chunks per stage
  constexpr int CPR = BITS == 4 ? 2 : 4;         // code chunks per row
  constexpr int WDMA = WCH / (64 * NW);          // code DMAs per wave per stage
  constexpr int BMT = 32 * RF;
  constexpr int XD = 4 * RF / NW;                // x DMAs per wave per stage
  constexpr int PER = XD + WDMA + 1;             // DMAs per wave per stage

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 31, fk = lane >> 5;
  const int KT = a.K / QBK;
  const _Float16* const x16 = reinterpret_cast<const _Float16*>(a.x);
  const uint4* const codes = reinterpret_cast<const uint4*>(a.codes) +
                             (long long)e * a.NW * a.K * BITS / 128;
  const uint32_t* const sbp = a.sb + (long long)e * a.NW * KT;
  // the weight row that tile row r holds; columns past N hold the last one's
  auto wrow = [&](int r) {
    int n = GATED ? n0 + 32 * (r >> 6) + (r & 31) : n0 + r;
    n = n < a.N ? n : a.N - 1;
    return GATED && (r & 32) ? n + a.N : n;
  };

  uint32_t xoff[XD], woff[WDMA];
#pragma unroll
  for (int i = 0; i < XD; ++i) {
    const int p = 64 * (XD * wave + i) + lane;
    const int row = p >> 3;
    const int c = (p & 7) ^ ((row >> 1) & 7);
    const int src = source_row(a, p0 + (row < rows ? row : rows - 1));
    xoff[i] = (uint32_t)(((long long)src * a.ldx + 8 * c) * 2);
  }
#pragma unroll
  for (int i = 0; i < WDMA; ++i) {
    const int p = 64 * (WDMA * wave + i) + lane;
    const int r = p / CPR;
    const int h = (p % CPR) ^ wswz<CPR>(r);
    woff[i] = (uint32_t)((wrow(r) * CPR + h) * 16);
  }
  const uint32_t soff = (uint32_t)wrow(64 * wave + lane) * 4u;

  // the stage's DMAs in three groups: the wave's x DMAs in two halves, then codes
  // and (s, b)
  auto issue_grp = [&](int g, int kt, const uint4* B) {
    if (g < 2) {
      const void* base = x16 + (long long)kt * QBK;
#pragma unroll
      for (int i = g ? XD / 2 : 0; i < (g ? XD : XD / 2); ++i)
        dma16_sb(base, xoff[i], lds_addr(B + 64 * (XD * wave + i)));
    } else {
      const void* wbase = codes + (long long)kt * a.NW * CPR;
#pragma unroll
      for (int i = 0; i < WDMA; ++i)
        dma16_sb(wbase, woff[i], lds_addr(B + BMT * 8 + 64 * (WDMA * wave + i)));
      dma4_sb(sbp + (long long)kt * a.NW, soff,
              lds_addr(reinterpret_cast<const uint32_t*>(B + BMT * 8 + WCH) + 64 * wave));
    }
  };

  floatx16_t acc[JT][RF];
#pragma unroll
  for (int j = 0; j < JT; ++j)
#pragma unroll
    for (int i = 0; i < RF; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.0f;

  uint4 wc[JT][CPR / 2];
  half2v s2[JT], b2[JT];
  uint4 wa[JT], xb[RF];
  auto load_ws = [&](const uint4* B, uint4 (&wcv)[JT][CPR / 2], half2v (&s2v)[JT],
                     half2v (&b2v)[JT]) {
    const uint4* W = B + BMT * 8;
    const uint32_t* S = reinterpret_cast<const uint32_t*>(B + BMT * 8 + WCH);
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      const int n = 32 * JT * wave + 32 * j + fr;
#pragma unroll
      for (int h = 0; h < CPR / 2; ++h) wcv[j][h] = W[wchunk<CPR>(n, fk * (CPR / 2) + h)];
      const uint32_t sb = S[n];
      s2v[j] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(sb, sb, 0x01000100u));
      b2v[j] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(sb, sb, 0x03020302u));
    }
  };
  auto deq = [&](const uint4 (&wcv)[JT][CPR / 2], const half2v (&s2v)[JT],
                 const half2v (&b2v)[JT], int j, int kk) -> uint4 {
    if constexpr (BITS == 4) {
      return deq_w4((&wcv[j][0].x)[kk], s2v[j], b2v[j]);
    } else {
      const uint32_t* w = &wcv[j][kk >> 1].x;
      return deq_w8(w[(kk & 1) * 2], w[(kk & 1) * 2 + 1], s2v[j], b2v[j]);
    }
  };
  // One stage, pipelined across the stage boundary: steps 0-2 read and dequantize
  // the next step's fragments beside the step's MFMAs and issue a DMA group of
  // stage kt + 2 into the buffer stage kt - 1 left; the wait and the barrier sit
  // before step 3, whose MFMAs carry the next stage's first fragments.
  auto body = [&](int kt, const uint4* C, const uint4* Nx, const uint4* Pv) {
    const int nk = kt + 2 < KT ? kt + 2 : KT - 1;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint4 wn_[JT], xn_[RF];
      uint4 wcn[JT][CPR / 2];
      half2v s2n[JT], b2n[JT];
      if (kk < 3) {
        issue_grp(kk, nk, Pv);
#pragma unroll
        for (int i = 0; i < RF; ++i) xn_[i] = C[swz8(32 * i + fr, 2 * (kk + 1) + fk)];
#pragma unroll
        for (int j = 0; j < JT; ++j) wn_[j] = deq(wc, s2, b2, j, kk + 1);
      } else {
        load_ws(Nx, wcn, s2n, b2n);
#pragma unroll
        for (int i = 0; i < RF; ++i) xn_[i] = Nx[swz8(32 * i + fr, fk)];
#pragma unroll
        for (int j = 0; j < JT; ++j) wn_[j] = deq(wcn, s2n, b2n, j, 0);
      }
#pragma unroll
      for (int i = 0; i < RF; ++i)
#pragma unroll
        for (int j = 0; j < JT; ++j)
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              __builtin_bit_cast(half8_t, wa[j]), __builtin_bit_cast(half8_t, xb[i]), acc[j][i], 0,
              0, 0);
      if (kk < 3) {
#pragma unroll
        for (int g = 0; g < RF; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // DS read
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // MFMA
        }
#pragma unroll
        for (int g = 0; g < RF; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x002, (32 + RF - 1) / RF, 0);   // VALU
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                    // MFMA
        }
      } else {
        constexpr int NDS = RF + JT * (CPR / 2) + JT;
        constexpr int VG = RF == 8 && CPR == 2 ? RF + 2 : RF < 4 ? 1 : 3 * RF / 4;
        constexpr int VPG = RF == 8 && CPR == 2 ? 4 : 6;   // VALU per group
        constexpr int DSM = 2 * RF - VG;
        constexpr int DPM = NDS / DSM, XTRA = NDS - DPM * DSM;   // reads per MFMA
#pragma unroll
        for (int g = 0; g < XTRA; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x100, DPM + 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int g = XTRA; g < DSM; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x100, DPM, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
#pragma unroll
        for (int g = 0; g < VG; ++g) {
          __builtin_amdgcn_sched_group_barrier(0x002, VPG, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (kk == 2) {
        ring_wait<PER>();                        // stage kt + 1 landed, kt done
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < JT; ++j) wa[j] = wn_[j];
#pragma unroll
      for (int i = 0; i < RF; ++i) xb[i] = xn_[i];
      if (kk == 3) {
#pragma unroll
        for (int j = 0; j < JT; ++j) {
#pragma unroll
          for (int h = 0; h < CPR / 2; ++h) wc[j][h] = wcn[j][h];
          s2[j] = s2n[j];
          b2[j] = b2n[j];
        }
      }
    }
  };
#pragma unroll
  for (int g = 0; g < 3; ++g) issue_grp(g, 0, st0);
#pragma unroll
  for (int g = 0; g < 3; ++g) issue_grp(g, KT > 1 ? 1 : 0, st1);
  ring_wait<PER>();
  load_ws(st0, wc, s2, b2);
#pragma unroll
  for (int i = 0; i < RF; ++i) xb[i] = st0[swz8(32 * i + fr, fk)];
#pragma unroll
  for (int j = 0; j < JT; ++j) wa[j] = deq(wc, s2, b2, j, 0);
  int kt = 0;
  for (; kt + 3 <= KT; kt += 3) {
    body(kt, st0, st1, st2);
    body(kt + 1, st1, st2, st0);
    body(kt + 2, st2, st0, st1);
  }
  if (KT - kt >= 1) body(kt, st0, st1, st2);
  if (KT - kt == 2) body(kt + 1, st1, st2, st0);
  ring_wait<0>();                                // drained; LDS free

  // Epilogue through LDS, each wave in a region of its own, two a stage (its
  // accesses complete in order: no barrier): up to 128 rows of 64 columns at a
  // time plain, all rows of 32 gated, chunks swizzled so that both ways are
  // conflict-free, whole row segments stored.
  constexpr int CH = GATED ? 4 : 8;              // 16-B chunks of a row segment
  constexpr int PF = GATED ? 2 * PP : PP;        // fragments of a part
  uint4* const E = (wave < 2 ? st0 : st1) + 32 * PF * CH * (wave & 1);
  uint2* const E2 = reinterpret_cast<uint2*>(E);
  auto swz = [&](int ml, int c) { return GATED ? swz4(ml, c) : swz8(ml, c); };
  constexpr int LR = 64 / CH;                    // rows a store instruction covers
  const int cl = lane % CH;
  const int n = n0 + 8 * CH * wave + 8 * cl;
#pragma unroll
  for (int h = 0; h < (RF + PF - 1) / PF; ++h) {
    constexpr int F = RF < PF ? RF : PF;
    const int HF = RF - PF * h < PF ? RF - PF * h : PF;
#pragma unroll
    for (int ii = 0; ii < F; ++ii) {
      if (ii >= HF) continue;
      const int i = PF * h + ii;
      const int ml = 32 * ii + fr;
#pragma unroll
      for (int j = 0; j < (GATED ? 1 : JT); ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = acc[j][i][4 * q + k];
            if constexpr (GATED) v[k] = silu_f(v[k]) * acc[1][i][4 * q + k];
          }
          uint2 o;
          o.x = pack_bf16x2_rne(v[0], v[1]);
          o.y = pack_bf16x2_rne(v[2], v[3]);
          E2[2 * swz(ml, 4 * j + q) + fk] = o;
        }
    }
#pragma unroll
    for (int r = 0; r < 32 * F / LR; ++r) {
      const int ml = LR * r + lane / CH;
      const uint4 v = E[swz(ml, cl)];
      const int row = 32 * PF * h + ml;
      if (ml < 32 * HF && row < rows && n < a.N)
        *reinterpret_cast<uint4*>(a.y + (long long)(p0 + row) * a.ldy + n) = v;
    }
  }
}

// Groups of more than 32 * MAX places are cut into the fewest tiles that hold them.
template <int BITS, bool GATED, int MAX>
__global__ __launch_bounds__(64 * NW, MAX == 8 ? 1 : MAX == 2 && BITS == 4 ? 3 : 2)
void experts_qtile_kernel(const ExpertsArgs a) {
  constexpr int CUT = 32 * MAX;
  constexpr int BNT = GATED ? QBN / 2 : QBN;     // output columns of a tile
  constexpr int STG0 = CUT * 8 + (BITS == 4 ? 512 : 1024) + QBN / 4;
  // the epilogue's rows at a time (32 each): two regions a stage
  constexpr int PP = MAX == 8 ? 4 : 2;
  constexpr int EPI = 2 * 32 * PP * 8;
  constexpr int STG = STG0 < EPI ? EPI : STG0;
  __shared__ uint4 st0[STG], st1[STG], st2[STG];
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
  const RowTile rt = row_tile<MAX == 8 ? 64 : 32>(rg.rows, tiles_m, tm);
  const int p0 = rg.p0 + rt.first, rows = rt.rows, n0 = tn * BNT;
  [&] {
    if constexpr (MAX >= 8)
      if (rows > 192) return experts_qtile<BITS, GATED, 8, PP>(a, st0, st1, st2, rg.e, p0, rows, n0);
    if constexpr (MAX >= 8)
      if (rows > 128) return experts_qtile<BITS, GATED, 6, PP>(a, st0, st1, st2, rg.e, p0, rows, n0);
    if constexpr (MAX >= 4)
      if (rows > (MAX == 8 ? 64 : 96))
        return experts_qtile<BITS, GATED, 4, PP>(a, st0, st1, st2, rg.e, p0, rows, n0);
    if constexpr (MAX == 4)
      if (rows > 64) return experts_qtile<BITS, GATED, 3, PP>(a, st0, st1, st2, rg.e, p0, rows, n0);
    if constexpr (MAX < 8)
      if (rows <= 32) return experts_qtile<BITS, GATED, 1, PP>(a, st0, st1, st2, rg.e, p0, rows, n0);
    experts_qtile<BITS, GATED, 2, PP>(a, st0, st1, st2, rg.e, p0, rows, n0);
  }();
  // Rows of x that no place names may hold anything: a row is reported by the tiles
  // that multiply it, one in each row of them (a tile has at most a place a thread).
  const int place = (int)threadIdx.x;
  if (tn == 0 && place < rows && a.beyond[source_row(a, p0 + place)] && a.range) *a.range = 1;
}

// x as fp16, and a byte a row: whether it holds a magnitude of 2^16 or more, inf or
// NaN. L lanes (a power of two, at most a wave) a row, 16 bytes a lane and step.
__global__ __launch_bounds__(256) void experts_f16_kernel(const uint16_t* __restrict__ x,
                                                          long long ldx, int rows, int K, int L,
                                                          uint16_t* __restrict__ y,
                                                          uint8_t* __restrict__ beyond) {
  const int lane = (int)threadIdx.x & 63, sub = lane & (L - 1);
  const long long r = (long long)blockIdx.x * (256 / L) + (int)threadIdx.x / L;
  if (r >= rows) return;
  uint32_t seen = 0;
  for (int k0 = 8 * sub; k0 < K; k0 += 32 * L) {
    uint4 v[4];                              // in flight together
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + 8 * L * u;
      if (k < K) v[u] = *reinterpret_cast<const uint4*>(x + r * ldx + k);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + 8 * L * u;
      if (k >= K) continue;
      seen = range_track4(seen, v[u]);
      *reinterpret_cast<uint4*>(y + r * K + k) =
          make_uint4(bf16x2_to_f16x2(v[u].x), bf16x2_to_f16x2(v[u].y), bf16x2_to_f16x2(v[u].z),
                     bf16x2_to_f16x2(v[u].w));
    }
  }
  const uint64_t all = __ballot(range_beyond(seen)) >> (lane & ~(L - 1));
  if (sub == 0) beyond[r] = (all & (~0ull >> (64 - L))) != 0;
}

// The taller cut of each type.
constexpr int tall(int bits) { return bits == 4 ? 4 : 8; }

template <int BITS, bool GATED>
void launch_max(const ExpertsArgs& a, int max, hipStream_t s) {
  const dim3 grid((unsigned)experts_tiles(BITS, GATED, max, a.n, a.E, a.N));
  if (max == 2)
    hipLaunchKernelGGL((experts_qtile_kernel<BITS, GATED, 2>), grid, dim3(64 * NW), 0, s, a);
  else
    hipLaunchKernelGGL((experts_qtile_kernel<BITS, GATED, tall(BITS)>), grid, dim3(64 * NW), 0, s,
                       a);
}

}  // namespace

hipError_t launch_experts_qtile(int bits, bool gated, const ExpertsArgs& a, int max,
                                hipStream_t s) {
  if (a.n <= 0 || a.N <= 0) return hipSuccess;
  if (a.K % 64 || a.N % 8 || a.NW != a.N * (gated ? 2 : 1) || a.E < 1 || a.fan < 1 ||
      a.x_rows < 1 || a.ldy % 8 || !a.beyond || (bits != 4 && bits != 8) ||
      (max != 2 && max != tall(bits)))
    return hipErrorInvalidValue;
  if (bits == 4)
    gated ? launch_max<4, true>(a, max, s) : launch_max<4, false>(a, max, s);
  else
    gated ? launch_max<8, true>(a, max, s) : launch_max<8, false>(a, max, s);
  return hipGetLastError();
}

hipError_t launch_experts_f16(const uint16_t* x, long long ldx, int rows, int K, uint16_t* y,
                              uint8_t* beyond, hipStream_t s) {
  if (rows <= 0) return hipSuccess;
  if (K < 64 || K % 64 || ldx % 8) return hipErrorInvalidValue;
  int L = 8;
  while (L < 64 && 16 * L <= K) L *= 2;
  const int rpb = 256 / L;
  hipLaunchKernelGGL(experts_f16_kernel, dim3((unsigned)((rows + (long long)rpb - 1) / rpb)),
                     dim3(256), 0, s, x, ldx, rows, K, L, y, beyond);
  return hipGetLastError();
}

hipError_t validate_experts_qtile_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {reinterpret_cast<const void*>(&experts_f16_kernel),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<4, false, 2>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<4, true, 2>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<8, false, 2>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<8, true, 2>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<4, false, 4>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<4, true, 4>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<8, false, 8>),
                       reinterpret_cast<const void*>(&experts_qtile_kernel<8, true, 8>)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
