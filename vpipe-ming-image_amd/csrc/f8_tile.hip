// The 8-bit products over many rows, plain or SwiGLU-gated, of one projection or of a
// mixture's groups: y[m] = sum over blocks b of 128 of xs[b][m] * ws[n / 128][b] *
// (x . w)_b.
//
// MFMA-bound. A workgroup takes 64*RF rows x 256 rows of the resident weights (gated:
// 128 columns, whose gate and up rows lie side by side in eights of 32), 8 wave64s
// in 2 x 4, each 32*RF rows x 64 weight rows: 2*RF x 4 tiles of
// v_mfma_f32_16x16x128_f8f6f4. A stage is a block of 128 of K, so each instruction's
// result is a whole block's sum: it starts from zero, and four fused multiply-adds take
// it into the f32 accumulators times both scales, in the shadow of the next ones (16
// of 32 cycles). A lane's four results are four columns of one row, so a row's scale
// is one register a row tile, times the weights' one scale.
//
// Stages go through an LDS ring filled by direct global->LDS DMA (x in rows of 128 bytes,
// chunks swizzled; the weights as they lie), with the rows' scales; the weights' scales
// are all taken at the start. One barrier a stage, before its last two row tiles: their
// operands are in registers by then, so the slot is free for the DMA, and the next
// stage's first operands are read under their matrix instructions.
//
// Measured: 8704 x [3840, 10240] 280 to 290 us (2360 to 2440 TFLOP/s), x [10240, 3840]
// 288 to 295; 4352 rows gated [10240, 3840] 298 to 303 (2260 to 2300), 203 rows 26 to 27;
// 34816 places of [64][2048, 1024] 110 to 113 (1310, 2.8 TB/s), gated of [64][1024, 2048] 191
// (1530). A stage of 256 rows is 1.65 us, 2600 TFLOP/s over the chip: the power limit (the
// matrix instruction alone 3400, with the sums, LDS and DMA 2914). Around a tile's stages
// 0.9 us go to its start, 0.8 to the first stage's arrival, 3 to the results (gated 5) and
// 1.2 to the change of workgroups, which short K feels. v_mfma_f32_32x32x64 has half the
// operand reads but no registers left for the sums (2441 against 2914 in the same loop);
// an s_setprio around the barrier and a stage's lines touched one ahead changed nothing.
#include <type_traits>

#include "common.h"
#include "f8.h"
#include "kernels.h"
#include "lds_ring.h"
#include "row_groups.h"

namespace ming {
namespace {

constexpr int TBN = 256, NW = 8;

template <int RF>
struct TileLds {
  static constexpr int kStages = RF >= 3 ? 2 : 3;
  static constexpr int kX = 64 * RF * 8, kW = TBN * 8, kS = 16 * RF;   // 16-byte units
  static constexpr int kStage = kX + kW + kS;
  static constexpr int kUnits = kStages * kStage + kF8TileBlocks / 2;
};

// One tile: rows p0 .. p0 + rows - 1, resident weight rows from 256 * tn of expert e.
template <int RF, bool GATED, bool GROUPED>
__device__ __forceinline__ void f8_tile(const F8Args& a, uint4* const ring, int e, int p0, int rows,
                                        int tn) {
  using L = TileLds<RF>;
  constexpr int NST = L::kStages, MF = 2 * RF, NF = 4;
  constexpr int XD = RF, WD = 4;           // DMAs a wave and stage, and one of scales
  // Of a stage's DMAs so many follow the barrier that frees its slot, the others lie
  // between the next stage's first steps: each holds its wave for some 20 cycles (512 x
  // [3840, 10240] in 256 rows 103.9 us, all at once 113.7).
  constexpr int kDma = XD + WD + 1, kPost = MF > 2 ? NF : kDma;
  constexpr int kEach = (kPost + NF - 1) / NF;
  float* const wsc = reinterpret_cast<float*>(ring + NST * L::kStage);

  const int tid = (int)threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int KB = a.KB;

  auto source = [&](int r) {               // x's row of tile row r
    int src = p0 + (r < rows ? r : rows - 1);
    if constexpr (GROUPED) {
      if (a.order) src = a.order[src] / a.fan;
      src = src < 0 ? 0 : src < a.x_rows ? src : a.x_rows - 1;
      return src;
    }
    return src - p0;
  };
  const uint8_t* const xbase = GROUPED ? a.x : a.x + (long long)p0 * a.ldx;
  const uint16_t* const sbase = GROUPED ? a.xs : a.xs + p0;
  const uint8_t* const wbase = a.w + e * a.w_expert + (long long)tn * (TBN * 128);
  // LDS chunk p of x's tile holds row p >> 3, logical chunk (p & 7) ^ swizzle
  auto chunk_of = [&](int p) { return (p & 7) ^ ((p >> 4) & 7); };
  uint32_t xrow[XD];
#pragma unroll
  for (int i = 0; i < XD; ++i)
    xrow[i] = (uint32_t)((long long)source((64 * (XD * wave + i) + lane) >> 3) * a.ldx);
  // W's 32 rows a wave are 4 KB of memory and of LDS, in the order of the lanes' operands.
  // A tile that ends the weights after 128 rows takes those twice.
  const int wrow = !GATED && TBN * tn + 32 * wave >= a.NR ? 32 * wave - 128 : 32 * wave;
  const uint32_t woff = (uint32_t)(16 * lane);
  // Scales of 64 rows a wave; more waves than that write some twice, the same values (a
  // branch here would split the stage, and the sums would be sunk past it). A lane's MF
  // rows of a wave's 16 MF lie side by side: dword c * MF + i is row 16 i + c.
  const int srow = 64 * (wave % RF), sd = srow + lane, si = sd % (16 * MF);
  const uint32_t soff =
      2u * (uint32_t)source(sd - si + 16 * (si % MF) + si / MF);
  const int klast = (a.K - 128 * (KB - 1)) / 16;       // the last block's chunks

  const uint8_t *xnext = xbase, *wnext = wbase + wrow * 128;
  const uint16_t* snext = sbase;
  int tnext = 0;
  // The DMAs of the stage that is next to be fetched, one at a time: 0 to XD - 1 x's, then
  // W's, then the scales'. Its bases move on by a stage at a time; past the last stage it
  // is read again into a slot nothing reads, so that every stage issues and waits alike.
  auto issue = [&](int q, const uint4* S) {
    if (q < XD) {
      // past K the weights are zeros: any chunk of x's own block will do
      const int ch = chunk_of(64 * (XD * wave + q) + lane), cut = tnext == KB - 1 ? klast : 8;
      dma16_sb(xnext, xrow[q] + (ch < cut ? 16 * ch : 0), lds_addr(S + 64 * (XD * wave + q)));
    } else if (q < XD + WD) {
      const uint32_t to = lds_addr(S + L::kX + 64 * WD * wave);
      switch (q - XD) {
        case 0: dma16_off<0>(wnext, woff, to); break;
        case 1: dma16_off<1024>(wnext, woff, to); break;
        case 2: dma16_off<2048>(wnext, woff, to); break;
        default: dma16_off<3 * 1024>(wnext, woff, to); break;
      }
    } else {
      dma2_sb(snext, soff, lds_addr(S + L::kX + L::kW) + 4 * srow);
      const bool more = tnext < KB - 1;
      tnext += more;
      xnext += more ? 128 : 0;
      wnext += more ? a.NR * 128ll : 0;
      snext += more ? a.ldxs : 0;
    }
  };

  // The weights' scales of all blocks, [KB][2]: of the tile's two blocks of rows, or gate's
  // and up's. By DMA too, before the others, so that every wait covers them and nothing
  // waits for them alone.
  {
    const float* const ws = a.ws + e * a.s_expert + 2 * tn;
    const int odd = 2 * tn + 1 < a.NB ? lane & 1 : 0;
    for (int i = 64 * wave; i < 2 * KB; i += 64 * NW) {
      const int k = (i + lane) >> 1;
      dma4_sb(ws, (uint32_t)(((k < KB ? k : KB - 1) * (long long)a.NB + odd) * 4),
              lds_addr(wsc + i));
    }
  }

  floatx4_t acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};

  // fragments: rows 16 apart keep their swizzle
  const int fx = (32 * RF * wm + c) * 8 + (g ^ (c >> 1)), fw = 64 * 8 * wn + lane;
  auto read_x = [&](const uint4* S, int i) {
    return F8Frag{S[fx + 128 * i], S[(fx ^ 4) + 128 * i]};
  };
  auto read_w = [&](const uint4* S, int j) {
    return F8Frag{S[L::kX + fw + 128 * j], S[L::kX + fw + 128 * j + 64]};
  };
  uint32_t sx[MF];
  float sw[2];
  auto read_s = [&](const uint4* S, int t) {
    const uint32_t* p =
        reinterpret_cast<const uint32_t*>(S + L::kX + L::kW) + 16 * MF * wm + MF * c;
#pragma unroll
    for (int i = 0; i < MF; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + i);
      sx[i] = v.x;
      sx[i + 1] = v.y;
    }
    const float* q = wsc + 2 * t + (GATED ? 0 : wn >> 1);
    sw[0] = q[0];
    sw[1] = GATED ? q[1] : 0.0f;
  };

  F8Frag w[NF], x[2];
  auto body = [&](auto ph, int t) {
    constexpr int PH = decltype(ph)::value;
    const uint4 *const S = ring + PH * L::kStage, *const Sn = ring + (PH + 1) % NST * L::kStage;
    const uint4* const Sl = ring + (PH + NST - 1) % NST * L::kStage;   // freed by stage t - 1
    float s[MF], u[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const float v = __uint_as_float(sx[i] << 16);
      s[i] = v * sw[0];
      u[i] = GATED ? v * sw[1] : 0.0f;
    }
    auto add = [&](int j, int i, const floatx4_t& d) {
      const float f = GATED && j >= 2 ? u[i] : s[i];
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(d[r], f, acc[j][i][r]);
    };
    constexpr int kSteps = MF > 2 ? MF - 2 : 1, kLate = (kDma - kPost + kSteps - 1) / kSteps;
    F8Frag xa = x[0], xb = x[1];
    floatx4_t dp[NF];
#pragma unroll
    for (int i = 0; i < MF - 2; ++i) {
      const F8Frag xn = read_x(S, i + 2);
      floatx4_t d[NF];
#pragma unroll
      for (int q = kPost + i * kLate; q < kPost + (i + 1) * kLate && q < kDma; ++q) issue(q, Sl);
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        d[j] = f8_mfma(w[j], xa);
        if (i > 0) add(j, i - 1, dp[j]);
      }
#pragma unroll
      for (int j = 0; j < NF; ++j) dp[j] = d[j];
      xa = xb;
      xb = xn;
      // a step's matrix instructions, each with a result of the step before
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);     // DS read
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // MFMA
        if (i > 0) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);   // VALU
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    ring_wait<(NST - 2) * kDma>();
    __builtin_amdgcn_sched_barrier(0);
    x[0] = read_x(Sn, 0);
    read_s(Sn, t + 1 < KB ? t + 1 : t);
    floatx4_t e0, e1;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NF; ++j) {
#pragma unroll
      for (int q = j * kEach; q < (j + 1) * kEach && q < kPost; ++q) issue(q, S);
      const floatx4_t d0 = f8_mfma(w[j], xa), d1 = f8_mfma(w[j], xb);
      if (MF > 2) add(j, MF > 2 ? MF - 3 : 0, dp[j]);
      w[j] = read_w(Sn, j);
      if (j > 0) {
        add(j - 1, MF - 2, e0);
        add(j - 1, MF - 1, e1);
      }
      e0 = d0;
      e1 = d1;
      __builtin_amdgcn_sched_barrier(0);
    }
    add(NF - 1, MF - 2, e0);
    add(NF - 1, MF - 1, e1);
    x[1] = read_x(Sn, 1);
  };

#pragma unroll
  for (int t = 0; t < NST; ++t) {
#pragma unroll
    for (int q = 0; q < kDma; ++q)
      // (the last one's later ones are stage 0's to issue)
      if (t < NST - 1 || q < kPost) issue(q, ring + t * L::kStage);
  }
  // stage 0 landed, and the weights' scales
  ring_wait<(NST - 2) * kDma + kPost>();
#pragma unroll
  for (int j = 0; j < NF; ++j) w[j] = read_w(ring, j);
  x[0] = read_x(ring, 0);
  x[1] = read_x(ring, 1);
  read_s(ring, 0);
  const std::integral_constant<int, 0> p0c{};
  const std::integral_constant<int, 1> p1c{};
  int t = 0;
  if constexpr (NST == 2) {
    for (; t + 2 <= KB; t += 2) {
      body(p0c, t);
      body(p1c, t + 1);
    }
    if (t < KB) body(p0c, t);
  } else {
    const std::integral_constant<int, 2> p2c{};
    for (; t + 3 <= KB; t += 3) {
      body(p0c, t);
      body(p1c, t + 1);
      body(p2c, t + 2);
    }
    if (KB - t >= 1) body(p0c, t);
    if (KB - t >= 2) body(p1c, t + 1);
  }
  ring_wait<0>();                          // drained; LDS free

  if constexpr (GATED) {
    // v = silu(gate) * up: fragments 0, 1 are the wave's 32 gate columns, 2, 3 the up
    // ones. A row's largest over the tile's 128 columns is a block's: over a lane's
    // columns, the four lane quarters, and the four waves side by side, by LDS. Then a
    // thread makes a row's scale and its reciprocal, once for the 16 lanes that divide by it
    // (NaN for a block that holds a NaN or an inf).
    uint32_t* const tops = reinterpret_cast<uint32_t*>(ring);            // [4][64 RF]
    uint4* const E = ring + RF * 64;                                      // [64 RF][8]
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = silu_f(acc[j][i][r]) * acc[j + 2][i][r];
          acc[j][i][r] = v;
          top = f8_top(top, v);
        }
      top = f8_top_quarters(top);
      if (g == 0) tops[64 * RF * wn + 32 * RF * wm + 16 * i + c] = top;
    }
    __syncthreads();
    if (tid < 64 * RF) {
      uint32_t top = tops[tid];
#pragma unroll
      for (int k = 1; k < 4; ++k) {
        const uint32_t v = tops[64 * RF * k + tid];
        top = top > v ? top : v;
      }
      const float tf = __uint_as_float(top);
      const uint32_t sb = f8_finite(tf) ? f8_scale_bits(tf) : kF8NanScale;
      if (tid < rows) a.hs[(long long)tn * a.ldhs + p0 + tid] = (uint16_t)sb;
      // (a thread's own entries: no other one reads them before the barrier)
      tops[tid] = sb << 16;
      tops[64 * RF + tid] = __float_as_uint(1.0f / __uint_as_float(sb << 16));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int row = 32 * RF * wm + 16 * i + c;
      const float s = __uint_as_float(tops[row]), y = __uint_as_float(tops[64 * RF + row]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const floatx4_t& v = acc[j][i];
        const uint32_t codes = f8_pack4(f8_quotient(v[0], s, y), f8_quotient(v[1], s, y),
                                        f8_quotient(v[2], s, y), f8_quotient(v[3], s, y));
        // chunk of 16 columns 2 wn + j, a lane quarter's dword
        reinterpret_cast<uint32_t*>(E)[(row * 8 + ((2 * wn + j) ^ ((row >> 1) & 7))) * 4 + g] =
            s == s ? codes : kF8Nan4;
      }
    }
    __syncthreads();
    const int ch = tid & 7, n = 128 * tn + 16 * ch;
    uint8_t* to = a.h + (long long)(p0 + (tid >> 3)) * a.ldh + n;
#pragma unroll
    for (int k = 0; k < RF; ++k, to += 64 * a.ldh) {
      const int row = 64 * k + (tid >> 3);
      if (row < rows && n < a.N)
        f8_store16(to, E[row * 8 + (ch ^ ((row >> 1) & 7))], a.stream);
    }
  } else {
    // each wave turns its 64 columns through its own part of LDS, then stores whole
    // 128-byte row pieces; 32 rows at a time, so that the first stores are on their way early
    uint4* const E = ring + 32 * RF * 8 * wave;
    uint2* const E2 = reinterpret_cast<uint2*>(E);
    const int nb = TBN * tn + 64 * wn;
    if (!GROUPED && a.bias) {
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const int n = nb + 16 * j + 4 * g;
        uint2 v = {0, 0};
        if (n < a.N) v = *reinterpret_cast<const uint2*>(a.bias + n);
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          acc[j][i][0] += bf16_lo(v.x);
          acc[j][i][1] += bf16_hi(v.x);
          acc[j][i][2] += bf16_lo(v.y);
          acc[j][i][3] += bf16_hi(v.y);
        }
      }
    }
    const int cl = lane & 7, n = nb + 8 * cl, first = 32 * RF * wm + (lane >> 3);
    uint16_t* to = a.y + (long long)(p0 + first) * a.ldy + n;
#pragma unroll
    for (int q = 0; q < RF; ++q) {
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 2 * q; i < 2 * q + 2; ++i) {
          const int row = 16 * i + c;
          const floatx4_t& v = acc[j][i];
          E2[(row * 8 + ((2 * j + (g >> 1)) ^ ((row >> 1) & 7))) * 2 + (g & 1)] =
              make_uint2(pack_bf16x2_rne(v[0], v[1]), pack_bf16x2_rne(v[2], v[3]));
        }
#pragma unroll
      for (int k = 4 * q; k < 4 * q + 4; ++k, to += 8 * a.ldy) {
        const int ml = 8 * k + (lane >> 3);
        const uint4 v = E[ml * 8 + (cl ^ ((ml >> 1) & 7))];
        if (first + 8 * k < rows && n < a.N) f8_store16(to, v, a.stream);
      }
    }
  }
}

template <int RF, bool GATED>
__global__ __launch_bounds__(64 * NW, 1) void f8_tile_kernel(const F8Args a) {
  __shared__ uint4 ring[TileLds<RF>::kUnits];
  constexpr int BM = 64 * RF;
  const int tiles_m = (a.n + BM - 1) / BM;
  int tm, tn;
  tile_of_block((int)blockIdx.x, tiles_m, (a.NR + TBN - 1) / TBN, &tm, &tn);
  const int p0 = BM * tm, left = a.n - p0;
  f8_tile<RF, GATED, false>(a, ring, 0, p0, left < BM ? left : BM, tn);
}

// The first `main` tiles of rows are of 256, the others of 128: a last round of the chip that
// is mostly empty takes half the time.
template <bool GATED>
__global__ __launch_bounds__(64 * NW, 1) void f8_mixed_kernel(const F8Args a, int main) {
  constexpr int kUnits = TileLds<4>::kUnits > TileLds<2>::kUnits ? TileLds<4>::kUnits
                                                                   : TileLds<2>::kUnits;
  __shared__ uint4 ring[kUnits];
  const int tiles_n = (a.NR + TBN - 1) / TBN, first = main * tiles_n, b = (int)blockIdx.x;
  int tm, tn;
  if (b < first) {
    tile_of_block(b, main, tiles_n, &tm, &tn);
    f8_tile<4, GATED, false>(a, ring, 0, 256 * tm, 256, tn);
  } else {
    tile_of_block(b - first, (a.n - 256 * main + 127) / 128, tiles_n, &tm, &tn);
    const int p0 = 256 * main + 128 * tm, left = a.n - p0;
    f8_tile<2, GATED, false>(a, ring, 0, p0, left < 128 ? left : 128, tn);
  }
}

// Groups of more than 64 * MAX places are cut into the fewest tiles that hold them.
template <int MAX, bool GATED>
__global__ __launch_bounds__(64 * NW, 1) void f8_group_tile_kernel(const F8Args a) {
  constexpr int CUT = 64 * MAX;
  constexpr int kUnits = TileLds<MAX>::kUnits > TileLds<2>::kUnits ? TileLds<MAX>::kUnits
                                                                     : TileLds<2>::kUnits;
  __shared__ uint4 ring[kUnits];
  const int tiles_n = (a.NR + TBN - 1) / TBN;
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
  const int p0 = rg.p0 + rt.first, rows = rt.rows;
  if constexpr (MAX >= 4) {
    if (rows > 192) return f8_tile<4, GATED, true>(a, ring, rg.e, p0, rows, tn);
    if (rows > 128) return f8_tile<3, GATED, true>(a, ring, rg.e, p0, rows, tn);
  }
  if (rows > 64)
    f8_tile<2, GATED, true>(a, ring, rg.e, p0, rows, tn);
  else
    f8_tile<1, GATED, true>(a, ring, rg.e, p0, rows, tn);
}

template <int RF>
void tile_launch(bool gated, const F8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)f8_tile_blocks(RF, false, a.n, a.E, a.NR));
  if (gated)
    hipLaunchKernelGGL((f8_tile_kernel<RF, true>), grid, dim3(64 * NW), 0, s, a);
  else
    hipLaunchKernelGGL((f8_tile_kernel<RF, false>), grid, dim3(64 * NW), 0, s, a);
}
template <int MAX>
void group_launch(bool gated, const F8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)f8_tile_blocks(MAX, true, a.n, a.E, a.NR));
  if (gated)
    hipLaunchKernelGGL((f8_group_tile_kernel<MAX, true>), grid, dim3(64 * NW), 0, s, a);
  else
    hipLaunchKernelGGL((f8_group_tile_kernel<MAX, false>), grid, dim3(64 * NW), 0, s, a);
}

}  // namespace

hipError_t launch_f8_tile(bool gated, bool grouped, const F8Args& a, int rf, int main,
                          hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  if (main < 0 || (main > 0 && (grouped || rf != 2 || 256ll * main >= a.n)))
    return hipErrorInvalidValue;
  if (a.N <= 0 || a.N % (gated ? 16 : 8) || a.K % 16 || a.KB > kF8TileBlocks || a.E < 1 || a.fan < 1)
    return hipErrorInvalidValue;
  if (main > 0) {
    const dim3 grid((unsigned)f8_mixed_blocks(main, a.n, a.NR));
    if (gated)
      hipLaunchKernelGGL((f8_mixed_kernel<true>), grid, dim3(64 * NW), 0, s, a, main);
    else
      hipLaunchKernelGGL((f8_mixed_kernel<false>), grid, dim3(64 * NW), 0, s, a, main);
    return hipGetLastError();
  }
  switch (grouped ? 10 + rf : rf) {
    case 1: tile_launch<1>(gated, a, s); break;
    case 2: tile_launch<2>(gated, a, s); break;
    case 3: tile_launch<3>(gated, a, s); break;
    case 4: tile_launch<4>(gated, a, s); break;
    case 12: group_launch<2>(gated, a, s); break;
    case 14: group_launch<4>(gated, a, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t validate_f8_tile_kernels() {
  hipFuncAttributes fa;
#define MING_F8_TILE(RF)                                          \
  reinterpret_cast<const void*>(&f8_tile_kernel<RF, false>),      \
      reinterpret_cast<const void*>(&f8_tile_kernel<RF, true>)
#define MING_F8_GROUP(MAX)                                        \
  reinterpret_cast<const void*>(&f8_group_tile_kernel<MAX, false>), \
      reinterpret_cast<const void*>(&f8_group_tile_kernel<MAX, true>)
  const void* fns[] = {MING_F8_TILE(1), MING_F8_TILE(2), MING_F8_TILE(3), MING_F8_TILE(4),
                       MING_F8_GROUP(2), MING_F8_GROUP(4),
                       reinterpret_cast<const void*>(&f8_mixed_kernel<false>),
                       reinterpret_cast<const void*>(&f8_mixed_kernel<true>)};
#undef MING_F8_TILE
#undef MING_F8_GROUP
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
