// The 8-bit products over few rows: y[m] = sum over blocks b of 128 of
// xs[b][m] * ws[n / 128][b] * (x . w)_b, plain or SwiGLU-gated, of one projection or
// of a mixture's groups.
//
// HBM-bound on the weights. A workgroup takes 16 * MF rows x 16 * NF columns; its
// eight waves take the K blocks in turn, each with operands straight from memory
// in the matrix instruction's own order: no barrier and no LDS before the waves'
// sums meet, so as many loads as registers hold are in flight. A block of K is one
// v_mfma_f32_16x16x128 a tile, whose f32 result joins the sum times both scales
// (f32: the scales are any, not the hardware's powers of two). Gated results go through
// f32 memory to f8_finish_kernel: a block's 128 columns are several workgroups'.
//
// Measured out of cold caches: one row x [3840, 3840] 4.6 us (4.0 in the kernel; 2.9 by
// bytes, the rest a launch's start and end), gated [10240, 3840] 15.1 (5.2 TB/s), eight rows 15.6;
// 8 x 8 places of [64][1024, 2048] gated 31.2 (5.5 TB/s). With weights in rows of 128
// bytes, 16 lines a load, the gated ones took 17.6 and 44; more than one block ahead a
// wave won nothing (occupancy); fp16 products, whose sums would be exact, cost 3 to 20%.
#include <algorithm>

#include "common.h"
#include "f8.h"
#include "kernels.h"
#include "row_groups.h"

namespace ming {
namespace {

constexpr int WK = 8;      // waves, each a share of K

template <int MF, int NF, bool GATED, bool GROUPED>
__global__ __launch_bounds__(64 * WK) void f8_rows_kernel(const F8Args a) {
  constexpr int NH = GATED ? 2 * NF : NF, TM = 16 * MF, TN = 16 * NF;
  __shared__ floatx4_t red[WK][MF * NH][64];
  const int lane = (int)threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

  const int tiles_n = (a.N + TN - 1) / TN;
  int e = 0, p0, rows, tn;
  auto spread = [&](int total) {           // an XCD takes a contiguous range
    const int b = (int)blockIdx.x, q = total / 8, rem = total % 8, xcd = b % 8;
    return b < total ? xcd * q + (xcd < rem ? xcd : rem) + b / 8 : -1;
  };
  if constexpr (GROUPED) {
    const RowGroup rg = find_group(
        a.offsets, a.E, a.n, [&](int r) { return (r + TM - 1) / TM * tiles_n; }, spread);
    if (rg.e < 0) return;
    const int tiles_m = (rg.rows + TM - 1) / TM;
    tn = rg.index / tiles_m;
    const int first = TM * (rg.index - tn * tiles_m);
    e = rg.e;
    p0 = rg.p0 + first;
    rows = rg.rows - first;
  } else {
    const int tiles_m = (a.n + TM - 1) / TM;
    const int v = spread(tiles_m * tiles_n);
    tn = v / tiles_m;
    p0 = TM * (v - tn * tiles_m);
    rows = a.n - p0;
  }
  rows = rows < TM ? rows : TM;
  const int n0 = tn * TN;

  const uint8_t* xp[MF];
  const uint16_t* sp[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int r = 16 * i + c;
    int src = p0 + (r < rows ? r : rows - 1);
    if constexpr (GROUPED) {
      if (a.order) src = a.order[src] / a.fan;
      src = src < 0 ? 0 : src < a.x_rows ? src : a.x_rows - 1;
    }
    xp[i] = a.x + (long long)src * a.ldx;
    sp[i] = a.xs + src;
  }
  const uint8_t* wp = a.w + e * a.w_expert + 16 * lane;
  const float* ws = a.ws + e * a.s_expert;
  int wr[NH];                              // resident rows of the fragments
#pragma unroll
  for (int j = 0; j < NF; ++j) {
    const int n = n0 + 16 * j;
    wr[j] = GATED ? f8_gate_row(n) : n;
    if constexpr (GATED) wr[NF + j] = wr[j] + 32;
  }
  const int sb = GATED ? 2 * (n0 >> 7) : n0 >> 7;

  struct Block {
    F8Frag w[NH], x[MF];
    float sx[MF], s0, s1;
  };
  auto load = [&](int kb, Block& b) {
    const uint8_t* p = wp + (long long)kb * a.NR * 128;
#pragma unroll
    for (int j = 0; j < NH; ++j) {
      b.w[j].lo = *reinterpret_cast<const uint4*>(p + wr[j] * 128);
      b.w[j].hi = *reinterpret_cast<const uint4*>(p + wr[j] * 128 + 1024);
    }
    // past K the weights are zeros, and any chunk of x's own block will do (not one
    // of other memory, whose NaN codes would count)
    const int k = 128 * kb, k0 = k + 16 * g;
    const int lo = k0 < a.K ? k0 : k, hi = k0 + 64 < a.K ? k0 + 64 : k;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      b.x[i].lo = *reinterpret_cast<const uint4*>(xp[i] + lo);
      b.x[i].hi = *reinterpret_cast<const uint4*>(xp[i] + hi);
      b.sx[i] = bf16_to_f32(sp[i][(long long)kb * a.ldxs]);
    }
    b.s0 = ws[(long long)kb * a.NB + sb];
    b.s1 = GATED ? ws[(long long)kb * a.NB + sb + 1] : 0.0f;
  };
  floatx4_t acc[NH][MF];
#pragma unroll
  for (int j = 0; j < NH; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto take = [&](const Block& b) {
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const float s0 = b.sx[i] * b.s0, s1 = b.sx[i] * b.s1;
#pragma unroll
      for (int j = 0; j < NH; ++j) {
        const floatx4_t d = f8_mfma(b.w[j], b.x[i]);
        const float s = GATED && j >= NF ? s1 : s0;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(d[r], s, acc[j][i][r]);
      }
    }
  };
  Block cur, nxt;
  if (wave < a.KB) load(wave, cur);
  for (int kb = wave; kb < a.KB; kb += WK) {
    if (kb + WK < a.KB) load(kb + WK, nxt);
    take(cur);
    cur = nxt;
  }
#pragma unroll
  for (int j = 0; j < NH; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) red[wave][j * MF + i][lane] = acc[j][i];
  __syncthreads();
  // the waves' sums in their order, a fragment a wave
  for (int f = wave; f < NF * MF; f += WK) {
    const int j = f / MF, m = 16 * (f - j * MF) + c, n = n0 + 16 * j + 4 * g;
    if (m >= rows || n >= a.N) continue;
    floatx4_t v = red[0][f][lane];
#pragma unroll
    for (int w = 1; w < WK; ++w) v += red[w][f][lane];
    if constexpr (GATED) {
      floatx4_t u = red[0][NF * MF + f][lane];
#pragma unroll
      for (int w = 1; w < WK; ++w) u += red[w][NF * MF + f][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = silu_f(v[r]) * u[r];
      *reinterpret_cast<floatx4_t*>(a.part + (long long)(p0 + m) * a.N + n) = v;
    } else {
      if (a.bias) {
        const uint2 b = *reinterpret_cast<const uint2*>(a.bias + n);
        v[0] += bf16_lo(b.x);
        v[1] += bf16_hi(b.x);
        v[2] += bf16_lo(b.y);
        v[3] += bf16_hi(b.y);
      }
      *reinterpret_cast<uint2*>(a.y + (long long)(p0 + m) * a.ldy + n) =
          make_uint2(pack_bf16x2_rne(v[0], v[1]), pack_bf16x2_rne(v[2], v[3]));
    }
  }
}

template <int CTRL>
__device__ __forceinline__ uint32_t f8_top_row(uint32_t top) {
  const uint32_t t = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, CTRL, 0xf, 0xf, false);
  return top > t ? top : t;
}

// Columns n .. n + 3 of a row's block b, lane l of the 32 that hold it (in: they exist;
// lanes without take part in the shuffles).
__device__ __forceinline__ void f8_store_block(const F8Args& a, int row, int b, int n, int l, bool in,
                                               const floatx4_t& v) {
  uint32_t top = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) top = f8_top(top, v[r]);
  top = f8_top_row<0x128>(top);            // row_ror by 8, 4, 2, 1, then the other row of 16
  top = f8_top_row<0x124>(top);
  top = f8_top_row<0x122>(top);
  top = f8_top_row<0x121>(top);
  const auto o = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = o[0] > o[1] ? o[0] : o[1];
  if (!in) return;
  const float t = __uint_as_float(top);
  const bool fine = f8_finite(t);
  const uint32_t sb = fine ? f8_scale_bits(t) : kF8NanScale;
  const float s = __uint_as_float(sb << 16), y = 1.0f / s;
  *reinterpret_cast<uint32_t*>(a.h + (long long)row * a.ldh + n) =
      fine ? f8_pack4(f8_quotient(v[0], s, y), f8_quotient(v[1], s, y), f8_quotient(v[2], s, y),
                      f8_quotient(v[3], s, y))
           : kF8Nan4;
  if (l == 0) a.hs[(long long)b * a.ldhs + row] = (uint16_t)sb;
}

// The gated results [n][N] in f32 into codes and scales: 32 lanes a block of 128. A
// dependent launch, 2 to 4.7 us of the above; the results are still in L2.
__global__ __launch_bounds__(256) void f8_finish_kernel(const F8Args a, int rows, int blocks) {
  const uint32_t unit = blockIdx.x * 8u + (threadIdx.x >> 5);
  const int l = (int)threadIdx.x & 31;
  const int b = (int)(unit / (uint32_t)rows), row = (int)(unit - (uint32_t)b * (uint32_t)rows);
  // rows before the first group and behind the last one stay as they are: part holds
  // nothing of theirs
  int first = 0, held = rows;
  if (a.offsets) {
    first = a.offsets[0];
    held = a.offsets[a.E];
  }
  const int n = 128 * b + 4 * l;
  floatx4_t v = {0.0f, 0.0f, 0.0f, 0.0f};  // (loaded beside held, not after it)
  if (b < blocks && n < a.N)
    v = *reinterpret_cast<const floatx4_t*>(a.part + (long long)row * a.N + n);
  f8_store_block(a, row, b, n, l, b < blocks && row >= first && row < held && n < a.N, v);
}

// Codes [halves * N][K] and scales [halves * blocks of N][KB] into the resident order,
// zeros past N and K: blocks of K outermost, then 16 rows (gated, f8_gate_row's), as the
// matrix instruction's lanes hold them: chunks g and g + 4 of row c for lane 16 g + c, the
// first ones of all lanes before the second ones. blockIdx.y is the expert.
__global__ void f8_repack_kernel(const uint8_t* codes, const float* scales, int N, int K, int halves,
                                 uint8_t* out, float* souts) {
  const int KB = (K + 127) / 128, nb = (N + 127) / 128, NR = halves * nb * 128;
  const long long total = (long long)KB * NR * 8, e = blockIdx.y;
  codes += e * halves * N * K;
  scales += e * halves * nb * KB;
  out += e * total * 16;
  souts += e * halves * nb * KB;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const int l = (int)(i & 63), ch = (l >> 4) + 4 * (int)((i >> 6) & 1);
    const long long q = i >> 7;              // 16 rows of a block
    const int kb = (int)(q / (NR / 16)), r = 16 * (int)(q % (NR / 16)) + (l & 15);
    int n = r, half = 0;
    if (halves == 2) {
      half = (r >> 5) & 1;
      n = 128 * (r >> 8) + 32 * ((r >> 6) & 3) + (r & 31);
    }
    const int k = 128 * kb + 16 * ch;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n < N && k < K)
      v = *reinterpret_cast<const uint4*>(codes + ((long long)half * N + n) * K + k);
    reinterpret_cast<uint4*>(out)[i] = v;
    // a block's scale beside its first row
    if (ch == 0 && (n & 127) == 0) {
      const int b = n >> 7;
      souts[(long long)kb * (halves * nb) + halves * b + half] =
          scales[(long long)(half * nb + b) * KB + kb];
    }
  }
}

template <int MF, int NF>
void rows_launch(bool gated, bool grouped, const F8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)f8_rows_blocks(16 * MF, 16 * NF, grouped, a.n, a.E, a.N));
  if constexpr (MF == 1) {
    if (grouped) {
      if (gated)
        hipLaunchKernelGGL((f8_rows_kernel<MF, NF, true, true>), grid, dim3(64 * WK), 0, s, a);
      else
        hipLaunchKernelGGL((f8_rows_kernel<MF, NF, false, true>), grid, dim3(64 * WK), 0, s, a);
      return;
    }
  }
  if (gated)
    hipLaunchKernelGGL((f8_rows_kernel<MF, NF, true, false>), grid, dim3(64 * WK), 0, s, a);
  else
    hipLaunchKernelGGL((f8_rows_kernel<MF, NF, false, false>), grid, dim3(64 * WK), 0, s, a);
}

}  // namespace

hipError_t launch_f8_repack(const uint8_t* codes, const float* scales, int experts, int N, int K,
                            int halves, uint8_t* out, float* souts, hipStream_t s) {
  if (experts < 1 || experts > 65535 || N <= 0 || K <= 0 || K % 16) return hipErrorInvalidValue;
  const long long units = (K + 127ll) / 128 * ((N + 127ll) / 128) * halves * 128 * 8;
  const long long each = (2048 + experts - 1) / experts;   // blocks, some 2048 in all
  hipLaunchKernelGGL(f8_repack_kernel,
                     dim3((unsigned)std::min(std::max(each, 32ll), (units + 255) / 256),
                          (unsigned)experts),
                     dim3(256), 0, s, codes, scales, N, K, halves, out, souts);
  return hipGetLastError();
}

hipError_t launch_f8_rows(bool gated, bool grouped, const F8Args& a, int mf, int nf,
                          hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  if (a.N <= 0 || a.N % (gated ? 16 : 8) || a.K % 16 || (gated && !a.part) || a.E < 1 || a.fan < 1)
    return hipErrorInvalidValue;
  switch (10 * mf + nf) {
    case 11: rows_launch<1, 1>(gated, grouped, a, s); break;
    case 12: rows_launch<1, 2>(gated, grouped, a, s); break;
    case 14: rows_launch<1, 4>(gated, grouped, a, s); break;
    case 24:
      if (grouped) return hipErrorInvalidValue;
      rows_launch<2, 4>(gated, false, a, s);
      break;
    default: return hipErrorInvalidValue;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !gated) return e;
  const int blocks = (a.N + 127) / 128;
  hipLaunchKernelGGL(f8_finish_kernel, dim3((unsigned)f8_finish_blocks(a.n, a.N)), dim3(256), 0, s, a,
                     a.n, blocks);
  return hipGetLastError();
}

hipError_t validate_f8_rows_kernels() {
  hipFuncAttributes fa;
#define MING_F8_ROWS(MF, NF)                                                    \
  reinterpret_cast<const void*>(&f8_rows_kernel<MF, NF, false, false>),         \
      reinterpret_cast<const void*>(&f8_rows_kernel<MF, NF, true, false>)
#define MING_F8_GROUPS(NF)                                                      \
  reinterpret_cast<const void*>(&f8_rows_kernel<1, NF, false, true>),           \
      reinterpret_cast<const void*>(&f8_rows_kernel<1, NF, true, true>)
  const void* fns[] = {reinterpret_cast<const void*>(&f8_finish_kernel),
                       reinterpret_cast<const void*>(&f8_repack_kernel), MING_F8_ROWS(1, 1),
                       MING_F8_ROWS(1, 2), MING_F8_ROWS(1, 4), MING_F8_ROWS(2, 4),
                       MING_F8_GROUPS(1), MING_F8_GROUPS(2), MING_F8_GROUPS(4)};
#undef MING_F8_GROUPS
#undef MING_F8_ROWS
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
