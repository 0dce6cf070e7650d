// Low-rank adapters that rows choose: the down-projection T = x . A^T of every
// row's own adapter. The up-projection runs in the projection's own launch.
#include "common.h"
#include "kernels.h"

namespace ming {
namespace {

// T[m] = strength * fold * (x[m] . A_a^T), a = ids[m]. A block takes 32 rows;
// the adapters among them (in any order) are found with ballots, and each
// adapter's 32-rank chunks are one v_mfma_f32_32x32x16_bf16 tile over all 32
// rows, of which only that adapter's rows are stored: requests' rows lie
// together, so a block has one or two adapters, and where every row has its own
// the time is that of reading their A. K is shared out over the eight waves by
// 64-groups, the sums meet in LDS and are added in wave order (no atomics).
// Where there are few row blocks, grid y shares out a block's chunks.
// Bound by the reads of x and, for few rows, of A.
constexpr int XW = 8;

__global__ __launch_bounds__(64 * XW) void row_xa_kernel(const RowXaArgs a) {
  __shared__ float red[XW][16][64];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 31, fk = lane >> 5;
  const int m0 = (int)blockIdx.x * 32;
  const int m = m0 + fr;
  // the row's adapter; both halves of the wave hold the same 32 rows
  int id = -1;
  float coef = 0.0f;
  if (m < a.M) {
    id = a.ids[m];
    coef = a.scale ? a.scale[m] : 1.0f;
    if (id < 0 || id >= a.cap || coef == 0.0f) id = -1;
    if (id >= 0) {
      if (a.table[id].r8 == 0) id = -1;
      else coef *= a.table[id].fold;
    }
  }
  if (blockIdx.y == 0 && wave == 0 && fk == 0 && m < a.M) a.rid[m] = id;
  const int KT = a.K / 64;
  const uint16_t* const xr = a.x + (long long)(m < a.M ? m : a.M - 1) * a.ldx + 8 * fk;
  uint64_t left = __ballot(id >= 0);
  int turn = 0;
  while (left) {
    const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    left &= ~__ballot(id == cur);
    const AdapterEntry e = a.table[cur];   // wave-uniform
    for (int ch = 0; ch < e.r8; ch += 32) {
      if (turn++ % (int)gridDim.y != (int)blockIdx.y) continue;
      const int rank = ch + fr < e.r8 ? ch + fr : e.r8 - 1;
      const uint16_t* const ar = e.A + (long long)rank * a.K + 8 * fk;
      floatx16_t acc;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
      for (int kt = wave; kt < KT; kt += XW) {
        uint4 xv[4], av[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          xv[kk] = *reinterpret_cast<const uint4*>(xr + 64 * kt + 16 * kk);
          av[kk] = *reinterpret_cast<const uint4*>(ar + 64 * kt + 16 * kk);
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, av[kk]),
                                                        __builtin_bit_cast(bf16x8_t, xv[kk]), acc,
                                                        0, 0, 0);
      }
      // lane (row fr, fk): ranks 8q + 4fk + 0..3 in registers 4q..4q+3
#pragma unroll
      for (int r = 0; r < 16; ++r) red[wave][r][lane] = acc[r];
      __syncthreads();
      // wave w sums registers 2w and 2w + 1, two ranks of a row
      float v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[i] = red[0][2 * wave + i][lane];
#pragma unroll
        for (int w = 1; w < XW; ++w) v[i] += red[w][2 * wave + i][lane];
      }
      const int r0 = ch + 8 * (wave >> 1) + 4 * fk + 2 * (wave & 1);
      if (id == cur) {
        const uint32_t o = r0 < e.r8 ? pack_bf16x2_rne(coef * v[0], coef * v[1]) : 0u;
        *reinterpret_cast<uint32_t*>(a.t + (long long)m * a.ldt + r0) = o;
      }
      __syncthreads();
    }
  }
}

// The up-projection on its own, in f32, for projections of few rows and for the
// routes without tiles of their own for it: a thread four columns of a row.
__global__ __launch_bounds__(256) void row_delta_kernel(const RowAdapters ra, int N, float* d) {
  const int m = (int)blockIdx.y;
  const int n = 4 * ((int)blockIdx.x * 256 + (int)threadIdx.x);
  if (n >= N) return;
  float s[4] = {-0.0f, -0.0f, -0.0f, -0.0f};
  const int a = ra.rid[m];
  if (a >= 0) {
    const AdapterEntry e = ra.table[a];
    const uint16_t* const t = ra.t + (long long)m * ra.ldt;
    const uint16_t* const b = e.B + (long long)n * e.r8;
    for (int k = 0; k < e.r8; k += 8) {
      const uint4 tv = *reinterpret_cast<const uint4*>(t + k);
      const uint32_t* const tp = &tv.x;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const uint4 bv = *reinterpret_cast<const uint4*>(b + v * e.r8 + k);
        const uint32_t* const bp = &bv.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[v] = fmaf(bf16_lo(tp[i]), bf16_lo(bp[i]), s[v]);
          s[v] = fmaf(bf16_hi(tp[i]), bf16_hi(bp[i]), s[v]);
        }
      }
    }
  }
  *reinterpret_cast<float4*>(d + (long long)m * N + n) = make_float4(s[0], s[1], s[2], s[3]);
}

__global__ void check_finite_kernel(const uint16_t* v, long long n, int* flag) {
  bool bad = false;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n;
       i += (long long)gridDim.x * blockDim.x)
    bad = bad || (v[i] & 0x7f80u) == 0x7f80u;
  if (bad) *flag = 1;
}

}  // namespace

hipError_t launch_row_xa(const RowXaArgs& a, hipStream_t s) {
  if (a.M <= 0) return hipSuccess;
  if (a.K % 64 || a.ldt % 32) return hipErrorInvalidValue;
  const int tiles = (a.M + 31) / 32;
  int y = 1;
  while (y < 32 && tiles * y < 512) y *= 2;
  hipLaunchKernelGGL(row_xa_kernel, dim3((unsigned)tiles, (unsigned)y), dim3(64 * XW), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_row_delta(const RowAdapters& r, int M, int N, float* d, hipStream_t s) {
  if (M <= 0 || N <= 0) return hipSuccess;
  if (N % 4) return hipErrorInvalidValue;
  // grid y holds 65535 rows
  for (int m = 0; m < M; m += 65535) {
    RowAdapters part = r;
    part.rid += m;
    part.t += (long long)m * r.ldt;
    hipLaunchKernelGGL(row_delta_kernel,
                       dim3((unsigned)((N / 4 + 255) / 256), (unsigned)(M - m < 65535 ? M - m : 65535)),
                       dim3(256), 0, s, part, N, d + (long long)m * N);
  }
  return hipGetLastError();
}

hipError_t launch_check_finite(const uint16_t* v, long long n, int* flag, hipStream_t s) {
  if (n <= 0) return hipSuccess;
  const long long blocks = (n + 1023) / 1024;
  hipLaunchKernelGGL(check_finite_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256),
                     0, s, v, n, flag);
  return hipGetLastError();
}

hipError_t validate_adapter_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {reinterpret_cast<const void*>(&row_xa_kernel),
                       reinterpret_cast<const void*>(&row_delta_kernel),
                       reinterpret_cast<const void*>(&check_finite_kernel)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
