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

// The adapter of row m and the factor of its T, -1 for none.
__device__ __forceinline__ int resolve(const RowXaArgs& a, int m, float* coef) {
  if (m >= a.M) return -1;
  const int id = a.ids[m];
  const float s = a.scale ? a.scale[m] : 1.0f;
  if (id < 0 || id >= a.cap || s == 0.0f || a.table[id].r8 == 0) return -1;
  *coef = s * a.table[id].fold;
  return id;
}

// The chunk list of row tile `tile` (at most 256 rows, a thread each): the chunks
// of each adapter where the tile's first row of it stands.
__device__ __forceinline__ void row_chunks(const RowXaArgs& a, int tile, int* ids, int* sums) {
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int mains = a.rows_main / 256;
  const int m0 = tile < mains ? 256 * tile : a.rows_main + (tile - mains) * a.rest;
  const int end = tile < mains ? m0 + 256 : m0 + a.rest;
  float unused;
  const int m = m0 + tid;
  const int id = tid < 256 && m < end ? resolve(a, m, &unused) : -1;
  if (tid < 256) ids[tid] = id;
  __syncthreads();
  bool first = id >= 0;
  const int4* const q = reinterpret_cast<const int4*>(ids);
  for (int r = 0; r < tid && r < 256; r += 4) {
    const int4 v = q[r >> 2];
    if (v.x == id || (r + 1 < tid && v.y == id) || (r + 2 < tid && v.z == id) ||
        (r + 3 < tid && v.w == id))
      first = false;
  }
  AdapterEntry e = {};
  if (first) e = a.table[id];
  const int chunks = first ? (e.r8 + 31) / 32 : 0;
  RowChunk* const out = reinterpret_cast<RowChunk*>(a.chunks) + (long long)tile * a.stride;
  int base = 0;
  for (int s = 0; s < a.slices; ++s) {     // chunk c of adapter id is slice (id + c) % slices'
    const int c0 = (s + a.slices - (id < 0 ? 0 : id) % a.slices) % a.slices;
    const int n = chunks > c0 ? (chunks - c0 + a.slices - 1) / a.slices : 0;
    int run = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(run, o, 64);
      if (lane >= o) run += v;
    }
    __syncthreads();                       // the last slice's sums are read
    if (lane == 63) sums[tid >> 6] = run;
    __syncthreads();
    int at = base + run - n;
    for (int w = 0; w < 4; ++w) {
      if (w < (tid >> 6)) at += sums[w];
      base += sums[w];
    }
    for (int i = 0; i < n; ++i) {
      const int c = c0 + i * a.slices;
      const int groups = e.r8 - 32 * c >= 32 ? 4 : (e.r8 - 32 * c) / 8;
      out[at + i] = RowChunk{e.B + 32 * c, id,
                             (uint32_t)e.r8 | (uint32_t)c << 12 | (uint32_t)(groups - 1) << 20};
    }
    if (tid == 0) a.counts[tile * a.slices + s] = base;
  }
  // T's row of zeros
  if (tile == 0)
    for (int i = tid; i < a.ldt; i += 64 * XW) a.t[(long long)a.M * a.ldt + i] = 0;
}

__global__ __launch_bounds__(64 * XW) void row_xa_kernel(const RowXaArgs a) {
  __shared__ __align__(16) float red[XW][16][64];
  const int xtiles = (a.M + 31) / 32;
  if ((int)blockIdx.x >= xtiles) {           // the lists' blocks
    if (blockIdx.y == 0)
      row_chunks(a, (int)blockIdx.x - xtiles, reinterpret_cast<int*>(&red[0][0][0]),
                 reinterpret_cast<int*>(&red[1][0][0]));
    return;
  }
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int fr = lane & 31, fk = lane >> 5;
  const int m0 = (int)blockIdx.x * 32;
  const int m = m0 + fr;
  // the row's adapter; both halves of the wave hold the same 32 rows
  float coef = 0.0f;
  const int id = resolve(a, m, &coef);
  if (a.xh) {
    // the fp16 copy of the block's rows, grid y sharing out the columns
    const int k8 = a.K / 8, c0 = k8 * (int)blockIdx.y / (int)gridDim.y;
    const int c1 = k8 * ((int)blockIdx.y + 1) / (int)gridDim.y;
    uint32_t seen = 0;
    for (int r = wave; r < 32 && m0 + r < a.M; r += XW)
      for (int c = c0 + lane; c < c1; c += 64) {
        const uint4 v = *reinterpret_cast<const uint4*>(a.x + (long long)(m0 + r) * a.ldx + 8 * c);
        seen = range_track4(seen, v);
        uint4 f;
        f.x = bf16x2_to_f16x2(v.x);
        f.y = bf16x2_to_f16x2(v.y);
        f.z = bf16x2_to_f16x2(v.z);
        f.w = bf16x2_to_f16x2(v.w);
        *reinterpret_cast<uint4*>(a.xh + (long long)(m0 + r) * a.K + 8 * c) = f;
      }
    range_report(a.range, seen);
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
  if (a.K % 64 || a.ldt % 32 || (a.counts && (a.rows_main % 256 || a.rest < 1 || a.rest > 256 || a.slices < 1)))
    return hipErrorInvalidValue;
  const int tiles = (a.M + 31) / 32;
  const int lists = a.counts ? row_tiles(a.M, a.rows_main, a.rest) : 0;
  int y = 1;
  while (y < 32 && tiles * y < 512) y *= 2;
  hipLaunchKernelGGL(row_xa_kernel, dim3((unsigned)(tiles + lists), (unsigned)y), dim3(64 * XW), 0,
                     s, a);
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
