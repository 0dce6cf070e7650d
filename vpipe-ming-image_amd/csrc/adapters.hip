// Low-rank adapters that rows choose: the down-projection T = x . A^T of every
// row's own adapter. The up-projection runs in the projection's own launch.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"
#include "row_xa.h"

namespace ming {
namespace {

constexpr int XW = 8;

// The chunk list of row tile `tile` (at most 256 rows, a thread each): the chunks
// of each adapter where the tile's first row of it stands, row_tile_chunks at most.
__device__ __forceinline__ void row_chunks(const RowXaArgs& a, int tile, int* ids, int* sums) {
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int mains = a.rows_main / 256;
  const int m0 = tile < mains ? 256 * tile : a.rows_main + (tile - mains) * a.rest;
  const int end = tile < mains ? m0 + 256 : m0 + a.rest;
  RowOf row = {-1, 0.0f, {}};
  if (tid < 256 && m0 + tid < end) row = resolve(a, m0 + tid);
  const int id = row.id;
  const AdapterEntry& e = row.e;
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
  const int chunks = first ? (e.r8 + 31) / 32 : 0;
  RowChunk* const out = reinterpret_cast<RowChunk*>(a.chunks) + (long long)tile * a.stride;
  int run = chunks;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(run, o, 64);
    if (lane >= o) run += v;
  }
  if (lane == 63) sums[tid >> 6] = run;
  __syncthreads();
  int at = run - chunks;
  for (int w = 0; w < (tid >> 6); ++w) at += sums[w];
  for (int c = 0; c < chunks; ++c) {
    const int groups = e.r8 - 32 * c >= 32 ? 4 : (e.r8 - 32 * c) / 8;
    out[at + c] = RowChunk{e.B + 32 * c, id,
                           (uint32_t)e.r8 | (uint32_t)c << 12 | (uint32_t)(groups - 1) << 20};
  }
  if (tid == 255) a.counts[tile] = at + chunks;
  // T's row of zeros
  if (tile == 0)
    for (int i = tid; i < a.ldt; i += 64 * XW) a.t[(long long)a.M * a.ldt + i] = 0;
}

__global__ __launch_bounds__(64 * XW) void row_xa_kernel(const RowXaArgs a) {
  __shared__ floatx4_t red[XW][64];
  __shared__ alignas(16) int ids[256];       // row_chunks reads four at a time
  __shared__ int sums[XW];
  const int xtiles = (a.M + 15) / 16;
  if ((int)blockIdx.x >= xtiles) {           // the lists' blocks
    if (blockIdx.y == 0) row_chunks(a, (int)blockIdx.x - xtiles, ids, sums);
    return;
  }
  row_xa_block<XW>(a, (int)blockIdx.x, (int)blockIdx.y, (int)gridDim.y, red);
}

// Up to NC chunks a pass; a pass walks K in steps of 512 through two LDS buffers,
// wave w the 64-group w of each, two steps' rows in flight under a step's MFMAs.
template <int NC>
__global__ __launch_bounds__(64 * XW, NC == 2 ? 4 : 2)
void row_xa_many_kernel(const RowXaArgs a) {
  constexpr int KS = 64 * XW;                // K a step
  __shared__ uint4 tile[2][32 * KS / 8];
  // the waves' sums take the first buffer's place after the walk
  floatx4_t (*const red)[2][64] = reinterpret_cast<floatx4_t (*)[2][64]>(&tile[0][0]);
  const int xtiles = (a.M + 31) / 32;
  if ((int)blockIdx.x >= xtiles) {
    if (blockIdx.y == 0)
      row_chunks(a, (int)blockIdx.x - xtiles, reinterpret_cast<int*>(&tile[0][0]),
                 reinterpret_cast<int*>(&tile[1][0]));
    return;
  }
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int m0 = (int)blockIdx.x * 32;
  const RowOf row = resolve(a, m0 + (lane & 31));
  const bool lead = blockIdx.y == 0;         // the passes go round grid y
  if (lead && wave == 0 && lane < 32 && m0 + lane < a.M) a.rid[m0 + lane] = row.id;
  const int KT = a.K / 64, steps = (a.K + KS - 1) / KS;
  uint32_t seen = 0;
  int cur[NC], r8[NC], ch[NC], held = 0;
  const uint4* A[NC];                        // this lane's; past the held ones any
#pragma unroll
  for (int i = 0; i < NC; ++i) A[i] = nullptr;
  int turn = 0;
  bool first = lead;
  auto pass = [&](auto count) {
    constexpr int C = decltype(count)::value;
    floatx4_t acc[C > 0 ? C : 1][2];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i][0] = acc[i][1] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int C1 = C > 0 ? C : 1;
    uint4 v0[4], v1[4], a0[C1][2], a1[C1][2];
    // the step's operands; past K the rows are zeros, so any will do
    auto load_a = [&](int s, uint4 (&av)[C1][2]) {
      const int kt = XW * s + wave < KT ? XW * s + wave : KT - 1;
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) av[i][h] = A[i][64 * (2 * kt + h)];
    };
    auto load = [&](int s, uint4 (&v)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a row's piece of the step, 16 bytes a lane
        const int r = m0 + 4 * wave + i;
        const int k = KS * s + 8 * lane;
        v[i] = k < a.K ? *reinterpret_cast<const uint4*>(
                             a.x + (long long)(r < a.M ? r : a.M - 1) * a.ldx + k)
                       : make_uint4(0, 0, 0, 0);
      }
    };
    auto step = [&](int s, uint4 (&v)[4], uint4 (&av)[C1][2], uint4 (&an)[C1][2]) {
      uint4* const buf = tile[s & 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // 16-byte piece c of row r lies at c ^ (r & 15)
        const int r = 4 * wave + i, k = KS * s + 8 * lane;
        buf[r * (KS / 8) + (lane ^ (r & 15))] = v[i];
        if (first && a.xh && m0 + r < a.M && k < a.K)
          *reinterpret_cast<uint4*>(a.xh + (long long)(m0 + r) * a.K + k) = to_f16(v[i], seen);
      }
      // the next step's operands and the rows of the one after it stay in flight
      // over the MFMAs
      if (s + 1 < steps) load_a(s + 1, an);
      __builtin_amdgcn_sched_barrier(0);
      if (s + 2 < steps) load(s + 2, v);
      // one barrier a step: the buffer written now was read two steps ago, before
      // the barrier between; it waits for LDS alone
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const uint4 xv = buf[(16 * b + c) * (KS / 8) + ((8 * wave + 4 * h + g) ^ c)];
#pragma unroll
          for (int i = 0; i < C; ++i) acc[i][b] = mfma_rows(av[i][h], xv, acc[i][b]);
        }
    };
    load(0, v0);
    load_a(0, a0);
    if (steps > 1) load(1, v1);
    for (int s = 0; s < steps; s += 2) {
      step(s, v0, a0, a1);
      if (s + 1 < steps) step(s + 1, v1, a1, a0);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (i >= held) break;
      __syncthreads();                       // the walk's reads, or the last chunk's, are done
      red[wave][0][lane] = acc[i][0];
      red[wave][1][lane] = acc[i][1];
      __syncthreads();
      if (wave < 2) {                        // wave b: rows 16b + c, columns ch + 4g ..
        floatx4_t t = red[0][wave][lane];
#pragma unroll
        for (int w = 1; w < XW; ++w) t += red[w][wave][lane];
        // the row's adapter is with lane 16b + c
        const int at = 16 * wave + c;
        const float coef = __shfl(row.coef, at, 64);
        if (__shfl(row.id, at, 64) == cur[i]) store_t(a, m0 + at, coef, r8[i], ch[i] + 4 * g, t);
      }
    }
    __syncthreads();
    first = false;
    held = 0;
  };
  each_chunk(row, [&](int id, int rank8, const uint4* p, int rank) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (i == held) {
        cur[i] = id;
        r8[i] = rank8;
        A[i] = chunk_lane(p, rank8, a.K, rank, lane);
        ch[i] = rank;
      }
#pragma unroll
    for (int i = 1; i < NC; ++i)
      if (i > held) A[i] = chunk_lane(p, rank8, a.K, rank, lane);
    if (++held == NC) {
      if (turn++ % (int)gridDim.y == (int)blockIdx.y) pass(std::integral_constant<int, NC>{});
      held = 0;
    }
  }, [&](int id, int rank8, int rank) {
    if (lead && wave == 7 && row.id == id && lane < 32) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        store_t(a, m0 + lane, 0.0f, rank8, rank + 4 * q, floatx4_t{0.0f, 0.0f, 0.0f, 0.0f});
    }
  });
  if (turn % (int)gridDim.y != (int)blockIdx.y) held = 0;
  if (NC > 2 && held > 1)
    pass(std::integral_constant<int, NC - 1>{});
  else if (held > 0)
    pass(std::integral_constant<int, 1>{});
  if (first && a.xh) {
    held = 0;
    pass(std::integral_constant<int, 0>{});
  }
  range_report(a.range, seen);
}

// A [rank][K] into [chunk of 16][K / 32][4][16][8], rows past it zero: the 16x16x32
// operand's lanes one after another.
__global__ void repack_adapter_kernel(const uint16_t* A, int rank, int K, uint16_t* out, long long n) {
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < n;
       i += (long long)gridDim.x * blockDim.x) {
    const int lane = (int)(i & 63);
    const long long s = i >> 6;              // (chunk, step)
    const int ch = (int)(s / (K / 32)), k = (int)(s % (K / 32)) * 32 + 8 * (lane >> 4);
    const int r = 16 * ch + (lane & 15);
    reinterpret_cast<uint4*>(out)[i] =
        r < rank ? *reinterpret_cast<const uint4*>(A + (long long)r * K + k) : make_uint4(0, 0, 0, 0);
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

int row_tile_chunks(int M, int rows_main, int rest, int cap, int ldt) {
  const int tallest = std::max(rows_main > 0 ? 256 : 0, M > rows_main ? rest : 0);
  return std::min({tallest, M, cap}) * (ldt / 32);
}

// The x.A's row tiles: of 32 rows, or of 16 where there are few.
static int row_xa_tiles(int M) {
  const int rows = M >= kRowXaMany ? 32 : 16;
  return (int)(((long long)M + rows - 1) / rows);
}

bool row_xa_fits(int M, int lists) {
  return one_launch((long long)row_xa_tiles(M) + lists, 64 * XW);
}

hipError_t launch_row_xa(const RowXaArgs& a, hipStream_t s) {
  if (a.M <= 0) return hipSuccess;
  if (a.K % 64 || a.ldt % 32 || (a.counts && (a.rows_main % 256 || a.rest < 1 || a.rest > 256)))
    return hipErrorInvalidValue;
  const int tiles = row_xa_tiles(a.M), cus = device_cus();
  const int lists = a.counts ? row_tiles(a.M, a.rows_main, a.rest) : 0;
  if (a.M >= kRowXaMany) {
    // ranks past 32 make it more than one pass over x: four chunks a pass then
    const dim3 grid((unsigned)(tiles + lists), tiles < cus / 2 ? 4u : tiles < cus ? 2u : 1u);
    if (a.ldt <= 32)
      hipLaunchKernelGGL(row_xa_many_kernel<2>, grid, dim3(64 * XW), 0, s, a);
    else
      hipLaunchKernelGGL(row_xa_many_kernel<4>, grid, dim3(64 * XW), 0, s, a);
    return hipGetLastError();
  }
  // a block a CU (two rounds of them, [500, 3840]: 14.6 us, one 9.0)
  const int y = tiles < cus / 64 ? 64 : tiles < cus ? cus / tiles : 1;
  hipLaunchKernelGGL(row_xa_kernel, dim3((unsigned)(tiles + lists), (unsigned)y), dim3(64 * XW), 0, s,
                     a);
  return hipGetLastError();
}

// Beside the split where its blocks have at most 10 us of 16-rank chunks each, were
// every row of a tile its own request: a chunk of K = 3840 takes 2 us, past 4096
// (where x is read again for each) half as long again; a launch of its own takes 5
// to 20 ([3840, 3840] dense, 37 rows of as many adapters of 16 to 64
// ranks: 26.2 us beside, 10.8 and 8.7 apart; 700 rows of 32 in turn: 83, 31 and 20;
// 37 rows of five requests, w4: 11.5 beside, 9.6 and 6 apart; [3840, 10240], 18 rows
// of six adapters of 64 and 128 ranks: 76.6 beside, 11.0 and 18.7 apart). Either way
// T has the same bits.
bool row_xa_beside(int ny, int M, int K, int held, int chunks) {
  if (ny <= 0) return false;
  if (held < 1) return true;
  const double chunk_us = K / 1920.0 * (K > 4096 ? 1.5 : 1.0);
  const double requests = std::min({16.0, (double)held, (double)M});
  return requests * chunks / held * chunk_us <= 10.0 * ny;
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

hipError_t launch_repack_adapter(const uint16_t* A, int rank, int K, uint16_t* out, hipStream_t s) {
  if (rank < 1 || K < 64 || K % 64) return hipErrorInvalidValue;
  const long long n = (long long)((rank + 15) / 16) * (K / 32) * 64;
  hipLaunchKernelGGL(repack_adapter_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, A,
                     rank, K, out, n);
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
                       reinterpret_cast<const void*>(&row_xa_many_kernel<2>),
                       reinterpret_cast<const void*>(&row_xa_many_kernel<4>),
                       reinterpret_cast<const void*>(&repack_adapter_kernel),
                       reinterpret_cast<const void*>(&row_delta_kernel),
                       reinterpret_cast<const void*>(&check_finite_kernel)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
