// Low-rank adapters that rows choose: the down-projection T = x . A^T of every
// row's own adapter. The up-projection runs in the projection's own launch.
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace ming {
namespace {

// T[m] = strength * fold * (x[m] . A_a^T), a = ids[m]. A block takes 16 or 32 rows;
// the adapters among them (in any order) are found with ballots, and each
// adapter's 16-rank chunks are v_mfma_f32_16x16x32_bf16 tiles over all the rows, of
// which only that adapter's are stored: requests' rows lie together, so a block
// has one or two adapters, and where every row has its own the time is that of
// reading their A. K is shared out over the eight waves by 64-groups, the sums
// meet in LDS and are added in wave order (no atomics). A is resident in the
// operand's own order (launch_repack_adapter): a wave's load is one run of 1 KB, of
// which lanes past the rank take no part.
//
// Two forms. Few rows (row_xa_kernel): 16 rows, a chunk a block and turn, operands
// straight from memory, all of a chunk's at once; grid y shares out the chunks. Bound by three memory
// latencies in a row (ids, table, A and x). Many rows (row_xa_many_kernel): x passes
// through LDS in whole 1 KB row pieces, read from memory once for two (or four)
// chunks and for the fp16 copy of x that a quantized projection multiplies. Bound by HBM, x
// once and its copy once ([8704, 3840]: 79 us with x from memory a lane's 16 bytes
// at a time).
constexpr int XW = 8;

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

// The chunk list of row tile `tile` (at most 256 rows, a thread each): the chunks
// of each adapter where the tile's first row of it stands.
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

__device__ __forceinline__ floatx4_t mfma16(const uint4& w, const uint4& x, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w),
                                                 __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
}

__global__ __launch_bounds__(64 * XW) void row_xa_kernel(const RowXaArgs a) {
  __shared__ floatx4_t red[XW][64];
  __shared__ int ids[256], sums[XW];
  const int xtiles = (a.M + 15) / 16;
  if ((int)blockIdx.x >= xtiles) {           // the lists' blocks
    if (blockIdx.y == 0) row_chunks(a, (int)blockIdx.x - xtiles, ids, sums);
    return;
  }
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int m0 = (int)blockIdx.x * 16, m = m0 + c;
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
  const RowOf row = resolve(a, m);           // the wave's quarters hold the same rows
  if (blockIdx.y == 0 && wave == 0 && lane < 16 && m < a.M) a.rid[m] = row.id;
  if (a.xh) {
    // the fp16 copy of the block's rows, grid y sharing out the columns
    const int k8 = a.K / 8, c0 = k8 * (int)blockIdx.y / (int)gridDim.y;
    const int c1 = k8 * ((int)blockIdx.y + 1) / (int)gridDim.y;
    uint32_t seen = 0;
    for (int r = wave; r < 16 && m0 + r < a.M; r += XW)
      for (int k = c0 + lane; k < c1; k += 64) {
        const uint4 v = *reinterpret_cast<const uint4*>(a.x + (long long)(m0 + r) * a.ldx + 8 * k);
        *reinterpret_cast<uint4*>(a.xh + (long long)(m0 + r) * a.K + 8 * k) = to_f16(v, seen);
      }
    range_report(a.range, seen);
  }
  int turn = 0;
  bool there = false;
  each_chunk(row, [&](int cur, int r8, const uint4* A, int ch) {
    if (turn++ % (int)gridDim.y != (int)blockIdx.y) return;
    const uint4* const ar = chunk_lane(A, r8, a.K, ch, lane);
    floatx4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = wave; k0 < KT; k0 += XW * U) {
      uint4 av[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kt = k0 + XW * u < KT ? k0 + XW * u : KT - 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) av[u][h] = ar[64 * (2 * kt + h)];
      }
      if (!there) load_x(k0);
      there = KT <= XW * U;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k0 + XW * u < KT) {
#pragma unroll
          for (int h = 0; h < 2; ++h) acc = mfma16(av[u][h], xv[u][h], acc);
        }
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
      floatx4_t v = red[0][lane];
#pragma unroll
      for (int w = 1; w < XW; ++w) v += red[w][lane];
      if (row.id == cur) store_t(a, m, row.coef, r8, ch + 4 * g, v);
    }
    __syncthreads();
  }, [&](int cur, int r8, int ch) {
    if (blockIdx.y == 0 && wave == 0 && row.id == cur)
      store_t(a, m, 0.0f, r8, ch + 4 * g, floatx4_t{0.0f, 0.0f, 0.0f, 0.0f});
  });
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
          for (int i = 0; i < C; ++i) acc[i][b] = mfma16(av[i][h], xv, acc[i][b]);
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

// From these rows on x passes through LDS.
constexpr int kRowXaMany = 768;

hipError_t launch_row_xa(const RowXaArgs& a, hipStream_t s) {
  if (a.M <= 0) return hipSuccess;
  if (a.K % 64 || a.ldt % 32 || (a.counts && (a.rows_main % 256 || a.rest < 1 || a.rest > 256 || a.slices < 1)))
    return hipErrorInvalidValue;
  const int tiles = (a.M + 31) / 32;
  const int lists = a.counts ? row_tiles(a.M, a.rows_main, a.rest) : 0;
  if (a.M >= kRowXaMany) {
    // ranks past 32 make it more than one pass over x: four chunks a pass then
    const dim3 grid((unsigned)(tiles + lists), tiles < 128 ? 4u : tiles < 256 ? 2u : 1u);
    if (a.ldt <= 32)
      hipLaunchKernelGGL(row_xa_many_kernel<2>, grid, dim3(64 * XW), 0, s, a);
    else
      hipLaunchKernelGGL(row_xa_many_kernel<4>, grid, dim3(64 * XW), 0, s, a);
    return hipGetLastError();
  }
  const int low = (a.M + 15) / 16;
  int y = 1;
  while (y < 32 && low * y < 512) y *= 2;
  hipLaunchKernelGGL(row_xa_kernel, dim3((unsigned)(low + lists), (unsigned)y), dim3(64 * XW), 0, s,
                     a);
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
