// What stands around a mixture's expert products: the router's top-k choice,
// the grouping of the choices by expert, and the weighted sum that brings the
// expert rows back to their tokens.
#include "common.h"
#include "kernels.h"

namespace ming {
namespace {

// ---- the router ------------------------------------------------------------
// Per row of logits l: scores s = softmax(l) or sigmoid(l), keys s + bias, the
// groups with the best sums of two keys, and of their experts the k largest
// keys. Scores and keys are in 64 bits: a choice is a comparison, and with
// 32-bit scores the rounding of an exponential would decide between experts
// whose logits differ. Ties go to the lowest index. A logit of -inf or NaN is
// never chosen.
//
// A wave per row, expert 64 i + lane in register i. A key is compared as the
// integer its bits order as (0: not to be chosen): one maximum over the wave is six
// DPP steps on the upper words, and six on the lower ones where two lanes share an
// upper; the winner is the lowest register whose ballot against it is not empty, so
// a choice costs no exchange of indices. Bound by that chain of dependent steps (k
// of them, about 0.15 us each), not by the logits' bytes: 8 rows, 8 of 256 experts in
// groups 6.9 us (9.0 with f64 maxima and a lane a group), 4099 rows, 6 of 60 4.6.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double old, double v) {
  const uint64_t o = __builtin_bit_cast(uint64_t, old), u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)o, (int)(uint32_t)u, CTRL, ROWS,
                                                  0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp((int)(o >> 32), (int)(u >> 32), CTRL, ROWS, 0xf,
                                                  false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// Over the wave; a lane without a source adds nothing to the maximum or the sum.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  auto step = [&](uint32_t o) { v = v > o ? v : o; };
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));   // row_shr 1, 2, 4, 8
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));   // row_bcast 15, 31
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double wave_add(double v) {
  v += dpp_f64<0x111, 0xf>(0.0, v);
  v += dpp_f64<0x112, 0xf>(0.0, v);
  v += dpp_f64<0x114, 0xf>(0.0, v);
  v += dpp_f64<0x118, 0xf>(0.0, v);
  v += dpp_f64<0x142, 0xa>(0.0, v);
  v += dpp_f64<0x143, 0xc>(0.0, v);
  return lane_f64(v, 63);
}
// The integers the values order as (no NaN).
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v);
  return u >> 31 ? ~u : u | 1u << 31;
}

template <int P>
__global__ __launch_bounds__(256) void topk_route_kernel(const RouteArgs a) {
  // [wave][expert]: logits, exponentials, scores, keys. The loops over a lane's
  // experts that hold an exponential or a division are not unrolled: one copy of
  // each in the code.
  __shared__ double gkeys[4][64 * P];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const long long row = (long long)blockIdx.x * 4 + wave;
  if (row >= a.rows) return;               // no barrier below: a wave is on its own
  const double none = -__builtin_inf();
  double* const mine = gkeys[wave];
  float l[P], bias[P];
  uint32_t may_choose = 0;                 // bit i: this lane's expert 64 i + lane
  float most = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = 64 * i + lane;
    l[i] = -__builtin_inff();
    bias[i] = a.bias && e < a.E ? a.bias[e] : 0.0f;
    if (e < a.E)
      l[i] = a.f32 ? reinterpret_cast<const float*>(a.logits)[row * a.ld + e]
                   : bf16_to_f32(reinterpret_cast<const uint16_t*>(a.logits)[row * a.ld + e]);
    // NaN is not larger than -inf; +inf is the largest finite value
    l[i] = l[i] > -__builtin_inff() ? fminf(l[i], 3.4028234663852886e38f) : -__builtin_inff();
    if (l[i] > -__builtin_inff()) may_choose |= 1u << i;
    most = fmaxf(most, l[i]);
    mine[64 * i + lane] = (double)l[i];
  }
  double top = 0.0, sum = 0.0;
  if (!a.sigmoid) {
    const uint32_t u = wave_max(ordered(most));
    top = (double)__uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u);
  }
#pragma unroll 1
  for (int i = 0; i < P; ++i) {
    const double v = mine[64 * i + lane];
    const double x = exp(a.sigmoid ? -v : v - top);
    mine[64 * i + lane] = x;
    if (may_choose >> i & 1) sum += x;
  }
  if (!a.sigmoid) sum = wave_add(sum);
  double s[P];
#pragma unroll 1
  for (int i = 0; i < P; ++i) {
    const double x = mine[64 * i + lane];
    mine[64 * i + lane] = a.sigmoid ? 1.0 / (1.0 + x) : x / sum;
  }
  double key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    s[i] = mine[64 * i + lane];
    key[i] = s[i] + (double)bias[i];
    // a key that is NaN (a bias that is) is never chosen either
    key[i] = (may_choose >> i & 1) && key[i] > none ? key[i] : none;
  }
  if (a.G > 1) {
    const int S = a.E / a.G;
#pragma unroll
    for (int i = 0; i < P; ++i) mine[64 * i + lane] = key[i];
    __builtin_amdgcn_wave_barrier();
    // L lanes a group find its two best keys
    int L = 1;
    while (2 * L * a.G <= 64) L *= 2;
    const int g = lane / L, q = lane % L;
    double b1 = none, b2 = none;
    if (g < a.G) {
#pragma unroll 4
      for (int j = q; j < S; j += L) {
        const double v = mine[g * S + j];
        b2 = fmax(b2, fmin(b1, v));
        b1 = fmax(b1, v);
      }
    }
    for (int o = 1; o < L; o *= 2) {
      const double o1 = __shfl_xor(b1, o, 64), o2 = __shfl_xor(b2, o, 64);
      b2 = fmax(fmin(b1, o1), fmax(b2, o2));
      b1 = fmax(b1, o1);
    }
    const double sc = b1 > none ? b1 + (b2 > none ? b2 : 0.0) : none;
    int better = 0;
#pragma unroll 1
    for (int h = 0; h < a.G; ++h) {
      const double o = lane_f64(sc, h * L);
      better += o > sc || (o == sc && h < g) ? 1 : 0;
    }
    // the experts of a group that may not
    if (g < a.G && !(sc > none && better < a.top_groups)) {
#pragma unroll 4
      for (int j = q; j < S; j += L) mine[g * S + j] = none;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < P; ++i) key[i] = 64 * i + lane < a.E ? mine[64 * i + lane] : none;
  }
#pragma unroll
  for (int i = 0; i < P; ++i) mine[64 * i + lane] = s[i];
  __builtin_amdgcn_wave_barrier();
  uint64_t u[P];
#pragma unroll
  for (int i = 0; i < P; ++i) u[i] = key[i] > none ? ordered(key[i]) : 0;
  int my_id = -1;                          // lane j: the row's choice j
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = u[0];
    int at = 0;                            // the lane's best, the lowest of equal ones
#pragma unroll
    for (int i = 1; i < P; ++i)
      if (u[i] > best) {
        best = u[i];
        at = i;
      }
    const uint32_t hi = wave_max((uint32_t)(best >> 32));
    if (hi == 0) break;                    // (an ordered key above -inf has an upper word)
    uint64_t those = __ballot((uint32_t)(best >> 32) == hi);
    if (those & (those - 1)) {             // lanes that share it: the lower word, then the index
      const uint32_t lo = wave_max((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
      const uint64_t m = (uint64_t)hi << 32 | lo;
      those = __ballot(best == m);
      for (int i = 0; i < P; ++i) {
        const uint64_t here = __ballot(best == m && at == i);
        if (here) {
          those = here;
          break;
        }
      }
    }
    const int w = __builtin_ctzll(those);
    const int i = __builtin_amdgcn_readlane(at, w);
    if (lane == j) my_id = 64 * i + w;
#pragma unroll
    for (int r = 0; r < P; ++r)
      if (r == i && lane == w) u[r] = 0;
  }
  double w = my_id >= 0 ? mine[my_id] : 0.0;
  if (a.normalize) {
    const double total = wave_add(w);
    w = total > 0.0 ? w / total : 0.0;
  }
  if (lane < a.k) {
    a.ids[row * a.k + lane] = my_id;
    a.weights[row * a.k + lane] = (float)(w * (double)a.scale);
  }
}

// ---- grouping ----------------------------------------------------------------
// A stable counting sort of n group ids: entry i of group g goes to offsets[g]
// + the number of earlier entries of g. Ids outside [0, G) count as a last
// group of their own, so the ends of `order` need no pass of their own.
//
// A block takes a contiguous part, each of its 16 waves a contiguous part of
// that, 64 entries at a time: the lanes with one id find each other with a
// ballot a bit of the id, so a rank is a population count and no atomic orders
// anything. Up to kGroupOne entries are one block and one launch; more take a
// launch that counts each block's groups and one that places: there each block
// adds up the counts of the blocks before it itself, which is less than a
// launch of its own. Bound by the launches and the chain inside them: 64 ids 3.8 us,
// 34816 of 64 groups 7.6 in two launches, 262144 10.0, of 1024 groups 30.
constexpr int GT = 1024, GW = GT / 64, GBINS = 1024 + 1;

__device__ __forceinline__ uint64_t lanes_with(int v, int bits, uint64_t active) {
  uint64_t peers = active;
  for (int b = 0; b < bits; ++b) {
    const uint64_t m = __ballot((v >> b) & 1);
    peers &= ((v >> b) & 1) ? m : ~m;
  }
  return peers;
}

// MODE 0: one block does it all; 1: counts only; 2: places by the counts.
template <int MODE>
__global__ __launch_bounds__(GT) void group_rows_kernel(const GroupRowsArgs a) {
  __shared__ uint32_t counts[GW * GBINS];  // [wave][bin]
  __shared__ uint32_t tot[GBINS + 63], pre[GBINS];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bins = a.G + 1;
  const long long b0 = (long long)blockIdx.x * a.chunk;
  const long long b1 = b0 + a.chunk < a.n ? b0 + a.chunk : a.n;
  const int part = (int)(((b1 - b0 + GT - 1) / GT) * 64);      // entries a wave
  const long long w0 = b0 + (long long)wave * part;
  const long long w1 = w0 + part < b1 ? w0 + part : b1;
  auto bin_of = [&](long long i) {
    const int id = a.ids[i];
    return id >= 0 && id < a.G ? id : a.G;
  };
  auto cnt = [&](int w, int g) -> uint32_t& { return counts[w * bins + g]; };
  // the wave's first batch, read once (while the counts of the blocks come in)
  const int first = w0 + lane < w1 ? bin_of(w0 + lane) : 0;
  for (int i = tid; i < GW * bins; i += GT) counts[i] = 0;
  if constexpr (MODE == 2)
    for (int g = tid; g < bins; g += GT) tot[g] = pre[g] = 0;
  __syncthreads();
  if constexpr (MODE == 2) {
    // the blocks' counts, one run of memory: all of them, and those before this one's;
    // eight reads of a thread at a time ([34816] of 1024 groups: 26.4 us a block's row
    // after the other)
    constexpr int UN = 8;
    const int total = (int)gridDim.x * bins, before = (int)blockIdx.x * bins;
    const int step = GT % bins;
    int g = tid % bins;
    for (int i = tid; i < total; i += GT * UN) {
      uint32_t v[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) v[u] = i + GT * u < total ? a.counts[i + GT * u] : 0;
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        if (v[u]) atomicAdd(&tot[g], v[u]);
        if (v[u] && i + GT * u < before) atomicAdd(&pre[g], v[u]);
        g += step;
        g = g >= bins ? g - bins : g;
      }
    }
  }
  if (w0 + lane < w1) atomicAdd(&cnt(wave, first), 1u);
  for (long long i = w0 + lane + 64; i < w1; i += 64) atomicAdd(&cnt(wave, bin_of(i)), 1u);
  __syncthreads();
  if constexpr (MODE == 1) {
    for (int g = tid; g < bins; g += GT) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < GW; ++w) t += cnt(w, g);
      a.counts[(long long)blockIdx.x * bins + g] = t;
    }
    return;
  }
  if constexpr (MODE == 0) {
    for (int g = tid; g < bins; g += GT) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < GW; ++w) t += cnt(w, g);
      tot[g] = t;
    }
    __syncthreads();
  }
  if (wave == 0) {                         // exclusive scan, a lane's bins in a row
    const int per = (bins + 63) / 64;
    uint32_t sum = 0;
    for (int j = 0; j < per; ++j)
      if (lane * per + j < bins) sum += tot[lane * per + j];
    uint32_t run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(run, o, 64);
      if (lane >= o) run += v;
    }
    run -= sum;
    for (int j = 0; j < per; ++j) {
      const int g = lane * per + j;
      if (g >= bins) break;
      const uint32_t t = tot[g];
      tot[g] = run;
      run += t;
    }
  }
  __syncthreads();
  for (int g = tid; g < bins; g += GT) {
    uint32_t at = tot[g];
    if (blockIdx.x == 0) a.offsets[g] = (int32_t)at;
    if constexpr (MODE == 2) at += pre[g];
#pragma unroll
    for (int w = 0; w < GW; ++w) {
      const uint32_t t = cnt(w, g);
      cnt(w, g) = at;
      at += t;
    }
  }
  __syncthreads();
  for (long long i0 = w0; i0 < w1; i0 += 64) {
    const long long i = i0 + lane;
    const bool live = i < w1;
    const int g = !live ? 0 : i0 == w0 ? first : bin_of(i);
    const uint64_t peers = lanes_with(g, a.bits, __ballot(live));
    if (live) {
      const int rank = __popcll(peers & ((1ull << lane) - 1));
      const uint32_t pos = cnt(wave, g) + (uint32_t)rank;
      __builtin_amdgcn_wave_barrier();
      if ((peers >> lane) == 1ull) cnt(wave, g) = pos + 1;     // the last of its group
      __builtin_amdgcn_wave_barrier();
      a.order[pos] = g < a.G ? (int32_t)i : -1;
      a.place[i] = g < a.G ? (int32_t)pos : -1;
    }
  }
}

// ---- the weighted sum -----------------------------------------------------------
// out[t] = bf16(add[t] + sum_j w[t][j] y[place[t k + j]]), f32 sums in the
// order of j, one rounding; a place outside [0, n) adds nothing, whatever its
// weight. Bound by HBM: every expert row is read once. tpr threads (a power of
// two) a token, 8 columns a thread and step, four rows' loads at a time. 4352 tokens
// of 8 rows of 2048, onto a row: 37 us, 4.8 TB/s.
__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
  const int tid = (int)threadIdx.x;
  const int sub = tid & (a.tpr - 1);
  const long long t = (long long)blockIdx.x * (256 / a.tpr) + tid / a.tpr;
  if (t >= a.tokens) return;
  const int32_t* const place = a.place + t * a.k;
  const float* const wt = a.weights + t * a.k;
  for (int c = 8 * sub; c < a.N; c += 8 * a.tpr) {
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      int p[4];
      float w[4];
      uint4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u < a.k ? j0 + u : a.k - 1;
        p[u] = place[j];
        w[u] = wt[j];
        if (p[u] < 0 || p[u] >= a.n || j0 + u >= a.k) p[u] = -1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (p[u] >= 0) v[u] = *reinterpret_cast<const uint4*>(a.y + (long long)p[u] * a.ldy + c);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (p[u] >= 0) {
          const uint32_t* vp = &v[u].x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[2 * e] = fmaf(w[u], bf16_lo(vp[e]), s[2 * e]);
            s[2 * e + 1] = fmaf(w[u], bf16_hi(vp[e]), s[2 * e + 1]);
          }
        }
    }
    if (a.add) {
      const uint4 v = *reinterpret_cast<const uint4*>(a.add + t * a.ldadd + c);
      const uint32_t* vp = &v.x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[2 * e] += bf16_lo(vp[e]);
        s[2 * e + 1] += bf16_hi(vp[e]);
      }
    }
    uint4 o;
    o.x = pack_bf16x2_rne(s[0], s[1]);
    o.y = pack_bf16x2_rne(s[2], s[3]);
    o.z = pack_bf16x2_rne(s[4], s[5]);
    o.w = pack_bf16x2_rne(s[6], s[7]);
    *reinterpret_cast<uint4*>(a.out + t * a.ldo + c) = o;
  }
}

}  // namespace

static long long route_blocks(long long rows) { return (rows + 3) / 4; }

bool route_fits(long long rows) { return one_launch(route_blocks(rows), 256); }

hipError_t launch_topk_route(const RouteArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.E < 1 || a.E > kRouteMaxExperts || a.G < 1 || a.G > 64 || a.E % a.G || a.k < 1 ||
      a.k > 64)
    return hipErrorInvalidValue;
  const dim3 grid((unsigned)route_blocks(a.rows));
  if (a.E <= 64)
    hipLaunchKernelGGL(topk_route_kernel<1>, grid, dim3(256), 0, s, a);
  else if (a.E <= 128)
    hipLaunchKernelGGL(topk_route_kernel<2>, grid, dim3(256), 0, s, a);
  else if (a.E <= 256)
    hipLaunchKernelGGL(topk_route_kernel<4>, grid, dim3(256), 0, s, a);
  else if (a.E <= 512)
    hipLaunchKernelGGL(topk_route_kernel<8>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(topk_route_kernel<16>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

// The blocks of n entries: one up to kGroupOne, else a batch of 64 a wave each as
// long as that is at most 128 blocks (each reads every block's counts). 34816 ids of
// 64 groups: 11.4 us in nine blocks of 4096, 7.6 in 34.
constexpr int kGroupOne = 4096;
static int group_chunk(long long n) {
  if (n <= kGroupOne) return (int)(n > 0 ? n : 1);
  return (int)((n + 128 * GT - 1) / (128 * GT) * GT);
}

size_t group_rows_bytes(long long n, int G) {
  if (n <= kGroupOne) return 0;
  const long long chunk = group_chunk(n);
  return (size_t)((n + chunk - 1) / chunk) * (size_t)(G + 1) * 4;
}

hipError_t launch_group_rows(GroupRowsArgs a, hipStream_t s) {
  if (a.n < 0 || a.G < 1 || a.G > kGroupMax) return hipErrorInvalidValue;
  a.chunk = group_chunk(a.n);
  a.bits = 32 - __builtin_clz((unsigned)a.G);
  if (a.n <= kGroupOne) {
    hipLaunchKernelGGL(group_rows_kernel<0>, dim3(1), dim3(GT), 0, s, a);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((a.n + a.chunk - 1) / a.chunk));
  hipLaunchKernelGGL(group_rows_kernel<1>, grid, dim3(GT), 0, s, a);
  hipLaunchKernelGGL(group_rows_kernel<2>, grid, dim3(GT), 0, s, a);
  return hipGetLastError();
}

static int combine_threads(int N) {
  int tpr = 1;
  while (tpr < 256 && tpr * 8 < N) tpr *= 2;
  return tpr;
}

long long combine_blocks(long long tokens, int N) {
  const int rpb = 256 / combine_threads(N);
  return (tokens + rpb - 1) / rpb;
}

hipError_t launch_combine(CombineArgs a, hipStream_t s) {
  if (a.tokens <= 0 || a.N <= 0) return hipSuccess;
  if (a.N % 8 || a.k < 1) return hipErrorInvalidValue;
  a.tpr = combine_threads(a.N);
  hipLaunchKernelGGL(combine_kernel, dim3((unsigned)combine_blocks(a.tokens, a.N)), dim3(256), 0, s,
                     a);
  return hipGetLastError();
}

hipError_t validate_routing_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {reinterpret_cast<const void*>(&topk_route_kernel<1>),
                       reinterpret_cast<const void*>(&topk_route_kernel<2>),
                       reinterpret_cast<const void*>(&topk_route_kernel<4>),
                       reinterpret_cast<const void*>(&topk_route_kernel<8>),
                       reinterpret_cast<const void*>(&topk_route_kernel<16>),
                       reinterpret_cast<const void*>(&group_rows_kernel<0>),
                       reinterpret_cast<const void*>(&group_rows_kernel<1>),
                       reinterpret_cast<const void*>(&group_rows_kernel<2>),
                       reinterpret_cast<const void*>(&combine_kernel)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
