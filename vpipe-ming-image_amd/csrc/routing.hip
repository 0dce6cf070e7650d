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
// A wave per row, expert 64 i + lane in register i. One maximum over the wave
// is six DPP steps; the winner is the lowest register whose ballot against it
// is not empty, so a choice costs no exchange of indices. Bound by that chain
// of dependent steps (k of them), not by the logits' bytes.
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
// Lanes without a source keep their own value (max) or add zero (sum).
__device__ __forceinline__ double wave_max(double v) {
  v = fmax(v, dpp_f64<0x111, 0xf>(v, v));   // row_shr 1, 2, 4, 8
  v = fmax(v, dpp_f64<0x112, 0xf>(v, v));
  v = fmax(v, dpp_f64<0x114, 0xf>(v, v));
  v = fmax(v, dpp_f64<0x118, 0xf>(v, v));
  v = fmax(v, dpp_f64<0x142, 0xa>(v, v));   // row_bcast 15, 31
  v = fmax(v, dpp_f64<0x143, 0xc>(v, v));
  return lane_f64(v, 63);
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

template <int P>
__global__ __launch_bounds__(256) void topk_route_kernel(const RouteArgs a) {
  __shared__ double gkeys[4][64 * P];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const long long row = (long long)blockIdx.x * 4 + wave;
  if (row >= a.rows) return;               // no barrier below: a wave is on its own
  const double none = -__builtin_inf();
  float l[P];
  double s[P], key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = 64 * i + lane;
    l[i] = -__builtin_inff();
    if (e < a.E)
      l[i] = a.f32 ? reinterpret_cast<const float*>(a.logits)[row * a.ld + e]
                   : bf16_to_f32(reinterpret_cast<const uint16_t*>(a.logits)[row * a.ld + e]);
    // NaN is not larger than -inf; +inf is the largest finite value
    l[i] = l[i] > -__builtin_inff() ? fminf(l[i], 3.4028234663852886e38f) : -__builtin_inff();
  }
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < P; ++i) s[i] = 1.0 / (1.0 + exp(-(double)l[i]));
  } else {
    double top = none, sum = 0.0;
#pragma unroll
    for (int i = 0; i < P; ++i) top = fmax(top, (double)l[i]);
    top = wave_max(top);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      s[i] = l[i] > -__builtin_inff() ? exp((double)l[i] - top) : 0.0;
      sum += s[i];
    }
    sum = wave_add(sum);
#pragma unroll
    for (int i = 0; i < P; ++i) s[i] = l[i] > -__builtin_inff() ? s[i] / sum : 0.0;
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = 64 * i + lane;
    key[i] = s[i];
    if (a.bias && e < a.E) key[i] += (double)a.bias[e];
    // a key that is NaN (a bias that is) is never chosen either
    key[i] = l[i] > -__builtin_inff() && key[i] > none ? key[i] : none;
  }
  if (a.G > 1) {
    const int S = a.E / a.G;
#pragma unroll
    for (int i = 0; i < P; ++i) gkeys[wave][64 * i + lane] = key[i];
    __builtin_amdgcn_wave_barrier();
    // lane g: its group's two best keys
    double b1 = none, b2 = none;
    if (lane < a.G) {
      for (int j = 0; j < S; ++j) {
        const double v = gkeys[wave][lane * S + j];
        b2 = fmax(b2, fmin(b1, v));
        b1 = fmax(b1, v);
      }
    }
    const double sc = b1 > none ? b1 + (b2 > none ? b2 : 0.0) : none;
    int better = 0;
    for (int g = 0; g < a.G; ++g) {
      const double o = lane_f64(sc, g);
      better += o > sc || (o == sc && g < lane) ? 1 : 0;
    }
    const uint64_t may = __ballot(lane < a.G && sc > none && better < a.top_groups);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int e = 64 * i + lane;
      if (e >= a.E || !((may >> (e / S)) & 1)) key[i] = none;
    }
  }
  int my_id = -1;                          // lane j: the row's choice j
  double my_s = 0.0, total = 0.0;
  for (int j = 0; j < a.k; ++j) {
    double m = key[0];
#pragma unroll
    for (int i = 1; i < P; ++i) m = fmax(m, key[i]);
    m = wave_max(m);
    if (!(m > none)) break;
    int e = -1;
    double sv = 0.0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint64_t at = __ballot(key[i] == m);
      if (e < 0 && at) {
        const int w = __builtin_ctzll(at);
        e = 64 * i + w;
        sv = lane_f64(s[i], w);
        if (lane == w) key[i] = none;
      }
    }
    total += sv;
    if (lane == j) {
      my_id = e;
      my_s = sv;
    }
  }
  if (lane < a.k) {
    double w = my_s;
    if (a.normalize) w = total > 0.0 ? w / total : 0.0;
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
// launch of its own.
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
  __shared__ uint32_t cnt[GW][GBINS];
  __shared__ uint32_t tot[GBINS + 63];
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
  for (int i = tid; i < GW * GBINS; i += GT) (&cnt[0][0])[i] = 0;
  __syncthreads();
  for (long long i = w0 + lane; i < w1; i += 64) atomicAdd(&cnt[wave][bin_of(i)], 1u);
  __syncthreads();
  if constexpr (MODE == 1) {
    for (int g = tid; g < bins; g += GT) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < GW; ++w) t += cnt[w][g];
      a.counts[(long long)blockIdx.x * bins + g] = t;
    }
    return;
  }
  uint32_t before[2] = {0, 0};             // of this block's group, in earlier blocks
  for (int g = tid, r = 0; g < bins; g += GT, ++r) {
    uint32_t t = 0;
    if constexpr (MODE == 0) {
#pragma unroll
      for (int w = 0; w < GW; ++w) t += cnt[w][g];
    } else {
#pragma unroll 8
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const uint32_t v = a.counts[(long long)b * bins + g];
        if (b < (int)blockIdx.x) before[r] += v;
        t += v;
      }
    }
    tot[g] = t;
  }
  __syncthreads();
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
  for (int g = tid, r = 0; g < bins; g += GT, ++r) {
    uint32_t at = tot[g];
    if (blockIdx.x == 0) a.offsets[g] = (int32_t)at;
    at += before[r];
#pragma unroll
    for (int w = 0; w < GW; ++w) {
      const uint32_t t = cnt[w][g];
      cnt[w][g] = at;
      at += t;
    }
  }
  __syncthreads();
  for (long long i0 = w0; i0 < w1; i0 += 64) {
    const long long i = i0 + lane;
    const bool live = i < w1;
    const int g = live ? bin_of(i) : 0;
    const uint64_t peers = lanes_with(g, a.bits, __ballot(live));
    if (live) {
      const int rank = __popcll(peers & ((1ull << lane) - 1));
      const uint32_t pos = cnt[wave][g] + (uint32_t)rank;
      __builtin_amdgcn_wave_barrier();
      if ((peers >> lane) == 1ull) cnt[wave][g] = pos + 1;     // the last of its group
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
// two) a token, 8 columns a thread and step.
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

hipError_t launch_topk_route(const RouteArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.E < 1 || a.E > kRouteMaxExperts || a.G < 1 || a.G > 64 || a.E % a.G || a.k < 1 ||
      a.k > 64)
    return hipErrorInvalidValue;
  const dim3 grid((unsigned)((a.rows + 3) / 4));
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

// The blocks of n entries: one up to kGroupOne, else 4096 entries each, at most
// 128 (each block reads every block's counts).
constexpr int kGroupOne = 4096;
static int group_chunk(long long n) {
  if (n <= kGroupOne) return (int)(n > 0 ? n : 1);
  const long long c = (n + 127) / 128;
  return (int)(c <= 4096 ? 4096 : (c + 1023) / 1024 * 1024);
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

hipError_t launch_combine(CombineArgs a, hipStream_t s) {
  if (a.tokens <= 0 || a.N <= 0) return hipSuccess;
  if (a.N % 8 || a.k < 1) return hipErrorInvalidValue;
  a.tpr = 1;
  while (a.tpr < 256 && a.tpr * 8 < a.N) a.tpr *= 2;
  const int rpb = 256 / a.tpr;
  hipLaunchKernelGGL(combine_kernel, dim3((unsigned)((a.tokens + rpb - 1) / rpb)), dim3(256), 0, s,
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
