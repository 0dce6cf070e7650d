// What makes the operands of the 8-bit products: rows of bf16 into e4m3 codes with
// a scale for each 128 columns, the same from an RMSNorm with the residual's
// addition before it, and weights in blocks of 128 x 128.
//
// One pass: everything between the loads and the stores is in registers. The quantizer is
// bound by HBM. The norm stays at a copy's 5.1 TB/s (an addition of two arrays reaches 6.0 to
// 6.2): a lane's 16 columns are two stores of 16 bytes to h and to y, so a wave's store takes
// every other 16 bytes, half of each line, and cannot go past the caches (46 -> 72 us).
// Measured out of cold caches: quantizing 8704 x 3840 16.1 us (6.2 TB/s), the norm of
// 8704 x 3840 with the residual 46.0 (5.1). Small ones take what a call costs the host:
// eight rows quantized 3.8 to 4.1 (2.5 in the kernel), a row's norm 4.6 to 5.0 (2.5), 203 x
// 2048 with y 4.6 to 5.0 (3.6).
#include "common.h"
#include "f8.h"
#include "kernels.h"

namespace ming {
namespace {

// 16 columns' codes by the scale of bits sb.
__device__ __forceinline__ uint4 f8_codes16(const float (&v)[16], uint32_t sb) {
  const float s = __uint_as_float(sb << 16), y = 1.0f / s;
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = f8_pack4(f8_quotient(v[4 * i], s, y), f8_quotient(v[4 * i + 1], s, y),
                    f8_quotient(v[4 * i + 2], s, y), f8_quotient(v[4 * i + 3], s, y));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

__device__ __forceinline__ void unpack8(const uint4& u, float* v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
  }
}
// The largest of the 8 lanes that hold a block of 128 columns.
__device__ __forceinline__ uint32_t top8(uint32_t t) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const uint32_t v = (uint32_t)__shfl_xor((int)t, o, 64);
    t = t > v ? t : v;
  }
  return t;
}

// A thread takes 16 columns, 8 threads a block of 128, `per` threads a row: a block's
// largest takes three shuffles, and a thread's codes are one store of 16 bytes.
__global__ __launch_bounds__(256) void f8_quantize_kernel(const F8QuantArgs a, int per) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = i / (uint32_t)per;
  const int c = (int)(i - row * (uint32_t)per);
  const bool in = row < (uint32_t)a.rows && 16 * c < a.D;
  float v[16];
  uint32_t top = 0;
  if (in) {
    const uint4* p = reinterpret_cast<const uint4*>(a.x + (long long)row * a.ldx + 16 * c);
    const uint4 u0 = p[0], u1 = p[1];
    unpack8(u0, v);
    unpack8(u1, v + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) top = f8_top(top, v[e]);
  }
  top = top8(top);
  if (!in) return;
  const float t = __uint_as_float(top);
  const bool fine = f8_finite(t);
  const uint32_t sb = fine ? f8_scale_bits(t) : kF8NanScale;
  f8_store16(a.codes + (long long)row * a.ldc + 16 * c,
             fine ? f8_codes16(v, sb) : make_uint4(kF8Nan4, kF8Nan4, kF8Nan4, kF8Nan4), a.stream);
  if ((c & 7) == 0) a.scales[(long long)(c >> 3) * a.lds + row] = (uint16_t)sb;
}

// A workgroup takes a row, 16 columns a thread: one pass over memory, the row stays in
// registers between the sum of squares and the codes. The codes are of the f32
// values, not of a bf16 norm: one rounding where two would do worse.
template <bool ADD>
__global__ __launch_bounds__(512) void f8_norm_kernel(const F8NormArgs a) {
  __shared__ float part[8];
  const int c = (int)threadIdx.x, row = (int)blockIdx.x;
  const bool in = 16 * c < a.D;
  float v[16], ss = 0.0f;
  uint4 u[2];
  if (in) {
    const uint4* p = reinterpret_cast<const uint4*>(a.x + (long long)row * a.ldx + 16 * c);
    u[0] = p[0];
    u[1] = p[1];
    unpack8(u[0], v);
    unpack8(u[1], v + 8);
    if constexpr (ADD) {
      const uint4* q = reinterpret_cast<const uint4*>(a.sub + (long long)row * a.ldsub + 16 * c);
      const uint4 s0 = q[0], s1 = q[1];
      float s[16];
      unpack8(s0, s);
      unpack8(s1, s + 8);
      // the sum is rounded to bf16 as it is stored: the norm is of what goes on
      uint32_t* up = &u[0].x;
#pragma unroll
      for (int e = 0; e < 8; ++e) up[e] = pack_bf16x2_rne(v[2 * e] + s[2 * e], v[2 * e + 1] + s[2 * e + 1]);
      uint4* h = reinterpret_cast<uint4*>(a.h + (long long)row * a.ldh + 16 * c);
      h[0] = u[0];
      h[1] = u[1];
      unpack8(u[0], v);
      unpack8(u[1], v + 8);
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) ss = fmaf(v[e], v[e], ss);
  }
  uint4 w0, w1;
  if (in) {
    const uint4* p = reinterpret_cast<const uint4*>(a.w + 16 * c);
    w0 = p[0];
    w1 = p[1];
  }
  ss = warp_sum(ss);
  const int waves = (int)blockDim.x >> 6;
  if (waves > 1) {
    if ((c & 63) == 0) part[c >> 6] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int i = 0; i < waves; ++i) ss += part[i];
  }
  const float inv = 1.0f / sqrtf(ss / (float)a.D + a.eps);
  uint32_t top = 0;
  if (in) {
    float w[16];
    unpack8(w0, w);
    unpack8(w1, w + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      v[e] = v[e] * inv * w[e];            // (inv * w may leave f32 where this does not)
      top = f8_top(top, v[e]);
    }
  }
  top = top8(top);
  if (!in) return;
  // not where the block holds inf or NaN, or the row's mean square does: inv is then 0
  // or NaN
  const float t = __uint_as_float(top);
  const bool fine = f8_finite(t) && inv > 0.0f;
  const uint32_t sb = fine ? f8_scale_bits(t) : kF8NanScale;
  *reinterpret_cast<uint4*>(a.codes + (long long)row * a.ldc + 16 * c) =
      fine ? f8_codes16(v, sb) : make_uint4(kF8Nan4, kF8Nan4, kF8Nan4, kF8Nan4);
  if ((c & 7) == 0) a.scales[(long long)(c >> 3) * a.lds + row] = (uint16_t)sb;
  if (a.y) {
    uint32_t y[8];
    // a row without a mean square has no norm: v would be zeros where inv is 0
#pragma unroll
    for (int e = 0; e < 8; ++e)
      y[e] = inv > 0.0f ? pack_bf16x2_rne(v[2 * e], v[2 * e + 1]) : kF8NanScale * 0x10001u;
    uint4* p = reinterpret_cast<uint4*>(a.y + (long long)row * a.ldy + 16 * c);
    p[0] = make_uint4(y[0], y[1], y[2], y[3]);
    p[1] = make_uint4(y[4], y[5], y[6], y[7]);
  }
}

// A workgroup takes 128 x 128 weights, half a row a thread. Their scale is an f32, as
// checkpoints hold it: a / 448; the codes go by 448 v / a (whose borders the rounding of
// the scale would move) as 512 times the quotient of 0.875 v, which stays below a.
__global__ __launch_bounds__(256) void f8_weight_kernel(const uint16_t* w, int N, int K,
                                                        uint8_t* codes, float* scales) {
  __shared__ uint32_t part[4];
  const int kb = (int)blockIdx.x, nb = (int)blockIdx.y;
  const int n = 128 * nb + ((int)threadIdx.x >> 1), k0 = 128 * kb + 64 * ((int)threadIdx.x & 1);
  const uint16_t* p = w + (long long)n * K + k0;
  uint32_t top = 0;
  float v[16];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n < N && k0 + 16 * j < K) {
      unpack8(reinterpret_cast<const uint4*>(p + 16 * j)[0], v);
      unpack8(reinterpret_cast<const uint4*>(p + 16 * j)[1], v + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) top = f8_top(top, v[e]);
    }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = (uint32_t)__shfl_xor((int)top, o, 64);
    top = top > t ? top : t;
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = top > part[i] ? top : part[i];
  const float t = __uint_as_float(top), m = fmaxf(t, kF8Least), y = 1.0f / m;
  const bool fine = f8_finite(t);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n < N && k0 + 16 * j < K) {
      unpack8(reinterpret_cast<const uint4*>(p + 16 * j)[0], v);
      unpack8(reinterpret_cast<const uint4*>(p + 16 * j)[1], v + 8);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = fine ? f8_pack4(512.0f * f8_quotient(0.875f * v[4 * i], m, y),
                               512.0f * f8_quotient(0.875f * v[4 * i + 1], m, y),
                               512.0f * f8_quotient(0.875f * v[4 * i + 2], m, y),
                               512.0f * f8_quotient(0.875f * v[4 * i + 3], m, y))
                    : kF8Nan4;
      *reinterpret_cast<uint4*>(codes + (long long)n * K + k0 + 16 * j) =
          make_uint4(o[0], o[1], o[2], o[3]);
    }
  if (threadIdx.x == 0)
    scales[(long long)nb * gridDim.x + kb] = fine ? m / kF8Most : __uint_as_float(0x7fc00000u);
}

int quant_threads(int D) { return (D + 127) / 128 * 8; }

}  // namespace

long long f8_quantize_blocks(long long rows, int D) {
  return (rows * quant_threads(D) + 255) / 256;
}

hipError_t launch_f8_quantize(const F8QuantArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.D <= 0 || a.D % 16 || !one_launch(f8_quantize_blocks(a.rows, a.D), 256))
    return hipErrorInvalidValue;
  hipLaunchKernelGGL(f8_quantize_kernel, dim3((unsigned)f8_quantize_blocks(a.rows, a.D)), dim3(256),
                     0, s, a, quant_threads(a.D));
  return hipGetLastError();
}

hipError_t launch_f8_norm(const F8NormArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.D <= 0 || a.D % 16 || a.D > 8192) return hipErrorInvalidValue;
  const dim3 grid((unsigned)a.rows), block((unsigned)((a.D + 1023) / 1024 * 64));
  if (a.sub)
    hipLaunchKernelGGL((f8_norm_kernel<true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((f8_norm_kernel<false>), grid, block, 0, s, a);
  return hipGetLastError();
}

hipError_t launch_f8_weight(const uint16_t* w, int N, int K, uint8_t* codes, float* scales,
                            hipStream_t s) {
  if (N <= 0 || K <= 0 || K % 16) return hipErrorInvalidValue;
  hipLaunchKernelGGL(f8_weight_kernel, dim3((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128)),
                     dim3(256), 0, s, w, N, K, codes, scales);
  return hipGetLastError();
}

hipError_t validate_f8_quant_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {reinterpret_cast<const void*>(&f8_quantize_kernel),
                       reinterpret_cast<const void*>(&f8_norm_kernel<true>),
                       reinterpret_cast<const void*>(&f8_norm_kernel<false>),
                       reinterpret_cast<const void*>(&f8_weight_kernel)};
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
