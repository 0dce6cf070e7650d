// The experts' products over ragged groups of rows: y[p] = x[row(p)] . W_e^T
// for the rows p of expert e's group, plain or SwiGLU-gated (kernels.h).
#include "common.h"
#include "kernels.h"
#include "row_groups.h"

namespace ming {
namespace {

__device__ __forceinline__ floatx4_t mfma16(const uint4& w, const uint4& x, floatx4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w),
                                                 __builtin_bit_cast(bf16x8_t, x), c, 0, 0, 0);
}
__device__ __forceinline__ float byte_f(uint32_t w, int i) { return (float)((w >> (8 * i)) & 0xffu); }
__device__ __forceinline__ float f16_lo(uint32_t u) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(u & 0xffffu));
}
__device__ __forceinline__ float f16_hi(uint32_t u) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
}

// One 64-group of weight row n, lane quarter g's 16 values as the A operands of two
// v_mfma_f32_16x16x32_bf16: dense weights as they are, w8 codes as the integers they
// hold, w4 codes as 16 more (0x4180 with the code in the upper four bits of its mantissa
// is that in bf16, so two codes are a v_perm; the group's bias takes the 16 scales off
// again, at sums of three times the codes' own: two bits of the f32 sums' 24, where the
// output keeps eight). Which k a quarter has is free as long as x's agree (x_at): they
// are what one wide load brings, with the lanes of a row side by side (w4 as two 4-byte
// loads a lane: [64][2048, 2048] gated, 8 places 13.9 us, 8.5 so).
template <int BITS>
struct Raw {
  uint4 v[BITS == 16 ? 2 : 1];
};
template <int BITS>
__device__ __forceinline__ void load_group(const ExpertsArgs& a, const void* w, int n, int kt,
                                           int g, Raw<BITS>& r) {
  if constexpr (BITS == 16) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(w) +
                                                    ((long long)kt * a.NW + n) * 64 + 8 * g);
    r.v[0] = p[0];
    r.v[1] = p[4];
  } else {
    // [kt][n][fk][kk] (w8: two words each): k 16 kk + 8 fk + 0..7, a quarter's kk 2 (g & 1)
    // and the next of fk g >> 1 in one load
    const uint32_t* p =
        static_cast<const uint32_t*>(w) + ((long long)kt * a.NW + n) * (2 * BITS) + BITS / 2 * g;
    if constexpr (BITS == 4) {
      const uint2 c = *reinterpret_cast<const uint2*>(p);
      r.v[0] = make_uint4(c.x, c.y, 0, 0);
    } else {
      r.v[0] = *reinterpret_cast<const uint4*>(p);
    }
  }
}
// k of quarter g's two 8-value pieces of x: the first, and how far the second.
template <int BITS>
__device__ __forceinline__ int x_at(int g) {
  return BITS == 16 ? 8 * g : 32 * (g & 1) + 8 * (g >> 1);
}
template <int BITS>
constexpr int kXStep = BITS == 16 ? 32 : 16;
template <int BITS>
__device__ __forceinline__ void operands(const Raw<BITS>& r, uint4& w0, uint4& w1) {
  if constexpr (BITS == 16) {
    w0 = r.v[0];
    w1 = r.v[1];
  } else {
    [[maybe_unused]] auto bytes = [](uint32_t c, uint32_t d) {
      uint4 o;
      o.x = pack_bf16x2_rne(byte_f(c, 0), byte_f(c, 1));
      o.y = pack_bf16x2_rne(byte_f(c, 2), byte_f(c, 3));
      o.z = pack_bf16x2_rne(byte_f(d, 0), byte_f(d, 1));
      o.w = pack_bf16x2_rne(byte_f(d, 2), byte_f(d, 3));
      return o;
    };
    if constexpr (BITS == 4) {
      // nibbles {k0,k4,k1,k5,k2,k6,k3,k7}: the even ones are k0..k3 by byte
      auto word = [](uint32_t c) {
        const uint32_t lo = ((c << 3) & 0x78787878u) | 0x80808080u;
        const uint32_t hi = ((c >> 1) & 0x78787878u) | 0x80808080u;
        return make_uint4(__builtin_amdgcn_perm(0x41414141u, lo, 0x05010400u),
                          __builtin_amdgcn_perm(0x41414141u, lo, 0x05030402u),
                          __builtin_amdgcn_perm(0x41414141u, hi, 0x05010400u),
                          __builtin_amdgcn_perm(0x41414141u, hi, 0x05030402u));
      };
      w0 = word(r.v[0].x);
      w1 = word(r.v[0].y);
    } else {
      w0 = bytes(r.v[0].x, r.v[0].y);
      w1 = bytes(r.v[0].z, r.v[0].w);
    }
  }
}

// ---- few rows an expert --------------------------------------------------------
// A block takes 16 output columns of one expert with rows, 16 of its rows at a
// time, its WK waves each a residue class of K's 64-groups; the sums meet in
// LDS and are added in class order, so the bits depend on K alone. Quantized
// weights multiply as integers: scale * sum(q x) + bias * sum(x) a group, in
// f32, the activations as the bf16 they are (no range limit). Bound by HBM:
// the weights of the experts that have rows, once (w4 and w8, by the loads beside
// them, x and scales: 6 and 5 weights a ps). Blocks of 16 (gated) or 32 columns leave
// thousands of them, so loads of many are in flight: [64][2048, 2048] dense, gated,
// 64 places 54 to 56 us, 303 MB at 5.5 TB/s; [60][2048, 1024] w8, 16 places 10.9.
//
// WK waves with U groups in flight, by K: 8 with 2 (4 cost registers, so waves: 20 to
// 55% longer), to K = 1024 with 1 ([60][2048, 1024] w8, 64 places 31.1 -> 26.0 us; K 7168
// 8% slower), to 512 4 waves ([64][2048, 512] w8 gated, 64 places 14.1, eight 19.4). CO
// 16-column tiles of the output by experts_rows_tiles.
template <int BITS, bool GATED, int WK, int U, int CO>
__global__ __launch_bounds__(64 * WK) void experts_rows_kernel(const ExpertsArgs a) {
  constexpr int CT = GATED ? 2 * CO : CO;  // column tiles: the outputs', then the up rows'
  const RowGroup rg =
      find_group(a.offsets, a.E, a.n, [](int) { return 1; }, [](int) { return (int)blockIdx.y; });
  if (rg.e < 0) return;
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16 * CO;
  const int KT = a.K / 64;
  const long long words = (long long)a.NW * a.K * BITS / 32;
  const void* const w = BITS == 16
                            ? (const void*)(a.w16 + (long long)rg.e * a.NW * a.K)
                            : (const void*)(a.codes + (long long)rg.e * words);
  const uint32_t* const sbp = a.sb + (long long)rg.e * a.NW * KT;
  const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
  __shared__ floatx4_t red[WK][CT][64];
  for (int r0 = 0; r0 < rg.rows; r0 += 16) {
    const bool row = c < rg.rows - r0;     // lanes past the rows multiply row r0, never store
    const int p = rg.p0 + r0 + (row ? c : 0);
    int src = p;
    if (a.order) {
      src = a.order[p] / a.fan;
      src = src < 0 ? 0 : src < a.x_rows ? src : a.x_rows - 1;
    }
    const uint16_t* const xr = a.x + (long long)src * a.ldx + x_at<BITS>(g);
    floatx4_t acc[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[t] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = wave; k0 < KT; k0 += WK * U) {
      Raw<BITS> wr[U][CT];
      uint4 x[U][2];
      [[maybe_unused]] uint4 sb[U][CT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kt = k0 + WK * u;
        if (kt < KT) {
          const uint4* xp = reinterpret_cast<const uint4*>(xr + 64 * kt);
          x[u][0] = xp[0];
          x[u][1] = xp[kXStep<BITS> / 8];
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            // columns past N (a multiple of 8) compute the last ones, never store
            const int n = n0 + 16 * (t % CO) + c;
            load_group<BITS>(a, w, (n < a.N ? n : a.N - 1) + t / CO * a.N, kt, g, wr[u][t]);
            if constexpr (BITS != 16) {
              const int ns = n0 + 16 * (t % CO) + 4 * g;
              sb[u][t] = *reinterpret_cast<const uint4*>(sbp + (long long)kt * a.NW + t / CO * a.N +
                                                         (ns < a.N ? ns : a.N - 4));
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k0 + WK * u < KT) {
          [[maybe_unused]] floatx4_t sx;
          const floatx4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (BITS != 16) sx = mfma16(ones, x[u][1], mfma16(ones, x[u][0], zero));
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            uint4 w0, w1;
            operands<BITS>(wr[u][t], w0, w1);
            if constexpr (BITS == 16) {
              acc[t] = mfma16(w0, x[u][0], acc[t]);
              acc[t] = mfma16(w1, x[u][1], acc[t]);
            } else {
              const floatx4_t d = mfma16(w1, x[u][1], mfma16(w0, x[u][0], zero));
              const uint32_t* sp = &sb[u][t].x;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float s = f16_lo(sp[r]);
                const float b = BITS == 4 ? __builtin_fmaf(-16.0f, s, f16_hi(sp[r])) : f16_hi(sp[r]);
                acc[t][r] += __builtin_fmaf(s, d[r], b * sx[r]);
              }
            }
          }
        }
      }
    }
    // lane (m = c, g): columns 4g + 0..3 of each 16, row m; wave t finishes tile t
#pragma unroll
    for (int t = 0; t < CT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    const int n = n0 + 16 * wave + 4 * g;
    if (wave < CO && row && n < a.N) {
      floatx4_t v = red[0][wave][lane];
#pragma unroll
      for (int j = 1; j < WK; ++j) v += red[j][wave][lane];
      if constexpr (GATED) {
        floatx4_t u = red[0][CO + wave][lane];
#pragma unroll
        for (int j = 1; j < WK; ++j) u += red[j][CO + wave][lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = silu_f(v[r]) * u[r];
      }
      *reinterpret_cast<uint2*>(a.y + (long long)(rg.p0 + r0 + c) * a.ldy + n) =
          make_uint2(pack_bf16x2_rne(v[0], v[1]), pack_bf16x2_rne(v[2], v[3]));
    }
    __syncthreads();                       // the sums are read: the next rows' may come
  }
}

template <int BITS, bool GATED, int WK, int U, int CO>
void rows_launch(const ExpertsArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.N + 16 * CO - 1) / (16 * CO)), (unsigned)(a.n < a.E ? a.n : a.E));
  hipLaunchKernelGGL((experts_rows_kernel<BITS, GATED, WK, U, CO>), grid, dim3(64 * WK), 0, s, a);
}

template <int BITS, bool GATED>
void rows_shape(const ExpertsArgs& a, hipStream_t s) {
  constexpr int CO = GATED ? 1 : 2;
  if (a.K <= 512)
    rows_launch<BITS, GATED, 4, 1, CO>(a, s);
  else if (a.K <= 1024)
    rows_launch<BITS, GATED, 8, 1, CO>(a, s);
  else if (experts_rows_tiles(device_cus(), BITS, GATED, a.E, a.N, a.K, a.n) == CO)
    rows_launch<BITS, GATED, 8, 2, CO>(a, s);
  else if constexpr (BITS == 16)
    rows_launch<BITS, GATED, 8, 2, 1>(a, s);
}

// w [NW][K] -> [K / 64][NW][64], 16 bytes a thread and step.
__global__ void repack_dense_kernel(const uint16_t* w, int NW, int K, uint16_t* out) {
  const long long total = (long long)NW * K / 8;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const int c = (int)(i & 7);
    const long long r = i >> 3;
    const int n = (int)(r % NW), kt = (int)(r / NW);
    reinterpret_cast<uint4*>(out)[i] =
        *reinterpret_cast<const uint4*>(w + (long long)n * K + 64 * kt + 8 * c);
  }
}

}  // namespace

// One gated (the up rows are a second one), 2 plain (1 is 7 to 30% longer up to K = 1024
// and with quantized weights, 4 as much). Dense plain ones past K = 1024 are 1 where
// blocks of 2 would leave CUs idle, and from K = 1536 on. Microseconds of 2 and 1:
// [64][1024, 1088 to 2048], one and 4 places (32 and 128 blocks of 2) 5.3 to 7.5 and 4.5 to
// 6.2; with more blocks, [64][1024, 1088], 16 places 8.8 and 9.4, [60][2048, 1088] 14.8 and
// 16.4, [60][2048, 1408] 18.8 and 20.2; [16][2048, 1536], 32 places 17.8 and 16.4, 64 21.5 and
// 23.1; [64][1024, 1792], 16 places 11.7 and 10.3; [128][512, 2048], 16 places 8.6 and 9.2;
// [16][2048, 4096], 16 places 36.3 and 31.0; [16][1024, 7168], 8 places 18.7 and 20.0, 16 38.9
// and 32.0.
int experts_rows_tiles(int cus, int bits, bool gated, int E, int N, int K, int n) {
  if (gated) return 1;
  if (bits != 16 || K <= 1024) return 2;
  return K >= 1536 || (long long)(n < E ? n : E) * ((N + 31) / 32) < cus ? 1 : 2;
}

hipError_t launch_repack_dense(const uint16_t* w, int NW, int K, uint16_t* out, hipStream_t s) {
  if (NW <= 0 || K <= 0 || K % 64) return hipErrorInvalidValue;
  const long long blocks = ((long long)NW * K / 8 + 255) / 256;
  hipLaunchKernelGGL(repack_dense_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256),
                     0, s, w, NW, K, out);
  return hipGetLastError();
}

hipError_t launch_experts_rows(int bits, bool gated, const ExpertsArgs& a, hipStream_t s) {
  if (a.n <= 0 || a.N <= 0) return hipSuccess;
  if (a.K % 64 || a.N % 8 || a.NW != a.N * (gated ? 2 : 1) || a.E < 1 || a.fan < 1 || a.x_rows < 1)
    return hipErrorInvalidValue;
  switch (bits) {
    case 4: gated ? rows_shape<4, true>(a, s) : rows_shape<4, false>(a, s); break;
    case 8: gated ? rows_shape<8, true>(a, s) : rows_shape<8, false>(a, s); break;
    case 16: gated ? rows_shape<16, true>(a, s) : rows_shape<16, false>(a, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t validate_experts_kernels() {
  hipFuncAttributes fa;
  const void* fns[] = {
#define MING_EXPERTS_ROWS(BITS)                                                   \
  reinterpret_cast<const void*>(&experts_rows_kernel<BITS, false, 4, 1, 2>),      \
      reinterpret_cast<const void*>(&experts_rows_kernel<BITS, false, 8, 1, 2>),  \
      reinterpret_cast<const void*>(&experts_rows_kernel<BITS, false, 8, 2, 2>),  \
      reinterpret_cast<const void*>(&experts_rows_kernel<BITS, true, 4, 1, 1>),   \
      reinterpret_cast<const void*>(&experts_rows_kernel<BITS, true, 8, 1, 1>),   \
      reinterpret_cast<const void*>(&experts_rows_kernel<BITS, true, 8, 2, 1>)
      reinterpret_cast<const void*>(&repack_dense_kernel),
      reinterpret_cast<const void*>(&experts_rows_kernel<16, false, 8, 2, 1>),
      MING_EXPERTS_ROWS(4), MING_EXPERTS_ROWS(8), MING_EXPERTS_ROWS(16)
#undef MING_EXPERTS_ROWS
  };
  for (const void* f : fns) {
    const hipError_t e = hipFuncGetAttributes(&fa, f);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ming
