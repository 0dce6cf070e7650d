// Host-side launch interface of the HIP kernels (internal to the library;
// the public boundary is include/ming_dit_amd.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ming {

// A launch holds 2^32 - 1 threads along x.
inline bool one_launch(long long blocks, int threads) { return blocks <= 0xffffffffll / threads; }

// ---- quantized / dense projection GEMM with the LoRA tail ------------------
//
// y[m][n] = sum_k x[m][k] W[n][k]  (+ sum_r T[m][seg.t_col0 + r] B[n][r])
//
// W is resident in the tiled layout built by repack_* (K-tile major):
//   bits 4:  codes[kt][n][8]  u32, nibble i of word j holds k = 8j + perm(i)
//            with perm = {0,2,4,6,1,3,5,7}
//   bits 8:  codes[kt][n][16] u32, byte i of word j holds k = 4j + i
//   bits 16: dense bf16 w[n][k] (the checkpoint's own layout)
//   sb[kt][n] = bf16 scale | bf16 bias << 16 (bits 4 and 8)
// T is the LoRA intermediate [M][ldt] bf16 (already scaled), B the
// segment's factors [N_seg][ldb] bf16, gathered per 8-wide rank group by
// `grp` (B column / 8, or -1 for a zero group).
constexpr int kQpBM = 256, kQpBN = 256, kQpBK = 64, kQpThreads = 256;
constexpr int kMaxSeg = 4;
constexpr int kMaxGroups = 512;   // 8-wide rank groups per call (4096 ranks)

struct QprojSeg {
  int n_begin;          // first output column of this segment
  int n_end;
  int t_col0;           // first T column of this segment's live ranks
  int chunks;           // live rank chunks of 32 (0: no adapter)
  int ldb;
  int grp0;             // first entry of this segment in grp[]
  const uint16_t* B;    // row (n - n_begin)
};

// A further projection of a merged launch: of the first one's shape, bits and
// ldy, one segment, its groups in the first one's grp[].
struct QprojMore {
  const uint32_t* codes;
  const uint32_t* sb;
  const uint16_t* w16;
  uint16_t* y;
  QprojSeg seg;
};

// Adapters that rows choose (adapters.hip): row m adds T[m] . B_a^T of adapter a
// = rid[m] (-1: none), T[m] = strength * fold * (x[m] . A_a^T) in bf16.
struct AdapterEntry {
  const uint16_t* A;    // in operand order (launch_repack_adapter), rows past the rank zero
  const uint16_t* B;    // [N][r8], columns past the rank zero
  int r8;               // rank padded to 8; 0: nothing bound
  float fold;
};
struct RowAdapters {
  const int32_t* rid;   // [M]
  const uint16_t* t;    // [M][ldt]
  int ldt;
  const AdapterEntry* table;
  // For the tile kernels' tails: per row tile the 32-rank chunks of the adapters
  // its rows name (RowChunk, `stride` a tile), how many, and T's row of zeros as a
  // byte offset from t.
  const uint4* chunks;
  const int32_t* counts;
  int stride;
  uint32_t zero;
};
// A chunk of a tile's tail as the kernels read it (one 16-byte scalar load).
struct RowChunk {
  const uint16_t* B;    // the adapter's factor at the chunk's first rank
  int32_t id;
  uint32_t shape;       // r8 | chunk << 12 | (live 8-rank groups - 1) << 20
};

struct RowXaArgs;

struct QprojArgs {
  const uint16_t* x;
  long long ldx;
  const uint32_t* codes;
  const uint32_t* sb;
  const uint16_t* w16;
  uint16_t* y;
  long long ldy;
  int M, N, K;
  const uint16_t* t;
  int ldt;
  int nseg;
  // optional SwiGLU gate: when g != nullptr the output is
  // y = bf16(silu(g) * bf16(x . W^T + LoRA)) (g bf16 [M][ldg], may equal y)
  const uint16_t* g;
  long long ldg;
  // optional fp16 copy of the (final) output, [M][ldyh], 16-byte aligned,
  // ldyh % 8 == 0: the next projection's fast-route input (fast kernel only)
  uint16_t* yh;
  long long ldyh;
  QprojSeg seg[kMaxSeg];
  int16_t grp[kMaxGroups];
  // fast route, split K (kslices > 1): f32 partials [kslices][M][N] in part,
  // summed in slice order by a second launch (N % 4 == 0)
  float* part;
  int kslices;
  int split_rf;         // rows per tile / 32 of a split launch (qproj_split_plan)
  // optional: set to 1 when an fp16 conversion of this launch (the general
  // kernel's x tiles, the fast epilogue's yh) met a bf16 value of magnitude
  // >= 2^16, inf or NaN (see range_report)
  int* range;
  // The paired gated launch (launch_qproj_pair): the weight above is the
  // gate projection (one segment, seg[0]) and (codes_u, sb_u, seg_u) the up
  // projection of the same shape, its groups in grp[] from seg_u.grp0, its
  // T columns in the same t; y = bf16(silu(bf16(gate)) * bf16(up)).
  const uint32_t* codes_u;
  const uint32_t* sb_u;
  QprojSeg seg_u;
  // a merged launch (launch_qproj_merged): nw projections over one x, the
  // second and third here; partials [nw][kslices][M][N]
  int nw;
  QprojMore more[2];
  // optional bias [N] bf16, added to the f32 result before the output's one
  // bf16 rounding (dense weights: ming_lin_bias)
  const uint16_t* bias;
  // optional f32 [M][N], added like the bias: what rows' own adapters add
  const float* delta;
  // rows' own adapters (no segments' adapters then): as a tail of the tiles
  // (launch_qproj_fast and launch_dense_fast) where counts is set, in the sum of a
  // K split where rid alone is
  RowAdapters rows;
};

// wide: bits 4/8 run with bf16 activations and the weight as a bf16 pair
// hi + lo (two passes over K): no fp16 anywhere, any finite input.
hipError_t launch_qproj(int bits, const QprojArgs& a, hipStream_t s, bool wide = false);

// Dense attention, head dim 128: O = softmax(scale * Q K^T) V per head.
// q, k: token-major rows (head h at column 128h); vt: V^T [NH][128][ldv]
// written by the launch from v (token-major), keys zero-padded to ldv (a
// multiple of 64 >= R); o: token-major [R][NH*128]. sl2 = scale * log2(e).
struct AttnArgs {
  const uint16_t* q;
  long long ldq;
  const uint16_t* k;
  long long ldk;
  const uint16_t* vt;
  int ldv;
  uint16_t* o;
  long long ldo;
  // optional per-head RMSNorm + RoPE of q, applied to the Q fragments as
  // they are loaded (launch_qk_norm_rope's arithmetic and bits): weight
  // qw[128], tables [R][64]; q is then the raw projection output
  const uint16_t* qw;
  const float* cos_t;
  const float* sin_t;
  float eps;
  // optional fp16 copy of O (the same bf16 values), [R][NH*128] at ldoh: the
  // fast projection route's input for the o-projection
  uint16_t* oh;
  long long ldoh;
  int* range;           // optional: raised as QprojArgs::range for oh
  int R, NH;
  float sl2;
};
hipError_t launch_attention(const AttnArgs& a, const uint16_t* v, long long ldv_in,
                            hipStream_t s);
hipError_t validate_attention_kernels();

// T[m][c] = bf16(coef[c/16] * sum_k x[m][k] A[row(c)][k]) for c < n_cols,
// row(c) = 16*grp[c/16] + c%16 (grp -1: a zero column). A is [R][K] bf16.
// Up to this many projections share one x.A launch (q, k, v; w1, w3).
constexpr int kMaxXaSources = 4;
// A tile of the fast x.A kernel: 64*mr rows x 64*cj columns.
struct XaTile {
  int mr, cj;
};
struct LoraXaArgs {
  const uint16_t* x;
  long long ldx;
  // A stacks [rows][K]: group entry g reads rows 8 * (g & 4095) + 0..7 of
  // A[g >> 12]; a negative entry is a zero (padding) group
  const uint16_t* A[kMaxXaSources];
  int K;
  int M;
  int n_cols;           // multiple of 64
  uint16_t* t;
  int ldt;
  int16_t grp[kMaxGroups];
  float coef[kMaxGroups];
  // optional (fast kernel only): the fp16 copy of x, [M][ldxh], 16-byte
  // aligned, ldxh % 8 == 0, written by the launch as it stages x (each
  // element once); range as in QprojArgs
  uint16_t* xh;
  long long ldxh;
  int* range;
  // optional (fast kernel only): bias [n_cols] bf16, T = bf16(coef * sum +
  // bias) -- the dense split-K GEMM's ming_lin_bias
  const uint16_t* bias;
  // or what rows' own adapters add (rid NULL: nothing); with one slice as the f32
  // plane [M][n_cols] of it
  RowAdapters rows;
  const float* delta;
  // fast kernel only: a dense weight's split-K GEMM. Column c is row c of
  // A[0], coefficient 1 (grp and coef unused), in tiles of `tile`
  bool ident;
  XaTile tile;
};
hipError_t launch_lora_xa(const LoraXaArgs& a, hipStream_t s);

// Repack the reference pack (codes [N][K*bits/32] u32 LSB-first,
// scales/biases bf16 [N][K/64]) into the tiled resident layout.
hipError_t launch_repack(int bits, const uint32_t* codes,
                         const uint16_t* scales, const uint16_t* biases,
                         int N, int K, uint32_t* codes_t, uint32_t* sb,
                         hipStream_t s);

// ---- norms and rotary --------------------------------------------------------
hipError_t launch_rmsnorm(const uint16_t* x, long long ldx, const uint16_t* w,
                          uint16_t* y, long long ldy, int rows, int D,
                          float eps, hipStream_t s);
// mode 0 plain; 1 also h = fp16(y); 2 h = bf16(h + tg * y) with tg = tanh(gate)
// in f32, y unused; 3 h = bf16(h + y) (see rmsnorm_kernel)
// `range` (optional, mode 1): raised as QprojArgs::range for the fp16 copy
hipError_t launch_rmsnorm_ex(int mode, const uint16_t* x, long long ldx, const uint16_t* w,
                             uint16_t* y, long long ldy, uint16_t* h, long long ldh,
                             const float* tg, int rows, int D, float eps,
                             hipStream_t s, int* range = nullptr);
// t[i] = tanhf(bf16 g[i]) for the two gates of a block's adaLN output:
// g = mods + n (gate_msa) and mods + 3n (gate_mlp) -> t[0, n) and t[n, 2n)
hipError_t launch_tanh_gates(const uint16_t* mods, int n, float* t, hipStream_t s);
// mods[4n] = bf16(mods + b) in place; nw1 = bf16(an1 * (1 + mods[0, n))),
// nw3 = bf16(fn1 * (1 + mods[2n, 3n))); t as launch_tanh_gates
// launch_adaln_glue over up to kGemvBatch blocks in one launch (grid y = entry).
struct GlueEntry {
  uint16_t* mods;
  const uint16_t* b;
  const uint16_t* an1;
  const uint16_t* fn1;
  uint16_t* nw1;
  uint16_t* nw3;
  float* t;
};
struct GlueBatch {
  int n;
  int count;
  GlueEntry e[32];
};
hipError_t launch_adaln_glue_batch(const GlueBatch& b, hipStream_t s);
hipError_t launch_adaln_glue(uint16_t* mods, int n, const uint16_t* b, const uint16_t* an1,
                             const uint16_t* fn1, uint16_t* nw1, uint16_t* nw3, float* t,
                             hipStream_t s);
hipError_t launch_rope_table(const int32_t* pt, const int32_t* ph,
                             const int32_t* pw, int n, int a0, int a1, int a2,
                             int head_dim, double theta, float* cos_t,
                             float* sin_t, hipStream_t s);
// h = bf16(h + (tg *) rmsnorm(sub) * wpost) then y = rmsnorm(h) * wpre and
// yh = fp16(y): the residual modes followed by mode 1, bit for bit, in one pass.
hipError_t launch_norm_residual_norm(const uint16_t* sub, long long lds, const uint16_t* wpost,
                                     uint16_t* h, long long ldh, const float* tg,
                                     const uint16_t* wpre, uint16_t* y, long long ldy,
                                     uint16_t* yh, long long ldyh, int rows, int D, float eps,
                                     hipStream_t s, int* range = nullptr);
// The same on k alone (the attention kernel norms q itself).
hipError_t launch_k_norm_rope(uint16_t* x, long long ld, int k_col, int rows, int n_heads,
                              const uint16_t* wk, const float* cos_t, const float* sin_t,
                              float eps, hipStream_t s);
// LlmOps::qk_norm_rope: heads [0, nq) then nk from column 0, norm when both
// weights are given, rotate-half of half-width rot_half (0, 32, 64) by
// tables [rows][rot_half].
hipError_t launch_llm_qk_norm_rope(uint16_t* x, long long ld, int rows, int nq, int nk,
                                   const uint16_t* wq, const uint16_t* wk, const float* cos_t,
                                   const float* sin_t, int rot_half, float eps, hipStream_t s);
hipError_t launch_qk_norm_rope(uint16_t* x, long long ld, int q_col,
                               int k_col, int rows, int n_heads,
                               const uint16_t* wq, const uint16_t* wk,
                               const float* cos_t, const float* sin_t,
                               float eps, hipStream_t s);

// ---- block glue and the pack quantizer (elementwise.hip) ----------------------
hipError_t launch_swiglu(const uint16_t* g, long long ldg, const uint16_t* u,
                         long long ldu, uint16_t* out, long long ldo, int rows,
                         int n, hipStream_t s);
hipError_t launch_residual(uint16_t* h, long long ldh, const uint16_t* gate,
                           const uint16_t* sub, long long lds, int rows, int n,
                           int gated, hipStream_t s);
hipError_t launch_modulate(const uint16_t* x, long long ldx,
                           const uint16_t* scale, uint16_t* y, long long ldy,
                           int rows, int n, hipStream_t s);
hipError_t launch_bias_act(uint16_t* y, long long ldy, const uint16_t* b,
                           uint16_t* out2, int rows, int n, int mode,
                           hipStream_t s);
hipError_t launch_ln_modulate(const uint16_t* x, long long ldx,
                              const uint16_t* scale, uint16_t* y,
                              long long ldy, int rows, int D, float eps,
                              hipStream_t s);
hipError_t launch_quantize(const float* w, int N, int K, int bits,
                           uint32_t* codes, uint16_t* scales, uint16_t* biases,
                           hipStream_t s);

// ---- projections over a handful of rows (gemv.hip) ----------------------------
// y[m][n] = bf16(sum_k x[m][k] W[n][k]) for m < M <= kGemvMaxM, W in the
// resident general layout (codes + sb for bits 4/8, w16 for bits 16).
constexpr int kGemvMaxM = 8;
struct GemvArgs {
  const uint16_t* x;
  long long ldx;
  const uint32_t* codes;
  const uint32_t* sb;
  const uint16_t* w16;
  uint16_t* y;
  long long ldy;
  int M, N, K;
  const uint16_t* bias;   // optional bias [N] bf16, added before the rounding
};
hipError_t launch_gemv(int bits, const GemvArgs& a, hipStream_t s);
// The same with what the rows' own adapters add (optional), before the rounding.
hipError_t launch_gemv_rows(int bits, const GemvArgs& a, const RowAdapters* ra, hipStream_t s);
// Up to kGemvBatch GEMVs of one shape over one x in one launch (grid y =
// entry): the per-block adaLN projections of a forward, each entry's bits
// those of launch_gemv on it.
constexpr int kGemvBatch = 32;
struct GemvEntry {
  const uint32_t* codes;
  const uint32_t* sb;
  const uint16_t* w16;
  uint16_t* y;
};
struct GemvBatch {
  GemvArgs base;       // x, ldx, ldy, M, N, K (the entry pointers unused)
  int count;
  GemvEntry e[kGemvBatch];
};
hipError_t launch_gemv_batch(int bits, const GemvBatch& b, hipStream_t s);
hipError_t validate_gemv_kernels();

// ---- the fast quantized route (qproj_fast.hip) --------------------------------
// x is fp16 (carrying bf16 values), a.codes / a.sb the fast resident layout.
// xa (a K split only): the rows' x.A in the same launch (qproj_rows_beside).
hipError_t launch_qproj_fast(int bits, const QprojArgs& a, hipStream_t s,
                             const RowXaArgs* xa = nullptr);
// Up to three projections over one x as one launch (the fields at QprojArgs::nw),
// each one's bits those of its own: the same K slices, tiles by the rounds of
// all. qproj_merge_pays: whether that is less time than one launch each.
hipError_t launch_qproj_merged(int bits, const QprojArgs& a, hipStream_t s);
bool qproj_merge_pays(int M, int N, int K, int nw);
// CUs of the current device, which the plans count rounds by (256 without one).
int device_cus();
// The rows of an unsplit launch: the first rows_main as 256-row tiles, the others
// as tiles of 32 * rf_rest, and the time that takes by the plan's model. Each
// output element is computed by the same MFMA sequence in every tile height, so
// the bits do not depend on the plan. tiles_n columns of tiles, stages of K (64)
// and the LoRA tail; pair: the paired launch (256, 192 and 128 rows).
struct RowPlan {
  int rows_main, rf_rest;
  double us;
};
RowPlan plan_rows(int M, int tiles_n, int stages, bool pair);
// K slices of a projection of few tiles, and its tile height (0: no split).
int qproj_split_plan(int M, int N, int K, int* rf);
// The tile height (rf) of nw projections' merged launch of those slices.
int qproj_merged_split_rf(int M, int N, int K, int kslices, int nw);
// The gate and up projections of a SwiGLU in one launch (the fields after
// `range` in QprojArgs): each 256 x 256 tile holds 128 columns of each, so
// the gate's output meets the up projection's in LDS and only
// y = bf16(silu(gate) * up) (and its fp16 copy yh) is written. Both weights
// one segment each with the same number of LoRA tail chunks, N % 8 == 0,
// y 16-byte aligned with ldy % 8 == 0; no K split.
hipError_t launch_qproj_pair(int bits, const QprojArgs& a, hipStream_t s);
hipError_t launch_repack_fast(int bits, const uint32_t* codes,
                              const uint16_t* scales, const uint16_t* biases,
                              int N, int K, uint32_t* codes_f, uint32_t* sbf,
                              int* inexact, hipStream_t s);
// x.A_live^T with split-K: `part` holds kslices * M * n_cols f32 (unused
// when kslices == 1).
int lora_xa_fast_slices(int M, int n_cols, int K);
// Bytes of f32 partials launch_lora_xa_fast needs for kslices > 1 (whole
// tiles per slice, in the kernel's accumulator order); 0 otherwise.
size_t lora_xa_part_bytes(int M, int n_cols, int K, int kslices);
size_t lora_xa_part_bytes(int M, int n_cols, int kslices, XaTile t);
XaTile xa_tile(int M, int n_cols, int K, int kslices);
// The same kernel as a plain split-K bf16 GEMM y = x . W^T of a dense W
// [N][K] of few tiles: its tile and slices, 0 slices where dense_fast.hip's
// kernel is the faster one.
struct DensePlan {
  XaTile tile;
  int slices;
};
DensePlan dense_split_plan(int M, int N, int K);
// Blocks for 16 rows' x.A that a split can take beside its own; 0: none.
int qproj_rows_beside(int M, int N, int kslices, int rf);
int dense_rows_beside(int M, int N, const DensePlan& p);
// xa: as launch_qproj_fast's, beside a dense weight's split.
hipError_t launch_lora_xa_fast(const LoraXaArgs& a, float* part, int kslices,
                               hipStream_t s, const RowXaArgs* xa = nullptr);
hipError_t launch_bf16_to_f16(const uint16_t* x, long long ldx, uint16_t* y,
                              long long ldy, int rows, int K, hipStream_t s,
                              int* range = nullptr);

// ---- the dense bf16 route (dense_fast.hip) ------------------------------------
// y = x . W^T (+ the LoRA tail), W = a.w16 [N][K] bf16, x bf16 at ldx, with
// a.bias or a.g (fused SwiGLU) as QprojArgs says. N % 8 == 0, K % 64 == 0; x,
// W, T and every B stack within 2 GiB of their base. rf: 64*rf rows a tile.
// With a.nw > 1, that many projections over one x as one launch (no bias, no
// gate), the others' w16, y and segment in a.more.
hipError_t launch_dense_fast(const QprojArgs& a, int rf, hipStream_t s);
// The tile height (rf) for nw projections of a shape, and whether one launch
// for them is less time than one each.
int dense_fast_rf(int M, int N, int nw = 1);
bool dense_merge_pays(int M, int N, int nw);
hipError_t validate_dense_fast_kernels();

// ---- many requests' adapters (adapters.hip) --------------------------------------
// rid[m] = ids[m] where it names a bound adapter and the row's strength is not
// zero, else -1; t[m][0, r32) = bf16(scale[m] * fold * x[m] . A^T), r32 the rank
// rounded up to 32 (zeros past the rank). ldt a multiple of 32.
struct RowXaArgs {
  const uint16_t* x;
  long long ldx;
  int M, K;
  const int32_t* ids;
  const float* scale;   // optional
  const AdapterEntry* table;
  int cap;
  int32_t* rid;
  uint16_t* t;
  int ldt;
  // optional: the chunk lists of row tiles (RowAdapters) of 256 rows up to
  // rows_main, then of `rest` rows, and T's row of zeros, row M
  uint4* chunks;
  int32_t* counts;
  int stride, rows_main, rest;
  // optional: the fp16 copy of x, [M][K], and the word it raises (QprojArgs::range)
  uint16_t* xh;
  int* range;
};
// Row tiles of the lists.
inline int row_tiles(int M, int rows_main, int rest) {
  return rows_main / 256 + (M > rows_main ? (M - rows_main + rest - 1) / rest : 0);
}
// Chunks a tile may need, RowXaArgs::stride: an adapter a row of the tallest tile at
// most, no more than the bank's `cap`, each of as many chunks as ldt holds. The lists'
// blocks write up to that many and rely on it.
int row_tile_chunks(int M, int rows_main, int rest, int cap, int ldt);
hipError_t launch_row_xa(const RowXaArgs& a, hipStream_t s);
// Whether its blocks, with `lists` of row tiles beside them, fit one launch.
bool row_xa_fits(int M, int lists);
// Below these rows launch_row_xa's blocks are 16 rows each, which a split
// projection can take beside its own.
constexpr int kRowXaMany = 768;
// Whether it does, with ny blocks for 16 rows, over a bank of `held` adapters of
// `chunks` 16-rank chunks.
bool row_xa_beside(int ny, int M, int K, int held, int chunks);
// d[m][n] = T[m] . B_a[n] in f32, a = rid[m]; -0 for rows without an adapter,
// which any sum takes without a change. N % 4 == 0.
hipError_t launch_row_delta(const RowAdapters& r, int M, int N, float* d, hipStream_t s);
// A [rank][K] into the x.A kernels' operand order, ranks rounded up to 16.
hipError_t launch_repack_adapter(const uint16_t* A, int rank, int K, uint16_t* out, hipStream_t s);
// *flag = 1 where any of n bf16 values is not finite
hipError_t launch_check_finite(const uint16_t* v, long long n, int* flag, hipStream_t s);
hipError_t validate_adapter_kernels();

// ---- a mixture's router, grouping and weighted sum (routing.hip) ---------------
constexpr int kRouteMaxExperts = 1024;
// Whether the router's blocks for them fit one launch: up to 2^26 - 4.
bool route_fits(long long rows);
struct RouteArgs {
  const void* logits;   // [rows][ld], f32 or bf16
  long long ld;
  int f32;
  const float* bias;    // optional [E], added to the scores for the choice alone
  long long rows;
  int E, k, G, top_groups;
  int sigmoid, normalize;
  float scale;
  int32_t* ids;         // [rows][k]
  float* weights;
};
hipError_t launch_topk_route(const RouteArgs& a, hipStream_t s);
constexpr int kGroupMax = 1024;
struct GroupRowsArgs {
  const int32_t* ids;   // [n]
  long long n;
  int G;
  int32_t* offsets;     // [G + 1]
  int32_t* order;       // [n]
  int32_t* place;       // [n]
  uint32_t* counts;     // group_rows_bytes(n, G)
  int chunk, bits;      // set by the launch
};
size_t group_rows_bytes(long long n, int G);
hipError_t launch_group_rows(GroupRowsArgs a, hipStream_t s);
struct CombineArgs {
  const uint16_t* y;
  long long ldy;
  int n;                // rows of y
  const int32_t* place; // [tokens][k]
  const float* weights;
  const uint16_t* add;  // optional
  long long ldadd;
  uint16_t* out;
  long long ldo;
  long long tokens;
  int k, N;
  int tpr;              // set by the launch
};
hipError_t launch_combine(CombineArgs a, hipStream_t s);
long long combine_blocks(long long tokens, int N);
hipError_t validate_routing_kernels();

// ---- the experts' ragged products (experts.hip) ---------------------------------
// Rows [offsets[e], offsets[e + 1]) of y are expert e's: y[p] = x[row(p)] .
// W_e^T with row(p) = order ? order[p] / fan : p, kept inside [0, x_rows). W is
// a stack of E projections of NW rows: NW = N, or gated 2 N, the gate's N rows
// before the up projection's, y = bf16(silu(gate) * up) of the f32 results.
// Weights: bits 16 w16 [E][K / 64][NW][64] (launch_repack_dense); bits 4 / 8 the fast
// resident layout (launch_repack_fast) an expert after another.
struct ExpertsArgs {
  const uint16_t* x;
  long long ldx;
  const uint32_t* codes;
  const uint32_t* sb;
  const uint16_t* w16;
  const int32_t* offsets;
  const int32_t* order;   // optional
  int E, fan, x_rows, n;
  int N, NW, K;
  uint16_t* y;
  long long ldy;
  // tiles of quantized stacks: a byte a row of x, 1 where its fp16 copy does not hold
  // it (launch_experts_f16), and the word raised for such a row that a place names
  const uint8_t* beyond;
  int* range;
};
// One projection [NW][K] into [K / 64][NW][64]: a stage of a tile is then one run
// of memory. In rows of a power of two the same 128 bytes of every row lie on a
// few of the memory's channels ([64][2048, 2048], 512 rows: 128.7 us by rows, 96.5
// with K = 2112).
hipError_t launch_repack_dense(const uint16_t* w, int NW, int K, uint16_t* out, hipStream_t s);
// few rows an expert, any weights (experts.hip)
hipError_t launch_experts_rows(int bits, bool gated, const ExpertsArgs& a, hipStream_t s);
// 16-column tiles of its blocks on a chip of `cus`, for n places of a stack of outputs
// N wide. The bits are the same.
int experts_rows_tiles(int cus, int bits, bool gated, int E, int N, int K, int n);
hipError_t validate_experts_kernels();
// dense weights, tiles (experts_tile.hip): groups cut every 64 * max places, max 2
// or 4; x_rows * ldx and NW * K below 2^30, y 16-byte aligned with ldy % 8 == 0
hipError_t launch_experts_tile(bool gated, const ExpertsArgs& a, int max, hipStream_t s);
hipError_t validate_experts_tile_kernels();
// w4 and w8, the same with x as its fp16 copy (experts_qtile.hip): groups cut
// every 32 * max places, max 2 or, of w4, 4, of w8, 8
hipError_t launch_experts_qtile(int bits, bool gated, const ExpertsArgs& a, int max,
                                hipStream_t s);
// That copy, y [rows][K], with ExpertsArgs::beyond.
hipError_t launch_experts_f16(const uint16_t* x, long long ldx, int rows, int K, uint16_t* y,
                              uint8_t* beyond, hipStream_t s);
hipError_t validate_experts_qtile_kernels();
// Blocks of the tiles: every group ends in at most one partial one.
inline long long experts_tiles(int bits, bool gated, int max, int n, int E, int N) {
  const int cut = (bits == 16 ? 64 : 32) * max, bn = gated ? 128 : 256;
  return (long long)(n / cut + (n < E ? n : E)) * ((N + bn - 1) / bn);
}
// Which of them takes n places of a stack of N weight rows: 0 the few-row kernel,
// else the tiles' cut (`max`). On the current device, or on a chip of `cus`.
int experts_cut(int E, int N, int K, int bits, int n);
int experts_cut_on(int cus, int E, int N, int K, int bits, int n);

// ---- 8-bit floating point with a scale a block of 128 (f8_quant.hip) --------------
// Whether outputs of that many bytes are stored past the caches: when most of them are out
// of the eight L2s of 4 MB before the next call asks for them. Alone, 8704 x [10240, 3840]
// takes 293 us against 319 and the quantizer of 8704 x 3840 16.1 against 19.7. norm, swiglu
// and lin in turn, storing every output so: 146 against 136 at 1024 rows (10 MB and 8 MB),
// 240 against 241 at 2048 (21 MB and 16 MB), 468 against 471 at 4352. Not for the norm, whose
// lanes store two halves of 32 bytes: 46 -> 72 us at 8704 x 3840.
inline int f8_streams(double bytes) { return bytes > 24.0 * 1048576; }
// Rows of bf16 into e4m3 codes, and scales [blocks of D][lds >= rows] in bf16.
// D % 16 == 0; x and codes 16-byte aligned, ldx % 8 == 0, ldc % 16 == 0.
struct F8QuantArgs {
  const uint16_t* x;
  long long ldx;
  int rows, D;
  uint8_t* codes;
  long long ldc;
  uint16_t* scales;
  long long lds;
  int stream;             // f8_streams of the codes
};
hipError_t launch_f8_quantize(const F8QuantArgs& a, hipStream_t s);
long long f8_quantize_blocks(long long rows, int D);
// h = bf16(x + sub) where sub is given (h may be x), else x; the codes and scales of
// v = h * rsqrt(mean(h^2) + eps) * w, and bf16(v) where y is given. D <= 8192.
struct F8NormArgs {
  const uint16_t* x;
  long long ldx;
  const uint16_t* sub;    // optional
  long long ldsub;
  uint16_t* h;            // with sub
  long long ldh;
  const uint16_t* w;
  uint16_t* y;            // optional
  long long ldy;
  uint8_t* codes;
  long long ldc;
  uint16_t* scales;
  long long lds;
  int rows, D;
  float eps;
};
hipError_t launch_f8_norm(const F8NormArgs& a, hipStream_t s);
// w [N][K] bf16 into codes [N][K] and f32 scales [blocks of N][blocks of K].
hipError_t launch_f8_weight(const uint16_t* w, int N, int K, uint8_t* codes, float* scales,
                            hipStream_t s);
hipError_t validate_f8_quant_kernels();

// ---- their products (f8_rows.hip) ------------------------------------------------------
// Row p of the output is x row p, or of a grouped call x row order[p] / fan (p itself
// without an order; kept inside [0, x_rows)) times the weights of p's group. w is
// resident as launch_f8_repack leaves it, an expert after another: [KB][NR / 16] pieces of
// 2 KB, NR rows padded to 128 a half, with scales [KB][NB].
struct F8Args {
  const uint8_t* x;
  long long ldx;
  const uint16_t* xs;     // [KB][ldxs]
  long long ldxs;
  const uint8_t* w;
  const float* ws;
  long long w_expert, s_expert;   // bytes and scales an expert
  int N, K, KB, NR, NB;
  int n;                  // rows, or places
  int stream;             // f8_streams of the output (the tiles heed it)
  // grouped
  const int32_t* offsets;
  const int32_t* order;   // optional
  int E, fan, x_rows;
  // plain
  const uint16_t* bias;   // optional
  uint16_t* y;
  long long ldy;
  // gated: codes and scales out
  uint8_t* h;
  long long ldh;
  uint16_t* hs;           // [blocks of N][ldhs]
  long long ldhs;
  // f32 sums on their way: of the few-row kernel's gated results [n][N], of the tiles'
  // slices of K (launch_f8_duo)
  float* part;
};
hipError_t launch_f8_repack(const uint8_t* codes, const float* scales, int experts, int N, int K,
                            int halves, uint8_t* out, float* souts, hipStream_t s);
// mf * 16 rows x nf * 16 columns a workgroup: 1 x 1, 1 x 2, 1 x 4 and, ungrouped, 2 x 4.
hipError_t launch_f8_rows(bool gated, bool grouped, const F8Args& a, int mf, int nf,
                          hipStream_t s);
// Blocks of tiles of tm rows x tn columns: every group ends in at most one partial one.
inline long long f8_rows_blocks(int tm, int tn, bool grouped, int n, int E, int N) {
  const long long tiles_m = grouped ? n / tm + (n < E ? n : E) : ((long long)n + tm - 1) / tm;
  return tiles_m * ((N + tn - 1) / tn);
}
inline long long f8_finish_blocks(int n, int N) {
  return ((long long)n * ((N + 127) / 128) + 7) / 8;
}
hipError_t validate_f8_rows_kernels();
// Many rows (f8_tile.hip): 64 * rf rows a tile, rf 1 to 4; over groups cut every 64 * rf
// places, rf 2 or 4. Up to kF8TileBlocks blocks of K; ungrouped ldx below 2^22, grouped
// x_rows * ldx below 2^31. main > 0 (ungrouped, rf 2): the first 256 * main rows in tiles
// of 256.
constexpr int kF8TileBlocks = 1024;
hipError_t launch_f8_tile(bool gated, bool grouped, const F8Args& a, int rf, int main,
                          hipStream_t s);
inline long long f8_mixed_blocks(int main, int n, int NR) {
  return (main + ((long long)n - 256ll * main + 127) / 128) * ((NR + 255) / 256);
}
inline long long f8_tile_blocks(int rf, bool grouped, int n, int E, int NR) {
  const int tm = 64 * rf;
  const long long tiles_m = grouped ? n / tm + (n < E ? n : E) : ((long long)n + tm - 1) / tm;
  return tiles_m * ((NR + 255) / 256);
}
hipError_t validate_f8_tile_kernels();
// Some hundred rows of a plain projection (f8_duo.hip), 64 x 128 a tile; with slices > 1
// K is cut into that many, whose sums meet in part [slices][f8_duo_blocks][64][128]. The
// limits as the tiles'.
hipError_t launch_f8_duo(const F8Args& a, int slices, hipStream_t s);
inline long long f8_duo_blocks(int n, int NR) { return ((long long)n + 63) / 64 * (NR / 128); }
hipError_t validate_f8_duo_kernels();
// Which kernel takes n rows (places) on a chip of `cus`: the few-row one with mf x nf
// fragments, f8_duo's with its slices, or tiles of rf behind `main` of 256 rows.
struct F8Plan {
  enum Kind { kRows, kDuo, kTiles } kind;
  int a, b;               // kRows mf, nf; kDuo slices; kTiles rf, main
};
F8Plan f8_plan(int cus, bool gated, bool grouped, int E, int NR, int KB, int n);

hipError_t validate_qproj_kernels();
hipError_t validate_qproj_fast_kernels();
hipError_t validate_norm_kernels();
hipError_t validate_elementwise_kernels();

}  // namespace ming
