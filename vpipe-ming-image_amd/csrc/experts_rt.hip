// Host side of the mixture's operators: the router, the grouping, the resident
// expert stacks with their ragged products, and the weighted sum.
#include <algorithm>
#include <cmath>
#include <new>
#include <string>

#include "../../include/ming_dit_amd.h"
#include "kernels.h"
#include "rt.h"

using ming::rt_fail;
using ming::rt_ok;

struct ming_experts {
  ming_ctx* ctx = nullptr;
  int E = 0, N = 0, K = 0, bits = 0;
  uint32_t* codes = nullptr;   // bits 4 / 8: the fast resident layout, an expert after another
  uint32_t* sb = nullptr;
  uint16_t* w16 = nullptr;     // bits 16: [E][K / 64][N][64]
};

namespace ming {

// Which kernel takes n places: 0 the few-row one, else the tiles, cut every
// 64 (dense) or 32 (quantized) * max places. The groups' sizes are on the device,
// so it goes by what an even router gives: live experts, rows of each. Of both the
// times below are fits (us) to [16 to 256][1024 to 4096, 1024 to 4096] at 8 to 384
// places out of cold caches; where they are close, so are the kernels.
//   few rows, dense: 2.5 + bytes / 5.9 TB/s, longer by the rows' own reads (swiglu
//     of [64][2048, 2048], 8 places: 14.6, the tiles 17.5); w4 and w8: 6 and 5
//     weights a ps ([60][2048, 1024], 16 places: 9.7 and 11.0, the tiles 13.6 and
//     15.4); a start a block; 16 rows a pass over the weights.
//   tiles: a start and the K stages of one, then the weights at 5.6 to 6.1 TB/s, a
//     round of the chip (one dense block a CU) at least that again (dense as above, 64
//     places: 74.1, few rows 68.8; 128: 85.4 and 89.6; w8 as above, 64: 25.0 and 26.3,
//     w4 19.7 and 23.3).
//     They have to win by 8%: x's fp16 copy grows with x.
// Cuts (low / tall, us): more rows a tile read the weights less often and, quantized,
// convert them less often; fewer fill the chip where there are few tiles. Dense, 128
// or 256 rows ([64][2048, 2048] gated, 96 rows an expert 99 / 103, 128: 125 / 110, 544:
// 311 / 283; [16][2048, 4096], 192 rows, 128 tall tiles: 65 / 94); w4, 64 rows and three
// blocks a CU or 128 and two ([128][1024, 2048] gated, 32 rows 41 / 43, 78: 70 / 57); w8, 64
// or 256 ([60][2048, 1024], 160 rows 63 / 62, all groups of 256: 86 / 74).
int experts_cut(int E, int N, int K, int bits, int n) {
  return experts_cut_on(device_cus(), E, N, K, bits, n);
}
int experts_cut_on(int cus, int E, int N, int K, int bits, int n) {
  const double live = E * (1.0 - std::exp(-(double)n / E)), rows = n / live;
  const double weights = live * N * (double)K, stages = K / 64.0, blocks = live * (N / 32.0);
  const double passes = rows > 8.0 ? rows / 16.0 + 0.5 : 1.0;
  double few, tile;
  if (bits == 16) {
    const double one = 256.0 * K * 2 / 6.1e6;            // a tile's weights, us
    const double all = live * ((N + 255) / 256), round = std::floor(all / cus) * cus;
    few = 2.5 + weights * 2 / 5.9e6 * (1.0 + rows / 40.0) * passes + 0.002 * blocks;
    tile = round * one + std::max(4.0 + 0.75 * stages, 2.5 + (all - round) * one);
  } else {
    few = 3.0 + weights / (bits == 4 ? 6.0e6 : 5.0e6) * passes + 0.0035 * blocks;
    tile = std::max(5.5 + 0.5 * stages, 7.0 + weights * (bits / 8.0 + 1.0 / 16) / 5.6e6);
  }
  if (few < 1.08 * tile) return 0;
  const int low = 2, tall = bits == 8 ? 8 : 4;
  const double from = bits == 16 ? 112.0 : bits == 4 ? 60.0 : 240.0;
  // tiles of the tall cut, of which every group ends in half a one on average
  const double each = std::max(1.0, rows / ((bits == 16 ? 64 : 32) * tall) + 0.5);
  return rows < from || live * each * ((N + 255) / 256) < cus * (180.0 / 256.0) ? low : tall;
}

}  // namespace ming

namespace {

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != dev) (void)hipSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
  }
};

hipStream_t stream_of(const ming_ctx* c) { return (hipStream_t)ming_ctx_stream(c); }
bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
int hip_fail(hipError_t e, const char* what) {
  return rt_fail(MING_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}
ming::Span row_span(const void* p, int64_t rows, int64_t ld, int64_t width) {
  return {p, rows, 2 * ld, 2 * width};
}
ming::Span flat_span(const void* p, int64_t bytes) { return {p, 1, bytes, bytes}; }

// One launch, timed when the context profiles.
template <class F>
int run(ming_ctx* c, ming::RtBucket b, double flops, double bytes, const char* what, F&& launch) {
  void* ev = nullptr;
  if (!ming::rt_profile_begin(c, &ev)) return hip_fail(hipErrorOutOfMemory, what);
  const hipError_t e = launch();
  const bool timed = ming::rt_profile_end(c, ev, b, flops, bytes);
  if (e != hipSuccess) return hip_fail(e, what);
  if (!timed) return hip_fail(hipErrorOutOfMemory, what);
  return MING_OK;
}

int products(const char* who, bool gated, ming_ctx* c, const ming_experts* ex, const uint16_t* x,
             int64_t ldx, int x_rows, const int32_t* order, int fan, const int32_t* offsets, int n,
             uint16_t* y, int64_t ldy, void* ws, size_t ws_bytes) {
  auto bad = [&](int code, const char* why) { return rt_fail(code, std::string(who) + ": " + why); };
  if (!c || !ex || (n > 0 && (!x || !offsets || !y))) return bad(MING_ERR_ARG, "null argument");
  if (ex->ctx != c) return bad(MING_ERR_ARG, "experts of another context");
  if (n < 0 || x_rows < 0 || fan < 1) return bad(MING_ERR_ARG, "a count out of range");
  // a group's rows are counted in ints, up to a tile past its end
  if (n > 1 << 30) return bad(MING_ERR_SHAPE, "n past 2^30, more places than a launch takes");
  const int N = gated ? ex->N / 2 : ex->N;
  if (gated && ex->N % 16 != 0)
    return bad(MING_ERR_SHAPE, "gate and up rows need N % 16 == 0");
  if (ldx < ex->K || ldx % 8 != 0 || ldy < N || ldy % 8 != 0)
    return bad(MING_ERR_SHAPE, "need ldx >= K and ldy >= the output's width, multiples of 8");
  if (!aligned(x, 16) || !aligned(y, 16) || !aligned(offsets, 4) || !aligned(order, 4))
    return bad(MING_ERR_ARG, "x and y must be 16-byte, offsets and order 4-byte aligned");
  if (n == 0) return rt_ok();
  if (x_rows == 0) return bad(MING_ERR_ARG, "places without rows of x");
  if (!order && x_rows < n) return bad(MING_ERR_SHAPE, "without an order x needs n rows");
  if (ldx > ((1ll << 30) - 1) / x_rows)
    return bad(MING_ERR_SHAPE, "x_rows * ldx must be below 2^30");
  DeviceGuard g(ming::rt_device(c));       // (the plan counts its CUs)
  // the quantized tiles multiply fp16, which the other routes are chosen against
  const int cut = ex->bits != 16 && ming::rt_route(c) != MING_ROUTE_AUTO ? 0
                  : ming::rt_experts_cut(c) >= 0
                      ? ming::rt_experts_cut(c)
                      : ming::experts_cut(ex->E, ex->N, ex->K, ex->bits, n);
  const size_t xh_bytes = cut ? ming_experts_workspace_bytes(ex, x_rows) : 0;
  if (xh_bytes > 0 && (!ws || !aligned(ws, 16)))
    return bad(MING_ERR_ARG, "ws must be given, 16-byte aligned");
  if (ws_bytes < xh_bytes)
    return rt_fail(MING_ERR_SHAPE, std::string(who) + ": the call needs " +
                                       std::to_string(xh_bytes) + " bytes of workspace, " +
                                       std::to_string(ws_bytes) + " given");
  if (cut && !ming::one_launch(ming::experts_tiles(ex->bits, gated, cut, n, ex->E, N),
                         ex->bits == 16 ? 512 : 256))
    return bad(MING_ERR_SHAPE, "more places times columns than one launch holds");
  // every block reads the plan and the rows by itself, while others store
  const ming::Span xs = row_span(x, x_rows, ldx, ex->K), ys = row_span(y, n, ldy, N);
  const ming::Span os = flat_span(order, order ? 4ll * n : 0), fs = flat_span(offsets, 4ll * (ex->E + 1));
  const ming::Span sc = flat_span(ws, (int64_t)xh_bytes);
  for (const ming::Span& in : {xs, os, fs})
    if (ming::spans_meet(in, ys) || ming::spans_meet(in, sc))
      return bad(MING_ERR_ARG, "x, order or offsets share memory with y or ws");
  if (ming::spans_meet(ys, sc)) return bad(MING_ERR_ARG, "y and ws share memory");
  ming::ExpertsArgs a{};
  a.x = x; a.ldx = ldx;
  a.codes = ex->codes; a.sb = ex->sb; a.w16 = ex->w16;
  a.offsets = offsets; a.order = order;
  a.E = ex->E; a.fan = fan; a.x_rows = x_rows; a.n = n;
  a.N = N; a.NW = ex->N; a.K = ex->K;
  a.y = y; a.ldy = ldy;
  const double flops = 2.0 * n * (double)ex->N * ex->K;
  const double wb = ex->bits == 16 ? 2.0 * ex->N * ex->K
                                   : (double)ex->N * ex->K * ex->bits / 8 + 4.0 * ex->N * (ex->K / 64);
  const int rc = run(
      c, ming::kRtExperts, flops, wb * std::min(n, ex->E) + 2.0 * x_rows * ex->K + 2.0 * n * N, who,
      [&] {
        if (cut == 0)
          return ming::launch_experts_rows(ex->bits, gated, a, stream_of(c));
        if (ex->bits == 16) return ming::launch_experts_tile(gated, a, cut, stream_of(c));
        // one conversion of x to fp16 for all experts' rows
        auto* xh = static_cast<uint16_t*>(ws);
        auto* beyond = static_cast<uint8_t*>(ws) + (size_t)x_rows * ex->K * 2;
        const hipError_t e =
            ming::launch_experts_f16(x, ldx, x_rows, ex->K, xh, beyond, stream_of(c));
        if (e != hipSuccess) return e;
        a.x = xh;
        a.ldx = ex->K;
        a.beyond = beyond;
        a.range = ming::rt_range_word(c);
        return ming::launch_experts_qtile(ex->bits, gated, a, cut, stream_of(c));
      });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, ex->bits, 2ull * (uint64_t)n * (uint64_t)ex->N * (uint64_t)ex->K);
  return rt_ok();
}

// What both creations check.
int check_stack(ming_ctx* c, int E, int N, int K) {
  if (!c) return rt_fail(MING_ERR_ARG, "ming_experts_create: null argument");
  if (E < 1 || E > ming::kGroupMax)
    return rt_fail(MING_ERR_SHAPE, "ming_experts_create: 1 to 1024 experts");
  if (N <= 0 || K <= 0 || K % 64 != 0 || N % 8 != 0)
    return rt_fail(MING_ERR_SHAPE, "ming_experts_create: need K % 64 == 0 and N % 8 == 0");
  if ((uint64_t)N * (uint64_t)K >= (1ull << 30))
    return rt_fail(MING_ERR_SHAPE, "ming_experts_create: an expert's N * K must be below 2^30");
  return MING_OK;
}

// Whether the context's kernels can read p where it is: its own device's memory. That
// of another device comes over by copies, which need no access from here.
bool own_memory(const ming_ctx* c, const void* p) {
  hipPointerAttribute_t at{};
  if (hipPointerGetAttributes(&at, p) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  return at.type == hipMemoryTypeDevice && at.device == ming::rt_device(c);
}

// Source memory that a stack's creation has on the device at a time where it has to
// bring it there: some experts, so that a stack can be as large as the memory.
constexpr size_t kStageBytes = 64u << 20;

}  // namespace

extern "C" {

int ming_topk_route(ming_ctx* c, const void* logits, int64_t ld, int logits_f32, const float* bias,
                    int rows, int n_experts, int top_k, int n_groups, int top_groups, int score,
                    int normalize, float scale, int32_t* ids, float* weights) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_topk_route: ") + why);
  };
  if (!c || (rows > 0 && (!logits || !ids || !weights)))
    return bad(MING_ERR_ARG, "null argument");
  if (rows < 0) return bad(MING_ERR_ARG, "rows < 0");
  if (!ming::route_fits(rows)) return bad(MING_ERR_SHAPE, "rows must be at most 2^26 - 4");
  if (score != MING_SCORE_SOFTMAX && score != MING_SCORE_SIGMOID)
    return bad(MING_ERR_ARG, "no such score");
  if (n_experts < 1 || n_experts > ming::kRouteMaxExperts || n_groups < 1 || n_groups > 64 ||
      n_experts % n_groups != 0)
    return bad(MING_ERR_SHAPE, "1 to 1024 experts in at most 64 equal groups");
  if (top_groups < 1 || top_groups > n_groups)
    return bad(MING_ERR_SHAPE, "top_groups must be 1 to n_groups");
  if (top_k < 1 || top_k > 64 || top_k > n_experts / n_groups * top_groups)
    return bad(MING_ERR_SHAPE, "top_k must be 1 to 64 and fit in the chosen groups");
  if (ld < n_experts) return bad(MING_ERR_SHAPE, "need ld >= n_experts");
  if (!aligned(logits, logits_f32 ? 4 : 2) || !aligned(bias, 4) || !aligned(ids, 4) ||
      !aligned(weights, 4))
    return bad(MING_ERR_ARG, "a misaligned pointer");
  if (rows == 0) return rt_ok();
  const int64_t el = logits_f32 ? 4 : 2;
  const ming::Span ls = {logits, rows, el * ld, el * n_experts};
  const ming::Span bs = flat_span(bias, bias ? 4ll * n_experts : 0);
  const ming::Span is = flat_span(ids, 4ll * rows * top_k), wt = flat_span(weights, 4ll * rows * top_k);
  if (ming::spans_meet(is, wt) || ming::spans_meet(ls, is) || ming::spans_meet(ls, wt) ||
      ming::spans_meet(bs, is) || ming::spans_meet(bs, wt))
    return bad(MING_ERR_ARG, "logits, bias, ids and weights must not share memory");
  DeviceGuard g(ming::rt_device(c));
  ming::RouteArgs a{};
  a.logits = logits; a.ld = ld; a.f32 = logits_f32 != 0; a.bias = bias;
  a.rows = rows; a.E = n_experts; a.k = top_k; a.G = n_groups; a.top_groups = top_groups;
  a.sigmoid = score == MING_SCORE_SIGMOID; a.normalize = normalize != 0; a.scale = scale;
  a.ids = ids; a.weights = weights;
  const int rc = run(c, ming::kRtRoute, 0.0, (double)rows * n_experts * (logits_f32 ? 4 : 2),
                     "ming_topk_route", [&] { return ming::launch_topk_route(a, stream_of(c)); });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, 0, 0);
  return rt_ok();
}

size_t ming_group_rows_workspace_bytes(int n, int n_groups) {
  if (n <= 0 || n > (1 << 30) || n_groups < 1 || n_groups > ming::kGroupMax) return 0;
  return ming::group_rows_bytes(n, n_groups);
}

int ming_group_rows(ming_ctx* c, const int32_t* ids, int n, int n_groups, int32_t* offsets,
                    int32_t* order, int32_t* place, void* ws, size_t ws_bytes) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_group_rows: ") + why);
  };
  if (n < 0 || n > (1 << 30)) return bad(MING_ERR_ARG, "n must be 0 to 2^30");
  if (!c || !offsets || (n > 0 && (!ids || !order || !place)))
    return bad(MING_ERR_ARG, "null argument");
  if (n_groups < 1 || n_groups > ming::kGroupMax)
    return bad(MING_ERR_SHAPE, "1 to 1024 groups");
  if (!aligned(ids, 4) || !aligned(offsets, 4) || !aligned(order, 4) || !aligned(place, 4))
    return bad(MING_ERR_ARG, "a misaligned pointer");
  const size_t need = ming::group_rows_bytes(n, n_groups);
  if (need > 0 && (!ws || !aligned(ws, 16)))
    return bad(MING_ERR_ARG, "ws must be given, 16-byte aligned");
  if (ws_bytes < need)
    return rt_fail(MING_ERR_SHAPE, "ming_group_rows: the call needs " + std::to_string(need) +
                                       " bytes of workspace, " + std::to_string(ws_bytes) +
                                       " given");
  const ming::Span all[5] = {flat_span(ids, 4ll * n), flat_span(offsets, 4ll * (n_groups + 1)),
                             flat_span(order, 4ll * n), flat_span(place, 4ll * n),
                             flat_span(ws, (int64_t)need)};
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < i; ++j)
      if (ming::spans_meet(all[i], all[j]))
        return bad(MING_ERR_ARG, "ids, offsets, order, place and ws must not share memory");
  DeviceGuard g(ming::rt_device(c));
  ming::GroupRowsArgs a{};
  a.ids = ids; a.n = n; a.G = n_groups;
  a.offsets = offsets; a.order = order; a.place = place;
  a.counts = static_cast<uint32_t*>(ws);
  const int rc = run(c, ming::kRtGroup, 0.0, 12.0 * n + 4.0 * n_groups, "ming_group_rows",
                     [&] { return ming::launch_group_rows(a, stream_of(c)); });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, 0, 0);
  return rt_ok();
}

int ming_experts_destroy(ming_experts* ex) {
  if (!ex) return rt_ok();
  DeviceGuard g(ming::rt_device(ex->ctx));
  (void)hipStreamSynchronize(stream_of(ex->ctx));
  if (ex->codes) (void)hipFree(ex->codes);
  if (ex->sb) (void)hipFree(ex->sb);
  if (ex->w16) (void)hipFree(ex->w16);
  ming::rt_release(ex->ctx);
  delete ex;
  return rt_ok();
}

int ming_experts_create_dense(ming_ctx* c, int n_experts, int N, int K, const uint16_t* w,
                              int src_on_device, ming_experts** out) {
  if (!out || !w) return rt_fail(MING_ERR_ARG, "ming_experts_create: null argument");
  *out = nullptr;
  if (const int rc = check_stack(c, n_experts, N, K)) return rc;
  if (src_on_device && !aligned(w, 16))
    return rt_fail(MING_ERR_ARG, "ming_experts_create: device weights must be 16-byte aligned");
  DeviceGuard g(ming::rt_device(c));
  auto* ex = new (std::nothrow) ming_experts();
  if (!ex) return rt_fail(MING_ERR_ALLOC, "ming_experts_create: out of memory");
  ex->ctx = c; ex->E = n_experts; ex->N = N; ex->K = K; ex->bits = 16;
  ming::rt_retain(c);
  const size_t one = (size_t)N * K;
  hipStream_t s = stream_of(c);
  void* stage = nullptr;                 // an expert's source, where it is elsewhere
  const bool direct = src_on_device && own_memory(c, w);
  const hipMemcpyKind kind = src_on_device ? hipMemcpyDefault : hipMemcpyHostToDevice;
  hipError_t e = hipMalloc(&ex->w16, (size_t)n_experts * one * 2);
  if (e == hipSuccess && !direct) e = hipMalloc(&stage, one * 2);
  for (int i = 0; i < n_experts && e == hipSuccess; ++i) {
    const uint16_t* src = w + i * one;
    if (stage) {
      e = hipMemcpyAsync(stage, src, one * 2, kind, s);
      src = static_cast<const uint16_t*>(stage);
    }
    if (e == hipSuccess) e = ming::launch_repack_dense(src, N, K, ex->w16 + i * one, s);
  }
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (stage) (void)hipFree(stage);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    ming_experts_destroy(ex);
    return e == hipErrorOutOfMemory
               ? rt_fail(MING_ERR_ALLOC, "ming_experts_create: device allocation failed")
               : hip_fail(e, "ming_experts_create");
  }
  *out = ex;
  return rt_ok();
}

int ming_experts_create(ming_ctx* c, int n_experts, int N, int K, int bits, int group,
                        const uint32_t* codes, const uint16_t* scales, const uint16_t* biases,
                        int src_on_device, ming_experts** out) {
  if (!out || !codes || !scales || !biases)
    return rt_fail(MING_ERR_ARG, "ming_experts_create: null argument");
  *out = nullptr;
  if (const int rc = check_stack(c, n_experts, N, K)) return rc;
  if (bits != 4 && bits != 8)
    return rt_fail(MING_ERR_SHAPE, "ming_experts_create: bits must be 4 or 8");
  if (group != 64) return rt_fail(MING_ERR_SHAPE, "ming_experts_create: group must be 64");
  DeviceGuard g(ming::rt_device(c));
  auto* ex = new (std::nothrow) ming_experts();
  if (!ex) return rt_fail(MING_ERR_ALLOC, "ming_experts_create: out of memory");
  ex->ctx = c; ex->E = n_experts; ex->N = N; ex->K = K; ex->bits = bits;
  ming::rt_retain(c);
  const size_t words = (size_t)N * K * bits / 32, pairs = (size_t)N * (K / 64);
  const size_t E = (size_t)n_experts;
  hipStream_t s = stream_of(c);
  // arrays that the repack can read are read where they are
  const bool direct = src_on_device && aligned(codes, 4) && aligned(scales, 2) &&
                      aligned(biases, 2) && own_memory(c, codes) && own_memory(c, scales) &&
                      own_memory(c, biases);
  const size_t some =
      direct ? E : std::clamp<size_t>(kStageBytes / (words * 4 + pairs * 4), 1, E);
  const hipMemcpyKind kind = src_on_device ? hipMemcpyDefault : hipMemcpyHostToDevice;
  uint32_t* dc = nullptr;
  uint16_t *ds = nullptr, *db = nullptr;
  int *flag = nullptr, inexact = 0;
  hipError_t e = hipMalloc(&ex->codes, E * words * 4);
  if (e == hipSuccess) e = hipMalloc(&ex->sb, E * pairs * 4);
  if (e == hipSuccess) e = hipMalloc(&flag, sizeof(int));
  if (e == hipSuccess && !direct) e = hipMalloc(&dc, some * words * 4);
  if (e == hipSuccess && !direct) e = hipMalloc(&ds, some * pairs * 2);
  if (e == hipSuccess && !direct) e = hipMalloc(&db, some * pairs * 2);
  if (e == hipSuccess) e = hipMemsetAsync(flag, 0, sizeof(int), s);
  for (size_t i0 = 0; i0 < E && e == hipSuccess; i0 += some) {
    const size_t n = std::min(some, E - i0);
    const uint32_t* sc = codes + i0 * words;
    const uint16_t *ss = scales + i0 * pairs, *sb = biases + i0 * pairs;
    if (!direct) {                         // (behind the repack of those before, in order)
      e = hipMemcpyAsync(dc, sc, n * words * 4, kind, s);
      if (e == hipSuccess) e = hipMemcpyAsync(ds, ss, n * pairs * 2, kind, s);
      if (e == hipSuccess) e = hipMemcpyAsync(db, sb, n * pairs * 2, kind, s);
      sc = dc; ss = ds; sb = db;
    }
    for (size_t i = 0; i < n && e == hipSuccess; ++i)
      e = ming::launch_repack_fast(bits, sc + i * words, ss + i * pairs, sb + i * pairs, N, K,
                                   ex->codes + (i0 + i) * words, ex->sb + (i0 + i) * pairs, flag,
                                   s);
  }
  if (e == hipSuccess) e = hipMemcpyAsync(&inexact, flag, sizeof(int), hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  for (void* p : {(void*)dc, (void*)ds, (void*)db, (void*)flag})
    if (p) (void)hipFree(p);
  if (e != hipSuccess || inexact) {
    (void)hipGetLastError();
    ming_experts_destroy(ex);
    if (inexact)
      return rt_fail(MING_ERR_RANGE,
                     "ming_experts_create: a scale or bias is not exact in fp16 (create the "
                     "stack from dense weights)");
    return e == hipErrorOutOfMemory
               ? rt_fail(MING_ERR_ALLOC, "ming_experts_create: device allocation failed")
               : hip_fail(e, "ming_experts_create");
  }
  *out = ex;
  return rt_ok();
}

int ming_experts_shape(const ming_experts* ex, int* n_experts, int* N, int* K, int* bits) {
  if (!ex) return rt_fail(MING_ERR_ARG, "ming_experts_shape: null argument");
  if (n_experts) *n_experts = ex->E;
  if (N) *N = ex->N;
  if (K) *K = ex->K;
  if (bits) *bits = ex->bits;
  return rt_ok();
}

size_t ming_experts_workspace_bytes(const ming_experts* ex, int x_rows) {
  // the fp16 copy of x that the tiles of a quantized stack multiply, a byte a row for
  // what it does not hold
  if (!ex || x_rows <= 0 || ex->bits == 16) return 0;
  return (size_t)x_rows * ex->K * 2 + ((size_t)x_rows + 15) / 16 * 16;
}

int ming_experts_lin(ming_ctx* c, const ming_experts* ex, const uint16_t* x, int64_t ldx,
                     int x_rows, const int32_t* order, int fan, const int32_t* offsets, int n,
                     uint16_t* y, int64_t ldy, void* ws, size_t ws_bytes) {
  return products("ming_experts_lin", false, c, ex, x, ldx, x_rows, order, fan, offsets, n, y, ldy,
                  ws, ws_bytes);
}

int ming_experts_swiglu(ming_ctx* c, const ming_experts* ex, const uint16_t* x, int64_t ldx,
                        int x_rows, const int32_t* order, int fan, const int32_t* offsets, int n,
                        uint16_t* y, int64_t ldy, void* ws, size_t ws_bytes) {
  return products("ming_experts_swiglu", true, c, ex, x, ldx, x_rows, order, fan, offsets, n, y,
                  ldy, ws, ws_bytes);
}

int ming_experts_combine(ming_ctx* c, const uint16_t* y, int64_t ldy, int n, const int32_t* place,
                         const float* weights, int tokens, int top_k, const uint16_t* add,
                         int64_t ldadd, uint16_t* out, int64_t ldo, int N) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_experts_combine: ") + why);
  };
  if (!c || (tokens > 0 && (!out || !place || !weights || (n > 0 && !y))))
    return bad(MING_ERR_ARG, "null argument");
  if (n < 0 || tokens < 0 || top_k < 1) return bad(MING_ERR_ARG, "a count out of range");
  // choices are counted in ints, four at a time
  if (top_k > 1 << 30) return bad(MING_ERR_SHAPE, "top_k must be at most 2^30");
  if (N <= 0 || N % 8 != 0 || (n > 0 && ldy < N) || ldo < N || (add && ldadd < N) ||
      ldy % 8 != 0 || ldo % 8 != 0 || (add && ldadd % 8 != 0))
    return bad(MING_ERR_SHAPE, "N and the strides must be multiples of 8, strides >= N");
  if (!aligned(y, 16) || !aligned(out, 16) || !aligned(add, 16) || !aligned(place, 4) ||
      !aligned(weights, 4))
    return bad(MING_ERR_ARG, "y, add and out must be 16-byte, place and weights 4-byte aligned");
  if (tokens == 0) return rt_ok();
  if (!ming::one_launch(ming::combine_blocks(tokens, N), 256))
    return bad(MING_ERR_SHAPE, "more tokens than one launch holds");
  const ming::Span outs = row_span(out, tokens, ldo, N);
  if (ming::spans_meet(row_span(y, n, ldy, N), outs))
    return bad(MING_ERR_ARG, "y and out share memory");
  if (ming::spans_meet(flat_span(place, 4ll * tokens * top_k), outs) ||
      ming::spans_meet(flat_span(weights, 4ll * tokens * top_k), outs))
    return bad(MING_ERR_ARG, "place or weights share memory with out");
  if (add && !(add == out && ldadd == ldo) && ming::spans_meet(row_span(add, tokens, ldadd, N), outs))
    return bad(MING_ERR_ARG, "add and out share memory but are not the same rows");
  DeviceGuard g(ming::rt_device(c));
  ming::CombineArgs a{};
  a.y = y; a.ldy = ldy; a.n = n; a.place = place; a.weights = weights;
  a.add = add; a.ldadd = ldadd; a.out = out; a.ldo = ldo;
  a.tokens = tokens; a.k = top_k; a.N = N;
  const int rc = run(c, ming::kRtCombine, 0.0,
                     2.0 * tokens * (double)N * (top_k + (add ? 2 : 1)), "ming_experts_combine",
                     [&] { return ming::launch_combine(a, stream_of(c)); });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, 0, 0);
  return rt_ok();
}

}  // extern "C"
