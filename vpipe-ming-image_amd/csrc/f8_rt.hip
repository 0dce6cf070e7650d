// Host side of the 8-bit floating-point operators: the quantizers, the norm, the
// resident projections and their products.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <new>
#include <string>

#include "../../include/ming_dit_amd.h"
#include "kernels.h"
#include "rt.h"

using ming::rt_fail;
using ming::rt_ok;
using ming::Span;

struct ming_f8 {
  ming_ctx* ctx = nullptr;
  int E = 0, N = 0, K = 0, halves = 0;
  int KB = 0, NR = 0, NB = 0;      // blocks of K, resident rows and scales a block of K
  uint8_t* codes = nullptr;        // [E][KB][NR][128], in 16 rows at a time
  float* scales = nullptr;         // [E][KB][NB], behind the codes in one allocation
};

namespace ming {

// Times (us) of n rows by each kernel's rounds of the chip, a workgroup a CU, fitted to
// widths of 512 to 10240 at K = 512 to 10240, 1 to 8704 rows, out of cold caches. The choice
// is then within 1% of the fastest one's time in the geometric mean of 279 shapes (worst
// 15%), over groups, whose sizes are on the device (what an even router gives), 2.5% of
// 156. rows: a start, the K blocks and a workgroup's end a round, and the weights' bytes
// (MB). Two halves: a start a round and its stages, with slices their sum's launch and
// bytes. Tiles: a start a round and its stages, which take longer where the chip is full.
namespace {
double rows_us(int i, bool gated, double wgs, int KB, double mb, int cus) {
  static const double kPlain[4][4] = {{3.32, 0.062, 0.000, 0.05}, {3.08, 0.074, 0.011, 0.17},
                                      {3.26, 0.100, 0.033, 0.30}, {1.85, 0.160, 0.035, 1.46}};
  static const double kGated[4][4] = {{6.33, 0.069, 0.031, 0.14}, {6.08, 0.087, 0.046, 0.41},
                                      {4.51, 0.149, 0.070, 1.83}, {3.52, 0.209, 0.067, 2.89}};
  const double* c = gated ? kGated[i] : kPlain[i];
  const double r = std::ceil(wgs / cus);
  return c[0] + r * (c[1] * KB + c[3]) + c[2] * mb;
}
double tiles_us(int rf, bool gated, long long tiles, int KB, int cus) {
  static const double kPlain[4][4] = {{1.20, 2.84, 0.439, 0.153}, {0.0, 4.66, 0.543, 0.317},
                                      {0.0, 4.58, 0.994, 0.322}, {0.20, 5.27, 1.063, 0.607}};
  static const double kGated[4][4] = {{1.31, 3.41, 0.455, 0.125}, {0.36, 5.63, 0.575, 0.241},
                                      {0.40, 6.04, 0.992, 0.332}, {0.53, 7.53, 1.123, 0.485}};
  const double* c = gated ? kGated[rf - 1] : kPlain[rf - 1];
  const double r = (double)((tiles + cus - 1) / cus), fill = std::min(1.0, (double)tiles / cus);
  return c[0] + r * (c[1] + KB * (c[2] + c[3] * fill));
}
constexpr int kRowShapes[4][2] = {{1, 1}, {1, 2}, {1, 4}, {2, 4}};

// Rows up to which a kernel with sums in the workspace is taken, which keeps the scan of
// workspace() short: tiles have won by then (groups: by some 40 rows each).
constexpr int kPartRows = 4096, kPartGroupRows = 64;

F8Plan group_plan(int cus, bool gated, int E, int NR, int KB, int rows_in) {
  // in steps of an eighth of a row a group, so that the scan has few sizes to look at
  const int step = std::max(1, E / 8), n = (rows_in + step - 1) / step * step;
  const int N = gated ? NR / 2 : NR, tiles_n = (NR + 255) / 256;
  const double live = E * (1.0 - std::exp(-(double)n / E)), rows = n / live;
  const double mb = live * NR * (double)KB * 128e-6;
  static const double kRows[2][3][4] = {
      {{3.34, 0.064, 0.000, 0.42}, {2.86, 0.060, 0.071, 0.68}, {2.33, 0.076, 0.097, 1.20}},
      {{5.80, 0.075, 0.052, 0.83}, {5.15, 0.125, 0.087, 0.91}, {3.97, 0.131, 0.146, 2.06}}};
  static const double kTile[2][3] = {{3.34, 0.131, 0.343}, {4.97, 0.115, 0.383}};
  F8Plan best{F8Plan::kTiles, 2, 0};
  {
    const double t = live * std::max(1.0, rows / 128 + (rows > 40 ? 0.5 : 0.0)) * tiles_n;
    const double h = std::min(2.0, std::ceil(rows / 64)), r = std::max(1.0, t / cus);
    const double* c = kTile[gated];
    double least = 1.05 * (r * (c[0] + KB * h * c[2]) + c[1] * mb);
    for (int i = 0; i < 3 && n <= kPartGroupRows * E; ++i) {
      const int nf = kRowShapes[i][1];
      const double w = live * (rows > 8 ? std::max(1.0, rows / 16 + 0.5) : 1.0) *
                       ((N + 16 * nf - 1) / (16 * nf));
      const double* q = kRows[gated][i];
      const double us = q[0] + std::max(1.0, w / cus) * (q[1] * KB + q[3]) + q[2] * mb;
      if (us < least) {
        best = {F8Plan::kRows, 1, nf};
        least = us;
      }
    }
  }
  // tall tiles read and start less often; low ones fill the chip where there are few
  if (best.kind == F8Plan::kTiles && rows >= 160.0 &&
      live * (rows / 256 + 0.5) * tiles_n >= 0.6 * cus)
    best.a = 4;
  return best;
}
}  // namespace

F8Plan f8_plan(int cus, bool gated, bool grouped, int E, int NR, int KB, int n) {
  if (KB > kF8TileBlocks) return {F8Plan::kRows, 1, 4};
  if (grouped) return group_plan(cus, gated, E, NR, KB, n);
  const int N = gated ? NR / 2 : NR;
  const double mb = NR * (double)KB * 128e-6;
  F8Plan best{F8Plan::kTiles, 4, 0};
  double least = 1e30;
  auto take = [&](double us, F8Plan p) {
    if (us < least) {
      best = p;
      least = us;
    }
  };
  for (int rf = 4; rf >= 1; --rf)
    take(tiles_us(rf, gated, f8_tile_blocks(rf, false, n, 1, NR), KB, cus), {F8Plan::kTiles, rf, 0});
  // whole rounds of 256-row tiles, and what is left of the rows in tiles of 128
  const int tiles_n = (NR + 255) / 256;
  const long long whole = (long long)(n / 256) * tiles_n / cus * cus / tiles_n;
  if (whole > 0 && 256 * whole < n)
    take(tiles_us(4, gated, whole * tiles_n, KB, cus) +
             tiles_us(2, gated, (n - 256 * whole + 127) / 128 * tiles_n, KB, cus),
         {F8Plan::kTiles, 2, (int)whole});
  for (int i = 0; i < 4 && n <= kPartRows; ++i) {
    const int mf = kRowShapes[i][0], nf = kRowShapes[i][1];
    const double wgs = (double)((n + 16ll * mf - 1) / (16 * mf)) * ((N + 16 * nf - 1) / (16 * nf));
    take(rows_us(i, gated, wgs, KB, mb, cus), {F8Plan::kRows, mf, nf});
  }
  if (!gated)
    for (int s = 1; s <= (n <= kPartRows ? 4 : 1) && s <= KB; ++s) {
      const long long tiles = f8_duo_blocks(n, NR) * s;
      const double r = (double)((tiles + cus - 1) / cus), stages = (KB + 2 * s - 1) / (2 * s);
      take(s == 1 ? 0.11 + r * (4.28 + 0.595 * stages)
                  : 4.60 + r * (2.33 + 0.531 * stages) + 0.418 * 0.0328 * tiles,
           {F8Plan::kDuo, s, 0});
    }
  return best;
}

}  // namespace ming

namespace {

struct DeviceGuard {
  int prev = -1;                           // the device to go back to, -1: none
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev == dev)
      prev = -1;
    else
      (void)hipSetDevice(dev);
  }
  ~DeviceGuard() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

hipStream_t stream_of(const ming_ctx* c) { return (hipStream_t)ming_ctx_stream(c); }
bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
int hip_fail(hipError_t e, const char* what) {
  return rt_fail(MING_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}
int blocks_of(int n) { return n / 128 + (n % 128 != 0); }
Span bf16_rows(const void* p, int64_t rows, int64_t ld, int64_t width) {
  return {p, rows, 2 * ld, 2 * width};
}
Span byte_rows(const void* p, int64_t rows, int64_t ld, int64_t width) { return {p, rows, ld, width}; }
Span flat(const void* p, int64_t bytes) { return {p, 1, bytes, bytes}; }
// Whether an output shares memory with another output or with an input.
bool shared(std::initializer_list<Span> ins, std::initializer_list<Span> outs) {
  for (const Span* o = outs.begin(); o != outs.end(); ++o) {
    for (const Span& i : ins)
      if (ming::spans_meet(i, *o)) return true;
    for (const Span* q = outs.begin(); q != o; ++q)
      if (ming::spans_meet(*q, *o)) return true;
  }
  return false;
}

// The rows, or places, of a call.
constexpr int kRowsMax = 1 << 28;

// A stride in elements of b bytes whose rows' last byte 64 bits hold.
bool stride_fits(int64_t ld) { return ld < (1ll << 30); }

// One launch (or a call's few), timed when the context profiles.
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

// Whether the context's kernels can read p where it is: its own device's memory.
bool own_memory(const ming_ctx* c, const void* p) {
  hipPointerAttribute_t at{};
  if (hipPointerGetAttributes(&at, p) != hipSuccess) {
    (void)hipGetLastError();
    return false;
  }
  return at.type == hipMemoryTypeDevice && at.device == ming::rt_device(c);
}

// The kernel that takes n rows of w on the current device. rt_set_f8_plan's choices: rf of
// the tiles (5: of 256 rows but for the last ones), 10 mf + nf of the few-row kernel, 100 *
// slices of f8_duo's.
ming::F8Plan plan_of(const ming_f8* w, bool grouped, int n) {
  using ming::F8Plan;
  const int set = ming::rt_f8_plan(w->ctx);
  if (set == 5 && !grouped && w->KB <= ming::kF8TileBlocks)
    return {F8Plan::kTiles, 2, (n - 1) / 256};
  if (set > 0 && set < 5 && w->KB <= ming::kF8TileBlocks) return {F8Plan::kTiles, set, 0};
  if (set >= 10 && set < 100) return {F8Plan::kRows, set / 10, set % 10};
  if (set >= 100 && !grouped && w->halves == 1 && w->KB <= ming::kF8TileBlocks)
    return {F8Plan::kDuo, std::min(set / 100, w->KB), 0};
  return ming::f8_plan(ming::device_cus(), w->halves == 2, grouped, w->E, w->NR, w->KB, n);
}
// f32 sums on their way (F8Args::part).
size_t part_bytes(const ming_f8* w, const ming::F8Plan& p, int n) {
  if (p.kind == ming::F8Plan::kRows) return w->halves == 2 ? (size_t)n * w->N * 4 : 0;
  return p.kind == ming::F8Plan::kDuo && p.a > 1
             ? (size_t)p.a * ming::f8_duo_blocks(n, w->NR) * (64 * 128 * 4)
             : 0;
}

// The most that a call of up to `rows` rows needs. A plan holds over 16 rows (a group's
// over a step) and what it needs grows with the rows, so each stretch's last ones do.
size_t workspace(const ming_f8* w, bool grouped, int rows) {
  auto need = [&](int n) { return part_bytes(w, plan_of(w, grouped, n), n); };
  size_t most = need(rows);
  const int step = grouped ? std::max(1, w->E / 8) : 16;
  const int last = std::min(rows, grouped ? ming::kPartGroupRows * w->E : ming::kPartRows);
  for (int n = step; n < last + step; n += step) {
    const int at = std::min(n, last);
    most = std::max(most, need(at));
    if (at > 1) most = std::max(most, need(at - 1));
  }
  return most;
}

// What a product's call brings.
struct Product {
  const char* who;
  bool gated, grouped;
  const uint8_t* x;
  int64_t ldx;
  const uint16_t* xs;
  int64_t ldxs;
  int x_rows;
  const int32_t* order;
  int fan;
  const int32_t* offsets;
  int n;
  const uint16_t* bias;
  uint16_t* y;           // plain
  int64_t ldy;
  uint8_t* h;            // gated
  int64_t ldh;
  uint16_t* hs;
  int64_t ldhs;
  void* ws;
  size_t ws_bytes;
};

int product(ming_ctx* c, const ming_f8* w, const Product& p) {
  auto bad = [&](int code, const char* why) {
    return rt_fail(code, std::string(p.who) + ": " + why);
  };
  if (!c || !w) return bad(MING_ERR_ARG, "null argument");
  if (w->ctx != c) return bad(MING_ERR_ARG, "weights of another context");
  if (p.n < 0 || p.x_rows < 0 || p.fan < 1) return bad(MING_ERR_ARG, "a count out of range");
  if ((w->halves == 2) != p.gated)
    return bad(MING_ERR_ARG, p.gated ? "the weights are not gated" : "the weights are gated");
  if (!p.grouped && w->E != 1) return bad(MING_ERR_ARG, "the weights are a stack of experts");
  if (p.n == 0) return rt_ok();
  if (!p.x || !p.xs || (p.grouped && !p.offsets) || (p.gated ? !p.h || !p.hs : !p.y))
    return bad(MING_ERR_ARG, "null argument");
  if (p.n > kRowsMax || p.x_rows > kRowsMax)
    return bad(MING_ERR_SHAPE, "at most 2^28 rows");
  if (p.x_rows == 0) return bad(MING_ERR_ARG, "places without rows of x");
  if (p.grouped && !p.order && p.x_rows < p.n)
    return bad(MING_ERR_SHAPE, "without an order x needs n rows");
  if (p.ldx < w->K || p.ldx % 16 != 0 || p.ldxs < p.x_rows)
    return bad(MING_ERR_SHAPE, "need ldx >= K, a multiple of 16, and ldxs >= the rows of x");
  // rows are addressed in 32 bits from the first (of a tile, where they lie in order)
  if (!stride_fits(p.ldxs) || p.ldx >= 1 << 22 ||
      (p.grouped && p.ldx > ((1ll << 31) - 1) / p.x_rows))
    return bad(MING_ERR_SHAPE, "need ldx below 2^22, ldxs below 2^30, and over groups x_rows * ldx "
                               "below 2^31");
  if (!aligned(p.x, 16) || !aligned(p.xs, 2) || !aligned(p.order, 4) || !aligned(p.offsets, 4))
    return bad(MING_ERR_ARG, "x must be 16-byte, its scales 2-byte, order and offsets 4-byte aligned");
  if (p.gated) {
    if (p.ldh < w->N || p.ldh % 16 != 0 || p.ldhs < p.n || !stride_fits(p.ldh) || !stride_fits(p.ldhs))
      return bad(MING_ERR_SHAPE, "need ldh >= N, a multiple of 16, and ldhs >= the rows, below 2^30");
    if (!aligned(p.h, 16) || !aligned(p.hs, 2))
      return bad(MING_ERR_ARG, "h must be 16-byte, its scales 2-byte aligned");
  } else {
    if (p.ldy < w->N || p.ldy % 8 != 0 || !stride_fits(p.ldy))
      return bad(MING_ERR_SHAPE, "need ldy >= N, a multiple of 8, below 2^30");
    if (!aligned(p.y, 16) || !aligned(p.bias, 8))
      return bad(MING_ERR_ARG, "y must be 16-byte, bias 8-byte aligned");
  }
  DeviceGuard g(ming::rt_device(c));       // (the plan counts its CUs)
  const ming::F8Plan plan = plan_of(w, p.grouped, p.n);
  const size_t need = part_bytes(w, plan, p.n);
  if (need > 0 && (!p.ws || !aligned(p.ws, 16)))
    return bad(MING_ERR_ARG, "ws must be given, 16-byte aligned");
  if (p.ws_bytes < need)
    return rt_fail(MING_ERR_SHAPE, std::string(p.who) + ": the call needs " + std::to_string(need) +
                                       " bytes of workspace, " + std::to_string(p.ws_bytes) +
                                       " given");
  using ming::F8Plan;
  const long long blocks =
      plan.kind == F8Plan::kTiles && plan.b > 0 ? ming::f8_mixed_blocks(plan.b, p.n, w->NR)
      : plan.kind == F8Plan::kTiles ? ming::f8_tile_blocks(plan.a, p.grouped, p.n, w->E, w->NR)
      : plan.kind == F8Plan::kDuo
          ? ming::f8_duo_blocks(p.n, w->NR) * plan.a
          : ming::f8_rows_blocks(16 * plan.a, 16 * plan.b, p.grouped, p.n, w->E, w->N);
  if (!ming::one_launch(blocks, 512) ||
      (plan.kind == F8Plan::kRows && !ming::one_launch(ming::f8_finish_blocks(p.n, w->N), 256)))
    return bad(MING_ERR_SHAPE, "more rows times columns than one launch holds");
  const Span out = p.gated ? byte_rows(p.h, p.n, p.ldh, w->N) : bf16_rows(p.y, p.n, p.ldy, w->N);
  const Span outs = bf16_rows(p.hs, p.gated ? blocks_of(w->N) : 0, p.ldhs, p.n);
  if (shared({byte_rows(p.x, p.x_rows, p.ldx, w->K), bf16_rows(p.xs, w->KB, p.ldxs, p.x_rows),
              flat(p.order, p.order ? 4ll * p.n : 0), flat(p.offsets, p.offsets ? 4ll * (w->E + 1) : 0),
              flat(p.bias, p.bias ? 2ll * w->N : 0)},
             {out, outs, flat(p.ws, (int64_t)need)}))
    return bad(MING_ERR_ARG, "inputs, outputs and ws must not share memory");
  ming::F8Args a{};
  a.x = p.x; a.ldx = p.ldx; a.xs = p.xs; a.ldxs = p.ldxs;
  a.w = w->codes; a.ws = w->scales;
  a.w_expert = (long long)w->KB * w->NR * 128;
  a.s_expert = (long long)w->KB * w->NB;
  a.N = w->N; a.K = w->K; a.KB = w->KB; a.NR = w->NR; a.NB = w->NB;
  a.n = p.n;
  a.stream = ming::f8_streams((p.gated ? 1.0 : 2.0) * p.n * w->N);
  a.offsets = p.offsets; a.order = p.order;
  a.E = w->E; a.fan = p.fan; a.x_rows = p.x_rows;
  a.bias = p.bias; a.y = p.y; a.ldy = p.ldy;
  a.h = p.h; a.ldh = p.ldh; a.hs = p.hs; a.ldhs = p.ldhs;
  a.part = static_cast<float*>(p.ws);
  const double wide = (double)w->N * w->halves, flops = 2.0 * p.n * wide * w->K;
  const double bytes = wide * w->K * std::min(p.n, w->E) + (double)p.x_rows * w->K +
                       (p.gated ? 1.0 : 2.0) * p.n * w->N;
  const int rc = run(c, p.gated ? ming::kRtF8Swiglu : ming::kRtF8Lin, flops, bytes, p.who, [&] {
    if (plan.kind == F8Plan::kTiles)
      return ming::launch_f8_tile(p.gated, p.grouped, a, plan.a, plan.b, stream_of(c));
    if (plan.kind == F8Plan::kDuo) return ming::launch_f8_duo(a, plan.a, stream_of(c));
    return ming::launch_f8_rows(p.gated, p.grouped, a, plan.a, plan.b, stream_of(c));
  });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, 8, 2ull * (uint64_t)p.n * (uint64_t)w->N * w->halves * (uint64_t)w->K);
  return rt_ok();
}

// Source memory that a creation has on the device at a time where it has to bring
// it there.
constexpr size_t kStageBytes = 64u << 20;

}  // namespace

extern "C" {

int ming_f8_quantize(ming_ctx* c, const uint16_t* x, int64_t ldx, int rows, int D, uint8_t* codes,
                     int64_t ldc, uint16_t* scales, int64_t lds) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_f8_quantize: ") + why);
  };
  if (!c || (rows > 0 && (!x || !codes || !scales))) return bad(MING_ERR_ARG, "null argument");
  if (rows < 0) return bad(MING_ERR_ARG, "rows < 0");
  if (D <= 0 || D % 16 != 0) return bad(MING_ERR_SHAPE, "need D % 16 == 0");
  if (rows == 0) return rt_ok();
  if (ldx < D || ldx % 8 != 0 || ldc < D || ldc % 16 != 0 || lds < rows || !stride_fits(ldx) ||
      !stride_fits(ldc) || !stride_fits(lds))
    return bad(MING_ERR_SHAPE, "need ldx >= D, a multiple of 8, ldc >= D, a multiple of 16, and "
                               "lds >= rows, below 2^30");
  if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(scales, 2))
    return bad(MING_ERR_ARG, "x and codes must be 16-byte, scales 2-byte aligned");
  if (!ming::one_launch(ming::f8_quantize_blocks(rows, D), 256))
    return bad(MING_ERR_SHAPE, "more rows than one launch holds");
  if (shared({bf16_rows(x, rows, ldx, D)},
             {byte_rows(codes, rows, ldc, D), bf16_rows(scales, blocks_of(D), lds, rows)}))
    return bad(MING_ERR_ARG, "x, codes and scales must not share memory");
  DeviceGuard g(ming::rt_device(c));
  const ming::F8QuantArgs a = {x,   ldx,    rows, D,  codes,
                               ldc, scales, lds,  ming::f8_streams(1.0 * rows * D)};
  const int rc = run(c, ming::kRtF8Quant, 0.0, 3.0 * rows * D, "ming_f8_quantize",
                     [&] { return ming::launch_f8_quantize(a, stream_of(c)); });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, 0, 0);
  return rt_ok();
}

int ming_f8_rmsnorm(ming_ctx* c, const uint16_t* x, int64_t ldx, const uint16_t* sub, int64_t ldsub,
                    uint16_t* h, int64_t ldh, const uint16_t* w, uint16_t* y, int64_t ldy,
                    uint8_t* codes, int64_t ldc, uint16_t* scales, int64_t lds, int rows, int D,
                    float eps) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_f8_rmsnorm: ") + why);
  };
  if (!c || (rows > 0 && (!x || !w || !codes || !scales))) return bad(MING_ERR_ARG, "null argument");
  if (rows < 0) return bad(MING_ERR_ARG, "rows < 0");
  if ((sub != nullptr) != (h != nullptr))
    return bad(MING_ERR_ARG, "sub and h are given together");
  if (D <= 0 || D % 16 != 0 || D > 8192) return bad(MING_ERR_SHAPE, "need D % 16 == 0 and D <= 8192");
  if (!(eps >= 1e-12f) || !(eps <= 1.0f)) return bad(MING_ERR_ARG, "eps must be 1e-12 to 1");
  if (rows == 0) return rt_ok();
  auto odd = [&](int64_t ld, int of) { return ld < D || ld % of != 0 || !stride_fits(ld); };
  if (odd(ldx, 8) || (sub && (odd(ldsub, 8) || odd(ldh, 8))) || (y && odd(ldy, 8)) || odd(ldc, 16) ||
      lds < rows || !stride_fits(lds))
    return bad(MING_ERR_SHAPE, "strides must be D at least, multiples of 8 (of codes 16), lds >= "
                               "rows, below 2^30");
  if (!aligned(x, 16) || !aligned(sub, 16) || !aligned(h, 16) || !aligned(w, 16) || !aligned(y, 16) ||
      !aligned(codes, 16) || !aligned(scales, 2))
    return bad(MING_ERR_ARG, "pointers must be 16-byte, scales 2-byte aligned");
  if (!ming::one_launch(rows, 512)) return bad(MING_ERR_SHAPE, "more rows than one launch holds");
  const Span xs = bf16_rows(x, rows, ldx, D), ss = bf16_rows(sub, rows, ldsub, D);
  const Span hs = bf16_rows(h, rows, ldh, D), ws = bf16_rows(w, 1, D, D);
  const Span ys = bf16_rows(y, rows, ldy, D), cs = byte_rows(codes, rows, ldc, D);
  const Span sc = bf16_rows(scales, blocks_of(D), lds, rows);
  // h may be x itself or sub itself: a thread reads both where it then writes
  const bool over_x = h == x && ldh == ldx, over_sub = h == sub && ldh == ldsub;
  if (shared({xs, ss, ws}, {ys, cs, sc}) || shared({ws}, {hs, ys, cs, sc}) ||
      (!over_x && ming::spans_meet(xs, hs)) || (!over_sub && ming::spans_meet(ss, hs)))
    return bad(MING_ERR_ARG, "inputs and outputs must not share memory (but h may be x or sub)");
  DeviceGuard g(ming::rt_device(c));
  const ming::F8NormArgs a = {x, ldx, sub, ldsub, h,   ldh,    w,   y,    ldy, codes,
                              ldc, scales, lds, rows, D, eps};
  const int rc = run(c, ming::kRtF8Norm, 0.0, (3.0 + (sub ? 4.0 : 0.0) + (y ? 2.0 : 0.0)) * rows * D,
                     "ming_f8_rmsnorm", [&] { return ming::launch_f8_norm(a, stream_of(c)); });
  if (rc != MING_OK) return rc;
  ming::rt_note_norm(c);
  return rt_ok();
}

int ming_f8_quantize_weight(ming_ctx* c, const uint16_t* w, int N, int K, uint8_t* codes,
                            float* scales) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_f8_quantize_weight: ") + why);
  };
  if (!c || !w || !codes || !scales) return bad(MING_ERR_ARG, "null argument");
  if (N <= 0 || K <= 0 || K % 16 != 0) return bad(MING_ERR_SHAPE, "need K % 16 == 0");
  if (blocks_of(N) > 65535) return bad(MING_ERR_SHAPE, "N must be at most 65535 * 128");
  if (!aligned(w, 16) || !aligned(codes, 16) || !aligned(scales, 4))
    return bad(MING_ERR_ARG, "w and codes must be 16-byte, scales 4-byte aligned");
  if (shared({bf16_rows(w, N, K, K)},
             {byte_rows(codes, N, K, K), flat(scales, 4ll * blocks_of(N) * blocks_of(K))}))
    return bad(MING_ERR_ARG, "w, codes and scales must not share memory");
  DeviceGuard g(ming::rt_device(c));
  const int rc = run(c, ming::kRtF8Quant, 0.0, 3.0 * N * K, "ming_f8_quantize_weight",
                     [&] { return ming::launch_f8_weight(w, N, K, codes, scales, stream_of(c)); });
  if (rc != MING_OK) return rc;
  ming::rt_note_rows(c, 0, 0);
  return rt_ok();
}

int ming_f8_destroy(ming_f8* w) {
  if (!w) return rt_ok();
  DeviceGuard g(ming::rt_device(w->ctx));
  (void)hipStreamSynchronize(stream_of(w->ctx));
  if (w->codes) (void)hipFree(w->codes);
  ming::rt_release(w->ctx);
  delete w;
  return rt_ok();
}

int ming_f8_create(ming_ctx* c, int n_experts, int N, int K, int gated, const uint8_t* codes,
                   const float* scales, int src_on_device, ming_f8** out) {
  auto bad = [](int code, const char* why) {
    return rt_fail(code, std::string("ming_f8_create: ") + why);
  };
  if (out) *out = nullptr;
  if (!c || !out || !codes || !scales) return bad(MING_ERR_ARG, "null argument");
  if (n_experts < 1 || n_experts > ming::kGroupMax) return bad(MING_ERR_SHAPE, "1 to 1024 experts");
  if (N <= 0 || K <= 0 || K % 16 != 0 || N % (gated ? 16 : 8) != 0)
    return bad(MING_ERR_SHAPE, "need K % 16 == 0 and N % 8 == 0, gated N % 16 == 0");
  const int halves = gated ? 2 : 1, nb = blocks_of(N), KB = blocks_of(K);
  if ((uint64_t)halves * nb * KB >= (1ull << 31) / (128 * 128))
    return bad(MING_ERR_SHAPE, "an expert's weights, padded to 128 rows and columns, must be below "
                               "2 GiB");
  DeviceGuard g(ming::rt_device(c));
  auto* w = new (std::nothrow) ming_f8();
  if (!w) return bad(MING_ERR_ALLOC, "out of memory");
  w->ctx = c; w->E = n_experts; w->N = N; w->K = K; w->halves = halves;
  w->KB = KB; w->NR = halves * nb * 128; w->NB = halves * nb;
  ming::rt_retain(c);
  const size_t E = (size_t)n_experts, one = (size_t)halves * N * K, ones = (size_t)halves * nb * KB;
  const size_t kept = (size_t)KB * w->NR * 128;
  hipStream_t s = stream_of(c);
  // arrays that the repack can read are read where they are
  const bool direct = src_on_device && aligned(codes, 16) && aligned(scales, 4) &&
                      own_memory(c, codes) && own_memory(c, scales);
  const size_t some = direct ? E : std::clamp<size_t>(kStageBytes / (one + 4 * ones), 1, E);
  const hipMemcpyKind kind = src_on_device ? hipMemcpyDefault : hipMemcpyHostToDevice;
  uint8_t* dc = nullptr;
  float* ds = nullptr;
  hipError_t e = hipMalloc(&w->codes, E * (kept + 4 * ones));
  if (e == hipSuccess) w->scales = reinterpret_cast<float*>(w->codes + E * kept);
  if (e == hipSuccess && !direct) e = hipMalloc(&dc, some * one);
  if (e == hipSuccess && !direct) e = hipMalloc(&ds, some * ones * 4);
  for (size_t i0 = 0; i0 < E && e == hipSuccess; i0 += some) {
    const size_t n = std::min(some, E - i0);
    const uint8_t* sc = codes + i0 * one;
    const float* ss = scales + i0 * ones;
    if (!direct) {                         // (behind the repack of those before, in order)
      e = hipMemcpyAsync(dc, sc, n * one, kind, s);
      if (e == hipSuccess) e = hipMemcpyAsync(ds, ss, n * ones * 4, kind, s);
      sc = dc;
      ss = ds;
    }
    if (e == hipSuccess)
      e = ming::launch_f8_repack(sc, ss, (int)n, N, K, halves, w->codes + i0 * kept,
                                 w->scales + i0 * ones, s);
  }
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (dc) (void)hipFree(dc);
  if (ds) (void)hipFree(ds);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    ming_f8_destroy(w);
    return e == hipErrorOutOfMemory ? bad(MING_ERR_ALLOC, "device allocation failed")
                                    : hip_fail(e, "ming_f8_create");
  }
  *out = w;
  return rt_ok();
}

int ming_f8_shape(const ming_f8* w, int* n_experts, int* N, int* K, int* gated) {
  if (!w) return rt_fail(MING_ERR_ARG, "ming_f8_shape: null argument");
  if (n_experts) *n_experts = w->E;
  if (N) *N = w->N;
  if (K) *K = w->K;
  if (gated) *gated = w->halves == 2;
  return rt_ok();
}

size_t ming_f8_workspace_bytes(const ming_f8* w, int rows) {
  if (!w || rows <= 0) return 0;
  rows = std::min(rows, kRowsMax);
  DeviceGuard g(ming::rt_device(w->ctx));
  const size_t grouped = workspace(w, true, rows);
  return w->E > 1 ? grouped : std::max(grouped, workspace(w, false, rows));
}

int ming_f8_lin(ming_ctx* c, const ming_f8* w, const uint8_t* x, int64_t ldx, const uint16_t* xs,
                int64_t ldxs, uint16_t* y, int64_t ldy, int M, const uint16_t* bias, void* ws,
                size_t ws_bytes) {
  Product p{};
  p.who = "ming_f8_lin";
  p.x = x; p.ldx = ldx; p.xs = xs; p.ldxs = ldxs;
  p.x_rows = p.n = M; p.fan = 1;
  p.bias = bias; p.y = y; p.ldy = ldy;
  p.ws = ws; p.ws_bytes = ws_bytes;
  return product(c, w, p);
}

int ming_f8_swiglu(ming_ctx* c, const ming_f8* w, const uint8_t* x, int64_t ldx, const uint16_t* xs,
                   int64_t ldxs, uint8_t* h, int64_t ldh, uint16_t* hs, int64_t ldhs, int M, void* ws,
                   size_t ws_bytes) {
  Product p{};
  p.who = "ming_f8_swiglu";
  p.gated = true;
  p.x = x; p.ldx = ldx; p.xs = xs; p.ldxs = ldxs;
  p.x_rows = p.n = M; p.fan = 1;
  p.h = h; p.ldh = ldh; p.hs = hs; p.ldhs = ldhs;
  p.ws = ws; p.ws_bytes = ws_bytes;
  return product(c, w, p);
}

int ming_f8_experts_lin(ming_ctx* c, const ming_f8* w, const uint8_t* x, int64_t ldx, const uint16_t* xs,
                        int64_t ldxs, int x_rows, const int32_t* order, int fan,
                        const int32_t* offsets, int n, uint16_t* y, int64_t ldy, void* ws,
                        size_t ws_bytes) {
  Product p{};
  p.who = "ming_f8_experts_lin";
  p.grouped = true;
  p.x = x; p.ldx = ldx; p.xs = xs; p.ldxs = ldxs;
  p.x_rows = x_rows; p.order = order; p.fan = fan; p.offsets = offsets; p.n = n;
  p.y = y; p.ldy = ldy;
  p.ws = ws; p.ws_bytes = ws_bytes;
  return product(c, w, p);
}

int ming_f8_experts_swiglu(ming_ctx* c, const ming_f8* w, const uint8_t* x, int64_t ldx,
                           const uint16_t* xs, int64_t ldxs, int x_rows, const int32_t* order, int fan,
                           const int32_t* offsets, int n, uint8_t* h, int64_t ldh, uint16_t* hs,
                           int64_t ldhs, void* ws, size_t ws_bytes) {
  Product p{};
  p.who = "ming_f8_experts_swiglu";
  p.gated = p.grouped = true;
  p.x = x; p.ldx = ldx; p.xs = xs; p.ldxs = ldxs;
  p.x_rows = x_rows; p.order = order; p.fan = fan; p.offsets = offsets; p.n = n;
  p.h = h; p.ldh = ldh; p.hs = hs; p.ldhs = ldhs;
  p.ws = ws; p.ws_bytes = ws_bytes;
  return product(c, w, p);
}

}  // extern "C"
