// Host side of the MXFP4 quantiser and the MXFP4 x MXFP4 matmul.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>

#include "mxfp4_args.h"
#include "rlxq.h"
#include "rlxq_internal.hpp"

namespace rlxq {

namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

// Groups of elements per thread of the row kernels: four once they still give
// 16 workgroups a CU (mx_quant_rows' figures).
int rows_ilp(int64_t groups) { return groups >= (int64_t)4096 * 1024 ? 4 : 1; }

// Workgroups of the preparation launch: a chunk of fragments each, and
// `wblocks` for the weights' scales.
int64_t frag_grid(const rlxq_mx_gemm_args& g, int rows, int64_t wblocks) { return (g.M + rows - 1) / rows * g.spans + wblocks; }

// The activations as fragments of `rows` rows (mxfp4_args.h); wblocks > 0:
// the weights' scales in the lane order of 32-row fragments beside them.
int quant_frag(rlxq_ctx* ctx, const rlxq_mx_gemm_args& g, const void* x, int x_dtype, int rows, uint8_t* xf,
               int wblocks, uint32_t* wsf, uint8_t* zero, void* stream) {
  rlxq_mx_quant_args a;
  std::memset(&a, 0, sizeof a);
  a.x = x;
  a.codes = xf;
  a.M = g.M;
  a.K = g.K;
  a.rows = rows;
  a.spans = g.spans;
  a.wblocks = wblocks;
  a.ws = g.ws;
  a.wsf = wsf;
  a.zero = zero;
  a.N = g.N;
  const char* name = x_dtype == RLXQ_BF16 ? "rlxq_mx_frag_bf16" : "rlxq_mx_frag_f32";
  hipFunction_t fn;
  int rc = get_fn(ctx, name, &fn);
  if (rc) return rc;
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)frag_grid(g, rows, wblocks)), dim3(256), 0, stream, args, name);
}

// Compiled tilings (kernel rlxq_mx_gemm_<name>), and what they cost: `span` us
// for 256 elements of one tile on a CU that is full of them, `solo` us where a
// tile has the CU to itself, `over` us a tile (prologue and stores).  `occ`
// tiles fit a CU (LDS).
struct MxCfg {
  const char* name;
  int BM, BN, waves, occ;
  double solo, span, over;
};
const MxCfg kMx[] = {{"m256n256", 256, 256, 8, 1, 0.0, 1.18, 11.1},
                     {"m128n128", 128, 128, 4, 2, 0.0, 0.52, 3.5},
                     {"m128n64", 128, 64, 2, 3, 0.44, 0.34, 2.3},
                     {"m64n64", 64, 64, 2, 4, 0.33, 0.25, 1.1}};

int span_splits(int spans, int splits) {   // K splits that all have spans
  if (splits > spans) splits = spans;
  const int per = (spans + splits - 1) / splits;
  return (spans + per - 1) / per;
}

// Tiling and K splits by the model above, the CUs filled evenly round by
// round, plus 3.3 us and 8 bytes per partial sum at 8.8 TB/s where K is split.
// Fitted to calls of 33 to 4096 rows, K 1056 to 12288 and N 2048 to 24576 on every
// tiling (RLXQ_MX_CFG).  It is not always the fastest: 384 x 4096 -> 24576 takes
// 51 us on the 256 x 256 tiles it picks and 42 on 128 x 128 ones, 197 x 4096 ->
// 6144 17.5 on 128 x 64 and 16.2 on 64 x 64.
const MxCfg& pick_tiling(int64_t m, int64_t k, int64_t n, int cus, int* splits) {
  const MxCfg* best = &kMx[0];
  double best_t = 1e300;
  const int spans = (int)((k + 255) / 256);
  for (const MxCfg& c : kMx) {
    const double tiles = (double)((m + c.BM - 1) / c.BM) * (double)((n + c.BN - 1) / c.BN);
    for (int sp : {1, 2, 3, 4, 6}) {
      if (sp > 1 && (sp > spans || tiles * sp > 4.0 * cus)) break;
      const int real = span_splits(spans, sp), per = (spans + real - 1) / real;
      const double n_cu = std::ceil(tiles * real / cus), full = std::floor(n_cu / c.occ), rest = n_cu - full * c.occ;
      auto round = [&](double g) { return g > 0 ? std::max(c.solo, g * c.span) * per + c.over * (0.5 + 0.5 * g) : 0.0; };
      double t = full * round(c.occ) + round(rest);
      if (real > 1) t += 3.3 + real * (double)m * (double)n * 8.0 / 8.8e6;
      if (t < best_t) best_t = t, best = &c, *splits = real;
    }
  }
  return *best;
}

int gemm_tiled(rlxq_ctx* ctx, rlxq_mx_gemm_args a, const void* x, int x_dtype, const MxCfg& c, int splits, void* stream) {
  a.spans = (int)((a.K + 255) / 256);
  a.splits = span_splits(a.spans, splits);
  const int64_t tiles_m = (a.M + c.BM - 1) / c.BM, tiles_n = (a.N + c.BN - 1) / c.BN;
  const int64_t xb = (a.M + 31) / 32, wb = (a.N + 31) / 32;
  const int64_t grid = 8 * ((tiles_m * tiles_n + 7) / 8), reduce = a.splits > 1 ? (a.M * a.N + 1023) / 1024 : 0;
  if (!grid_fits(frag_grid(a, 32, wb), 256) || !grid_fits(grid, 64 * c.waves) || !grid_fits(reduce, 256))
    return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: M, K and N need a launch of 2^32 work-items or more");
  const size_t b_xf = round256((size_t)xb * a.spans * RLXQ_MX_CHUNK), b_ws = (size_t)wb * a.spans * 256;
  const size_t b_z = round256((size_t)wb), b_part = a.splits > 1 ? (size_t)a.splits * a.M * a.N * 4 : 0;
  void* ws = nullptr;
  int rc;
  if ((rc = workspace(ctx, b_xf + b_ws + b_z + b_part, &ws, stream))) return rc;
  uint8_t* p = static_cast<uint8_t*>(ws);
  uint32_t* wsf = reinterpret_cast<uint32_t*>(p + b_xf);
  uint8_t* zero = p + b_xf + b_ws;
  if ((rc = quant_frag(ctx, a, x, x_dtype, 32, p, (int)wb, wsf, zero, stream))) return rc;
  a.xf = p;
  a.wsf = wsf;
  a.zero = zero;
  a.part = reinterpret_cast<float*>(p + b_xf + b_ws + b_z);
  char name[48];
  std::snprintf(name, sizeof name, "rlxq_mx_gemm_%s", c.name);
  hipFunction_t fn;
  if ((rc = get_fn(ctx, name, &fn))) return rc;
  void* args[] = {&a};
  if ((rc = launch(ctx, fn, dim3((unsigned)grid, (unsigned)a.splits), dim3(64 * c.waves), (size_t)(c.BM + c.BN) * (256 + 16), stream,
                   args, name)))
    return rc;
  if (a.splits > 1) {
    if ((rc = get_fn(ctx, "rlxq_mx_reduce", &fn))) return rc;
    if ((rc = launch(ctx, fn, dim3((unsigned)reduce), dim3(256), 0, stream, args, "rlxq_mx_reduce"))) return rc;
    ctx->last_kernel = name;
  }
  return RLXQ_OK;
}

// At most 32 rows: the kernel that streams the weights through registers.
//   - 32 weight rows a workgroup where that still gives 192 of them, else 16
//     (1 row, K = 4096, N = 6144: 5.8 us and 6.0; N = 4096: 5.6 and 4.9).
//   - Eight waves; sixteen where the workgroups are no more than the CUs and K
//     is long enough for them (4 rows, 12288 -> 4096: 11.4 and 10.6 us); four for
//     more than 16 rows on 32 weight rows (32 rows, 4096 -> 24576: 24.9 and 20.3).
//   - The activations quantised in the kernel up to 24576 of them: a launch less
//     (1 row, 4096 -> 24576: 12.8 us against 15.6; 2 of 12288: 11.1 and 12.0; 4 of
//     12288: 13.9 and 12.1).
int gemm_decode(rlxq_ctx* ctx, rlxq_mx_gemm_args a, const void* x, int x_dtype, void* stream) {
  a.spans = (int)((a.K + 511) / 512);
  const int cus = ctx->cu_count > 0 ? ctx->cu_count : 256;
  const int mt = a.M > 16 ? 2 : 1;
  const int nt = (a.N + 31) / 32 >= 3 * cus / 4 ? 2 : 1;
  const bool fused = mt == 1 && a.M * a.K <= 24576;
  int waves = nt == 2 && mt == 2 ? 4 : 8;
  if (nt == 1 && (a.N + 15) / 16 <= cus && (fused || a.spans >= 16)) waves = 16;
  const int64_t grid = (a.N + 16 * nt - 1) / (16 * nt);
  if (!grid_fits(grid, 64 * waves) || (!fused && !grid_fits(frag_grid(a, 16, 0), 256)))
    return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: M, K and N need a launch of 2^32 work-items or more");
  char name[48];
  if (fused) {
    std::snprintf(name, sizeof name, "rlxq_mx_dec_n%d_f%s", nt, x_dtype == RLXQ_BF16 ? "bf16" : "f32");
    a.x = x;
  } else {
    std::snprintf(name, sizeof name, "rlxq_mx_dec_n%dm%d", nt, mt);
    void* ws = nullptr;
    int rc = workspace(ctx, (size_t)mt * a.spans * RLXQ_MX_CHUNK, &ws, stream);
    if (rc) return rc;
    a.xf = static_cast<uint8_t*>(ws);
    if ((rc = quant_frag(ctx, a, x, x_dtype, 16, static_cast<uint8_t*>(ws), 0, nullptr, nullptr, stream))) return rc;
  }
  hipFunction_t fn;
  int rc = get_fn(ctx, name, &fn);
  if (rc) return rc;
  const size_t lds = (size_t)waves * nt * mt * 1024 + (fused ? (size_t)((a.spans * a.M * 272 + 15) & ~15) : 0);
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)grid), dim3(64 * waves), lds, stream, args, name);
}

}  // namespace

// Values of MXFP4 rows with E8M0 scales (rlxq_dequantize).
int mx_dequantize(rlxq_ctx* ctx, const void* codes, const void* scales, int64_t rows, int64_t k, float* out, void* stream) {
  rlxq_mx_quant_args a;
  std::memset(&a, 0, sizeof a);
  a.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  a.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  a.M = rows;
  a.K = k;
  hipFunction_t fn;
  const int u = rows_ilp(rows * (k / 4));
  int rc = get_fn(ctx, u == 1 ? "rlxq_mx_dequant_u1" : "rlxq_mx_dequant_u4", &fn);
  if (rc) return rc;
  const int64_t grid = (rows * (k / 4) + 256 * u - 1) / (256 * u);
  if (!grid_fits(grid, 256)) return fail(ctx, RLXQ_E_SHAPE, "dequantize: 2^36 weights or more");
  void* args[] = {&a, &out};
  return launch(ctx, fn, dim3((unsigned)grid), dim3(256), 0, stream, args, "dequantize");
}

}  // namespace rlxq

using namespace rlxq;

extern "C" {

int rlxq_quantize_mxfp4(rlxq_ctx* ctx, const void* x, int x_dtype, int64_t m, int64_t k, uint8_t* codes,
                        uint8_t* scales, void* stream) {
  if (!ctx) return RLXQ_E_NULL;
  ctx->last_error.clear();
  // with no rows nothing is read or written: the pointers may be NULL then
  if (m > 0 && (!x || !codes || !scales)) return fail(ctx, RLXQ_E_NULL, "quantize_mxfp4: null pointer");
  if (m < 0 || k <= 0 || m > 0x7fffffff || k > 0x7fffffff)
    return fail(ctx, RLXQ_E_SHAPE, "quantize_mxfp4: need 0 <= m < 2^31 and 0 < k < 2^31");
  if (k % 32) return fail(ctx, RLXQ_E_ALIGN, "quantize_mxfp4: K must be a multiple of 32");
  if (x_dtype != RLXQ_F32 && x_dtype != RLXQ_BF16) return fail(ctx, RLXQ_E_DTYPE, "quantize_mxfp4: x_dtype");
  if (!aligned(x, 16)) return fail(ctx, RLXQ_E_ALIGN, "quantize_mxfp4: x must be 16-byte aligned");
  if (!aligned(codes, 16)) return fail(ctx, RLXQ_E_ALIGN, "quantize_mxfp4: codes must be 16-byte aligned");
  if (m == 0) return RLXQ_OK;
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(ctx, RLXQ_E_HIP, "quantize_mxfp4: hipSetDevice");
  rlxq_mx_quant_args a;
  std::memset(&a, 0, sizeof a);
  a.x = x;
  a.codes = codes;
  a.scales = scales;
  a.M = m;
  a.K = k;
  const int u = rows_ilp(m * (k / 8));
  char name[32];
  std::snprintf(name, sizeof name, "rlxq_mx_quant_%s_u%d", x_dtype == RLXQ_BF16 ? "bf16" : "f32", u);
  hipFunction_t fn;
  int rc = get_fn(ctx, name, &fn);
  if (rc) return rc;
  const int64_t grid = (m * (k / 8) + 256 * u - 1) / (256 * u);
  if (!grid_fits(grid, 256)) return fail(ctx, RLXQ_E_SHAPE, "quantize_mxfp4: 2^37 elements or more");
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)grid), dim3(256), 0, stream, args, name);
}

int rlxq_mxfp4_gemm(rlxq_ctx* ctx, const void* x, int x_dtype, const uint8_t* w, const uint8_t* w_scales, int64_t m,
                    int64_t k, int64_t n, void* y, int y_dtype, void* stream) {
  if (!ctx) return RLXQ_E_NULL;
  ctx->last_error.clear();
  // with no rows nothing is read or written: x and y may be NULL then
  if (!w || !w_scales || (m > 0 && (!x || !y))) return fail(ctx, RLXQ_E_NULL, "mxfp4_gemm: null pointer");
  if (m < 0 || k <= 0 || n <= 0) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: need m >= 0, k > 0, n > 0");
  if (m > 0x7fffffff || n > 0x7fffffff || k > (1 << 24))
    return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: K above 2^24 or M, N above 2^31");
  if (k % 32) return fail(ctx, RLXQ_E_ALIGN, "mxfp4_gemm: K must be a multiple of 32");
  if (x_dtype != RLXQ_F32 && x_dtype != RLXQ_BF16) return fail(ctx, RLXQ_E_DTYPE, "mxfp4_gemm: x_dtype");
  if (y_dtype != RLXQ_F32 && y_dtype != RLXQ_BF16) return fail(ctx, RLXQ_E_DTYPE, "mxfp4_gemm: y_dtype");
  if (!aligned(x, 16)) return fail(ctx, RLXQ_E_ALIGN, "mxfp4_gemm: x must be 16-byte aligned");
  if (!aligned(w, 16)) return fail(ctx, RLXQ_E_ALIGN, "mxfp4_gemm: w must be 16-byte aligned");
  if (m == 0) return RLXQ_OK;
  DeviceGuard g(ctx->device);
  if (!g.ok()) return fail(ctx, RLXQ_E_HIP, "mxfp4_gemm: hipSetDevice");

  rlxq_mx_gemm_args a;
  std::memset(&a, 0, sizeof a);
  a.w = w;
  a.ws = w_scales;
  a.y = y;
  a.M = m;
  a.N = n;
  a.K = k;
  a.y_bf16 = y_dtype == RLXQ_BF16;
  a.vec = n % (y_dtype == RLXQ_BF16 ? 8 : 4) == 0 && aligned(y, 16);
  // RLXQ_MX_CFG=<tiling>[,<K splits>] selects a tiled kernel (tuning sweeps and
  // the per-variant tests)
  if (const char* e = std::getenv("RLXQ_MX_CFG")) {
    const std::string s(e), nm = s.substr(0, s.find(','));
    const int sp = s.size() > nm.size() ? std::max(1, std::atoi(s.c_str() + nm.size() + 1)) : 1;
    for (const auto& c : kMx)
      if (nm == c.name) return gemm_tiled(ctx, a, x, x_dtype, c, sp, stream);
    return fail(ctx, RLXQ_E_NOKERNEL, "mxfp4_gemm: RLXQ_MX_CFG names no compiled tiling");
  }
  // (17 to 32 rows too: the tiles' preparation and LDS ring start slower than
  // the weights stream, 4096 -> 4096 8.2 us against 11.9)
  if (m <= 32) return gemm_decode(ctx, a, x, x_dtype, stream);
  int splits = 1;
  const MxCfg& c = pick_tiling(m, k, n, ctx->cu_count > 0 ? ctx->cu_count : 256, &splits);
  return gemm_tiled(ctx, a, x, x_dtype, c, splits, stream);
}

}  // extern "C"
