// Host side of the MXFP4 quantiser and the MXFP4 x MXFP4 matmul.
#include <hip/hip_runtime_api.h>

#include <algorithm>
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
  const int64_t grid = (g.M + rows - 1) / rows * g.spans + wblocks;
  if (grid > 0x7fffffff) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: x too large");
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)grid), dim3(256), 0, stream, args, name);
}

struct MxCfg {
  const char* name;
  int BM, BN, waves;
};
// Compiled tilings (kernel rlxq_mx_gemm_<name>).
const MxCfg kMx[] = {{"m256n256", 256, 256, 4}, {"m256n256w8", 256, 256, 8}, {"m128n128", 128, 128, 4},
                     {"m128n256", 128, 256, 4}, {"m64n64", 64, 64, 2},       {"m64n128", 64, 128, 2},
                     {"m128n64", 128, 64, 2},   {"m32n64", 32, 64, 1}};

int gemm_tiled(rlxq_ctx* ctx, rlxq_mx_gemm_args a, const void* x, int x_dtype, const MxCfg& c, int splits, void* stream) {
  a.spans = (int)((a.K + 255) / 256);
  if (splits > a.spans) splits = a.spans;
  const int per = (a.spans + splits - 1) / splits;
  a.splits = (a.spans + per - 1) / per;
  const int64_t tiles_m = (a.M + c.BM - 1) / c.BM, tiles_n = (a.N + c.BN - 1) / c.BN;
  if (tiles_m * tiles_n > 0x7ffffff0) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: too many tiles");
  const int64_t xb = (a.M + 31) / 32, wb = (a.N + 31) / 32;
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
  const int64_t grid = 8 * ((tiles_m * tiles_n + 7) / 8);
  if ((rc = launch(ctx, fn, dim3((unsigned)grid, (unsigned)a.splits), dim3(64 * c.waves), (size_t)(c.BM + c.BN) * (256 + 16), stream,
                   args, name)))
    return rc;
  if (a.splits > 1) {
    if ((rc = get_fn(ctx, "rlxq_mx_reduce", &fn))) return rc;
    const int64_t blocks = (a.M * a.N + 1023) / 1024;
    if (blocks > 0x7fffffff) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: output too large");
    if ((rc = launch(ctx, fn, dim3((unsigned)blocks), dim3(256), 0, stream, args, "rlxq_mx_reduce"))) return rc;
    ctx->last_kernel = name;
  }
  return RLXQ_OK;
}

}  // namespace

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
  const char* name = x_dtype == RLXQ_BF16 ? "rlxq_mx_quant_bf16" : "rlxq_mx_quant_f32";
  hipFunction_t fn;
  int rc = get_fn(ctx, name, &fn);
  if (rc) return rc;
  const int64_t grid = (m * (k / 8) + 255) / 256;
  if (grid > 0x7fffffff) return fail(ctx, RLXQ_E_SHAPE, "quantize_mxfp4: more than 2^42 elements");
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
  int rc;
  if (const char* e = std::getenv("RLXQ_MX_CFG")) {
    int i = -1, sp = 1;
    if (std::sscanf(e, "%d,%d", &i, &sp) >= 1 && i >= 0 && i < 8) return gemm_tiled(ctx, a, x, x_dtype, kMx[i], sp, stream);
  }
  const int64_t tiles_n = (n + 15) / 16, tiles_m = (m + 15) / 16;
  if (tiles_m > 65535) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: too many rows");
  a.spans = (int)((k + 511) / 512);
  a.splits = 1;
  void* ws = nullptr;
  if ((rc = workspace(ctx, (size_t)tiles_m * a.spans * RLXQ_MX_CHUNK, &ws, stream))) return rc;
  a.xf = static_cast<uint8_t*>(ws);
  if ((rc = quant_frag(ctx, a, x, x_dtype, 16, static_cast<uint8_t*>(ws), 0, nullptr, nullptr, stream))) return rc;
  hipFunction_t fn;
  const char* name = "rlxq_mx_dec_n1m1";
  if ((rc = get_fn(ctx, name, &fn))) return rc;
  const int waves = 8;
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)tiles_n, (unsigned)tiles_m), dim3(64 * waves), (size_t)waves * 1024, stream, args,
                name);
}

}  // extern "C"
