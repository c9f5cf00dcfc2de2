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

// The activations as fragments of `rows` rows (mxfp4_args.h).
int quant_frag(rlxq_ctx* ctx, const void* x, int x_dtype, int64_t m, int64_t k, int rows, int spans, uint8_t* xf,
               void* stream) {
  rlxq_mx_quant_args a;
  std::memset(&a, 0, sizeof a);
  a.x = x;
  a.codes = xf;
  a.M = m;
  a.K = k;
  a.rows = rows;
  a.spans = spans;
  const char* name = x_dtype == RLXQ_BF16 ? "rlxq_mx_frag_bf16" : "rlxq_mx_frag_f32";
  hipFunction_t fn;
  int rc = get_fn(ctx, name, &fn);
  if (rc) return rc;
  const int64_t threads = m * spans * (64 / rows * 16);
  if ((threads + 255) / 256 > 0x7fffffff) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: x too large");
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, args, name);
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

  const int64_t tiles_n = (n + 15) / 16, tiles_m = (m + 15) / 16;
  if (tiles_m > 65535) return fail(ctx, RLXQ_E_SHAPE, "mxfp4_gemm: too many rows");
  const int spans = (int)((k + 511) / 512);
  const size_t xf_bytes = round256((size_t)tiles_m * spans * RLXQ_MX_CHUNK);
  void* ws = nullptr;
  int rc;
  if ((rc = workspace(ctx, xf_bytes, &ws, stream))) return rc;
  uint8_t* xf = static_cast<uint8_t*>(ws);
  if ((rc = quant_frag(ctx, x, x_dtype, m, k, 16, spans, xf, stream))) return rc;

  rlxq_mx_gemm_args a;
  std::memset(&a, 0, sizeof a);
  a.xf = xf;
  a.w = w;
  a.ws = w_scales;
  a.y = y;
  a.M = m;
  a.N = n;
  a.K = k;
  a.spans = spans;
  a.splits = 1;
  a.y_bf16 = y_dtype == RLXQ_BF16;
  hipFunction_t fn;
  const char* name = "rlxq_mx_dec_n1m1";
  if ((rc = get_fn(ctx, name, &fn))) return rc;
  const int waves = 8;
  void* args[] = {&a};
  return launch(ctx, fn, dim3((unsigned)tiles_n, (unsigned)tiles_m), dim3(64 * waves), (size_t)waves * 1024, stream, args,
                name);
}

}  // extern "C"
