// Host side of the operators around a served batch's packed products: low-rank
// adapters, the residual norm, sampling.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>

#include "lora_args.h"
#include "resnorm_args.h"
#include "rlxq.h"
#include "rlxq_internal.hpp"
#include "sample_args.h"

using namespace rlxq;

namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool act_dtype(int d) { return d == RLXQ_F32 || d == RLXQ_BF16; }
// Whether p holds whole elements of dtype d.
bool element_aligned(const void* p, int d) { return aligned(p, d == RLXQ_BF16 ? 2 : 4); }

int run_kernel(rlxq_ctx* ctx, const char* name, int64_t grid, int threads, size_t lds, void* args, void* stream) {
  hipFunction_t fn;
  int rc = get_fn(ctx, name, &fn);
  if (rc) return rc;
  void* kargs[] = {args};
  return launch(ctx, fn, dim3((unsigned)grid), dim3(threads), lds, stream, kargs, name);
}

}  // namespace

extern "C" {

int rlxq_lora_matmul(rlxq_ctx* ctx, const void* x, int x_dtype, const int32_t* ids, const void* a, const void* b,
                     int ab_dtype, const int32_t* ranks, const float* scales, const int64_t* seg_ends, int64_t segs,
                     int64_t m, int64_t k, int64_t n, int64_t rank, int64_t num_adapters, const void* base, void* y,
                     int y_dtype, void* stream) {
  if (!ctx) return RLXQ_E_NULL;
  ctx->last_error.clear();
  if (m < 0 || n < 0 || k <= 0) return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: need m >= 0, n >= 0, k > 0");
  if (m > (1 << 24) || n > (1 << 24) || k > (1 << 24))
    return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: m, k and n up to 2^24");
  if (rank <= 0 || rank > RLXQ_LORA_MAX_RANK || rank % 8) return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: rank is a multiple of 8 up to 256");
  if (num_adapters <= 0 || num_adapters > RLXQ_LORA_MAX_ADAPTERS)
    return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: 1 to 16384 adapters");
  if (k % 8) return fail(ctx, RLXQ_E_ALIGN, "lora_matmul: K must be a multiple of 8");
  if (!act_dtype(x_dtype)) return fail(ctx, RLXQ_E_DTYPE, "lora_matmul: x_dtype");
  if (!act_dtype(ab_dtype)) return fail(ctx, RLXQ_E_DTYPE, "lora_matmul: ab_dtype");
  if (!act_dtype(y_dtype)) return fail(ctx, RLXQ_E_DTYPE, "lora_matmul: y_dtype");
  rlxq_lora_args g;
  std::memset(&g, 0, sizeof g);
  if (seg_ends) {
    if (segs < 1 || segs > RLXQ_LORA_SEGS) return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: 1 to 4 segments");
    for (int64_t i = 0; i < segs; i++) {
      if (seg_ends[i] < (i ? seg_ends[i - 1] : 0) || seg_ends[i] > n)
        return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: segment ends must rise from 0 to n");
      g.ends[i] = seg_ends[i];
    }
    if (g.ends[segs - 1] != n) return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: the last segment must end at n");
  } else {
    if (segs != 1) return fail(ctx, RLXQ_E_NULL, "lora_matmul: seg_ends of several segments");
    g.ends[0] = n;
  }
  if (m == 0 || n == 0) return RLXQ_OK;   // nothing is read or written
  if (!x || !ids || !a || !b || !y) return fail(ctx, RLXQ_E_NULL, "lora_matmul: null pointer");
  if (!aligned(x, 16) || !aligned(a, 16) || !aligned(b, 16))
    return fail(ctx, RLXQ_E_ALIGN, "lora_matmul: x, a and b must be 16-byte aligned");
  if (!element_aligned(y, y_dtype) || !element_aligned(base, y_dtype) || !aligned(ids, 4) || !aligned(ranks, 4) ||
      !aligned(scales, 4))
    return fail(ctx, RLXQ_E_ALIGN, "lora_matmul: base, y, ids, ranks and scales must be element aligned");
  DeviceGuard dg(ctx->device);
  if (!dg.ok()) return fail(ctx, RLXQ_E_HIP, "lora_matmul: hipSetDevice");
  g.x = x;
  g.ids = ids;
  g.a = a;
  g.b = b;
  g.ranks = ranks;
  g.scales = scales;
  g.base = base;
  g.y = y;
  g.M = m;
  g.K = k;
  g.N = n;
  g.R = (int32_t)rank;
  g.E = (int32_t)num_adapters;
  g.S = (int32_t)segs;
  const bool xb = x_dtype == RLXQ_BF16, ab = ab_dtype == RLXQ_BF16, yb = y_dtype == RLXQ_BF16;
  // every workgroup finds its tile among up to 256 ids, a launch of the list less (bf16,
  // rank 32, 64 rows of 16 adapters 4096 -> 6144 12.5 us against 16.9, 256 of 48 23.0
  // against 24.2), unless columns are many and adapters few: a workgroup a row and 256
  // columns then is mostly for nothing (192 rows -> 24576, 16 adapters 31.1 against
  // 26.8, 48 34.6 against 53; 256 rows of 4 33.8 against 23.0)
  const bool many = m > RLXQ_LORA_FEW || (m * n > (3 << 20) && 8 * num_adapters <= m);
  const int cus = ctx->cu_count > 0 ? ctx->cu_count : 256;
  const int64_t per = yb ? 8 : 4;   // elements of 16 bytes
  g.vec = n % per == 0 && aligned(base, 16) && aligned(y, 16);
  for (int64_t i = 0; i < segs; i++) g.vec = g.vec && g.ends[i] % per == 0;
  g.copy = base != y;
  // tiles: a row each may lead one of 16, or whole tiles from the list and one more for
  // each adapter (and for the rows without one)
  const int64_t used = std::min<int64_t>(num_adapters, m);
  const int64_t tiles = many ? m / RLXQ_LORA_ROWS + std::min<int64_t>(num_adapters + 1, m) : m;
  g.max_tiles = (int32_t)tiles;
  // v: slices of K until there is a workgroup a CU (few rows, whose workgroups are
  // small: six), of 512 elements at least; no more than eight, which every workgroup of y
  // adds up (33 rows 12288 -> 4096, 24 slices 19.6, 8 17.4).  A call with 1, 2, 4 and 8
  // slices: 4096 bf16 rows 4096 -> 24576 of rank 64 168 us, 173, 180, 193 (the rule: 1);
  // 1500 f32 rows 4096 -> 4096 of rank 256 124, 121, 121, 138 (2); 777 of rank 128 55, 41,
  // 34, 36 (6: 37); 300 bf16 rows 4096 -> 6144 of rank 16 32, 23, 19, 19 (8)
  const int64_t sr = segs * rank;
  g.jblocks = (int32_t)((sr + (many ? 63 : 15)) / (many ? 64 : 16));
  const int64_t rows_wgs = many ? (m + RLXQ_LORA_ROWS - 1) / RLXQ_LORA_ROWS : used;
  const int64_t likely = rows_wgs * g.jblocks;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>({many ? (cus + likely - 1) / likely : 6 * cus / likely, k / 512, RLXQ_LORA_SPLITS}));
  g.kslice = (int32_t)(((k + want - 1) / want + 127) / 128 * 128);
  g.splits = (int32_t)((k + g.kslice - 1) / g.kslice);
  // y: 256 columns a workgroup, or up to 1024 while there are four workgroups a CU (4096
  // rows -> 24576 256 198 us of a call, 512 170, 1024 164, 2048 185; 777 rows -> 4096 48, 55, 67)
  g.cols = 256;
  while (g.cols < 1024 && rows_wgs * (n / (2 * g.cols)) >= 4 * cus) g.cols *= 2;
  int64_t cb = 0;
  for (int64_t i = 0; i < segs; i++) {
    g.cfirst[i] = (int32_t)cb;
    cb += (g.ends[i] - (i ? g.ends[i - 1] : 0) + g.cols - 1) / g.cols;
  }
  g.cblocks = (int32_t)cb;
  const int64_t shrink = tiles * g.jblocks * g.splits, expand = tiles * cb;
  if (!grid_fits(shrink, 256) || !grid_fits(expand, 256))
    return fail(ctx, RLXQ_E_SHAPE, "lora_matmul: m, n and rank need a launch of 2^32 work-items or more");
  const size_t b_v = ((size_t)(g.splits * m * sr) * 4 + 255) & ~(size_t)255;
  const size_t b_tiles = many ? (size_t)tiles * sizeof(rlxq_lora_tile) : 0;
  void* ws = nullptr;
  int rc = workspace(ctx, b_v + b_tiles + (many ? (size_t)m * 4 : 0), &ws, stream);
  if (rc) return rc;
  g.v = static_cast<float*>(ws);
  g.tiles = reinterpret_cast<rlxq_lora_tile*>(static_cast<char*>(ws) + b_v);
  g.order = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + b_v + b_tiles);
  static const char* const kDt[2] = {"f32", "bf16"};
  const char* size = many ? "many" : "few";
  char name[48];
  if (many && (rc = run_kernel(ctx, "rlxq_lora_sort", 1, 1024, (size_t)(num_adapters + 1) * 4, &g, stream))) return rc;
  std::snprintf(name, sizeof name, "rlxq_lora_shrink_%s_%s_%s", kDt[xb], kDt[ab], size);
  if ((rc = run_kernel(ctx, name, shrink, 256, 0, &g, stream))) return rc;
  const size_t pieces = ab ? 3 : 2;   // of v, a lane (lr_expand)
  const int steps = rank <= 32 ? 1 : (rank <= 64 ? 2 : (rank <= 128 ? 4 : 8));
  std::snprintf(name, sizeof name, "rlxq_lora_expand_%s_%s_%s_s%d", kDt[ab], kDt[yb], size, steps);
  return run_kernel(ctx, name, expand, 256, (size_t)((rank + 31) / 32) * (many ? RLXQ_LORA_ROWS / 16 : 1) * pieces * 1024, &g, stream);
}

int rlxq_residual_norm(rlxq_ctx* ctx, const void* block, int block_dtype, const void* resid, int resid_dtype,
                       const void* gate, int gate_dtype, int64_t gate_rows, const void* post_weight,
                       const void* pre_weight, int weight_dtype, float weight_offset, float scale, float eps,
                       int64_t rows, int64_t hidden, void* sum, void* y, int y_dtype, void* stream) {
  if (!ctx) return RLXQ_E_NULL;
  ctx->last_error.clear();
  if (rows < 0 || hidden <= 0) return fail(ctx, RLXQ_E_SHAPE, "residual_norm: need rows >= 0, hidden > 0");
  if (hidden > (1 << 24)) return fail(ctx, RLXQ_E_SHAPE, "residual_norm: hidden up to 2^24");
  if (!grid_fits(rows, 1024)) return fail(ctx, RLXQ_E_SHAPE, "residual_norm: rows need a launch of 2^32 work-items or more");
  if ((block && !act_dtype(block_dtype)) || !act_dtype(resid_dtype) || (gate && !act_dtype(gate_dtype)) ||
      ((post_weight || pre_weight) && !act_dtype(weight_dtype)) || (y && !act_dtype(y_dtype)))
    return fail(ctx, RLXQ_E_DTYPE, "residual_norm: dtypes are f32 or bf16");
  if (!(eps >= 0.0f)) return fail(ctx, RLXQ_E_SHAPE, "residual_norm: eps must be >= 0");
  if (gate && (gate_rows <= 0 || (rows > 0 && (gate_rows > rows || rows % gate_rows))))
    return fail(ctx, RLXQ_E_SHAPE, "residual_norm: gate_rows must divide rows");
  if (rows == 0) return RLXQ_OK;   // nothing is read or written
  if (!block && !resid) return fail(ctx, RLXQ_E_NULL, "residual_norm: neither block nor resid");
  if (!block && (gate || post_weight)) return fail(ctx, RLXQ_E_NULL, "residual_norm: gate and post_weight need block");
  if (!sum && !y) return fail(ctx, RLXQ_E_NULL, "residual_norm: neither sum nor y");
  if ((y == nullptr) != (pre_weight == nullptr)) return fail(ctx, RLXQ_E_NULL, "residual_norm: y and pre_weight go together");
  if (!element_aligned(block, block_dtype) || !element_aligned(resid, resid_dtype) || !element_aligned(gate, gate_dtype) ||
      !element_aligned(post_weight, weight_dtype) || !element_aligned(pre_weight, weight_dtype) ||
      !element_aligned(sum, resid_dtype) || !element_aligned(y, y_dtype))
    return fail(ctx, RLXQ_E_ALIGN, "residual_norm: pointers must be element aligned");
  DeviceGuard dg(ctx->device);
  if (!dg.ok()) return fail(ctx, RLXQ_E_HIP, "residual_norm: hipSetDevice");
  rlxq_resnorm_args g;
  std::memset(&g, 0, sizeof g);
  g.block = block;
  g.resid = resid;
  g.gate = gate;
  g.post_w = post_weight;
  g.pre_w = pre_weight;
  g.sum = sum;
  g.y = y;
  g.M = rows;
  g.H = hidden;
  g.gate_span = gate ? rows / gate_rows : 1;
  g.alpha = scale;
  g.eps = eps;
  g.w_off = weight_offset;
  g.block_bf16 = block_dtype == RLXQ_BF16;
  g.resid_bf16 = resid_dtype == RLXQ_BF16;
  g.gate_bf16 = gate_dtype == RLXQ_BF16;
  g.w_bf16 = weight_dtype == RLXQ_BF16;
  g.y_bf16 = y_dtype == RLXQ_BF16;
  bool vec = hidden % 8 == 0 && hidden <= 16384;
  for (const void* p : {block, resid, gate, post_weight, pre_weight, static_cast<const void*>(sum), static_cast<const void*>(y)})
    vec = vec && aligned(p, 16);
  if (!vec) return run_kernel(ctx, "rlxq_resnorm_any", rows, 256, 0, &g, stream);
  // pieces of eight a thread: two with many rows (512 of 5120 f32, a call with one piece
  // 10.4 us, two 11.1; 2048 of 8192 bf16 31.1 against 28.7, four 30.6)
  const int cus = ctx->cu_count > 0 ? ctx->cu_count : 256;
  const int64_t pieces = hidden / 8;
  const int ch = pieces > 1024 ? 4 : (pieces <= 64 || rows <= 2 * cus ? 1 : 2);
  const int threads = (int)(((pieces + ch - 1) / ch + 63) / 64 * 64);
  static const char* const kDt[2] = {"f32", "bf16"};
  char name[40];
  std::snprintf(name, sizeof name, "rlxq_resnorm_%s_%s_c%d", kDt[block ? g.block_bf16 : 0], kDt[g.resid_bf16], ch);
  return run_kernel(ctx, name, rows, threads, 0, &g, stream);
}

int rlxq_sample(rlxq_ctx* ctx, const void* logits, int logits_dtype, int64_t rows, int64_t vocab,
                const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, const float* u,
                int32_t* tokens, float* probs, void* stream) {
  if (!ctx) return RLXQ_E_NULL;
  ctx->last_error.clear();
  if (rows < 0 || vocab <= 0) return fail(ctx, RLXQ_E_SHAPE, "sample: need rows >= 0, vocab > 0");
  if (vocab > RLXQ_SAMPLE_MAX_VOCAB) return fail(ctx, RLXQ_E_SHAPE, "sample: vocab up to 2^20");
  if (!grid_fits(rows, 1024)) return fail(ctx, RLXQ_E_SHAPE, "sample: rows need a launch of 2^32 work-items or more");
  if (!act_dtype(logits_dtype)) return fail(ctx, RLXQ_E_DTYPE, "sample: logits_dtype");
  if (rows == 0) return RLXQ_OK;   // nothing is read or written
  if (!logits || !u || !tokens) return fail(ctx, RLXQ_E_NULL, "sample: null pointer");
  if (!element_aligned(logits, logits_dtype) || !aligned(temperature, 4) || !aligned(top_k, 4) || !aligned(top_p, 4) ||
      !aligned(min_p, 4) || !aligned(u, 4) || !aligned(tokens, 4) || !aligned(probs, 4))
    return fail(ctx, RLXQ_E_ALIGN, "sample: pointers must be element aligned");
  DeviceGuard dg(ctx->device);
  if (!dg.ok()) return fail(ctx, RLXQ_E_HIP, "sample: hipSetDevice");
  rlxq_sample_args g;
  std::memset(&g, 0, sizeof g);
  g.logits = logits;
  g.temperature = temperature;
  g.top_k = top_k;
  g.top_p = top_p;
  g.min_p = min_p;
  g.u = u;
  g.tokens = tokens;
  g.probs = probs;
  g.M = rows;
  g.V = (int32_t)vocab;
  g.bf16 = logits_dtype == RLXQ_BF16;
  const bool bf = logits_dtype == RLXQ_BF16;
  const int lead = bf ? 7 : 3;   // elements ahead of the row in its first 16 bytes, at most
  g.chunks = (int32_t)((vocab + lead + RLXQ_SAMPLE_CHUNK - 1) / RLXQ_SAMPLE_CHUNK);
  // rows in batches whose chunks take up to 128 MB of scratch
  const int64_t row_bytes = g.chunks * (int64_t)(sizeof(rlxq_sample_chunk) + RLXQ_SAMPLE_BINS * (8 + 2));
  const int cus = ctx->cu_count > 0 ? ctx->cu_count : 256;
  const int64_t batch = std::min<int64_t>(rows, std::max<int64_t>(1, (128 << 20) / row_bytes));
  const size_t b_heads = ((size_t)(batch * g.chunks) * sizeof(rlxq_sample_chunk) + 255) & ~(size_t)255;
  void* ws = nullptr;
  int rc = workspace(ctx, b_heads + (size_t)(batch * g.chunks) * RLXQ_SAMPLE_BINS * (8 + 2), &ws, stream);
  if (rc) return rc;
  g.heads = static_cast<rlxq_sample_chunk*>(ws);
  g.masses = reinterpret_cast<uint64_t*>(static_cast<char*>(ws) + b_heads);
  g.counts = reinterpret_cast<uint16_t*>(g.masses + batch * g.chunks * RLXQ_SAMPLE_BINS);
  for (int64_t at = 0; at < rows; at += batch) {
    g.M = std::min(batch, rows - at);
    // A chunk a workgroup, or up to three while there are six workgroups a CU.  It
    // matters little; a call with 1, 2, 3, 4 and 6 chunks: 256 bf16 rows of 128000
    // without borders 51 us, 44, 45, 44, 48 (the rule: 3); 1024 f32 rows of 50257 93, 92,
    // 92, 100, 95 (3); 512 of 32000 40, 39, 41, 40, 46 (2); 64 of 151936 24, 25, 26, 26, 29 (1)
    g.per = (int32_t)std::max<int64_t>(1, std::min<int64_t>(3, g.M * g.chunks / (6 * cus)));
    g.logits = static_cast<const char*>(logits) + at * vocab * (bf ? 2 : 4);
    if (temperature) g.temperature = temperature + at;
    if (top_k) g.top_k = top_k + at;
    if (top_p) g.top_p = top_p + at;
    if (min_p) g.min_p = min_p + at;
    g.u = u + at;
    g.tokens = tokens + at;
    if (probs) g.probs = probs + at;
    const int64_t hist = g.M * ((g.chunks + g.per - 1) / g.per);
    if ((rc = run_kernel(ctx, bf ? "rlxq_sample_hist_bf16" : "rlxq_sample_hist_f32", hist, RLXQ_SAMPLE_CHUNK / 16, 0, &g, stream)) ||
        (rc = run_kernel(ctx, bf ? "rlxq_sample_pick_bf16" : "rlxq_sample_pick_f32", g.M, 512, 0, &g, stream)))
      return rc;
  }
  return RLXQ_OK;
}

}  // extern "C"
