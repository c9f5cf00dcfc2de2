// Low-rank adapters of many requests beside a shared projection:
//   y[i, n] = base[i, n] + s[e] sum_{r < rank[e]} B[e, n, r] v[i, g(n), r],
//   v[i, g, r] = sum_k A[e, g R + r, k] x[i, k],   e = ids[i],
// g(n) the segment of column n.  v stays f32.
#include "common.hip.h"
#include "lora_args.h"

namespace rlxq {

RLXQ_DEV float lr_ld(const void* p, int bf16, int64_t i) {
  return bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
// Rank of adapter e: what lies past it in A and B is never multiplied.
RLXQ_DEV int lr_rank(const rlxq_lora_args& a, int e) {
  if (!a.ranks) return a.R;
  const int r = a.ranks[e];
  return r < 0 ? 0 : (r > a.R ? a.R : r);
}

}  // namespace rlxq

using namespace rlxq;

// v: a wave per row and row of A.
extern "C" __global__ __launch_bounds__(256) void rlxq_lora_shrink(rlxq_lora_args a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), sr = (int64_t)a.S * a.R;
  if (w >= a.M * sr) return;
  const int64_t i = w / sr, j = w - i * sr;
  const int e = a.ids[i];
  if (e < 0 || e >= a.E || (int)(j % a.R) >= lr_rank(a, e)) return;
  float s = 0.f;
  for (int64_t k = threadIdx.x & 63; k < a.K; k += 64)
    s = __fmaf_rn(lr_ld(a.x, a.x_bf16, i * a.K + k), lr_ld(a.a, a.ab_bf16, (e * sr + j) * a.K + k), s);
  s = group_sum<64>(s);
  if ((threadIdx.x & 63) == 0) a.v[w] = a.scales ? s * a.scales[e] : s;
}

// y: a thread per output.
extern "C" __global__ __launch_bounds__(256) void rlxq_lora_expand(rlxq_lora_args a) {
  const int64_t o = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (o >= a.M * a.N) return;
  const int64_t i = o / a.N, n = o - i * a.N;
  const int e = a.ids[i];
  float s = a.base ? lr_ld(a.base, a.y_bf16, o) : 0.f;
  if (e < 0 || e >= a.E) {   // base's bits
    if (a.y_bf16) reinterpret_cast<uint16_t*>(a.y)[o] = a.base ? reinterpret_cast<const uint16_t*>(a.base)[o] : 0;
    else reinterpret_cast<float*>(a.y)[o] = s;
    return;
  }
  {
    int g = 0;
    while (n >= a.ends[g]) g++;
    const float* v = a.v + (i * a.S + g) * a.R;
    const int rank = lr_rank(a, e);
    float d = 0.f;
    for (int r = 0; r < rank; r++) d = __fmaf_rn(v[r], lr_ld(a.b, a.ab_bf16, ((int64_t)e * a.N + n) * a.R + r), d);
    s += d;
  }
  if (a.y_bf16) reinterpret_cast<uint16_t*>(a.y)[o] = (uint16_t)f32_to_bf16_bits(s);
  else reinterpret_cast<float*>(a.y)[o] = s;
}
