// Residual norm: the norms after one block and before the next, with the gate
// and the residual sum between them, in one pass over the rows.
//
//   t = block;  t *= (o + post_w) / sqrt(mean t^2 + eps)   (post_w given)
//   h = resid + alpha * gate * t                           -> sum
//   y = h * (o + pre_w) / sqrt(mean h^2 + eps)             (pre_w given)
//
// f32 arithmetic and statistics; sum and y are each rounded once, from the f32
// h (y's norm is that of the unrounded sum).
#include "common.hip.h"
#include "resnorm_args.h"

namespace rlxq {

RLXQ_DEV float rn_ld(const void* p, int bf16, int64_t i) {
  return bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
RLXQ_DEV void rn_st(void* p, int bf16, int64_t i, float v) {
  if (bf16) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16_bits(v);
  else reinterpret_cast<float*>(p)[i] = v;
}

// Sum over the workgroup (every thread gets it), the waves' sums in order.
template <int WAVES>
RLXQ_DEV float rn_block_sum(float v, float* red) {
  v = group_sum<64>(v);
  if constexpr (WAVES == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; w++) s += red[w];
  __syncthreads();
  return s;
}

}  // namespace rlxq

using namespace rlxq;

// Any width and alignment: a workgroup a row, the row read again for each
// statistic.  Every thread writes the elements it alone reads, last, so sum
// may be resid and y may be block.
extern "C" __global__ __launch_bounds__(256) void rlxq_resnorm_any(rlxq_resnorm_args a) {
  __shared__ float red[4];
  const int64_t r = blockIdx.x, row = r * a.H, grow = r / a.gate_span * a.H;
  float post = 1.f, pre = 1.f;
  if (a.block && a.post_w) {
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < a.H; c += 256) {
      const float t = rn_ld(a.block, a.block_bf16, row + c);
      ss += t * t;
    }
    post = 1.0f / sqrtf(rn_block_sum<4>(ss, red) / (float)a.H + a.eps);
  }
  auto h_at = [&](int64_t c) {
    float h = a.resid ? rn_ld(a.resid, a.resid_bf16, row + c) : 0.f;
    if (a.block) {
      float t = rn_ld(a.block, a.block_bf16, row + c);
      if (a.post_w) t *= post * (a.w_off + rn_ld(a.post_w, a.w_bf16, c));
      if (a.gate) t *= rn_ld(a.gate, a.gate_bf16, grow + c);
      h += a.alpha * t;
    }
    return h;
  };
  if (a.pre_w) {
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < a.H; c += 256) {
      const float h = h_at(c);
      ss += h * h;
    }
    pre = 1.0f / sqrtf(rn_block_sum<4>(ss, red) / (float)a.H + a.eps);
  }
  for (int64_t c = threadIdx.x; c < a.H; c += 256) {
    const float h = h_at(c);
    if (a.sum) rn_st(a.sum, a.resid_bf16, row + c, h);
    if (a.pre_w) rn_st(a.y, a.y_bf16, row + c, h * pre * (a.w_off + rn_ld(a.pre_w, a.w_bf16, c)));
  }
}
