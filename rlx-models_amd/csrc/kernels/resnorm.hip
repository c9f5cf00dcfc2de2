// Residual norm: the norms after one block and before the next, with the gate
// and the residual sum between them, in one pass over the rows.
//
//   t = block;  t *= (o + post_w) / sqrt(mean t^2 + eps)   (post_w given)
//   h = resid + alpha * gate * t                           -> sum
//   y = h * (o + pre_w) / sqrt(mean h^2 + eps)             (pre_w given)
//
// f32 arithmetic and statistics; sum and y are each rounded once, from the f32
// h (y's norm is that of the unrounded sum).
//
// Bound by memory: 16384 x 4096 bf16 in 107 us for 537 MB, the rate of a copy (with
// its workgroups going on from row to row, the next row on its way, it took 134); 197 x 5120 in 6.0, one row in 2.6, by the latency of two sums.
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

namespace rlxq {

// Eight elements as loaded, and as floats.
template <int BF>
struct RnRaw {
  uint4 q[BF ? 1 : 2];
};
template <int BF>
RLXQ_DEV RnRaw<BF> rn_raw(const void* p, int64_t i) {
  RnRaw<BF> r;
  const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + i * (BF ? 2 : 4));
  r.q[0] = s[0];
  if constexpr (!BF) r.q[1] = s[1];
  return r;
}
template <int BF>
RLXQ_DEV void rn_unpack(const RnRaw<BF>& r, float* v) {
  if constexpr (BF) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int j = 0; j < 4; j++) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  } else {
    const uint32_t w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = __uint_as_float(w[j]);
  }
}
RLXQ_DEV void rn_ld8(const void* p, int bf16, int64_t i, float* v) {
  if (bf16) rn_unpack<1>(rn_raw<1>(p, i), v);
  else rn_unpack<0>(rn_raw<0>(p, i), v);
}
RLXQ_DEV void rn_st8(void* p, int bf16, int64_t i, const float* v) {
  if (bf16) {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// Sum over the workgroup; the waves' sums lie in red, whose half alternates
// (`turn`), so one barrier separates two sums.
RLXQ_DEV float rn_sum(float v, float (*red)[16], int& turn) {
  const int waves = blockDim.x >> 6;
  v = group_sum<64>(v);
  if (waves == 1) return v;
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < waves; w++) s += red[turn][w];
  return s;
}

// A row of whole 16-byte pieces a workgroup, in registers: CH pieces of eight a
// thread, all of block and resid on their way before the first sum; the weights and
// the gate are loaded where they are used.
template <int BB, int RB, int CH>
RLXQ_DEV void rn_row(const rlxq_resnorm_args& a) {
  __shared__ float red[2][16];
  int turn = 0;
  const int t = threadIdx.x, step = 8 * blockDim.x;
  const int64_t r = blockIdx.x;
  const float inv_h = 1.0f / (float)a.H;
  bool on[CH];
  RnRaw<BB> xb[CH];
  RnRaw<RB> xr[CH];
#pragma unroll
  for (int c = 0; c < CH; c++) {
    on[c] = 8 * t + c * step < a.H;
    const int64_t i = r * a.H + 8 * t + c * step;
    if (a.block && on[c]) xb[c] = rn_raw<BB>(a.block, i);
    if (a.resid && on[c]) xr[c] = rn_raw<RB>(a.resid, i);
  }
  float h[CH][8], res[CH][8];
#pragma unroll
  for (int c = 0; c < CH; c++) {
#pragma unroll
    for (int j = 0; j < 8; j++) h[c][j] = 0.f, res[c][j] = 0.f;
    if (a.block && on[c]) rn_unpack<BB>(xb[c], h[c]);
    if (a.resid && on[c]) rn_unpack<RB>(xr[c], res[c]);
  }
  if (a.block) {
    float post = a.alpha;
    if (a.post_w) {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < CH; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) ss += h[c][j] * h[c][j];
      post *= 1.0f / sqrtf(rn_sum(ss, red, turn) * inv_h + a.eps);
    }
    const int64_t grow = a.gate ? r / a.gate_span * a.H : 0;
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const int i = 8 * t + c * step;
      float w[8];
      if (!on[c]) continue;
      if (a.post_w) {
        rn_ld8(a.post_w, a.w_bf16, i, w);
#pragma unroll
        for (int j = 0; j < 8; j++) h[c][j] *= a.w_off + w[j];
      }
      if (a.gate) {
        rn_ld8(a.gate, a.gate_bf16, grow + i, w);
#pragma unroll
        for (int j = 0; j < 8; j++) h[c][j] *= w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; j++) h[c][j] = res[c][j] + post * h[c][j];
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
      for (int j = 0; j < 8; j++) h[c][j] = res[c][j];
  }
  if (a.sum) {
#pragma unroll
    for (int c = 0; c < CH; c++)
      if (on[c]) rn_st8(a.sum, RB, r * a.H + 8 * t + c * step, h[c]);
  }
  if (a.pre_w) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
      for (int j = 0; j < 8; j++) ss += h[c][j] * h[c][j];
    const float pre = 1.0f / sqrtf(rn_sum(ss, red, turn) * inv_h + a.eps);
#pragma unroll
    for (int c = 0; c < CH; c++) {
      if (!on[c]) continue;
      const int i = 8 * t + c * step;
      float w[8];
      rn_ld8(a.pre_w, a.w_bf16, i, w);
#pragma unroll
      for (int j = 0; j < 8; j++) w[j] = h[c][j] * pre * (a.w_off + w[j]);
      rn_st8(a.y, a.y_bf16, r * a.H + i, w);
    }
  }
}

}  // namespace rlxq

#define RLXQ_RN(B, R, bn, rn)                                                                                              \
  extern "C" __global__ __launch_bounds__(1024) void rlxq_resnorm_##bn##_##rn##_c1(rlxq_resnorm_args a) { rn_row<B, R, 1>(a); } \
  extern "C" __global__ __launch_bounds__(512) void rlxq_resnorm_##bn##_##rn##_c2(rlxq_resnorm_args a) { rn_row<B, R, 2>(a); }  \
  extern "C" __global__ __launch_bounds__(512) void rlxq_resnorm_##bn##_##rn##_c4(rlxq_resnorm_args a) { rn_row<B, R, 4>(a); }
RLXQ_RN(0, 0, f32, f32)
RLXQ_RN(0, 1, f32, bf16)
RLXQ_RN(1, 0, bf16, f32)
RLXQ_RN(1, 1, bf16, bf16)
