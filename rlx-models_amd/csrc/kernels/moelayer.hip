// The whole routed-expert layer: router product, top-k with softmax weights,
// and the experts' products for a few tokens.
//
//   l[r, e] = sum_h x[r, h] R[e, h]
//   e_j, p_j = the top_k largest logits of the row (ties to the lower expert),
//              exp(l - max) / sum over all experts of exp(l - max)
//   a[r, j] = silu(g) * u,  g, u = gate and up rows of expert e_j times x[r]
//   y[r] = sum_j p_j * (down rows of expert e_j times a[r, j])
#include "gemv_core.hip.h"
#include "moe_args.h"

namespace rlxq {

// ------------------------------------------------------------ router product
// A logit's sum runs in f64 and is rounded once: which experts a row takes
// then does not depend on the order of the sum (its 2 E H operations a row are
// nothing beside the experts').  A wave takes EB experts and RB rows, its
// lanes four consecutive elements of every 256.
template <bool BF16>
RLXQ_DEV void load4(const void* p, int64_t i, double (&v)[4]) {
  if constexpr (BF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
    v[0] = __uint_as_float(u.x << 16);
    v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16);
    v[3] = __uint_as_float(u.y & 0xffff0000u);
  } else {
    const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  }
}

RLXQ_DEV double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Workgroup = one wave per (EB experts, RB rows); grid (experts, rows).
template <bool XBF, bool RBF, int EB, int RB>
RLXQ_DEV void moe_logits_body(const rlxq_moe_logits_args& a) {
  const int lane = threadIdx.x;
  const int e0 = blockIdx.x * EB;
  const int64_t r0 = (int64_t)blockIdx.y * RB;
  double acc[EB][RB];
#pragma unroll
  for (int i = 0; i < EB; i++)
#pragma unroll
    for (int q = 0; q < RB; q++) acc[i][q] = 0.;
  for (int64_t h = 4 * lane; h < a.H; h += 256) {
    double w[EB][4];
#pragma unroll
    for (int i = 0; i < EB; i++) load4<RBF>(a.router, (int64_t)(e0 + i < a.E ? e0 + i : a.E - 1) * a.H + h, w[i]);
#pragma unroll
    for (int q = 0; q < RB; q++) {
      double v[4];
      load4<XBF>(a.x, (r0 + q < a.rows ? r0 + q : a.rows - 1) * a.H + h, v);
#pragma unroll
      for (int i = 0; i < EB; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[i][q] = fma(w[i][c], v[c], acc[i][q]);
    }
  }
#pragma unroll
  for (int i = 0; i < EB; i++)
#pragma unroll
    for (int q = 0; q < RB; q++) {
      const double s = wave_sum(acc[i][q]);
      if (lane == 0 && e0 + i < a.E && r0 + q < a.rows) a.logits[(r0 + q) * a.E + e0 + i] = (float)s;
    }
}

// --------------------------------------------------------------------- top-k
RLXQ_DEV uint32_t wave_umax(uint32_t v) {
  auto m = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
  v = m(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
  v = m(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
  v = m(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));
  v = m(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));
  const uint32_t r0 = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), r1 = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t r2 = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), r3 = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  return m(m(r0, r1), m(r2, r3));
}

// Floats in their order as unsigned keys, all above 0 (-0 as 0).
RLXQ_DEV uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Top-k of one row by a wave: lane j < top_k ends with the j-th expert and its
// weight.  NPER * 64 >= E.  A row with no softmax (a NaN or +inf logit, or
// nothing but -inf) takes experts 0 .. top_k - 1 with weight NaN.
template <int NPER>
RLXQ_DEV void pick_row(const float* __restrict__ l, int E, int top_k, bool renorm, int& id, float& prob) {
  const int lane = threadIdx.x & 63;
  float v[NPER];
  uint32_t key[NPER];
  float mx = -INFINITY, s = 0.f;
#pragma unroll
  for (int i = 0; i < NPER; i++) {
    const int e = lane + 64 * i;
    v[i] = e < E ? l[e] : -INFINITY;
    key[i] = e < E ? order_key(v[i]) : 0u;
    mx = fmaxf(mx, v[i]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
#pragma unroll
  for (int i = 0; i < NPER; i++) s += expf(v[i] - mx);
  s = lane_group_sum<64>(s);
  if (!(s < INFINITY) || !(mx < INFINITY) || !(mx > -INFINITY)) {
    id = lane;
    prob = __uint_as_float(0x7fc00000u);
    return;
  }
  float kept = 0.f;
  id = 0;
  prob = 0.f;
  for (int j = 0; j < top_k; j++) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < NPER; i++) best = best > key[i] ? best : key[i];
    best = wave_umax(best);
    int pick = -1;
#pragma unroll
    for (int i = NPER - 1; i >= 0; i--) {
      const uint64_t b = __ballot(key[i] == best);
      if (b) pick = 64 * i + __builtin_ctzll(b);
    }
    const uint32_t u = best & 0x80000000u ? best & 0x7fffffffu : ~best;
    const float p = expf(__uint_as_float(u) - mx) / s;
    kept += p;
    if (lane == j) {
      id = pick;
      prob = p;
    }
#pragma unroll
    for (int i = 0; i < NPER; i++)
      if (lane + 64 * i == pick) key[i] = 0u;
  }
  if (renorm) prob /= kept;
}

template <int NPER>
RLXQ_DEV void moe_pick_body(const rlxq_moe_pick_args& a) {
  const int64_t r = blockIdx.x;
  int id;
  float p;
  pick_row<NPER>(a.logits + r * a.E, a.E, a.top_k, a.renorm != 0, id, p);
  if ((int)threadIdx.x < a.top_k) {
    a.ids[r * a.top_k + threadIdx.x] = id;
    a.probs[r * a.top_k + threadIdx.x] = p;
  }
}

}  // namespace rlxq

// rlxq_moe_logits_<x>_<router>_e<EB>r<RB>
#define RLXQ_LOGITS(XN, XBF, RN, RBF)                                                                               \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_logits_##XN##_##RN##_e1r4(rlxq_moe_logits_args a) {     \
    rlxq::moe_logits_body<XBF, RBF, 1, 4>(a);                                                                       \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_logits_##XN##_##RN##_e4r8(rlxq_moe_logits_args a) {     \
    rlxq::moe_logits_body<XBF, RBF, 4, 8>(a);                                                                       \
  }
RLXQ_LOGITS(f32, false, f32, false)
RLXQ_LOGITS(bf16, true, f32, false)
RLXQ_LOGITS(f32, false, bf16, true)
RLXQ_LOGITS(bf16, true, bf16, true)

#define RLXQ_PICK(NPER)                                                                                \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_pick_k##NPER(rlxq_moe_pick_args a) {       \
    rlxq::moe_pick_body<NPER>(a);                                                                      \
  }
RLXQ_PICK(1)
RLXQ_PICK(2)
RLXQ_PICK(4)
RLXQ_PICK(16)
