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

// One wave: experts eb EB .., rows rb RB ...
template <bool XBF, bool RBF, int EB, int RB>
RLXQ_DEV void moe_logits_body(const rlxq_moe_logits_args& a, int eb, int64_t rb) {
  const int lane = threadIdx.x;
  const int e0 = eb * EB;
  const int64_t r0 = rb * RB;
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

// ------------------------------------------------------- rows as f16 planes
// Four elements of a block per lane, eight lanes a block: the block's scale,
// its planes and sums (moe_args.h).  v is zero where there is no element.
struct PlaneQuad {
  uint2 hi, lo;
  float inv, sum, sum16;   // (the same in the block's eight lanes)
};
RLXQ_DEV PlaneQuad plane_quad(const float (&x)[4], bool want_lo) {
  PlaneQuad r;
  const float s = (x[0] + x[1]) + (x[2] + x[3]);
  r.sum = group8_sum(s);
  r.sum16 = group4_sum(s);   // (lanes 0..3: of the first 16 elements)
  const float amax = group8_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
  // 2^e: amax 2^-e in [2^14, 2^15); the float's own exponent bits.  (An infinity
  // or a NaN stays what it is under any scale.)
  int e = (int)(__float_as_uint(amax) >> 23) - 127 - 14;
  e = amax < INFINITY ? (e < -126 ? -126 : e) : 0;
  const float sc = __uint_as_float((uint32_t)(127 - e) << 23);
  r.inv = __uint_as_float((uint32_t)(127 + e) << 23);
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float v = x[i] * sc;
    h[i] = f32_to_f16_bits(v);
    l[i] = want_lo ? f32_to_f16_bits(v - f16_bits_to_f32(h[i])) : 0u;
  }
  r.hi = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  r.lo = make_uint2(l[0] | (l[1] << 16), l[2] | (l[3] << 16));
  return r;
}

// Router logits (workgroups 0 .. lblocks - 1, one wave each) and, beside them,
// the prepared rows.
template <bool XBF, bool RBF>
RLXQ_DEV void moe_prep_body(const rlxq_moe_prep_args& a) {
  if ((int)blockIdx.x < a.lblocks) {
    moe_logits_body<XBF, RBF, 1, 4>(a.r, blockIdx.x % a.r.E, blockIdx.x / a.r.E);
    return;
  }
  const int64_t i = (int64_t)(blockIdx.x - a.lblocks) * 64 + threadIdx.x, n4 = a.r.rows * a.r.H / 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (i < n4) {   // (H is whole blocks: uniform over a block's lanes)
    double d[4];
    load4<XBF>(a.r.x, 4 * i, d);
#pragma unroll
    for (int q = 0; q < 4; q++) v[q] = (float)d[q];
  }
  const PlaneQuad p = plane_quad(v, !XBF);
  if (i >= n4) return;
  reinterpret_cast<uint2*>(a.hi)[i] = p.hi;
  if (!XBF) reinterpret_cast<uint2*>(a.lo)[i] = p.lo;
  if ((threadIdx.x & 7) == 0) reinterpret_cast<float4*>(a.meta)[i >> 3] = make_float4(p.inv, p.sum, p.sum16, 0.f);
}

// ------------------------------------------------- products for few tokens
// A weight row is spread over L = 2^log2l lanes of a wave, lane li holding units
// li, li + L, ... (NU of them; a unit is one or two 32-weight blocks), the same
// units of the activation row in its registers; 64 / L rows go at once.  Codes
// become exact f16 integers (the offset of the bit pattern subtracted), so the
// products with the f16 planes are exact in v_dot2_f32_f16 and a block's sum is
// an f32 sum of its 32 (64 with the lo plane) products, which then takes the
// block's scale (times the activation block's power of two) and, for formats
// with a minimum, the minimum times the block's sum of activations.

// f16 pairs of block bl of a unit in the scheme's order, exact integers.
template <int SCH>
RLXQ_DEV void block_f16(const uint32_t* dw, int bl, uint32_t* pw, const UnpackK& k) {
  if constexpr (SCH == SCH_MXFP4) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      pw[4 * i + 0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(dw[i], 1.0f, 0));
      pw[4 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(dw[i], 1.0f, 1));
      pw[4 * i + 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(dw[i], 1.0f, 2));
      pw[4 * i + 3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(dw[i], 1.0f, 3));
    }
  } else {
    block_pairs<SCH>(dw, bl, pw, k);   // f16 1024 + code (8-bit codes; k.magic makes it so for nibbles)
    constexpr float off = SCH == SCH_Q4_0 ? 1032.f : SCH == SCH_Q3_K ? 1028.f : SCH == SCH_Q6_K ? 1056.f
                          : (SCH == SCH_Q8_0 || SCH == SCH_Q8_K) ? 1152.f : 1024.f;
    const rlxq_f16x2_t o = {(_Float16)off, (_Float16)off};
#pragma unroll
    for (int t = 0; t < 16; t++) {
      // (Q5_K, Q2_K and Q3_K pairs come as bf16 128 + code)
      if constexpr (SCH == SCH_Q5_K || SCH == SCH_Q2_K || SCH == SCH_Q3_K) pw[t] ^= 0x43004300u ^ 0x64006400u;
      pw[t] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(rlxq_f16x2_t, pw[t]) - o);
    }
  }
}

// Natural f16 pairs (x[2i], x[2i+1]) of a block in the scheme's pair order.
template <int SCH>
RLXQ_DEV void planes_from_raw(const uint32_t* R, uint32_t* X) {
  // (byte codes and the 2 to 6-bit K-quants pair as Q4_K's nibbles do)
  constexpr int AS = SCH == SCH_MXFP4 || SCH == SCH_Q4_0 || SCH == SCH_Q4_1 ? SCH : SCH_Q4_K;
  pairs_from_raw<AS>(R, X);
}

template <int SCH, int NU, int NPL>
struct FewX {
  static constexpr int NB = NU * Unit<SCH>::BLOCKS;
  uint32_t h[NB][16], l[NPL == 2 ? NB : 1][16];
  float inv[NB], sum[NB], sum16[half_scales<SCH>() ? NB : 1];

  // The lane's blocks of a row: planes hi / lo [K] and meta [K / 32][4].
  RLXQ_DEV void load(const uint16_t* hi, const uint16_t* lo, const float* meta, const int* uc, const bool* uok) {
#pragma unroll
    for (int c = 0; c < NU; c++)
#pragma unroll
      for (int bl = 0; bl < Unit<SCH>::BLOCKS; bl++) {
        const int i = c * Unit<SCH>::BLOCKS + bl, b = uc[c] * Unit<SCH>::BLOCKS + bl;
        uint32_t R[16];
        auto plane = [&](const uint16_t* p, uint32_t* X) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const uint4 v = reinterpret_cast<const uint4*>(p + 32 * b)[q];
            R[4 * q] = v.x; R[4 * q + 1] = v.y; R[4 * q + 2] = v.z; R[4 * q + 3] = v.w;
          }
          planes_from_raw<SCH>(R, X);
        };
        plane(hi, h[i]);
        if constexpr (NPL == 2) plane(lo, l[i]);
        const float4 m = reinterpret_cast<const float4*>(meta)[b];
        // (a unit past the row's end repeats the last one, times zero)
        inv[i] = uok[c] ? m.x : 0.f;
        sum[i] = uok[c] ? m.y : 0.f;
        if constexpr (half_scales<SCH>()) sum16[i] = uok[c] ? m.z : 0.f;
        if (!uok[c]) {
#pragma unroll
          for (int t = 0; t < 16; t++) {
            h[i][t] = 0u;
            if constexpr (NPL == 2) l[i][t] = 0u;
          }
        }
      }
  }
};

template <int SCH, int NU>
struct FewW {
  uint32_t dw[NU][Unit<SCH>::DW];
  uint32_t sc[SCH == SCH_MXFP4 ? NU : 1];

  // A lane's units of the packed row at p (MXFP4: its scale bytes at s).
  RLXQ_DEV void load(const uint8_t* p, const uint8_t* s, const int* uc) {
#pragma unroll
    for (int c = 0; c < NU; c++) {
      load_unit_at<SCH>(dw[c], p, uc[c]);
      if constexpr (SCH == SCH_MXFP4) sc[c] = s[uc[c]];
    }
  }
};

// The lane's part of a weight row times the activation row.
template <int SCH, int NU, int NPL>
RLXQ_DEV float few_dot(const FewW<SCH, NU>& w, const FewX<SCH, NU, NPL>& x, const int* uc, const UnpackK& kc) {
  constexpr int BLOCKS = Unit<SCH>::BLOCKS;
  float acc = 0.f;
#pragma unroll
  for (int c = 0; c < NU; c++)
#pragma unroll
    for (int bl = 0; bl < BLOCKS; bl++) {
      const int i = c * BLOCKS + bl;
      uint32_t pw[16];
      block_f16<SCH>(w.dw[c], bl, pw, kc);
      if constexpr (half_scales<SCH>()) {   // a scale (and minimum) per 16 weights
        float d, d2, m = 0.f, m2 = 0.f;
        if constexpr (SCH == SCH_Q6_K) block_scales<SCH>(w.dw[c], bl, d, d2, uc[c]);
        else block_scales_half<SCH>(w.dw[c], d, d2, m, m2);
        float c0 = 0.f, c1 = 0.f;
#pragma unroll
        for (int t = 0; t < 8; t++) {
          c0 = dot2_f16(pw[t], x.h[i][t], c0);
          c1 = dot2_f16(pw[8 + t], x.h[i][8 + t], c1);
          if constexpr (NPL == 2) {
            c0 = dot2_f16(pw[t], x.l[i][t], c0);
            c1 = dot2_f16(pw[8 + t], x.l[i][8 + t], c1);
          }
        }
        acc = fmaf(d * x.inv[i], c0, acc);
        acc = fmaf(d2 * x.inv[i], c1, acc);
        if constexpr (SCH == SCH_Q2_K) {
          acc = fmaf(m, x.sum16[i], acc);
          acc = fmaf(m2, x.sum[i] - x.sum16[i], acc);
        }
      } else {
        float d, m = 0.f;
        if constexpr (SCH == SCH_MXFP4) d = e8m0_to_f32(w.sc[c]);
        else block_scales<SCH>(w.dw[c], bl, d, m, uc[c]);
        float c0 = 0.f, c1 = 0.f;
#pragma unroll
        for (int t = 0; t < 16; t++) {
          c0 = dot2_f16(pw[t], x.h[i][t], c0);
          if constexpr (NPL == 2) c1 = dot2_f16(pw[t], x.l[i][t], c1);
        }
        acc = fmaf(d * x.inv[i], NPL == 2 ? c0 + c1 : c0, acc);
        if constexpr (SCH == SCH_Q4_1 || SCH == SCH_Q4_K || SCH == SCH_Q5_K) acc = fmaf(m, x.sum[i], acc);
      }
    }
  return acc;
}

// Sum over aligned groups of L = 2^log2l lanes (4 .. 64), in every lane of the
// group; the branches are uniform.
RLXQ_DEV float few_sum(float v, int log2l) {
  v = group4_sum(v);
  if (log2l == 2) return v;
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xF, 0xF, false));
  if (log2l == 3) return v;
  v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xF, 0xF, false));
  if (log2l == 4) return v;
  const float r0 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 0));
  const float r1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16));
  const float r2 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 32));
  const float r3 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 48));
  if (log2l == 5) return (threadIdx.x & 32) ? r2 + r3 : r0 + r1;
  return (r0 + r1) + (r2 + r3);
}

RLXQ_DEV UnpackK f16_unpack_consts() {
  UnpackK k{0x000F000Fu, 0x64006400u};
  asm volatile("" : "+v"(k.mask), "+v"(k.magic));
  return k;
}

constexpr int FEW_ENTRIES = 256;   // most (row, slot) pairs of a call

// gate|up and SwiGLU.  Every workgroup routes all rows itself (a wave a row:
// the grid is one round of workgroups, so the layer pays for it once, where a
// launch of its own would cost more), then the waves share the (entry, group of
// columns) steps evenly.  Workgroup 0 leaves the routing for the down launch.
template <int SCH, int NU, int NPL>
RLXQ_DEV void moe_few_gate_up(const rlxq_moe_few_args& a) {
  __shared__ int32_t ids[FEW_ENTRIES];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int n = a.rows * a.top_k;
  for (int r = wv; r < a.rows; r += nw) {
    int id;
    float p;
    const float* l = a.logits + (int64_t)r * a.E;
    if (a.E <= 128) pick_row<2>(l, a.E, a.top_k, a.renorm != 0, id, p);
    else if (a.E <= 256) pick_row<4>(l, a.E, a.top_k, a.renorm != 0, id, p);
    else pick_row<16>(l, a.E, a.top_k, a.renorm != 0, id, p);
    if (lane < a.top_k) {
      const int i = r * a.top_k + lane;
      ids[i] = id;
      if (blockIdx.x == 0) {
        a.ids[i] = id;
        a.probs[i] = p;
        if (a.ids2) a.ids2[i] = id;
        if (a.probs2) a.probs2[i] = p;
      }
    }
  }
  __syncthreads();
  const int L = 1 << a.log2l, RP = 64 >> a.log2l;
  const int g = lane >> a.log2l, li = lane & (L - 1);
  const int U = a.H / 32 / Unit<SCH>::BLOCKS;
  int uc[NU];
  bool uok[NU];
#pragma unroll
  for (int c = 0; c < NU; c++) {
    const int u = li + L * c;
    uok[c] = u < U;
    uc[c] = uok[c] ? u : U - 1;
  }
  const UnpackK kc = f16_unpack_consts();
  const int steps = (a.I + RP - 1) / RP;   // of an entry
  const int64_t total = (int64_t)n * steps, waves = (int64_t)gridDim.x * nw, w = (int64_t)blockIdx.x * nw + wv;
  int64_t s = total * w / waves;
  const int64_t s_end = total * (w + 1) / waves;
  while (s < s_end) {
    const int ent = (int)(s / steps), c0 = (int)(s - (int64_t)ent * steps);
    const int c1 = (int)(s_end - (int64_t)ent * steps < steps ? s_end - (int64_t)ent * steps : steps);
    const int e = __builtin_amdgcn_readfirstlane(ids[ent]), r = ent / a.top_k;
    const uint8_t* base = a.bank + (int64_t)e * 2 * a.I * a.rb;
    const uint8_t* sbase = SCH == SCH_MXFP4 ? a.scales + (int64_t)e * 2 * a.I * (a.H / 32) : nullptr;
    FewW<SCH, NU> gate[2], up[2];
    auto load = [&](int c, int slot) {
      int col = c * RP + g;
      col = col < a.I ? col : a.I - 1;
      gate[slot].load(base + (int64_t)col * a.rb, sbase + (int64_t)col * (a.H / 32), uc);
      up[slot].load(base + (int64_t)(a.I + col) * a.rb, sbase + (int64_t)(a.I + col) * (a.H / 32), uc);
    };
    FewX<SCH, NU, NPL> x;
    load(c0, 0);
    x.load(a.hi + (int64_t)r * a.H, NPL == 2 ? a.lo + (int64_t)r * a.H : nullptr, a.meta + (int64_t)r * (a.H / 32) * 4, uc, uok);
    auto step = [&](int c, int slot) {
      const float gv = few_sum(few_dot<SCH, NU, NPL>(gate[slot], x, uc, kc), a.log2l);
      const float uv = few_sum(few_dot<SCH, NU, NPL>(up[slot], x, uc, kc), a.log2l);
      const int col = c * RP + g;
      if (li == 0 && col < a.I) a.act[(int64_t)ent * a.I + col] = gv / (1.f + expf(-gv)) * uv;
    };
    int c = c0;
    for (; c + 1 < c1; c += 2) {   // (the next step's weights while this one is multiplied)
      load(c + 1, 1);
      step(c, 0);
      if (c + 2 < c1) load(c + 2, 0);
      step(c + 1, 1);
    }
    if (c < c1) step(c, 0);
    s = (int64_t)ent * steps + c1;
  }
}

// down and the weighted sum, a workgroup per (row, tile of columns): the row's
// top_k activation vectors become planes in LDS, the waves share the slots
// (waves / top_k of them per slot, each a part of the tile), and the slots are
// added in slot order.  slots at once: top_k up to the waves, else all in turns.
template <int SCH, int NU>
RLXQ_DEV void moe_few_down(const rlxq_moe_few_args& a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int r = blockIdx.x / a.tiles, c_beg = (blockIdx.x % a.tiles) * a.tile;
  const int c_end = c_beg + a.tile < a.H ? c_beg + a.tile : a.H;
  const int K = a.I, nb = K / 32;
  uint16_t* hi = reinterpret_cast<uint16_t*>(few_lds);            // [top_k][K]
  uint16_t* lo = hi + a.top_k * K;
  float* meta = reinterpret_cast<float*>(lo + a.top_k * K);       // [top_k][nb][4]
  float* vals = meta + a.top_k * nb * 4;                          // [top_k][tile]

  const int L = 1 << a.log2l, RP = 64 >> a.log2l;
  const int g = lane >> a.log2l, li = lane & (L - 1);
  const int U = nb / Unit<SCH>::BLOCKS;
  int uc[NU];
  bool uok[NU];
#pragma unroll
  for (int c = 0; c < NU; c++) {
    const int u = li + L * c;
    uok[c] = u < U;
    uc[c] = uok[c] ? u : U - 1;
  }
  const UnpackK kc = f16_unpack_consts();
  // wave -> slot and part of the tile
  const int parts = nw / a.top_k > 1 ? nw / a.top_k : 1;
  const int j0 = wv / parts, part = wv - j0 * parts, jstep = nw / parts;
  const int psize = ((a.tile + parts - 1) / parts + RP - 1) / RP * RP;   // whole steps
  const int p_beg = c_beg + part * psize, p_end = p_beg + psize < c_end ? p_beg + psize : c_end;

  FewW<SCH, NU> w[2];
  auto load = [&](int e, int col, int slot) {
    col += g;
    col = col < a.H ? col : a.H - 1;
    w[slot].load(a.bank + ((int64_t)e * a.H + col) * a.rb,
                 SCH == SCH_MXFP4 ? a.scales + ((int64_t)e * a.H + col) * nb : nullptr, uc);
  };
  int j = j0;
  int e = j < a.top_k ? __builtin_amdgcn_readfirstlane(a.ids[r * a.top_k + j]) : 0;
  if (j < a.top_k && p_beg < p_end) load(e, p_beg, 0);
  // the row's activation vectors as planes
  const float* act = a.act + (int64_t)r * a.top_k * K;
  const int n4 = a.top_k * K / 4;
  for (int i0 = 0; i0 < n4; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < n4) {
      const float4 u = reinterpret_cast<const float4*>(act)[i];
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
    const PlaneQuad p = plane_quad(v, true);
    if (i < n4) {
      reinterpret_cast<uint2*>(hi)[i] = p.hi;
      reinterpret_cast<uint2*>(lo)[i] = p.lo;
      if ((i & 7) == 0) reinterpret_cast<float4*>(meta)[i >> 3] = make_float4(p.inv, p.sum, p.sum16, 0.f);
    }
  }
  __syncthreads();
  for (; j < a.top_k; j += jstep) {
    if (j != j0) {
      e = __builtin_amdgcn_readfirstlane(a.ids[r * a.top_k + j]);
      if (p_beg < p_end) load(e, p_beg, 0);
    }
    FewX<SCH, NU, 2> x;
    x.load(hi + j * K, lo + j * K, meta + j * nb * 4, uc, uok);
    auto step = [&](int col, int slot) {
      const float v = few_sum(few_dot<SCH, NU, 2>(w[slot], x, uc, kc), a.log2l);
      if (li == 0 && col + g < p_end) vals[j * a.tile + col + g - c_beg] = v;
    };
    int c = p_beg;
    for (; c + RP < p_end; c += 2 * RP) {
      load(e, c + RP, 1);
      step(c, 0);
      if (c + 2 * RP < p_end) load(e, c + 2 * RP, 0);
      step(c + RP, 1);
    }
    if (c < p_end) step(c, 0);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < c_end - c_beg; c += blockDim.x) {
    float s = 0.f;
    for (int q = 0; q < a.top_k; q++) s = fmaf(a.probs[r * a.top_k + q], vals[q * a.tile + c], s);
    const int64_t o = (int64_t)r * a.H + c_beg + c;
    if (a.y_bf16) reinterpret_cast<uint16_t*>(a.y)[o] = (uint16_t)f32_to_bf16_bits(s);
    else reinterpret_cast<float*>(a.y)[o] = s;
  }
}

}  // namespace rlxq

#if RLXQ_PART_IS(0)
// rlxq_moe_logits_<x>_<router>_e<EB>r<RB>; rlxq_moe_prep_<x>_<router>
#define RLXQ_LOGITS(XN, XBF, RN, RBF)                                                                               \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_logits_##XN##_##RN##_e1r4(rlxq_moe_logits_args a) {     \
    rlxq::moe_logits_body<XBF, RBF, 1, 4>(a, blockIdx.x, blockIdx.y);                                               \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_logits_##XN##_##RN##_e4r8(rlxq_moe_logits_args a) {     \
    rlxq::moe_logits_body<XBF, RBF, 4, 8>(a, blockIdx.x, blockIdx.y);                                               \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_prep_##XN##_##RN(rlxq_moe_prep_args a) {                \
    rlxq::moe_prep_body<XBF, RBF>(a);                                                                               \
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
#endif

// rlxq_moefew_gu_<scheme>_u<NU>_p<planes>, rlxq_moefew_dn_<scheme>_u<NU>
#define RLXQ_FEW_U(SNAME, SCH, NU)                                                                       \
  extern "C" __global__ __launch_bounds__(512) void rlxq_moefew_gu_##SNAME##_u##NU##_p1(rlxq_moe_few_args a) { \
    rlxq::moe_few_gate_up<SCH, NU, 1>(a);                                                                \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(512) void rlxq_moefew_gu_##SNAME##_u##NU##_p2(rlxq_moe_few_args a) { \
    rlxq::moe_few_gate_up<SCH, NU, 2>(a);                                                                \
  }                                                                                                      \
  extern "C" __global__ __launch_bounds__(512) void rlxq_moefew_dn_##SNAME##_u##NU(rlxq_moe_few_args a) { \
    rlxq::moe_few_down<SCH, NU>(a);                                                                      \
  }
// (units of two blocks: at most two per lane, which covers K = 8192 as four of
// one do)
#define RLXQ_FEW1(SNAME, SCH) \
  RLXQ_FEW_U(SNAME, SCH, 1)   \
  RLXQ_FEW_U(SNAME, SCH, 2)   \
  RLXQ_FEW_U(SNAME, SCH, 3)   \
  RLXQ_FEW_U(SNAME, SCH, 4)
#define RLXQ_FEW2(SNAME, SCH) \
  RLXQ_FEW_U(SNAME, SCH, 1)   \
  RLXQ_FEW_U(SNAME, SCH, 2)
#if RLXQ_PART_IS(1)
RLXQ_FEW1(mxfp4, SCH_MXFP4)
RLXQ_FEW1(q4_1, SCH_Q4_1)
#endif
#if RLXQ_PART_IS(2)
RLXQ_FEW2(q4_k, SCH_Q4_K)
RLXQ_FEW2(q4_0, SCH_Q4_0)
RLXQ_FEW2(q8_0, SCH_Q8_0)
#endif
#if RLXQ_PART_IS(3)
RLXQ_FEW1(q6_k, SCH_Q6_K)
RLXQ_FEW2(q5_k, SCH_Q5_K)
#endif
#if RLXQ_PART_IS(4)
RLXQ_FEW1(q3_k, SCH_Q3_K)
#endif
#if RLXQ_PART_IS(5)
RLXQ_FEW1(q2_k, SCH_Q2_K)
RLXQ_FEW1(q8_k, SCH_Q8_K)
#endif
