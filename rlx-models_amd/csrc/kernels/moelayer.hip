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

// Sum over the wave (lanes of a row of 16 by DPP moves of the halves, the four
// rows through readlane), the same in every lane.
template <int CTRL>
RLXQ_DEV double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
RLXQ_DEV double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
RLXQ_DEV double wave_sum(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  v += dpp_f64<0x140>(v);
  return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
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

RLXQ_DEV float wave_fmax(float v) {
  v = group8_max(v);
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xF, 0xF, false)));
  auto at = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
  return fmaxf(fmaxf(at(0), at(16)), fmaxf(at(32), at(48)));
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
  mx = wave_fmax(mx);
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

// ------------------------------------------------------- rows as records
// Order of a scheme's codes within a block (moe_args.h).
template <int SCH>
RLXQ_DEV constexpr int few_order() {
  return SCH == SCH_MXFP4 ? 0 : (SCH == SCH_Q4_0 || SCH == SCH_Q4_1) ? 1 : 2;
}

// Four elements 4 q .. 4 q + 3 of a block per lane, eight lanes (q = lane & 7) a
// block, into the block's record; all lanes of the wave take part.
RLXQ_DEV void put_record(uint8_t* rec, const float (&x)[4], int planes, int order, bool active) {
  const int q = threadIdx.x & 7;
  const float s = (x[0] + x[1]) + (x[2] + x[3]);
  const float sum = group8_sum(s), sum16 = group4_sum(s);   // (lanes 0..3: of the first 16 elements)
  const float amax = group8_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
  // 2^e: amax 2^-e in [2^14, 2^15), from the float's exponent bits (an infinity
  // or a NaN stays what it is under any scale)
  int e = (int)(__float_as_uint(amax) >> 23) - 127 - 14;
  e = amax < INFINITY ? (e < -126 ? -126 : e) : 0;
  const float sc = __uint_as_float((uint32_t)(127 - e) << 23);
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float v = x[i] * sc;
    h[i] = f32_to_f16_bits(v);
    l[i] = f32_to_f16_bits(v - f16_bits_to_f32(h[i]));
  }
  if (!active) return;
  // the lane's two pairs and their places among the block's 16
  const int near = order == 0 ? 1 : 2;   // (4q, 4q + near)
  const int t0 = order == 1 ? (q < 4 ? 4 * q : 4 * (q - 4) + 1) : 2 * q, t1 = order == 1 ? t0 + 2 : t0 + 1;
  uint32_t* r = reinterpret_cast<uint32_t*>(rec);
  r[t0] = h[0] | ((near == 1 ? h[1] : h[2]) << 16);
  r[t1] = (near == 1 ? h[2] : h[1]) | (h[3] << 16);
  if (planes == 2) {
    r[16 + t0] = l[0] | ((near == 1 ? l[1] : l[2]) << 16);
    r[16 + t1] = (near == 1 ? l[2] : l[1]) | (l[3] << 16);
  }
  if (q == 0) {
    float* m = reinterpret_cast<float*>(rec + 64 * planes);
    m[0] = __uint_as_float((uint32_t)(127 + e) << 23);
    m[1] = sum;
    m[2] = sum16;
    m[3] = 0.f;
  }
}

// Router logits (the first lblocks workgroups: an expert and four rows, H over
// the four waves) and, beside them, the prepared rows.
template <bool XBF, bool RBF>
RLXQ_DEV void moe_prep_body(const rlxq_moe_prep_args& a) {
  constexpr int RB = 4;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  if ((int)blockIdx.x < a.lblocks) {
    __shared__ double part[4][RB];
    const int e = blockIdx.x % a.r.E;
    const int64_t r0 = (int64_t)(blockIdx.x / a.r.E) * RB;
    double acc[RB] = {0., 0., 0., 0.};
#pragma unroll 2
    for (int64_t h = 4 * threadIdx.x; h < a.r.H; h += 1024) {
      double w[4], v[RB][4];
      load4<RBF>(a.r.router, (int64_t)e * a.r.H + h, w);
#pragma unroll
      for (int q = 0; q < RB; q++)
        if (r0 + q < a.r.rows) load4<XBF>(a.r.x, (r0 + q) * a.r.H + h, v[q]);   // (uniform)
#pragma unroll
      for (int q = 0; q < RB; q++)
        if (r0 + q < a.r.rows) {
#pragma unroll
          for (int c = 0; c < 4; c++) acc[q] = fma(w[c], v[q][c], acc[q]);
        }
    }
#pragma unroll
    for (int q = 0; q < RB; q++) {
      if (r0 + q >= a.r.rows) break;
      const double s = wave_sum(acc[q]);
      if (lane == 0) part[wv][q] = s;
    }
    __syncthreads();
    const int q = threadIdx.x;
    if (q < RB && r0 + q < a.r.rows)
      a.r.logits[(r0 + q) * a.r.E + e] = (float)((part[0][q] + part[1][q]) + (part[2][q] + part[3][q]));
    return;
  }
  const int64_t i = (int64_t)(blockIdx.x - a.lblocks) * 256 + threadIdx.x, n4 = a.r.rows * a.r.H / 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (i < n4) {   // (H is whole blocks: uniform over a block's lanes)
    double d[4];
    load4<XBF>(a.r.x, 4 * i, d);
#pragma unroll
    for (int q = 0; q < 4; q++) v[q] = (float)d[q];
  }
  constexpr int P = XBF ? 1 : 2;
  put_record(a.rec + (i >> 3) * RLXQ_FEW_REC(P), v, P, a.order, i < n4);
}

// ------------------------------------------------- products for few tokens
// A weight row is spread over L = 2^log2l lanes of a wave, lane li taking units
// li, li + L, ... (a unit is one or two 32-weight blocks) against the activation
// rows' records in LDS; 64 / L rows go at once.  Codes become exact f16 integers
// (the offset of the bit pattern subtracted), so the products with the f16
// planes are exact in v_dot2_f32_f16 and a block's sum is an f32 sum of its 32
// (64 with the remainders) products, which then takes the block's scale (times
// the activation block's power of two) and, for formats with a minimum, the
// minimum times the block's sum of activations.

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

template <int SCH>
struct FewW {
  uint32_t dw[Unit<SCH>::DW];
  uint32_t sc;
  // unit u of the packed row at p (MXFP4: its scale byte among those at s)
  RLXQ_DEV void load(const uint8_t* p, const uint8_t* s, int u) {
    load_unit_at<SCH>(dw, p, u);
    if constexpr (SCH == SCH_MXFP4) sc = s[u];
  }
};

// One block's record in registers.
template <int NPL>
struct FewRec {
  uint32_t h[16], l[NPL == 2 ? 16 : 1];
  float4 me;
  RLXQ_DEV void load(const uint8_t* rec, bool uok) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const uint4 v = reinterpret_cast<const uint4*>(rec)[q];
      h[4 * q] = v.x; h[4 * q + 1] = v.y; h[4 * q + 2] = v.z; h[4 * q + 3] = v.w;
      if constexpr (NPL == 2) {
        const uint4 z = reinterpret_cast<const uint4*>(rec)[4 + q];
        l[4 * q] = z.x; l[4 * q + 1] = z.y; l[4 * q + 2] = z.z; l[4 * q + 3] = z.w;
      }
    }
    // (a unit past the row's end repeats the last one, times zero)
    me = uok ? reinterpret_cast<const float4*>(rec)[4 * NPL] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
};

// A block of a weight row: exact f16 codes, multipliers of its code sum (of its
// halves') and of its activations' sum (halves').
template <int SCH>
struct FewBlk {
  uint32_t pw[16];
  float d, d2, mn, m2;
  RLXQ_DEV void decode(const FewW<SCH>& w, int bl, int u, const UnpackK& kc) {
    block_f16<SCH>(w.dw, bl, pw, kc);
    d2 = mn = m2 = 0.f;
    if constexpr (SCH == SCH_MXFP4) d = e8m0_to_f32(w.sc);
    else if constexpr (SCH == SCH_Q6_K) block_scales<SCH>(w.dw, bl, d, d2, u);
    else if constexpr (half_scales<SCH>()) block_scales_half<SCH>(w.dw, d, d2, mn, m2);
    else block_scales<SCH>(w.dw, bl, d, mn, u);
  }
  template <int NPL>
  RLXQ_DEV void add(const FewRec<NPL>& x, float& s) const {
    float c0 = 0.f, c1 = 0.f;   // (two chains: the halves, hi and lo, or even and odd pairs)
#pragma unroll
    for (int t = 0; t < 16; t++) {
      if constexpr (half_scales<SCH>()) {
        float& c = t < 8 ? c0 : c1;
        c = dot2_f16(pw[t], x.h[t], c);
        if constexpr (NPL == 2) c = dot2_f16(pw[t], x.l[t], c);
      } else if constexpr (NPL == 2) {
        c0 = dot2_f16(pw[t], x.h[t], c0);
        c1 = dot2_f16(pw[t], x.l[t], c1);
      } else {
        float& c = t & 1 ? c1 : c0;
        c = dot2_f16(pw[t], x.h[t], c);
      }
    }
    if constexpr (half_scales<SCH>()) {
      s = fmaf(d * x.me.x, c0, s);
      s = fmaf(d2 * x.me.x, c1, s);
      if constexpr (SCH == SCH_Q2_K) {
        s = fmaf(mn, x.me.z, s);
        s = fmaf(m2, x.me.y - x.me.z, s);
      }
    } else {
      s = fmaf(d * x.me.x, c0 + c1, s);
      if constexpr (SCH == SCH_Q4_1 || SCH == SCH_Q4_K || SCH == SCH_Q5_K) s = fmaf(mn, x.me.y, s);
    }
  }
};

// A unit's part of R weight rows (w[0 .. R - 1], unit u) times MT activation
// rows (records of the unit's first block at x + m * xld).  One activation row:
// its record stays in registers and the weight rows are decoded in turn; more:
// the weight rows are decoded once and the records pass.  (The empty statements
// keep the products where they stand: the compiler would gather them behind the
// reads of all records, in as many registers, and run them for absent rows.)
template <int SCH, int NPL, int R, int MT>
RLXQ_DEV void few_unit(const FewW<SCH> (&w)[R], const uint8_t* x, int xld, int cnt, int u, bool uok, const UnpackK& kc,
                       float (&acc)[R][MT]) {
#pragma unroll
  for (int bl = 0; bl < Unit<SCH>::BLOCKS; bl++) {
    if constexpr (MT == 1) {
      FewRec<NPL> rec;
      rec.load(x + bl * RLXQ_FEW_REC(NPL), uok);
#pragma unroll
      for (int r = 0; r < R; r++) {
        FewBlk<SCH> b;
        b.decode(w[r], bl, u, kc);
        b.add(rec, acc[r][0]);
        asm volatile("" : "+v"(acc[r][0]));
      }
    } else {
      FewBlk<SCH> b[R];
#pragma unroll
      for (int r = 0; r < R; r++) b[r].decode(w[r], bl, u, kc);
#pragma unroll
      for (int m = 0; m < MT; m++) {
        if (m > 0 && m >= cnt) break;   // (uniform)
        FewRec<NPL> rec;
        rec.load(x + m * xld + bl * RLXQ_FEW_REC(NPL), uok);
#pragma unroll
        for (int r = 0; r < R; r++) {
          b[r].add(rec, acc[r][m]);
          asm volatile("" : "+v"(acc[r][m]));
        }
      }
    }
  }
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
  auto at = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
  const float r0 = at(0), r1 = at(16), r2 = at(32), r3 = at(48);
  if (log2l == 5) return (threadIdx.x & 32) ? r2 + r3 : r0 + r1;
  return (r0 + r1) + (r2 + r3);
}

RLXQ_DEV UnpackK f16_unpack_consts() {
  UnpackK k{0x000F000Fu, 0x64006400u};
  asm volatile("" : "+v"(k.mask), "+v"(k.magic));
  return k;
}

// Columns c_first, c_first + c_step, ... below c_end of a slab (64 / L columns at
// each) times the rows whose records start at x (MT of them, xld apart, cnt in
// use).  R = 2: a column is gate row col and up row col + up.  The steps (column,
// unit) run as one sequence with the weights of D - 1 steps ahead in registers;
// past the last step the loads repeat its column (a load under a condition would
// make the compiler wait for all the others).  begin() requests the first; run()
// needs the records in LDS.
template <int SCH, int NPL, int R, int MT>
struct FewCols {
  static constexpr int D0 = 48 / (R * Unit<SCH>::DW), D = D0 < 1 ? 1 : D0 > 4 ? 4 : D0;   // (48 registers of weights)
  FewW<SCH> ring[D][R];
  const uint8_t* base;
  const uint8_t* sbase;
  int64_t rb;
  int up, nbs, U, c_first, c_step, c_end, log2l, nchunk, S;
  const uint8_t *lp[R], *ls[R];   // the rows of the column being loaded
  int l_col, l_j;

  RLXQ_DEV void load(FewW<SCH> (&w)[R]) {   // the next step's weights
    if (l_j == 0) {
      const int col = l_col < c_end ? l_col : c_end - 1;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int64_t n = col + (r ? up : 0);
        lp[r] = base + n * rb;
        ls[r] = SCH == SCH_MXFP4 ? sbase + n * nbs : nullptr;
      }
    }
    int u = (threadIdx.x & ((1 << log2l) - 1)) + (l_j << log2l);
    u = u < U ? u : U - 1;
#pragma unroll
    for (int r = 0; r < R; r++) w[r].load(lp[r], ls[r], u);
    if (++l_j == nchunk) {
      l_j = 0;
      l_col += c_step;
    }
  }
  RLXQ_DEV void begin() {
    nchunk = (U + (1 << log2l) - 1) >> log2l;
    S = c_first < c_end ? (c_end - c_first + c_step - 1) / c_step * nchunk : 0;
    l_col = c_first + ((threadIdx.x & 63) >> log2l);
    l_j = 0;
#pragma unroll
    for (int d = 0; d < D - 1; d++) load(ring[d]);
  }
  template <class Emit>
  RLXQ_DEV void run(const uint8_t* x, int xld, int cnt, const UnpackK& kc, Emit emit) {
    const int lane = threadIdx.x & 63, li = lane & ((1 << log2l) - 1);
    float acc[R][MT];
    int col = c_first + (lane >> log2l), j = 0;
    for (int s0 = 0; s0 < S; s0 += D) {
#pragma unroll
      for (int d = 0; d < D; d++) {
        const int s = s0 + d;
        load(ring[(d + D - 1) % D]);
        if (s < S) {
          if (j == 0) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
              for (int m = 0; m < MT; m++) acc[r][m] = 0.f;
          }
          const int u = li + (j << log2l);
          const bool uok = u < U;
          const int uc = uok ? u : U - 1;
          few_unit<SCH, NPL, R, MT>(ring[d], x + uc * (Unit<SCH>::BLOCKS * RLXQ_FEW_REC(NPL)), xld, cnt, uc, uok, kc, acc);
          if (++j == nchunk) {
#pragma unroll
            for (int m = 0; m < MT; m++) {
              if (m > 0 && m >= cnt) break;
              float v[R];
#pragma unroll
              for (int r = 0; r < R; r++) v[r] = few_sum(acc[r][m], log2l);
              if (li == 0 && col < c_end) emit(m, col, v);
            }
            j = 0;
            col += c_step;
          }
        }
      }
    }
  }
};

constexpr int FEW_ENTRIES = 256;   // most (row, slot) pairs of a call (of at most 32 rows)

// gate|up and SwiGLU.  Every workgroup routes all rows itself (a wave a row:
// the grid is one round of workgroups, so the layer pays for it once, where a
// launch of its own would cost more).  The entries of one expert are cut into
// chunks of MT, and the workgroups share the (chunk, columns) evenly; a chunk's
// rows are copied to LDS and its weights read once for all of them.  Workgroup
// 0 leaves the routing for the down launch.
template <int SCH, int NPL, int MT>
RLXQ_DEV void moe_few_gate_up(const rlxq_moe_few_args& a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];   // MT rows of records
  __shared__ __attribute__((aligned(16))) int32_t ids[FEW_ENTRIES];
  // (MT > 1; a chunk holds at least one entry)
  __shared__ uint32_t mask[MT > 1 ? 1024 : 1];
  __shared__ int32_t first[MT > 1 ? 1024 : 1], member[MT > 1 ? FEW_ENTRIES * MT : 1], wsum[8];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int n = a.rows * a.top_k, nb = a.H / 32, xld = nb * RLXQ_FEW_REC(NPL);
  auto stage = [&](int m, int r) {
    const uint4* src = reinterpret_cast<const uint4*>(a.rec + (int64_t)r * xld);
    uint4* dst = reinterpret_cast<uint4*>(few_lds + m * xld);
    for (int i = threadIdx.x; i < xld / 16; i += blockDim.x) dst[i] = src[i];
  };
  if (a.rows == 1) stage(0, 0);   // (the only row: ahead of the routing)
  if constexpr (MT > 1) {
    for (int i = threadIdx.x; i < a.E; i += blockDim.x) mask[i] = 0u;
    for (int i = threadIdx.x; i < n * MT; i += blockDim.x) member[i] = -1;
  }
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
  int chunks = n;
  if constexpr (MT > 1) {
    // a row takes an expert once: an expert's entries are the bits of a mask of
    // rows, an entry's rank among them the bits below its row's
    for (int i = threadIdx.x; i < n; i += blockDim.x) atomicOr(&mask[ids[i]], 1u << (i / a.top_k));
    __syncthreads();
    // chunk offsets: exclusive sum over the experts, four a thread
    int c4[4], t = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int e = 4 * threadIdx.x + q;
      c4[q] = e < a.E ? (__popc(mask[e]) + MT - 1) / MT : 0;
      t += c4[q];
    }
    int inc = t;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(inc, off, 64);
      if (lane >= off) inc += o;
    }
    if (lane == 63) wsum[wv] = inc;
    __syncthreads();
    int off = inc - t;
    chunks = 0;
    for (int q = 0; q < nw; q++) {
      off += q < wv ? wsum[q] : 0;
      chunks += wsum[q];
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int e = 4 * threadIdx.x + q;
      if (e < a.E) first[e] = off;
      off += c4[q];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int e = ids[i], rank = __popc(mask[e] & ((1u << (i / a.top_k)) - 1));
      member[(first[e] + rank / MT) * MT + rank % MT] = i;
    }
    __syncthreads();
  }
  const int RP = 64 >> a.log2l;
  const UnpackK kc = f16_unpack_consts();
  // steps of a chunk: groups of RP columns
  const int steps = (a.I + RP - 1) / RP;
  const int64_t total = (int64_t)chunks * steps;
  int64_t s = total * blockIdx.x / gridDim.x;
  const int64_t s_end = total * (blockIdx.x + 1) / gridDim.x;
  bool again = false;
  while (s < s_end) {   // (uniform over the workgroup)
    const int ch = (int)(s / steps), c0 = (int)(s - (int64_t)ch * steps);
    const int64_t left = s_end - (int64_t)ch * steps;
    const int c1 = (int)(left < steps ? left : steps);
    int ent[MT], cnt = 1;
    if constexpr (MT > 1) {
      cnt = 0;
#pragma unroll
      for (int m = 0; m < MT; m++) {
        ent[m] = __builtin_amdgcn_readfirstlane(member[ch * MT + m]);
        cnt += ent[m] >= 0 ? 1 : 0;
      }
    } else {
      ent[0] = ch;
    }
    const int e = __builtin_amdgcn_readfirstlane(ids[ent[0]]);
    FewCols<SCH, NPL, 2, MT> f;
    f.base = a.bank + (int64_t)e * 2 * a.I * a.rb;
    f.sbase = SCH == SCH_MXFP4 ? a.scales + (int64_t)e * 2 * a.I * nb : nullptr;
    f.rb = a.rb;
    f.up = a.I;
    f.nbs = nb;
    f.U = nb / Unit<SCH>::BLOCKS;
    f.log2l = a.log2l;
    f.c_first = (c0 + wv) * RP;
    f.c_step = nw * RP;
    f.c_end = c1 * RP < a.I ? c1 * RP : a.I;
    f.begin();
    if (a.rows > 1) {
      if (again) __syncthreads();   // (the rows before are no longer read)
#pragma unroll
      for (int m = 0; m < MT; m++)
        if (m < cnt) stage(m, ent[m] / a.top_k);
      __syncthreads();
    }
    f.run(few_lds, xld, cnt, kc, [&](int m, int col, const float (&v)[2]) {
      int en = ent[0];
#pragma unroll
      for (int q = 1; q < MT; q++) en = m == q ? ent[q] : en;
      a.act[(int64_t)en * a.I + col] = v[0] / (1.f + expf(-v[0])) * v[1];   // silu(g) * u
    });
    again = true;
    s = (int64_t)ch * steps + c1;
  }
}

// down and the weighted sum, a workgroup per (row, tile of columns): the row's
// top_k activation vectors become records in LDS, the waves share the slots
// (waves / top_k of them per slot, each a part of the tile; more slots than
// waves in turns), and the slots are added in slot order.  Workgroups of one
// column tile are dealt to one XCD (workgroup b runs on XCD b % 8), whose L2
// then holds the rows of an expert that several tokens take.
template <int SCH>
RLXQ_DEV void moe_few_down(const rlxq_moe_few_args& a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int x8 = blockIdx.x & 7, q8 = blockIdx.x >> 3;
  const int r = q8 % a.rows, tn = q8 / a.rows * 8 + x8;
  if (tn >= a.tiles) return;
  const int c_beg = tn * a.tile, c_end = c_beg + a.tile < a.H ? c_beg + a.tile : a.H;
  const int K = a.I, nb = K / 32;
  constexpr int REC = RLXQ_FEW_REC(2);
  float* vals = reinterpret_cast<float*>(few_lds + (size_t)a.top_k * nb * REC);   // [top_k][tile]
  const int RP = 64 >> a.log2l;
  const UnpackK kc = f16_unpack_consts();
  const int parts = nw / a.top_k > 1 ? nw / a.top_k : 1;
  const int part = wv % parts, jstep = nw / parts;

  FewCols<SCH, 2, 1, 1> f;
  f.rb = a.rb;
  f.up = 0;
  f.nbs = nb;
  f.U = nb / Unit<SCH>::BLOCKS;
  f.log2l = a.log2l;
  f.c_first = c_beg + part * RP;
  f.c_step = parts * RP;
  f.c_end = c_end;
  auto begin = [&](int j) {
    const int e = __builtin_amdgcn_readfirstlane(a.ids[r * a.top_k + j]);
    f.base = a.bank + (int64_t)e * a.H * a.rb;
    f.sbase = SCH == SCH_MXFP4 ? a.scales + (int64_t)e * a.H * nb : nullptr;
    f.begin();
  };
  const int j0 = wv / parts;
  if (j0 < a.top_k) begin(j0);
  const float* act = a.act + (int64_t)r * a.top_k * K;
  const int n4 = a.top_k * K / 4;
  for (int i0 = 0; i0 < n4; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < n4) {
      const float4 u = reinterpret_cast<const float4*>(act)[i];
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
    put_record(few_lds + (i >> 3) * REC, v, 2, few_order<SCH>(), i < n4);
  }
  __syncthreads();
  for (int j = j0; j < a.top_k; j += jstep) {
    if (j != j0) begin(j);
    f.run(few_lds + (size_t)j * nb * REC, 0, 1, kc, [&](int, int col, const float (&v)[1]) { vals[j * a.tile + col - c_beg] = v[0]; });
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
  extern "C" __global__ __launch_bounds__(256) void rlxq_moe_prep_##XN##_##RN(rlxq_moe_prep_args a) {                \
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

// rlxq_moefew_gu_<scheme>_p<planes>_m<entries a pass>, rlxq_moefew_dn_<scheme>
#define RLXQ_FEW_GU(SNAME, SCH, P, M)                                                                          \
  extern "C" __global__ __launch_bounds__(512) void rlxq_moefew_gu_##SNAME##_p##P##_m##M(rlxq_moe_few_args a) { \
    rlxq::moe_few_gate_up<SCH, P, M>(a);                                                                       \
  }
#define RLXQ_FEW(SNAME, SCH)                                                                      \
  RLXQ_FEW_GU(SNAME, SCH, 1, 1)                                                                   \
  RLXQ_FEW_GU(SNAME, SCH, 2, 1)                                                                   \
  RLXQ_FEW_GU(SNAME, SCH, 1, 2)                                                                   \
  RLXQ_FEW_GU(SNAME, SCH, 2, 2)                                                                   \
  RLXQ_FEW_GU(SNAME, SCH, 1, 4)                                                                   \
  RLXQ_FEW_GU(SNAME, SCH, 2, 4)                                                                   \
  extern "C" __global__ __launch_bounds__(512) void rlxq_moefew_dn_##SNAME(rlxq_moe_few_args a) { \
    rlxq::moe_few_down<SCH>(a);                                                                   \
  }
#if RLXQ_PART_IS(1)
RLXQ_FEW(mxfp4, SCH_MXFP4)
RLXQ_FEW(q4_1, SCH_Q4_1)
#endif
#if RLXQ_PART_IS(2)
RLXQ_FEW(q4_k, SCH_Q4_K)
RLXQ_FEW(q4_0, SCH_Q4_0)
#endif
#if RLXQ_PART_IS(3)
RLXQ_FEW(q6_k, SCH_Q6_K)
RLXQ_FEW(q8_0, SCH_Q8_0)
#endif
#if RLXQ_PART_IS(4)
RLXQ_FEW(q3_k, SCH_Q3_K)
RLXQ_FEW(q5_k, SCH_Q5_K)
#endif
#if RLXQ_PART_IS(5)
RLXQ_FEW(q2_k, SCH_Q2_K)
RLXQ_FEW(q8_k, SCH_Q8_K)
#endif
