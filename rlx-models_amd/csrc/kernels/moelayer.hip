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

// Inclusive sum over a wave's lanes: within rows of 16, then across them.
RLXQ_DEV int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // a row's last lane to the next row; to the upper half
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
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
  id = 0;
  uint32_t mine = 0;   // lane j: the j-th key
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
    if (lane == j) {
      id = pick;
      mine = best;
    }
#pragma unroll
    for (int i = 0; i < NPER; i++)
      if (lane + 64 * i == pick) key[i] = 0u;
  }
  const float f = __uint_as_float(mine & 0x80000000u ? mine & 0x7fffffffu : ~mine);
  prob = lane < top_k ? expf(f - mx) / s : 0.f;
  if (renorm) prob /= lane_group_sum<64>(prob);
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
    m[0] = order == 0 ? __int_as_float(e) : __uint_as_float((uint32_t)(127 + e) << 23);
    m[1] = sum;
    m[2] = sum16;
    m[3] = 0.f;
  }
}

// Router logits (the first lblocks workgroups: an expert and four rows, H over
// the four waves) and, beside them, the prepared rows.  Latency: 3.6 us for a
// row, 5.5 for 16 (2048 elements, 128 experts).
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

// A block of a weight row: exact f16 codes, multipliers of its code sum (of its
// halves') and of its activations' sum (halves').
// MXFP4: the scale stays an exponent that is added to the record factor's: the
// two powers of two need not have an f32 product (2^127 of zero codes on rows
// beyond 2^15 made NaN of a zero).  Byte 0, a scale of zero, is an exponent that
// leaves nothing of any finite sum; 255 reads as 254 (e8m0_to_f32).
template <int SCH>
struct FewBlk {
  uint32_t pw[16];
  float d, d2, mn, m2;
  int e;
  RLXQ_DEV void decode(const FewW<SCH>& w, int bl, int u, const UnpackK& kc) {
    block_f16<SCH>(w.dw, bl, pw, kc);
    d = d2 = mn = m2 = 0.f;
    e = 0;
    if constexpr (SCH == SCH_MXFP4) e = w.sc == 0u ? -1024 : (int)(w.sc < 254u ? w.sc : 254u) - 127;
    else if constexpr (SCH == SCH_Q6_K) block_scales<SCH>(w.dw, bl, d, d2, u);
    else if constexpr (half_scales<SCH>()) block_scales_half<SCH>(w.dw, d, d2, mn, m2);
    else block_scales<SCH>(w.dw, bl, d, mn, u);
  }
  // the codes times 32 f16 activations (a plane of a record), added to c
  // (two chains: the block's halves, or even and odd pairs)
  RLXQ_DEV void dots(const uint32_t (&h)[16], float (&c)[2]) const {
#pragma unroll
    for (int t = 0; t < 16; t++) {
      float& q = c[half_scales<SCH>() ? t / 8 : t % 2];
      q = dot2_f16(pw[t], h[t], q);
    }
  }
  // the block's sum of products from its code sums and the record's factors
  RLXQ_DEV float finish(const float (&c)[2], const float4& me, float s) const {
    if constexpr (SCH == SCH_MXFP4) {
      s += __builtin_amdgcn_ldexpf(c[0] + c[1], e + __float_as_int(me.x));
    } else if constexpr (half_scales<SCH>()) {
      s = fmaf(d * me.x, c[0], s);
      s = fmaf(d2 * me.x, c[1], s);
      if constexpr (SCH == SCH_Q2_K) {
        s = fmaf(mn, me.z, s);
        s = fmaf(m2, me.y - me.z, s);
      }
    } else {
      s = fmaf(d * me.x, c[0] + c[1], s);
      if constexpr (SCH == SCH_Q4_1 || SCH == SCH_Q4_K || SCH == SCH_Q5_K) s = fmaf(mn, me.y, s);
    }
    return s;
  }
};

// A unit's part of R weight rows (w[0 .. R - 1], unit u) times MT activation
// rows (records of the unit's first block at x + m * xld): the weight rows are
// decoded once, and the records pass a plane at a time.  (The empty statements
// keep the products where they stand: the compiler would gather them behind the
// reads of all planes, in as many registers, and run them for absent rows.)  A
// lane past the row's end repeats the last unit and leaves its sum alone: times
// zero, an infinity would stay.
template <int SCH, int NPL, int R, int MT>
RLXQ_DEV void few_unit(const FewW<SCH> (&w)[R], const uint8_t* x, int xld, int cnt, int u, bool uok, const UnpackK& kc,
                       float (&acc)[R][MT]) {
#pragma unroll
  for (int bl = 0; bl < Unit<SCH>::BLOCKS; bl++) {
    FewBlk<SCH> b[R];
#pragma unroll
    for (int r = 0; r < R; r++) b[r].decode(w[r], bl, u, kc);
#pragma unroll
    for (int m = 0; m < MT; m++) {
      if (m > 0 && m >= cnt) break;   // (uniform)
      const uint4* rec = reinterpret_cast<const uint4*>(x + m * xld + bl * RLXQ_FEW_REC(NPL));
      float c[R][2];
#pragma unroll
      for (int r = 0; r < R; r++) c[r][0] = c[r][1] = 0.f;
#pragma unroll
      for (int pl = 0; pl < NPL; pl++) {
        uint32_t h[16];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint4 v = rec[4 * pl + q];
          h[4 * q] = v.x; h[4 * q + 1] = v.y; h[4 * q + 2] = v.z; h[4 * q + 3] = v.w;
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
          b[r].dots(h, c[r]);
          asm volatile("" : "+v"(c[r][0]), "+v"(c[r][1]));
        }
      }
      const float4 me = reinterpret_cast<const float4*>(rec)[4 * NPL];
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float s = b[r].finish(c[r], me, acc[r][m]);
        acc[r][m] = uok ? s : acc[r][m];
      }
    }
  }
}

// Sum over aligned groups of 2^log2l lanes (8 or 16), in every lane of the
// group; the branch is uniform.
RLXQ_DEV float few_sum(float v, int log2l) {
  v = group8_sum(v);
  if (log2l == 4) v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xF, 0xF, false));
  return v;
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
  // steps in 48 registers of weights (one step ahead of the wide units, which
  // exceed them, cost more in waves than it hid: Q6_K, 8 rows, 48 -> 50 us)
  static constexpr int D0 = 48 / (R * Unit<SCH>::DW), D = D0 < 1 ? 1 : D0 > 4 ? 4 : D0;
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
// chunks of MT, and the workgroups share the (chunk, columns) by cost; a chunk's
// rows are copied to LDS and its weights read once for all of them.  Workgroup
// 0 leaves the routing for the down launch.
// (2048 -> 2 x 768, 8 of 128 experts) MXFP4, 1 row: 8.4 us, of which some 6 to the
// first product.  16 rows: 39 us for 191 MB past L2, 53 of them rows of experts
// that a second entry reads again; Q4_K, 4 rows: 18 us for 53 MB.  VALU busy half
// of the time, LDS a tenth; three quarters of decoding and dot products left out
// (both launches, a timing experiment) were worth 8 of the layer's 67 us at 16
// rows, so most of what separates it from its bytes is elsewhere.
template <int SCH, int NPL, int MT>
RLXQ_DEV void moe_few_gate_up(const rlxq_moe_few_args& a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];   // MT rows of records
  __shared__ __attribute__((aligned(16))) int32_t ids[FEW_ENTRIES];
  // (MT > 1; a chunk holds at least one entry)
  __shared__ uint32_t mask[MT > 1 ? 1024 : 1];
  __shared__ int32_t first[MT > 1 ? 1024 : 1], member[MT > 1 ? FEW_ENTRIES * MT : 1], wsum[4], cut[4];
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
  // Entries in chunks of up to MT of one expert, and the workgroup's share of the
  // (chunk, step) pairs in sequence: from step c_lo of chunk ch_lo up to step c_hi
  // of chunk ch_hi.  A step, a group of RP columns, of a chunk of m entries counts
  // 1 + m (counted alike, 16 rows at MT 4 took 75 us instead of 68).
  const int RP = 64 >> a.log2l, steps = (a.I + RP - 1) / RP;
  int ch_lo, c_lo, ch_hi, c_hi;
  if constexpr (MT == 1) {
    const int total = n * steps, share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    const int s0 = min(share * (int)blockIdx.x, total), s1 = min(s0 + share, total);
    ch_lo = s0 / steps, c_lo = s0 - ch_lo * steps;
    ch_hi = s1 / steps, c_hi = s1 - ch_hi * steps;
  } else {
    // a row takes an expert once: an expert's entries are the bits of a mask of
    // rows, an entry's rank among them the bits below its row's
    const float inv_k = 1.f / (float)a.top_k;
    auto row_of = [&](int i) { return (int)(((float)i + 0.5f) * inv_k); };   // (i < 256, top_k <= 64: exact)
    for (int i = threadIdx.x; i < n; i += blockDim.x) atomicOr(&mask[ids[i]], 1u << row_of(i));
    __syncthreads();
    // before each expert, in one sum over them (four a thread): chunks << 16 | entries
    int at[4], t = 0, cnt[4] = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int e = 4 * threadIdx.x + q;
      if (e < a.E) cnt[q] = __popc(mask[e]);
      at[q] = t;
      t += ((cnt[q] + MT - 1) / MT) << 16 | cnt[q];
    }
    const int inc = wave_scan(t);
    if (lane == 63 && wv < 4) wsum[wv] = inc;
    __syncthreads();
    int before = inc - t, all = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      before += q < wv ? wsum[q] : 0;
      all += wsum[q];
    }
    all = __builtin_amdgcn_readfirstlane(all);
    const int total = ((all >> 16) + (all & 0xFFFF)) * steps, share = (total + (int)gridDim.x - 1) / (int)gridDim.x;
    const int s0 = min(share * (int)blockIdx.x, total), s1 = min(s0 + share, total);
#pragma unroll
    for (int q = 0; q < 4; q++) {
      if (cnt[q] == 0) continue;
      const int p = before + at[q], chunks = (cnt[q] + MT - 1) / MT;
      first[4 * threadIdx.x + q] = p >> 16;
      const int lo = ((p >> 16) + (p & 0xFFFF)) * steps, span = (chunks + cnt[q]) * steps;
#pragma unroll
      for (int side = 0; side < 2; side++) {
        const int rel = (side ? s1 : s0) - lo;
        if (rel < 0 || rel >= span) continue;
        const int k = rel / ((MT + 1) * steps);   // (the chunks before an expert's last are full)
        cut[2 * side] = (p >> 16) + k;
        cut[2 * side + 1] = (rel - k * (MT + 1) * steps) / (min(MT, cnt[q] - k * MT) + 1);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int e = ids[i], rank = __popc(mask[e] & ((1u << row_of(i)) - 1));
      member[(first[e] + rank / MT) * MT + rank % MT] = i;
    }
    __syncthreads();
    // (no expert holds the end of the sequence)
    ch_lo = s0 < total ? __builtin_amdgcn_readfirstlane(cut[0]) : all >> 16;
    c_lo = s0 < total ? __builtin_amdgcn_readfirstlane(cut[1]) : 0;
    ch_hi = s1 < total ? __builtin_amdgcn_readfirstlane(cut[2]) : all >> 16;
    c_hi = s1 < total ? __builtin_amdgcn_readfirstlane(cut[3]) : 0;
  }
  const UnpackK kc = f16_unpack_consts();
  bool again = false;
  for (int ch = ch_lo; ch <= ch_hi; ch++) {   // (uniform over the workgroup)
    const int c0 = ch == ch_lo ? c_lo : 0, c1 = ch == ch_hi ? c_hi : steps;
    if (c0 >= c1) continue;
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
  }
}

// down and the weighted sum, a workgroup per (row, tile of columns): the row's
// top_k activation vectors become records in LDS, the waves share the slots
// (waves / top_k of them per slot, each a part of the tile; more slots than
// waves in turns), and the slots are added in slot order.  Workgroups of one
// column tile are dealt to one XCD (workgroup b runs on XCD b % 8), whose L2
// then holds the rows of an expert that several tokens take.  (768 -> 2048, 8 of
// 128) MXFP4, 16 rows: 25.9 us, 73 MB read past L2 of 114 MB in all, VALU busy half
// of the time, LDS a quarter (a lane reads a record of 144 bytes for each block of
// one weight row); Q6_K, 4 rows: 16.6 us for 40 MB.
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
    rlxq::moe_logits_body<XBF, RBF, 1, 4>(a, blockIdx.y, blockIdx.x);                                               \
  }                                                                                                                 \
  extern "C" __global__ __launch_bounds__(64) void rlxq_moe_logits_##XN##_##RN##_e4r8(rlxq_moe_logits_args a) {     \
    rlxq::moe_logits_body<XBF, RBF, 4, 8>(a, blockIdx.y, blockIdx.x);                                               \
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
