// MXFP4 (OCP microscaling FP4): float rows to codes and scales, and the linear
// layer of MXFP4 weights on activations quantised in the same call (W4A4).
//
// Quantiser.  A block is 32 consecutive elements of a row.  Its scale is the
// smallest power of two 2^e with 6 * 2^e >= amax (6 is the largest E2M1
// value), stored as the byte e + 127 (127 for a block of zeros or one with an
// infinity or a NaN); a code is the nearest E2M1 value of v / 2^e, ties to the
// even mantissa, sign kept, +-6 for what is not finite
// (crates/rlx-models-core/src/mxfp4_pack.rs:64-128, 196-250).  With amax =
// 1.m * 2^q the scale's exponent is q - 2 where 1.m <= 1.5, else q - 1, read
// off the float's bits; v / 2^e and its rounding are one instruction, exact.
//
// Matmul.  y[m, n] = sum over blocks of 2^(bx - 127) 2^(bw - 127) * sum of the
// 32 code products: v_mfma_scale_f32_*_f8f6f4 with both operands in FP4 takes
// 16 code bytes (one block) and one scale byte per lane and operand.  A lane
// owns four consecutive blocks of a row (64 code bytes, one dword of scales),
// one per MFMA: which blocks of K meet in one MFMA does not matter as long as
// both operands agree.  Products are exact and sums are f32.
#include "common.hip.h"
#include "mxfp4_args.h"

namespace rlxq {

typedef int32_t mx_i32x8_t __attribute__((ext_vector_type(8)));
typedef float mx_f32x4_t __attribute__((ext_vector_type(4)));

// Largest bit pattern of |v| over the four lanes of a quad (for floats the
// order of the patterns is the order of the magnitudes, infinities and NaN
// last).
RLXQ_DEV uint32_t quad_umax(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false);
  v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false);
  return v > o ? v : o;
}

// Eight elements of a block (a quarter of it per lane of a quad) -> their
// codes, element 0 in the low nibble of the dword, and the block's scale
// byte.  NAN_SCALE: a block with an infinity or a NaN gets the byte 255 (a NaN
// for the scaled MFMA) in place of 127.
template <bool NAN_SCALE>
RLXQ_DEV uint32_t mx_quant8(const float (&v)[8], uint32_t& byte) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
    a = a > u ? a : u;
  }
  a = quad_umax(a);
  const bool finite = a < 0x7f800000u;
  int e = (int)(a >> 23) - 2 + ((a & 0x7fffffu) > 0x400000u ? 1 : 0);
  e = e > 0 ? e : 0;
  const uint32_t b = a != 0u && finite ? (uint32_t)e : 127u;
  const float s = __uint_as_float(b << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
  if (b == 0u) c = 0u;   // (scale byte 0 reads as 0)
  if (!finite) {         // a NaN keeps its sign, as an infinity does
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t u = __float_as_uint(v[i]);
      if ((u & 0x7fffffffu) > 0x7f800000u) c = (c & ~(15u << (4 * i))) | ((7u | (u >> 31 << 3)) << (4 * i));
    }
  }
  byte = NAN_SCALE && !finite ? 255u : b;
  return c;
}

template <bool BF16>
RLXQ_DEV void mx_load8(const void* x, int64_t i, float (&v)[8]) {
  if constexpr (BF16) {
    const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int q = 0; q < 4; q++) {
      v[2 * q] = __uint_as_float(w[q] << 16);
      v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + i);
    const float4 a = p[0], b = p[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

// Row-major codes and scales: rows are whole blocks, so the matrix is one
// list of blocks, a quad of lanes each.
template <bool BF16>
RLXQ_DEV void mx_quant_rows(const rlxq_mx_quant_args& a) {
  const int64_t n8 = a.M * a.K / 8;   // groups of eight elements
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n8) return;   // (n8 is a multiple of 4: quads stay whole)
  float v[8];
  mx_load8<BF16>(a.x, i * 8, v);
  uint32_t b;
  const uint32_t c = mx_quant8<false>(v, b);
  reinterpret_cast<uint32_t*>(a.codes)[i] = c;
  if ((threadIdx.x & 3) == 0) a.scales[i >> 2] = (uint8_t)b;
}

// The matmul's activation fragments (mxfp4_args.h); the blocks past K of the
// last span are zeros.
template <bool BF16>
RLXQ_DEV void mx_quant_frag(const rlxq_mx_quant_args& a) {
  const int R = a.rows, G8 = 64 / R * 16;   // eights in a span
  const int64_t per = (int64_t)a.spans * G8;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.M * per) return;
  const int64_t m = i / per, e8 = i - m * per;
  const int span = (int)(e8 / G8), t = (int)(e8 - (int64_t)span * G8);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (e8 * 8 < a.K) mx_load8<BF16>(a.x, m * a.K + e8 * 8, v);   // (K is whole blocks: uniform over a quad)
  uint32_t b;
  const uint32_t c = mx_quant8<true>(v, b);
  const int blk = t >> 2, lane = (blk >> 2) * R + (int)(m % R), j = blk & 3;
  uint8_t* p = a.codes + ((m / R) * a.spans + span) * (int64_t)RLXQ_MX_CHUNK;
  *reinterpret_cast<uint32_t*>(p + 1024 * j + 16 * lane + 4 * (t & 3)) = c;
  if ((t & 3) == 0) p[4096 + 4 * lane + j] = (uint8_t)b;
}

// Four scale bytes of weights as the MFMA takes them: 255 reads as 2^127
// (e8m0_to_f32), which is byte 254.
RLXQ_DEV uint32_t mx_scales(uint32_t s) {
  const uint32_t f = ((s & 0x7f7f7f7fu) + 0x01010101u) & s & 0x80808080u;
  return s - (f >> 7);
}
// Whether one of the four bytes is 0 (a scale of zero).
RLXQ_DEV bool mx_has_zero(uint32_t s) { return ((s - 0x01010101u) & ~s & 0x80808080u) != 0u; }

// The scale bytes of blocks b0 .. b0 + 3 of a row of nb blocks (blocks past
// the end repeat the last one: their activations' codes are zero).
RLXQ_DEV uint32_t mx_load_scales(const uint8_t* row, int b0, int nb) {
  uint32_t s;
  if (b0 + 4 <= nb) {
    __builtin_memcpy(&s, row + b0, 4);
  } else {
    s = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) s |= (uint32_t)row[b0 + j < nb ? b0 + j : nb - 1] << (8 * j);
  }
  return s;
}

template <int OP>
RLXQ_DEV mx_f32x4_t mx_mfma16(const uint4& a, const uint4& b, mx_f32x4_t c, uint32_t sa, uint32_t sb) {
  const mx_i32x8_t av = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const mx_i32x8_t bv = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, OP, (int)sa, OP, (int)sb);
}

// Few rows: a wave takes NT tiles of 16 weight rows (the MFMA's first operand,
// straight from memory to registers) and MT tiles of 16 activation rows; the
// waves of the workgroup take the spans of 512 elements in turn and their sums
// meet in LDS.  Grid: (weight tiles, activation tiles, K splits).
template <int NT, int MT>
RLXQ_DEV void mx_dec_body(const rlxq_mx_gemm_args& a) {
  extern __shared__ float mx_red[];   // [waves][NT * MT][256]
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int row = lane & 15, g = lane >> 4;
  const int nb = (int)(a.K / 32);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const uint8_t* wr[NT];
  const uint8_t* sr[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    int64_t n = n0 + 16 * t + row;
    n = n < a.N ? n : a.N - 1;
    wr[t] = a.w + n * (a.K / 2);
    sr[t] = a.ws + n * nb;
  }
  mx_f32x4_t acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int q = 0; q < MT; q++) acc[t][q] = mx_f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int per = (a.spans + a.splits - 1) / a.splits;
  const int s0 = (int)blockIdx.z * per, s1 = s0 + per < a.spans ? s0 + per : a.spans;
  for (int s = s0 + wv; s < s1; s += nw) {
    const int b0 = 16 * s + 4 * g;
    uint4 wc[NT][4];
    uint32_t wsc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int b = b0 + j < nb ? b0 + j : nb - 1;
        wc[t][j] = *reinterpret_cast<const uint4*>(wr[t] + 16 * (int64_t)b);
      }
      wsc[t] = mx_load_scales(sr[t], b0, nb);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      if (mx_has_zero(wsc[t])) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (((wsc[t] >> (8 * j)) & 0xffu) == 0u) wc[t][j] = make_uint4(0u, 0u, 0u, 0u);
      }
      wsc[t] = mx_scales(wsc[t]);
    }
#pragma unroll
    for (int q = 0; q < MT; q++) {
      const uint8_t* xp = a.xf + ((m0 / 16 + q) * (int64_t)a.spans + s) * RLXQ_MX_CHUNK;
      uint4 xc[4];
      uint32_t xs = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) xc[j] = make_uint4(0u, 0u, 0u, 0u);
      if (m0 + 16 * q + row < a.M) {
#pragma unroll
        for (int j = 0; j < 4; j++) xc[j] = *reinterpret_cast<const uint4*>(xp + 1024 * j + 16 * lane);
        xs = *reinterpret_cast<const uint32_t*>(xp + 4096 + 4 * lane);
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        acc[t][q] = mx_mfma16<0>(wc[t][0], xc[0], acc[t][q], wsc[t], xs);
        acc[t][q] = mx_mfma16<1>(wc[t][1], xc[1], acc[t][q], wsc[t], xs);
        acc[t][q] = mx_mfma16<2>(wc[t][2], xc[2], acc[t][q], wsc[t], xs);
        acc[t][q] = mx_mfma16<3>(wc[t][3], xc[3], acc[t][q], wsc[t], xs);
      }
    }
  }
  // D: lane holds rows (weight rows) 4 g .. 4 g + 3 of column (activation row)
  // lane & 15; word i of tile (t, q) is weight row i / 16, activation row i % 16
  float* mine = mx_red + wv * (NT * MT * 256);
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int q = 0; q < MT; q++)
#pragma unroll
      for (int r = 0; r < 4; r++) mine[(t * MT + q) * 256 + (4 * g + r) * 16 + row] = acc[t][q][r];
  __syncthreads();
  for (int i = threadIdx.x; i < NT * MT * 256; i += blockDim.x) {
    // neighbouring threads take neighbouring columns of y
    const int q = i / (NT * 256), m = (i / (NT * 16)) & 15, n = i % (NT * 16);
    const int64_t mm = m0 + 16 * q + m, nn = n0 + n;
    if (mm >= a.M || nn >= a.N) continue;
    const float* p = mx_red + ((n >> 4) * MT + q) * 256 + (n & 15) * 16 + m;
    float s = 0.f;
    for (int v = 0; v < nw; v++) s += p[v * (NT * MT * 256)];
    if (a.splits > 1) a.part[((int64_t)blockIdx.z * a.M + mm) * a.N + nn] = s;
    else if (a.y_bf16) reinterpret_cast<uint16_t*>(a.y)[mm * a.N + nn] = (uint16_t)f32_to_bf16_bits(s);
    else reinterpret_cast<float*>(a.y)[mm * a.N + nn] = s;
  }
}

}  // namespace rlxq

extern "C" __global__ __launch_bounds__(256) void rlxq_mx_quant_bf16(rlxq_mx_quant_args a) { rlxq::mx_quant_rows<true>(a); }
extern "C" __global__ __launch_bounds__(256) void rlxq_mx_quant_f32(rlxq_mx_quant_args a) { rlxq::mx_quant_rows<false>(a); }
extern "C" __global__ __launch_bounds__(256) void rlxq_mx_frag_bf16(rlxq_mx_quant_args a) { rlxq::mx_quant_frag<true>(a); }
extern "C" __global__ __launch_bounds__(256) void rlxq_mx_frag_f32(rlxq_mx_quant_args a) { rlxq::mx_quant_frag<false>(a); }

extern "C" __global__ __launch_bounds__(512) void rlxq_mx_dec_n1m1(rlxq_mx_gemm_args a) { rlxq::mx_dec_body<1, 1>(a); }
