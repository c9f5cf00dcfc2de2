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
// list of blocks, a quad of lanes each, ILP groups of eight elements per
// thread.  Bytes bound it: 24576 x 4096 in bf16 (254 MB) 46 us with four groups
// in flight and streaming stores, 59 with one; f32 80 and 102.  Small matrices
// take one (16 x 4096: 2.7 us against 3.5; the reader's caches keep the codes).
template <bool BF16, int ILP>
RLXQ_DEV void mx_quant_rows(const rlxq_mx_quant_args& a) {
  const int64_t n8 = a.M * a.K / 8;   // groups of eight elements (a multiple of 4: quads stay whole)
  const int64_t i0 = (int64_t)blockIdx.x * (256 * ILP) + threadIdx.x;
  float v[ILP][8];
#pragma unroll
  for (int u = 0; u < ILP; u++)
    if (i0 + 256 * u < n8) mx_load8<BF16>(a.x, (i0 + 256 * u) * 8, v[u]);
#pragma unroll
  for (int u = 0; u < ILP; u++) {
    const int64_t i = i0 + 256 * u;
    if (i >= n8) continue;
    uint32_t b;
    const uint32_t c = mx_quant8<false>(v[u], b);
    if constexpr (ILP > 1) __builtin_nontemporal_store(c, reinterpret_cast<uint32_t*>(a.codes) + i);
    else reinterpret_cast<uint32_t*>(a.codes)[i] = c;
    if ((threadIdx.x & 3) == 0) a.scales[i >> 2] = (uint8_t)b;
  }
}

// The values of codes and E8M0 scale bytes, four per thread and step: 1 KB of
// consecutive floats per wave and store (24576 x 4096 in 73 us, 456 MB).
template <int ILP>
RLXQ_DEV void mx_dequant_rows(const rlxq_mx_quant_args& a, float* out) {
  const int64_t n4 = a.M * a.K / 4;
  const int64_t i0 = (int64_t)blockIdx.x * (256 * ILP) + threadIdx.x;
  uint32_t c[ILP], b[ILP];
#pragma unroll
  for (int u = 0; u < ILP; u++) {
    const int64_t i = i0 + 256 * u < n4 ? i0 + 256 * u : n4 - 1;
    c[u] = reinterpret_cast<const uint16_t*>(a.codes)[i];
    b[u] = a.scales[i >> 3];
  }
#pragma unroll
  for (int u = 0; u < ILP; u++) {
    if (i0 + 256 * u >= n4) continue;
    const float s = e8m0_to_f32(b[u]);
    const rlxq_f32x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.0f, 0);
    const rlxq_f32x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.0f, 1);
    const mx_f32x4_t v = {lo.x * s, lo.y * s, hi.x * s, hi.y * s};
    if constexpr (ILP > 1) __builtin_nontemporal_store(v, reinterpret_cast<mx_f32x4_t*>(out) + i0 + 256 * u);
    else reinterpret_cast<mx_f32x4_t*>(out)[i0 + 256 * u] = v;
  }
}

// Four scale bytes of weights as the MFMA takes them: 255 reads as 2^127
// (e8m0_to_f32), which is byte 254.
RLXQ_DEV uint32_t mx_scales(uint32_t s) {
  const uint32_t f = ((s & 0x7f7f7f7fu) + 0x01010101u) & s & 0x80808080u;
  return s - (f >> 7);
}
// Whether one of the four bytes is 0 (a scale of zero).
RLXQ_DEV bool mx_has_zero(uint32_t s) { return ((s - 0x01010101u) & ~s & 0x80808080u) != 0u; }

// The scale bytes of 32 weight rows (one workgroup), a dword per lane and span
// of 256 elements in the lane order of the fragments: the matmul then reads
// whole lines of them.  255 becomes 254 (mx_scales), blocks past K get 127.
// zero[rb] tells whether one of the row block's bytes is 0.
RLXQ_DEV void mx_scale_frag(const rlxq_mx_quant_args& a, int rb) {
  const int nb = (int)(a.K / 32);
  bool zero = false;
  for (int i = threadIdx.x; i < a.spans * 32; i += blockDim.x) {
    const int span = i >> 5, row = i & 31;
    int64_t n = (int64_t)rb * 32 + row;
    n = n < a.N ? n : a.N - 1;
    const uint8_t* p = a.ws + n * nb + 8 * span;
    uint64_t v;   // the span's eight bytes of the row
    if (8 * span + 8 <= nb) {
      __builtin_memcpy(&v, p, 8);
    } else {
      v = 0x7f7f7f7f7f7f7f7full;
      for (int j = 0; 8 * span + j < nb; j++) v = (v & ~(0xffull << (8 * j))) | ((uint64_t)p[j] << (8 * j));
    }
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    zero = zero || mx_has_zero(lo) || mx_has_zero(hi);
    uint32_t* o = a.wsf + ((int64_t)rb * a.spans + span) * 64 + row;
    o[0] = mx_scales(perm_b32(hi, lo, 0x05040100u));    // blocks 0, 1, 4, 5
    o[32] = mx_scales(perm_b32(hi, lo, 0x07060302u));   // blocks 2, 3, 6, 7
  }
  const bool any = __syncthreads_or(zero) != 0;
  if (threadIdx.x == 0) a.zero[rb] = any ? 1 : 0;
}

// The matmul's activation fragments (mxfp4_args.h), a workgroup per chunk: the
// threads follow the chunk's code dwords, so a wave stores 256 consecutive
// bytes and a quad reads a block.  Zeros for the blocks past K and the rows
// past M.
template <bool BF16>
RLXQ_DEV void mx_quant_frag(const rlxq_mx_quant_args& a) {
  if ((int)blockIdx.x < a.wblocks) {   // (the weights' scales beside them)
    mx_scale_frag(a, blockIdx.x);
    return;
  }
  const int R = a.rows, c = blockIdx.x - a.wblocks;
  const int rb = c / a.spans, span = c - rb * a.spans;
  const int lane = threadIdx.x >> 2, row = lane % R, g = lane / R;
  const int64_t m = (int64_t)rb * R + row;
  uint8_t* p = a.codes + (int64_t)c * RLXQ_MX_CHUNK;
  float v[4][8];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int blk = R == 16 ? 4 * g + j : 4 * (j >> 1) + 2 * g + (j & 1);
    const int64_t e = (int64_t)span * (64 / R * 128) + 32 * blk + 8 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < 8; i++) v[j][i] = 0.f;
    if (m < a.M && e < a.K) mx_load8<BF16>(a.x, m * a.K + e, v[j]);   // (K is whole blocks)
  }
  uint32_t sc = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t b;
    reinterpret_cast<uint32_t*>(p)[256 * j + threadIdx.x] = mx_quant8<true>(v[j], b);
    sc |= b << (8 * j);
  }
  if ((threadIdx.x & 3) == 0) *reinterpret_cast<uint32_t*>(p + 4096 + threadIdx.x) = sc;
}

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
// straight from memory to registers, the next span's while this one is
// multiplied) and MT tiles of 16 activation rows; the waves of the workgroup
// take the spans of 512 elements in turn and their sums meet in LDS.  Weight
// bytes bound it: 64 consecutive code bytes and four scale bytes per lane and
// span, four MFMAs per 4 KB.
// FUSED (MT == 1): the workgroup quantises the activation rows itself, into
// LDS, while its first weights are on the way (no launch ahead of this one);
// else they come as fragments from the preparation launch.
template <int NT, int MT, bool FUSED, bool XBF>
RLXQ_DEV void mx_dec_body(const rlxq_mx_gemm_args& a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t mx_dec_lds[];
  float* red = reinterpret_cast<float*>(mx_dec_lds);   // [waves][NT * MT][256], behind the activations
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int row = lane & 15, g = lane >> 4;
  const int nb = (int)(a.K / 32);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);
  const int M = FUSED ? (int)a.M : 0;
  const uint8_t* wr[NT];
  const uint8_t* sr[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    int64_t n = n0 + 16 * t + row;
    n = n < a.N ? n : a.N - 1;
    wr[t] = a.w + n * (a.K / 2);
    sr[t] = a.ws + n * nb;
  }
  struct Buf {
    uint4 c[NT][4];
    uint32_t s[NT];
  };
  auto load = [&](int s, Buf& w) {
    const int b0 = 16 * s + 4 * g;
    if (16 * s + 16 <= nb) {
#pragma unroll
      for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int j = 0; j < 4; j++) w.c[t][j] = *reinterpret_cast<const uint4*>(wr[t] + 16 * (int64_t)(b0 + j));
        __builtin_memcpy(&w.s[t], sr[t] + b0, 4);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; t++) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          w.c[t][j] = *reinterpret_cast<const uint4*>(wr[t] + 16 * (int64_t)(b0 + j < nb ? b0 + j : nb - 1));
        w.s[t] = mx_load_scales(sr[t], b0, nb);
      }
    }
  };
  Buf cur;
  if (wv < a.spans) load(wv, cur);
  if constexpr (FUSED) {
    // row m, span s: 64 code bytes and a dword of scales per lane group g, at
    // (s M + m) 272 + 68 g
    const int per = a.spans * 64;   // eights of a row, whole spans
    for (int i = threadIdx.x; i < M * per; i += blockDim.x) {
      const int m = i / per, e8 = i - m * per, blk = e8 >> 2;
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (e8 * 8 < a.K) mx_load8<XBF>(a.x, (int64_t)m * a.K + e8 * 8, v);
      uint32_t b;
      const uint32_t c = mx_quant8<true>(v, b);
      uint8_t* p = mx_dec_lds + ((blk >> 4) * M + m) * 272 + 68 * ((blk >> 2) & 3);
      *reinterpret_cast<uint32_t*>(p + 16 * (blk & 3) + 4 * (e8 & 3)) = c;
      if ((e8 & 3) == 0) p[64 + (blk & 3)] = (uint8_t)b;
    }
    red = reinterpret_cast<float*>(mx_dec_lds + ((a.spans * M * 272 + 15) & ~15));
    __syncthreads();
  }
  mx_f32x4_t acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int q = 0; q < MT; q++) acc[t][q] = mx_f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int s = wv; s < a.spans; s += nw) {
    Buf nxt;
    if (s + nw < a.spans) load(s + nw, nxt);
    uint4 xc[MT][4];
    uint32_t xs[MT];
#pragma unroll
    for (int q = 0; q < MT; q++) {
      xs[q] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) xc[q][j] = make_uint4(0u, 0u, 0u, 0u);
      if (16 * q + row < a.M) {
        if constexpr (FUSED) {
          const uint32_t* p = reinterpret_cast<const uint32_t*>(mx_dec_lds + (s * M + row) * 272 + 68 * g);
#pragma unroll
          for (int j = 0; j < 4; j++) xc[q][j] = make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
          xs[q] = p[16];
        } else {
          const uint8_t* xp = a.xf + (q * (int64_t)a.spans + s) * RLXQ_MX_CHUNK;
#pragma unroll
          for (int j = 0; j < 4; j++) xc[q][j] = *reinterpret_cast<const uint4*>(xp + 1024 * j + 16 * lane);
          xs[q] = *reinterpret_cast<const uint32_t*>(xp + 4096 + 4 * lane);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) {
      if (mx_has_zero(cur.s[t])) {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (((cur.s[t] >> (8 * j)) & 0xffu) == 0u) cur.c[t][j] = make_uint4(0u, 0u, 0u, 0u);
      }
      const uint32_t sw = mx_scales(cur.s[t]);
#pragma unroll
      for (int q = 0; q < MT; q++) {
        acc[t][q] = mx_mfma16<0>(cur.c[t][0], xc[q][0], acc[t][q], sw, xs[q]);
        acc[t][q] = mx_mfma16<1>(cur.c[t][1], xc[q][1], acc[t][q], sw, xs[q]);
        acc[t][q] = mx_mfma16<2>(cur.c[t][2], xc[q][2], acc[t][q], sw, xs[q]);
        acc[t][q] = mx_mfma16<3>(cur.c[t][3], xc[q][3], acc[t][q], sw, xs[q]);
      }
    }
    cur = nxt;
  }
  // D: lane holds weight rows 4 g .. 4 g + 3 of activation row lane & 15; word
  // 16 n + m of tile (t, q) is weight row n, activation row m
  float* mine = red + wv * (NT * MT * 256);
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
    const int64_t mm = 16 * q + m, nn = n0 + n;
    if (mm >= a.M || nn >= a.N) continue;
    const float* p = red + ((n >> 4) * MT + q) * 256 + (n & 15) * 16 + m;
    float s = 0.f;
    for (int v = 0; v < nw; v++) s += p[v * (NT * MT * 256)];
    if (a.y_bf16) reinterpret_cast<uint16_t*>(a.y)[mm * a.N + nn] = (uint16_t)f32_to_bf16_bits(s);
    else reinterpret_cast<float*>(a.y)[mm * a.N + nn] = s;
  }
}

// ------------------------------------------------------------- many rows
typedef float mx_f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t mx_u32x4_t __attribute__((ext_vector_type(4)));

// c += a . b for 32 x 32 outputs and 64 elements, byte OP of the scales.  As the
// instruction itself, so that it stays where it is written between the LDS
// reads and the loads around it (the compiler moves the builtin past both).
// The compiler then does not see what the instruction asks for: two wait
// states behind a vector instruction that writes one of its operands (masked
// weights straight in front of it gave wrong sums without them; behind another
// MFMA they cost nothing), and mx_mfma_done() ahead of any other use of c.
template <int OP>
RLXQ_DEV void mx_mfma32(mx_f32x16_t& c, const uint4& a, const uint4& b, uint32_t sa, uint32_t sb) {
  const mx_u32x4_t av = {a.x, a.y, a.z, a.w}, bv = {b.x, b.y, b.z, b.w};
  asm volatile("s_nop 1\n\tv_mfma_scale_f32_32x32x64_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] "
               "cbsz:4 blgp:4"
               : "+a"(c)
               : "v"(av), "v"(bv), "v"(sa), "v"(sb), "n"(OP & 1), "n"(OP >> 1));
}
RLXQ_DEV void mx_mfma_done() { asm volatile("s_nop 15\n\ts_nop 15"); }

// 64 lanes x 16 (or 4) bytes from base + off + I into LDS at dst + I (base and
// dst wave-uniform).  Written as the instruction itself: the compiler cannot
// tell the buffer that is being filled from the one being read and would wait
// for the fill ahead of every LDS read.  mx_loads_wait() waits for all but the
// wave's last N loads; nothing else does.
// The instruction takes dst from M0, which the compiler may use for its own
// between any two statements: each load sets it itself, one wait state ahead.
template <int I>
RLXQ_DEV void mx_to_lds16(uint32_t dst, const uint8_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 offset:%2"
               : : "v"(off), "s"(base), "n"(I), "s"(dst) : "memory", "m0");
}
template <int I>
RLXQ_DEV void mx_to_lds4(uint32_t dst, const uint8_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1 offset:%2"
               : : "v"(off), "s"(base), "n"(I), "s"(dst) : "memory", "m0");
}
template <int N>
RLXQ_DEV void mx_loads_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}
// p, the same in every lane, in scalar registers.
RLXQ_DEV const uint8_t* mx_uniform(const uint8_t* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
  return reinterpret_cast<const uint8_t*>(((uint64_t)hi << 32) | lo);
}
RLXQ_DEV uint32_t mx_lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }

// One output tile of 32 TM WGM activation rows x 32 TN WGN weight rows by
// WGM x WGN waves, in stages of 128 elements (64 code bytes a row).  Both
// operands go from memory straight into LDS, three stages ahead of the one
// being multiplied, in a ring of four: the activations' fragments as they are
// (a wave reads lane-consecutive 16 bytes), the weights as rows of four
// 16-byte pieces, piece p of row r at slot p ^ (r >> 1 & 3), which spreads the
// eight lanes that read one piece of eight rows over all banks.  Scales come a
// span (two stages) at a time, a dword per lane and 32 rows.
// A stage is two MFMA steps.  While one step's MFMAs run, the fragments of the
// next are read and the loads of the stage three ahead are issued, one or two
// between any two MFMAs; the workgroup meets once a stage, between the steps:
// behind that barrier the next stage is in LDS and the last one has been read.
// The weights are the MFMA's first operand, so that a lane's results are four
// consecutive columns of y.
// MASKED: weight blocks whose scale byte is 0 are read as zero codes.
template <int WGM, int WGN, int TM, int TN, bool MASKED>
RLXQ_DEV void mx_gemm_tile(const rlxq_mx_gemm_args& a, int tm, int tn, uint8_t* mx_lds) {
  constexpr int BM = 32 * TM * WGM, BN = 32 * TN * WGN, NW = WGM * WGN;
  constexpr int STAGE = (BM + BN) * 64, XB = BM / 32, WB = BN / 32, SCALES = (XB + WB) * 256;
  constexpr int LX = BM * 64 / 1024 / NW, LW = BN * 64 / 1024 / NW;   // 1 KB loads per wave and stage
  constexpr int LS = (XB + WB) / NW;   // 256 B scale loads per wave and span
  static_assert(LX * NW * 1024 == BM * 64 && LW * NW * 1024 == BN * 64 && LS * NW == XB + WB, "whole loads per wave");
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wv / WGN, wn = wv % WGN;
  const int row = lane & 31, g = lane >> 5;
  const int nb = (int)(a.K / 32);
  const int64_t kb = a.K / 2;
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int xb_last = (int)((a.M + 31) / 32) - 1, wb_last = (int)((a.N + 31) / 32) - 1;
  const int per = (a.spans + a.splits - 1) / a.splits;
  const int s0 = __builtin_amdgcn_readfirstlane((int)blockIdx.y * per);
  const int s1 = __builtin_amdgcn_readfirstlane(s0 + per < a.spans ? s0 + per : a.spans);

  // ---- loads.  A wave fills LX KB of the activations' part of a ring slot
  // and LW KB of the weights', each one run of LDS at immediate offsets,
  // which move the source too (the lanes' offsets undo that).
  // Its LX KB are whole halves of row blocks' fragments: 2 KB each.
  static_assert(LX % 2 == 0, "whole row blocks per wave");
  constexpr int XP = LX / 2;
  const uint32_t l16 = 16 * lane, l4 = 4 * lane;
  const uint8_t* xp[XP];   // row block q's fragments (its half-chunk of the next stage to load), less 2048 q
#pragma unroll
  for (int q = 0; q < XP; q++) {
    const int rb = tm * XB + wv * XP + q;
    xp[q] = mx_uniform(a.xf + ((int64_t)(rb < xb_last ? rb : xb_last) * a.spans + s0) * RLXQ_MX_CHUNK - 2048 * q);
  }
  // weight pieces of this lane (rows clamped to N): piece (lane & 3) ^ .. of
  // row lane >> 2 of each 16; blocks past K read the row's last one (the
  // activations are zero there): `back` in the stage that K ends in
  // (offsets are unsigned: the base never passes that stage)
  const int piece = (lane & 3) ^ ((lane >> 3) & 3), u_end = __builtin_amdgcn_readfirstlane((nb - 1) / 4);
  uint32_t wo[LW];
  const int over = 4 * u_end + piece - (nb - 1);
  const uint32_t back = over > 0 ? 16 * over : 0;
#pragma unroll
  for (int i = 0; i < LW; i++) {
    int64_t n = n0 + (wv * LW + i) * 16 + (lane >> 2);
    n = n < a.N ? n : a.N - 1;
    wo[i] = (uint32_t)((n - n0) * kb) + 16 * piece + 1024 * (LW - 1 - i);
  }
  const uint8_t* wbase = mx_uniform(a.w + n0 * kb - 1024 * (LW - 1));
  // scales: the wave's run i of 256 B is row block wv LS + i of the
  // activations, then of the weights
  const uint8_t* sp_[LS];
  int sstep[LS];
#pragma unroll
  for (int i = 0; i < LS; i++) {
    const int c = wv * LS + i;
    const bool sx = c < XB;
    const int rb = sx ? tm * XB + c : tn * WB + c - XB, last = sx ? xb_last : wb_last;
    sstep[i] = sx ? RLXQ_MX_CHUNK : 256;
    const uint8_t* b = sx ? a.xf + 4096 : reinterpret_cast<const uint8_t*>(a.wsf);
    sp_[i] = mx_uniform(b + (int64_t)(rb < last ? rb : last) * a.spans * sstep[i] - 256 * i);
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(mx_lds_addr(mx_lds));
  const uint32_t x_dst = lds0 + 1024 * wv * LX, w_dst = lds0 + BM * 64 + 1024 * wv * LW;
  const uint32_t s_dst = lds0 + 4 * STAGE + 256 * wv * LS;
  const uint8_t* wp = wbase;   // of the next stage to load
  bool w_end = false;          // that stage is the one K ends in
  // before the loads of stage u (past the last stage: that one again)
  const int u_last = 2 * s1 - 1;
  auto stage_w = [&](int u) {
    u = u < u_last ? u : u_last;
    w_end = u >= u_end;
    wp = wbase + 64 * (int64_t)(w_end ? u_end : u);
  };
  // load i (0 .. LX + LW - 1) of the stage into ring slot `slot`
  auto load_codes = [&](auto ii, int slot) {
    constexpr int i = decltype(ii)::value;
    if constexpr (i < LX) {
      mx_to_lds16<1024 * i>(x_dst + slot * STAGE, xp[i / 2], l16);
    } else {
      mx_to_lds16<1024 * (i - LX)>(w_dst + slot * STAGE, wp, wo[i - LX] - (w_end ? back : 0));
    }
  };
  // the activations' pointers from a stage (half h of a span) to the next;
  // past the last stage they stay
  auto next_x = [&](int u, int h) {
    const int d = u < u_last ? (h ? RLXQ_MX_CHUNK - 2048 : 2048) : 0;
#pragma unroll
    for (int q = 0; q < XP; q++) xp[q] += d;
  };
  auto load_scales = [&](auto ii, int sp) {   // run i of span sp's scales
    constexpr int i = decltype(ii)::value;
    mx_to_lds4<256 * i>(s_dst + (sp & 1) * SCALES, sp_[i] + (int64_t)(sp < s1 ? sp : s1 - 1) * sstep[i], l4);
  };
  mx_f32x16_t acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[j][i][r] = 0.f;

  // ---- fragments.  Stages of even spans are in slots 0 and 1, of odd ones in
  // 2 and 3: `half` is the byte offset of the span's pair of slots.
  uint4 xf[2][TM], wf[2][TN];
  uint32_t xc[TM], wc[TN], xn[TM], wn_[TN];
  const uint8_t* xl = mx_lds + wm * TM * 2048 + l16;
  const uint8_t* wl = mx_lds + BM * 64 + (wn * TN * 32 + row) * 64;
  const uint32_t wpc[2] = {(uint32_t)(((2 * g) ^ ((row >> 1) & 3)) << 4), (uint32_t)(((2 * g + 1) ^ ((row >> 1) & 3)) << 4)};
  // fragment q of MFMA step k (0..3) of a span
  auto read_frag = [&](auto kk, auto qq, uint32_t half) {
    constexpr int k = decltype(kk)::value, q = decltype(qq)::value;
    constexpr int slot = (k >> 1) * STAGE;
    if constexpr (q < TM) xf[k & 1][q] = *reinterpret_cast<const uint4*>(xl + half + (slot + q * 2048 + 1024 * (k & 1)));
    else wf[k & 1][q - TM] = *reinterpret_cast<const uint4*>(wl + half + wpc[k & 1] + (slot + (q - TM) * 2048));
  };
  auto read_scale = [&](auto qq, int sp) {
    constexpr int q = decltype(qq)::value;
    const uint8_t* st = mx_lds + 4 * STAGE + (sp & 1) * SCALES + l4;
    if constexpr (q < TM) xn[q] = *reinterpret_cast<const uint32_t*>(st + wm * TM * 256 + q * 256);
    else wn_[q - TM] = *reinterpret_cast<const uint32_t*>(st + (XB + wn * TN) * 256 + (q - TM) * 256);
  };
  auto take_scales = [&]() {
#pragma unroll
    for (int i = 0; i < TM; i++) xc[i] = xn[i];
#pragma unroll
    for (int j = 0; j < TN; j++) wc[j] = wn_[j];
  };
  // The MFMAs of step k with `A` other actions spread between them.
  auto step = [&](auto kk, auto nact, auto act) {
    constexpr int k = decltype(kk)::value, A = decltype(nact)::value, Q = TM * TN;
    static_for<Q>([&](auto qq) {
      constexpr int q = decltype(qq)::value, j = q / TM, i = q % TM;
      if constexpr (MASKED && i == 0) {
        if (((wc[j] >> (8 * k)) & 0xffu) == 0u) wf[k & 1][j] = make_uint4(0u, 0u, 0u, 0u);
      }
      mx_mfma32<k>(acc[j][i], wf[k & 1][j], xf[k & 1][i], wc[j], xc[i]);
      static_for<A>([&](auto aa) {
        constexpr int x = decltype(aa)::value;
        if constexpr (x * Q / A == q) act(aa);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  constexpr int LC = LX + LW, F = TM + TN;

  static_for<LS>([&](auto i) { load_scales(i, s0); });
  static_for<3>([&](auto uu) {
    constexpr int u = decltype(uu)::value;
    if constexpr (u == 2) static_for<LS>([&](auto i) { load_scales(i, s0 + 1); });
    stage_w(2 * s0 + u);
    static_for<LC>([&](auto i) { load_codes(i, u); });
    next_x(2 * s0 + u, u & 1);
  });
  mx_loads_wait<2 * LC + LS>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  static_for<F>([&](auto q) { read_scale(q, s0); });
  static_for<F>([&](auto q) { read_frag(std::integral_constant<int, 0>{}, q, 0); });
  take_scales();
  for (int sp = s0; sp < s1; sp++) {
    const uint32_t half = ((sp - s0) & 1) * (2 * STAGE);
    const int slots = 2 * ((sp - s0) & 1);
    static_for<2>([&](auto hh) {   // stage u = 2 sp + h, in slot slots + h
      constexpr int h = decltype(hh)::value;
      const int u = 2 * sp + h;
      constexpr std::integral_constant<int, 2 * h> k0{};
      constexpr std::integral_constant<int, 2 * h + 1> k1{};
      constexpr std::integral_constant<int, h == 0 ? 2 : 0> k2{};
      // first step; meanwhile the second's fragments, then the stage three on
      stage_w(u + 3);
      step(k0, std::integral_constant<int, F + LC>{}, [&](auto aa) {
        constexpr int x = decltype(aa)::value;
        if constexpr (x < F) read_frag(k1, aa, half);
        else load_codes(std::integral_constant<int, x - F>{}, h == 0 ? (slots + 3) & 3 : slots);
      });
      next_x(u + 3, 1 - h);
      if constexpr (h == 1) static_for<LS>([&](auto i) { load_scales(i, sp + 2); });
      mx_loads_wait<2 * LC + LS>();   // stage u + 1 has landed; this wave has read stage u
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      // second step; meanwhile the first fragments (and scales) of the next stage
      step(k1, std::integral_constant<int, F * (h + 1)>{}, [&](auto aa) {
        constexpr int x = decltype(aa)::value;
        if constexpr (x < F) read_frag(k2, aa, h == 0 ? half : half ^ (2 * STAGE));
        else read_scale(std::integral_constant<int, x - F>{}, sp + 1);
      });
      if constexpr (h == 1) take_scales();
    });
  }
  // (the loads past the last stage: none may land in another workgroup's LDS)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  mx_mfma_done();
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++) asm volatile("" : "+a"(acc[j][i]));   // (no use of them moves ahead of it)

  // A lane holds activation row (column of the MFMA's result) lane & 31 and
  // weight rows 8 q + 4 g .. + 3 of each tile: four consecutive outputs.  A
  // whole tile goes out through the wave's own part of LDS, 32 rows at a time,
  // as whole runs of 32 TN outputs (straight from the registers a store would
  // hold 32 runs of 16 or 32 bytes).
  const int64_t mw = m0 + wm * TM * 32, nw = n0 + wn * TN * 32;
  const bool whole = m0 + BM <= a.M && n0 + BN <= a.N && a.vec;
  const bool bf = a.splits == 1 && a.y_bf16;
  uint8_t* yb = reinterpret_cast<uint8_t*>(a.splits > 1 ? a.part + (int64_t)blockIdx.y * a.M * a.N : a.y);
  constexpr int EROW = 32 * TN * 4 + 16;   // bytes of a staged row (16 more: rows start in different banks)
  static_assert(NW * 32 * EROW <= 4 * STAGE, "staging fits the ring");
  uint8_t* est = mx_lds + wv * (32 * EROW);
  __syncthreads();   // (every wave has read its last fragments)
  auto tiles = [&](auto bfc) {
    constexpr bool BF = decltype(bfc)::value;
    constexpr int ES = BF ? 2 : 4;
#pragma unroll
    for (int i = 0; i < TM; i++) {
#pragma unroll
      for (int j = 0; j < TN; j++) {
        mx_f32x16_t v = acc[j][i];
        asm volatile("" : "+v"(v) : : "memory");   // (one tile at a time out of the accumulators)
        if (whole) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            uint8_t* d = est + row * EROW + (32 * j + 8 * q + 4 * g) * ES;
            if constexpr (BF)
              *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v[4 * q], v[4 * q + 1]), pack_bf16x2(v[4 * q + 2], v[4 * q + 3]));
            else
              *reinterpret_cast<float4*>(d) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          }
        } else if (mw + 32 * i + row < a.M) {
          const int64_t o = (mw + 32 * i + row) * a.N + nw + 32 * j + 4 * g;
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const int d = 8 * (r / 4) + r % 4;
            if (nw + 32 * j + 4 * g + d >= a.N) continue;
            if constexpr (BF) reinterpret_cast<uint16_t*>(yb)[o + d] = (uint16_t)f32_to_bf16_bits(v[r]);
            else reinterpret_cast<float*>(yb)[o + d] = v[r];
          }
        }
      }
      if (whole) {
        // (the wave's own LDS: its stores are done before its reads)
        constexpr int PER = 32 * TN * ES / 16, RPI = 64 / PER;   // lanes per row, rows per store
        static_assert(PER <= 64, "a row per store at least");
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int q = 0; q < 32 / RPI; q++) {
          const int r = q * RPI + lane / PER, c = 16 * (lane % PER);
          const uint4 v = *reinterpret_cast<const uint4*>(est + r * EROW + c);
          *reinterpret_cast<uint4*>(yb + ((mw + 32 * i + r) * a.N + nw) * ES + c) = v;
        }
      }
    }
  };
  if (bf) tiles(std::true_type{});
  else tiles(std::false_type{});
}

template <int WGM, int WGN, int TM, int TN>
RLXQ_DEV void mx_gemm_body(const rlxq_mx_gemm_args& a) {
  extern __shared__ __attribute__((aligned(1024))) uint8_t mx_lds[];
  constexpr int BM = 32 * TM * WGM, BN = 32 * TN * WGN;
  const int tiles_m = (int)((a.M + BM - 1) / BM), tiles_n = (int)((a.N + BN - 1) / BN);
  int tm, tn;
  if (!tile_of(blockIdx.x, tiles_m, tiles_n, 4, tm, tn)) return;
  const int wb_last = (int)((a.N + 31) / 32) - 1;
  bool zero = false;
#pragma unroll
  for (int j = 0; j < BN / 32; j++) {
    const int rb = tn * (BN / 32) + j;
    zero = zero || a.zero[rb < wb_last ? rb : wb_last] != 0;
  }
  if (__builtin_amdgcn_readfirstlane(zero ? 1 : 0)) mx_gemm_tile<WGM, WGN, TM, TN, true>(a, tm, tn, mx_lds);
  else mx_gemm_tile<WGM, WGN, TM, TN, false>(a, tm, tn, mx_lds);
}

// y = the K splits' partial sums, added in split order.
RLXQ_DEV void mx_reduce_body(const rlxq_mx_gemm_args& a) {
  const int64_t total = a.M * a.N;
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 4;
  if (i >= total) return;
  if (i + 4 <= total && a.vec) {
    float4 s = *reinterpret_cast<const float4*>(a.part + i);
    for (int p = 1; p < a.splits; p++) {
      const float4 v = *reinterpret_cast<const float4*>(a.part + p * total + i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    if (a.y_bf16) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.y) + i) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
    else *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.y) + i) = s;
    return;
  }
  for (int64_t j = i; j < i + 4 && j < total; j++) {
    float s = a.part[j];
    for (int p = 1; p < a.splits; p++) s += a.part[p * total + j];
    if (a.y_bf16) reinterpret_cast<uint16_t*>(a.y)[j] = (uint16_t)f32_to_bf16_bits(s);
    else reinterpret_cast<float*>(a.y)[j] = s;
  }
}

}  // namespace rlxq

extern "C" __global__ __launch_bounds__(256) void rlxq_mx_reduce(rlxq_mx_gemm_args a) { rlxq::mx_reduce_body(a); }
#define RLXQ_MX_GEMM(NAME, WGM, WGN, TM, TN)                                                             \
  extern "C" __global__ __launch_bounds__(64 * WGM * WGN) void rlxq_mx_gemm_##NAME(rlxq_mx_gemm_args a) { \
    rlxq::mx_gemm_body<WGM, WGN, TM, TN>(a);                                                             \
  }
RLXQ_MX_GEMM(m256n256, 2, 4, 4, 2)
RLXQ_MX_GEMM(m128n128, 2, 2, 2, 2)
RLXQ_MX_GEMM(m128n64, 2, 1, 2, 2)
RLXQ_MX_GEMM(m64n64, 1, 2, 2, 1)

// rlxq_mx_quant_<x>_u<groups per thread>
#define RLXQ_MX_ROWS(U)                                                                                                \
  extern "C" __global__ __launch_bounds__(256) void rlxq_mx_quant_bf16_u##U(rlxq_mx_quant_args a) {                    \
    rlxq::mx_quant_rows<true, U>(a);                                                                                   \
  }                                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void rlxq_mx_quant_f32_u##U(rlxq_mx_quant_args a) {                     \
    rlxq::mx_quant_rows<false, U>(a);                                                                                  \
  }                                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void rlxq_mx_dequant_u##U(rlxq_mx_quant_args a, float* out) {           \
    rlxq::mx_dequant_rows<U>(a, out);                                                                                  \
  }
RLXQ_MX_ROWS(1)
RLXQ_MX_ROWS(4)
extern "C" __global__ __launch_bounds__(256) void rlxq_mx_frag_bf16(rlxq_mx_quant_args a) { rlxq::mx_quant_frag<true>(a); }
extern "C" __global__ __launch_bounds__(256) void rlxq_mx_frag_f32(rlxq_mx_quant_args a) { rlxq::mx_quant_frag<false>(a); }


// rlxq_mx_dec_<weight tiles>_<activation tiles>, _f<type>: quantising itself
#define RLXQ_MX_DEC(NAME, NT, MT, FUSED, XBF, WAVES)                                                      \
  extern "C" __global__ __launch_bounds__(64 * WAVES) void rlxq_mx_dec_##NAME(rlxq_mx_gemm_args a) {      \
    rlxq::mx_dec_body<NT, MT, FUSED, XBF>(a);                                                      \
  }
RLXQ_MX_DEC(n1m1, 1, 1, false, false, 16)
RLXQ_MX_DEC(n2m1, 2, 1, false, false, 8)
RLXQ_MX_DEC(n1m2, 1, 2, false, false, 16)
RLXQ_MX_DEC(n2m2, 2, 2, false, false, 8)
RLXQ_MX_DEC(n1_fbf16, 1, 1, true, true, 16)
RLXQ_MX_DEC(n2_fbf16, 2, 1, true, true, 8)
RLXQ_MX_DEC(n1_ff32, 1, 1, true, false, 16)
RLXQ_MX_DEC(n2_ff32, 2, 1, true, false, 8)
