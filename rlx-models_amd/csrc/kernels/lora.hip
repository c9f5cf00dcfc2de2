// Low-rank adapters of many requests beside a shared projection:
//   y[i, n] = base[i, n] + s[e] sum_{r < rank[e]} B[e, n, r] v[i, g(n), r],
//   v[i, g, r] = sum_k A[e, g R + r, k] x[i, k],   e = ids[i],
// g(n) the segment of column n.
//
// Rows of one adapter are taken together, in tiles: of up to RLXQ_LORA_FEW rows
// every workgroup finds its tile of 16 among the ids itself (a launch less), for
// more a launch of one workgroup sorts the rows and cuts them into tiles of 32.
// Two launches then: v (K over the waves of a workgroup and, where the
// workgroups would be few, over workgroups), then y.  Both put the adapter's rows
// on the long side of a 16x16 MFMA tile and the activation rows on the other, so
// the results of one activation row lie on one lane: v leaves as 16-byte pieces,
// y's columns are dealt to the tiles so that a lane holds 16 neighbouring ones.
//
// Types: the bf16 MFMA, f32 x and A as three bf16 terms each (all of their bits).
// v stays f32; against bf16 B it takes part as three bf16 terms, all of its bits
// (base may cancel what two would round).  Sums are f32, y is rounded once.
//
// What bounds it: many adapters at few rows, their bytes (64 rows of 48 adapters of
// rank 64, 4096 -> 24576: v 13.4 us for 50 MB, y 41.9 for 157, 3.7 TB/s); one
// adapter at one row, the two launches (4.0 and 7.0 us); prompts, base and y (4096
// rows of 8 adapters, 4096 -> 24576: sort 8 us, v 31, y 138 for 458 MB, 3.3 TB/s; 134
// with two terms of v).
// Tried on y of the last: tiles of 16, 64 and 128 rows (217, 172 and 193 us of the call
// against 173; 777 f32 rows of rank 128, 64 rows 41.8, 32 35.9), B's sharers on one XCD
// (145 us against 136: fewer columns at a time reach fewer memory channels), B's
// next rows not ahead of their use and accesses past the caches (within 3%).
#include "common.hip.h"
#include "lora_args.h"

namespace rlxq {

typedef float lr_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 lr_bf8 __attribute__((ext_vector_type(8)));

// Rank of adapter e: what lies past it in A and B is never multiplied.
RLXQ_DEV int lr_rank(const rlxq_lora_args& a, int e) {
  if (!a.ranks) return a.R;
  const int r = a.ranks[e];
  return r < 0 ? 0 : (r > a.R ? a.R : r);
}

// Eight neighbouring elements: as loaded (bf16), or as floats.
template <bool BF>
struct LrFrag {
  uint4 q[BF ? 1 : 2];
};
template <bool BF>
RLXQ_DEV LrFrag<BF> lr_zero() {
  LrFrag<BF> f;
  f.q[0] = make_uint4(0, 0, 0, 0);
  if constexpr (!BF) f.q[1] = f.q[0];
  return f;
}
// From element i of p.
template <bool BF>
RLXQ_DEV LrFrag<BF> lr_load(const void* p, int64_t i) {
  LrFrag<BF> f;
  const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + i * (BF ? 2 : 4));
  f.q[0] = s[0];
  if constexpr (!BF) f.q[1] = s[1];
  return f;
}
// The first n of the eight, the others zero.
template <bool BF>
RLXQ_DEV void lr_keep(LrFrag<BF>& f, int n) {
  uint32_t* w = reinterpret_cast<uint32_t*>(f.q);
#pragma unroll
  for (int j = 0; j < (BF ? 4 : 8); j++) {
    if (BF) w[j] = n >= 2 * j + 2 ? w[j] : (n == 2 * j + 1 ? w[j] & 0xffffu : 0u);
    else w[j] = n > j ? w[j] : 0u;
  }
}
// acc += the products of 32 k: lane l holds row (a) or column (b) l % 16, k 8 (l /
// 16) .. + 7 of them.  The f32 MFMA takes four k at a time; which four is the same
// on both sides.
template <bool BF>
RLXQ_DEV lr_f4 lr_mfma(const LrFrag<BF>& a, const LrFrag<BF>& b, lr_f4 acc) {
  if constexpr (BF) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lr_bf8, a.q[0]), __builtin_bit_cast(lr_bf8, b.q[0]), acc,
                                                   0, 0, 0);
  } else {
    const float* x = reinterpret_cast<const float*>(a.q);
    const float* y = reinterpret_cast<const float*>(b.q);
#pragma unroll
    for (int j = 0; j < 8; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], acc, 0, 0, 0);
    return acc;
  }
}

constexpr int kLrThreads = 256;
constexpr int kLrFrags = RLXQ_LORA_ROWS / 16;   // of a tile from the list

// Tile `index`: its rows into LDS, its adapter (-1: none) and number.  False:
// there is no such tile.  Every thread of the workgroup calls it.
template <bool LIST>
RLXQ_DEV bool lr_tile(const rlxq_lora_args& a, int index, int* rows, uint64_t* masks, int& e, int& count) {
  const int t = threadIdx.x;
  if constexpr (LIST) {
    const rlxq_lora_tile tile = a.tiles[index];
    e = tile.e, count = tile.count;
    if (count <= 0) return false;
    if (t < count) rows[t] = a.order[tile.start + t];
  } else {
    // row `index` leads a tile if the rows of its adapter ahead of it fill whole ones
    e = a.ids[index];
    e = e >= 0 && e < a.E ? e : -1;
    int mine = t < a.M ? a.ids[t] : -2;
    if (t < a.M) mine = mine >= 0 && mine < a.E ? mine : -1;
    const uint64_t m = __ballot(mine == e);
    if ((t & 63) == 0) masks[t >> 6] = m;
    __syncthreads();
    int lead = 0, ahead = 0, all = 0;
    for (int w = 0; w < kLrThreads / 64; w++) {
      const uint64_t q = masks[w];
      const int n = __popcll(q);
      lead += w < index >> 6 ? n : (w == index >> 6 ? __popcll(q & ((1ull << (index & 63)) - 1)) : 0);
      ahead += w < t >> 6 ? n : (w == t >> 6 ? __popcll(q & ((1ull << (t & 63)) - 1)) : 0);
      all += n;
    }
    if (lead & 15) return false;
    count = all - lead < 16 ? all - lead : 16;
    if (mine == e && ahead >= lead && ahead < lead + 16) rows[ahead - lead] = t;
  }
  __syncthreads();
  return true;
}

// Eight f32 as three bf16 terms that add up to them: a float's 24 significant bits
// cut into eights (cut, not rounded: no term can exceed the float).
RLXQ_DEV void lr_cut(const LrFrag<false>& f, uint4* term) {
  uint32_t v[8] = {f.q[0].x, f.q[0].y, f.q[0].z, f.q[0].w, f.q[1].x, f.q[1].y, f.q[1].z, f.q[1].w};
#pragma unroll
  for (int s = 0; s < 3; s++) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      w[j] = perm_b32(v[2 * j + 1], v[2 * j], 0x07060302u);   // the upper halves
#pragma unroll
      for (int i = 2 * j; i < 2 * j + 2; i++)
        v[i] = __float_as_uint(__uint_as_float(v[i]) - __uint_as_float(v[i] & 0xffff0000u));
    }
    term[s] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// The bf16 terms of a fragment: itself, or three.
template <bool BF>
struct LrTerms {
  uint4 t[BF ? 1 : 3];
};
template <bool BF>
RLXQ_DEV LrTerms<BF> lr_terms(const LrFrag<BF>& f) {
  LrTerms<BF> r;
  if constexpr (BF) r.t[0] = f.q[0];
  else lr_cut(f, r.t);
  return r;
}
// acc += the products of 32 k, term by term (of the last ones, 2^-30 of the first
// at most, none).
template <bool AB, bool XB>
RLXQ_DEV lr_f4 lr_products(const LrTerms<AB>& a, const LrTerms<XB>& x, lr_f4 acc) {
#pragma unroll
  for (int i = 0; i < (AB ? 1 : 3); i++)
#pragma unroll
    for (int j = 0; j < (XB ? 1 : 3); j++)
      if (i + j < 4)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lr_bf8, a.t[i]), __builtin_bit_cast(lr_bf8, x.t[j]), acc,
                                                      0, 0, 0);
  return acc;
}

// v of 16 FR rows and 16 RT rows of A, one slice of K: the waves take a quarter
// of it each and join their sums in LDS.
template <bool XB, bool AB, bool LIST, int FR, int RT>
RLXQ_DEV void lr_shrink(const rlxq_lora_args& a) {
  __shared__ int rows[RLXQ_LORA_ROWS];
  __shared__ uint64_t masks[4];
  __shared__ lr_f4 part[4][RT * FR][64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  static_assert(FR == (LIST ? kLrFrags : 1), "a workgroup takes a whole tile");
  int e, count;
  if (!lr_tile<LIST>(a, blockIdx.x / (a.jblocks * a.splits), rows, masks, e, count) || e < 0) return;
  const int other = blockIdx.x % (a.jblocks * a.splits);
  const int split = other % a.splits, sr = a.S * a.R, j0 = other / a.splits * 16 * RT;
  const int rank = lr_rank(a, e), col = lane & 15, kk = 8 * (lane >> 4);
  int64_t xrow[FR], arow[RT];
  bool xon[FR], aon[RT];
#pragma unroll
  for (int f = 0; f < FR; f++) {
    xon[f] = 16 * f + col < count;
    xrow[f] = xon[f] ? (int64_t)rows[16 * f + col] * a.K : 0;
  }
#pragma unroll
  for (int j = 0; j < RT; j++) {
    const int row = j0 + 16 * j + col;
    aon[j] = row < sr && row % a.R < rank;
    arow[j] = ((int64_t)e * sr + (aon[j] ? row : 0)) * a.K;
  }
  const int64_t k0 = (int64_t)split * a.kslice, k_end = k0 + a.kslice < a.K ? k0 + a.kslice : a.K;
  const int64_t quarter = (a.kslice / 4 + 31) / 32 * 32;
  const int64_t w0 = k0 + wave * quarter, w1 = w0 + quarter < k_end ? w0 + quarter : k_end;
  lr_f4 acc[RT][FR];
#pragma unroll
  for (int j = 0; j < RT; j++)
#pragma unroll
    for (int f = 0; f < FR; f++) acc[j][f] = (lr_f4){0.f, 0.f, 0.f, 0.f};
  constexpr int U = FR * RT == 1 ? 4 : (XB && AB ? 2 : 1);   // steps of 32 whose loads are on their way together
  LrFrag<XB> xf[U][FR];
  LrFrag<AB> af[U][RT];
  auto fetch = [&](int64_t k) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int64_t at = k + 32 * u + kk;
      const bool in = at < w1;   // (K is whole eights)
#pragma unroll
      for (int f = 0; f < FR; f++) xf[u][f] = in && xon[f] ? lr_load<XB>(a.x, xrow[f] + at) : lr_zero<XB>();
#pragma unroll
      for (int j = 0; j < RT; j++) af[u][j] = in && aon[j] ? lr_load<AB>(a.a, arow[j] + at) : lr_zero<AB>();
    }
  };
  for (int64_t k = w0; k < w1; k += 32 * U) {
    fetch(k);
#pragma unroll
    for (int u = 0; u < U; u++) {
      LrTerms<XB> xt[FR];
#pragma unroll
      for (int f = 0; f < FR; f++) xt[f] = lr_terms<XB>(xf[u][f]);
#pragma unroll
      for (int j = 0; j < RT; j++) {
        const LrTerms<AB> at = lr_terms<AB>(af[u][j]);
#pragma unroll
        for (int f = 0; f < FR; f++) acc[j][f] = lr_products<AB, XB>(at, xt[f], acc[j][f]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < RT; j++)
#pragma unroll
    for (int f = 0; f < FR; f++) part[wave][j * FR + f][lane] = acc[j][f];
  __syncthreads();
  // (lane: row 16 f + lane % 16 of the tile, rows 16 j + 4 (lane / 16) .. + 3 of A)
  for (int i = wave; i < RT * FR; i += 4) {
    const int row = 16 * (i % FR) + col, j = j0 + 16 * (i / FR) + 4 * (lane >> 4);
    if (row >= count || j >= sr) continue;
    const lr_f4 s = (part[0][i][lane] + part[1][i][lane]) + (part[2][i][lane] + part[3][i][lane]);
    *reinterpret_cast<lr_f4*>(a.v + ((int64_t)split * a.M + rows[row]) * sr + j) = s;
  }
}

// The column that row p of tile q of a wave's 64 columns stands for: chosen so that
// a lane's results (rows 4 g .. 4 g + 3 of every tile, g = lane / 16) make 16-byte
// pieces, neighbouring ones in neighbouring g.  Piece u of a lane starts at column
// lr_piece and is tile u (f32), or tiles 2 u and 2 u + 1 (bf16).
template <bool YB>
RLXQ_DEV int lr_column(int q, int p) {
  return YB ? 32 * (q >> 1) + 8 * (p >> 2) + 4 * (q & 1) + (p & 3) : 16 * q + p;
}
template <bool YB>
RLXQ_DEV int lr_piece(int u, int g) {
  return YB ? 32 * u + 8 * g : 16 * u + 4 * g;
}

// y of a tile's rows and a.cols columns of one segment, ranks up to 32 STEPS.  A
// wave takes 64 columns at a time, their rows of B in registers (the next ones asked
// for where two sets fit), and goes through the tile's rows 16 at a time against
// them.  v lies in LDS as the MFMA takes it, made once for the workgroup while the
// first of B is on its way.  base is asked for in the step that adds it, after B's
// next rows, and the build waits for both ahead of the step's first MFMA.
template <bool BB, bool YB, bool LIST, int STEPS>
RLXQ_DEV void lr_expand(const rlxq_lora_args& a) {
  constexpr int FR = LIST ? kLrFrags : 1;
  constexpr int NT = BB ? 3 : 2;   // 16-byte pieces of v a lane and 32 k (f32: the eight floats)
  constexpr bool AHEAD = STEPS <= 2;
  constexpr int P = YB ? 2 : 4, ES = YB ? 2 : 4;   // pieces of a lane's 16 columns
  extern __shared__ uint4 lds[];              // [steps][FR][NT][64]
  __shared__ int rows[RLXQ_LORA_ROWS];
  __shared__ uint64_t masks[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int cb = blockIdx.x % a.cblocks;
  int e, count;
  if (!lr_tile<LIST>(a, blockIdx.x / a.cblocks, rows, masks, e, count)) return;
  int seg = 0;
  while (seg + 1 < a.S && cb >= a.cfirst[seg + 1]) seg++;
  const int64_t c0 = (seg ? a.ends[seg - 1] : 0) + (int64_t)(cb - a.cfirst[seg]) * a.cols;
  const int64_t c1 = c0 + a.cols < a.ends[seg] ? c0 + a.cols : a.ends[seg];
  if (e < 0) {   // base's bits
    if (!a.copy) return;
    const int per = a.vec ? 16 / ES : 1, n = (int)(c1 - c0) / per;
    for (int i = t; i < count * n; i += kLrThreads) {
      const int64_t o = (int64_t)rows[i / n] * a.N + c0 + (int64_t)(i % n) * per;
      if (a.vec)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.y) + o * ES) =
            a.base ? *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.base) + o * ES) : make_uint4(0, 0, 0, 0);
      else if (YB)
        reinterpret_cast<uint16_t*>(a.y)[o] = a.base ? reinterpret_cast<const uint16_t*>(a.base)[o] : 0;
      else
        reinterpret_cast<uint32_t*>(a.y)[o] = a.base ? reinterpret_cast<const uint32_t*>(a.base)[o] : 0;
    }
    return;
  }
  const int rank = lr_rank(a, e), sr = a.S * a.R, col = lane & 15, g = lane >> 4, kk = 8 * g;
  LrFrag<BB> bf[STEPS][4], bn[AHEAD ? STEPS : 1][4];
  auto fetch = [&](LrFrag<BB>(&dst)[STEPS][4], int64_t c) {
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int64_t n = c + lr_column<YB>(q, col);
      const bool on = n < c1;
      const int64_t row = ((int64_t)e * a.N + (on ? n : c0)) * a.R;
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        const int r = 32 * s + kk;
        dst[s][q] = on && r < rank ? lr_load<BB>(a.b, row + r) : lr_zero<BB>();
      }
    }
  };
  fetch(bf, c0 + 64 * wave);
  int64_t yrow[FR];
  bool on[FR];
#pragma unroll
  for (int f = 0; f < FR; f++) {
    on[f] = 16 * f + col < count;
    yrow[f] = on[f] ? (int64_t)rows[16 * f + col] * a.N : 0;
  }
  const float scale = a.scales ? a.scales[e] : 1.0f;
  const int steps = (rank + 31) / 32, frags = (count + 15) / 16;
  for (int i = t; i < steps * frags * 64; i += kLrThreads) {
    const int l = i & 63, f = (i >> 6) % frags, s = (i >> 6) / frags, r = 32 * s + 8 * (l >> 4), row = 16 * f + (l & 15);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = 0.f;
    if (row < count && r < rank) {
      const float* p = a.v + (int64_t)rows[row] * sr + seg * a.R + r;
      const int64_t step = a.M * sr;
      // (slices in order; past the last: the last, not added.  The build has a slice's
      // loads behind the one before it: as many round trips as slices)
      float4 lo[RLXQ_LORA_SPLITS], hi[RLXQ_LORA_SPLITS];
#pragma unroll
      for (int q = 0; q < RLXQ_LORA_SPLITS; q++) {
        const float* at = p + (q < a.splits ? q : a.splits - 1) * step;
        lo[q] = reinterpret_cast<const float4*>(at)[0], hi[q] = reinterpret_cast<const float4*>(at)[1];
      }
#pragma unroll
      for (int q = 0; q < RLXQ_LORA_SPLITS; q++) {
        if (q >= a.splits) break;
        v[0] += lo[q].x, v[1] += lo[q].y, v[2] += lo[q].z, v[3] += lo[q].w;
        v[4] += hi[q].x, v[5] += hi[q].y, v[6] += hi[q].z, v[7] += hi[q].w;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = r + j < rank ? v[j] * scale : 0.f;
    }
    uint4* d = lds + (s * FR + f) * NT * 64 + l;
    LrFrag<false> whole;
    whole.q[0] = __builtin_bit_cast(uint4, make_float4(v[0], v[1], v[2], v[3]));
    whole.q[1] = __builtin_bit_cast(uint4, make_float4(v[4], v[5], v[6], v[7]));
    if constexpr (BB) {
      uint4 term[3];
      lr_cut(whole, term);
#pragma unroll
      for (int q = 0; q < NT; q++) d[q * 64] = term[q];
    } else {
      d[0] = whole.q[0];
      d[64] = whole.q[1];
    }
  }
  __syncthreads();
  constexpr int kStep = 64 * (kLrThreads / 64);
  for (int64_t c = c0 + 64 * wave; c < c1; c += kStep) {
    if constexpr (!AHEAD) {
      if (c != c0 + 64 * wave) fetch(bf, c);
    } else if (c + kStep < c1) {
      fetch(bn, c + kStep);
    }
    uint4 bq[FR][P];
    bool whole[P];
#pragma unroll
    for (int u = 0; u < P; u++) {
      whole[u] = a.vec && c + lr_piece<YB>(u, g) < c1;   // (with vec, segments are whole pieces)
#pragma unroll
      for (int f = 0; f < FR; f++) {
        bq[f][u] = make_uint4(0, 0, 0, 0);
        if (a.base && whole[u] && on[f])
          bq[f][u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.base) +
                                                     (yrow[f] + c + lr_piece<YB>(u, g)) * ES);
      }
    }
    if (rank & 7) {   // what lies past the rank in its eight
#pragma unroll
      for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int q = 0; q < 4; q++)
          if (rank - 32 * s - kk < 8) lr_keep<BB>(bf[s][q], rank - 32 * s - kk);
    }
#pragma unroll
    for (int f = 0; f < FR; f++) {
      if (f >= frags) break;
      lr_f4 acc[4];
#pragma unroll
      for (int q = 0; q < 4; q++) acc[q] = (lr_f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        if (s >= steps) break;
        const uint4* d = lds + (s * FR + f) * NT * 64 + lane;
        if constexpr (BB) {
#pragma unroll
          for (int w = 0; w < NT; w++) {
            LrFrag<BB> vf;
            vf.q[0] = d[w * 64];
#pragma unroll
            for (int q = 0; q < 4; q++) acc[q] = lr_mfma<BB>(bf[s][q], vf, acc[q]);
          }
        } else {
          LrFrag<BB> vf;
          vf.q[0] = d[0];
          vf.q[1] = d[64];
#pragma unroll
          for (int q = 0; q < 4; q++) acc[q] = lr_mfma<BB>(bf[s][q], vf, acc[q]);
        }
      }
      if (!on[f]) continue;
#pragma unroll
      for (int u = 0; u < P; u++) {
        const int64_t n = c + lr_piece<YB>(u, g);
        if (whole[u]) {
          uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.y) + (yrow[f] + n) * ES);
          if constexpr (YB) {
            const uint32_t w[4] = {bq[f][u].x, bq[f][u].y, bq[f][u].z, bq[f][u].w};
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
              o[j] = pack_bf16x2(__uint_as_float(w[j] << 16) + acc[2 * u + (j >> 1)][2 * j & 3],
                                 __uint_as_float(w[j] & 0xffff0000u) + acc[2 * u + (j >> 1)][(2 * j & 3) + 1]);
            *d = make_uint4(o[0], o[1], o[2], o[3]);
          } else {
            const float4 w = __builtin_bit_cast(float4, bq[f][u]);
            *d = __builtin_bit_cast(uint4, make_float4(w.x + acc[u][0], w.y + acc[u][1], w.z + acc[u][2], w.w + acc[u][3]));
          }
          continue;
        }
#pragma unroll
        for (int j = 0; j < 16 / P; j++) {
          if (n + j >= c1) break;
          const int64_t o = yrow[f] + n + j;
          if constexpr (YB) {
            const float w = a.base ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.base)[o]) : 0.f;
            reinterpret_cast<uint16_t*>(a.y)[o] = (uint16_t)f32_to_bf16_bits(w + acc[2 * u + (j >> 2)][j & 3]);
          } else {
            const float w = a.base ? reinterpret_cast<const float*>(a.base)[o] : 0.f;
            reinterpret_cast<float*>(a.y)[o] = w + acc[u][j & 3];
          }
        }
      }
    }
    if constexpr (AHEAD) {
#pragma unroll
      for (int s = 0; s < STEPS; s++)
#pragma unroll
        for (int q = 0; q < 4; q++) bf[s][q] = bn[s][q];
    }
  }
}

}  // namespace rlxq

using namespace rlxq;

namespace rlxq {
// count[e]++ by every active lane, and the number it had: prompts are runs of
// one adapter, so the first lanes' adapters are counted a wave at a time.
RLXQ_DEV int lr_take(int* count, int e) {
  for (int turn = 0; turn < 2; turn++) {
    const int first = __builtin_amdgcn_readfirstlane(e);
    const uint64_t same = __ballot(e == first);
    if (e == first) {
      const int at = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
      int base = 0;
      if (at == 0) base = atomicAdd(&count[first], __popcll(same));
      return __builtin_amdgcn_readfirstlane(base) + at;
    }
  }
  return atomicAdd(&count[e], 1);
}
}  // namespace rlxq

// The rows by adapter (those without one last), cut into tiles of up to 32: one
// workgroup; LDS holds a counter for each adapter.  The order of an adapter's
// rows is that of the counters' atomics; no result depends on it.
extern "C" __global__ __launch_bounds__(1024) void rlxq_lora_sort(rlxq_lora_args a) {
  extern __shared__ int count[];   // [E + 1]: rows, then where the next one goes
  __shared__ int red[2][16];
  constexpr int kRows = RLXQ_LORA_ROWS;
  const int t = threadIdx.x, n = a.E + 1;
  for (int e = t; e < n; e += 1024) count[e] = 0;
  __syncthreads();
  for (int64_t i = t; i < a.M; i += 1024) {
    const int e = a.ids[i];
    (void)lr_take(count, e >= 0 && e < a.E ? e : a.E);
  }
  __syncthreads();
  // a run of adapters a thread: rows and tiles ahead of it
  const int per = (n + 1023) / 1024, lo = t * per, hi = lo + per < n ? lo + per : n;
  int rows = 0, tiles = 0;
  for (int e = lo; e < hi; e++) rows += count[e], tiles += (count[e] + kRows - 1) / kRows;
  int ri = rows, ti = tiles;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int ro = __shfl_up(ri, off, 64), to = __shfl_up(ti, off, 64);
    if ((t & 63) >= off) ri += ro, ti += to;
  }
  if ((t & 63) == 63) red[0][t >> 6] = ri, red[1][t >> 6] = ti;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < 16; w++) {
    if (w < t >> 6) ri += red[0][w], ti += red[1][w];
    all += red[1][w];
  }
  int start = ri - rows, tile = ti - tiles;
  for (int e = lo; e < hi; e++) {
    const int c = count[e];
    for (int at = 0; at < c; at += kRows) a.tiles[tile++] = {e < a.E ? e : -1, start + at, c - at < kRows ? c - at : kRows, 0};
    count[e] = start;
    start += c;
  }
  for (int i = all + t; i < a.max_tiles; i += 1024) a.tiles[i] = {-1, 0, 0, 0};
  __syncthreads();
  for (int64_t i = t; i < a.M; i += 1024) {
    const int e = a.ids[i];
    a.order[lr_take(count, e >= 0 && e < a.E ? e : a.E)] = (int)i;
  }
}

// _few: tiles of 16 rows that every workgroup finds; _many: of 32 from the list
#define RLXQ_LORA_SHRINK(X, A, xn, an)                                                                                  \
  extern "C" __global__ __launch_bounds__(256) void rlxq_lora_shrink_##xn##_##an##_few(rlxq_lora_args a) {                \
    lr_shrink<X, A, false, 1, 1>(a);                                                                                    \
  }                                                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void rlxq_lora_shrink_##xn##_##an##_many(rlxq_lora_args a) {               \
    lr_shrink<X, A, true, kLrFrags, 4>(a);                                                                                     \
  }
RLXQ_LORA_SHRINK(true, true, bf16, bf16)
RLXQ_LORA_SHRINK(true, false, bf16, f32)
RLXQ_LORA_SHRINK(false, true, f32, bf16)
RLXQ_LORA_SHRINK(false, false, f32, f32)
#define RLXQ_LORA_EXPAND1(B, Y, bn, yn, st)                                                                             \
  extern "C" __global__ __launch_bounds__(256) void rlxq_lora_expand_##bn##_##yn##_few_s##st(rlxq_lora_args a) {          \
    lr_expand<B, Y, false, st>(a);                                                                                      \
  }                                                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void rlxq_lora_expand_##bn##_##yn##_many_s##st(rlxq_lora_args a) {         \
    lr_expand<B, Y, true, st>(a);                                                                                       \
  }
#define RLXQ_LORA_EXPAND(B, Y, bn, yn) \
  RLXQ_LORA_EXPAND1(B, Y, bn, yn, 1) RLXQ_LORA_EXPAND1(B, Y, bn, yn, 2) RLXQ_LORA_EXPAND1(B, Y, bn, yn, 4) RLXQ_LORA_EXPAND1(B, Y, bn, yn, 8)
RLXQ_LORA_EXPAND(true, true, bf16, bf16)
RLXQ_LORA_EXPAND(true, false, bf16, f32)
RLXQ_LORA_EXPAND(false, true, f32, bf16)
RLXQ_LORA_EXPAND(false, false, f32, f32)
