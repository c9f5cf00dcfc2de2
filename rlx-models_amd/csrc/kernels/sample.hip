// A token per row of logits l, from a given random number u, under temperature
// T, top-k, top-p and min-p.
//
// w_j = exp((l_j - max l) / T).  In the order of falling logits, equal ones by
// rising index: K the first top_k; P the shortest prefix of K whose mass is at
// least top_p times K's, never empty; M those with w >= min_p.  All three are
// prefixes of that order, so what is kept is everything at or ahead of one
// element, the border (key, index).  The token is the lowest index whose sum of
// kept w over it and all lower indices exceeds u times the whole kept sum.
//
// Whether a border or a sum falls on one side or the other of a number decides
// whole tokens: weights are f64, and sums are f64 in a fixed order, or
// fixed-point integers where they go through atomics (the same in any order).
#include "common.hip.h"
#include "sample_args.h"

namespace rlxq {

// exp(x) for x <= 0: 2^n 2^f with n the integer nearest x / ln 2; 2^f by its
// Taylor series about 0, whose first term left out is below (ln 2 / 2)^13 / 13! =
// 2e-16.  exp(0) is exactly 1.
RLXQ_DEV double exp_neg(double x) {
  if (x < -700.0) return 0.0;
  const double t = x * 1.4426950408889634, n = __builtin_rint(t), f = (t - n) * 0.6931471805599453;
  double p = 1.0 / 479001600;
  p = __builtin_fma(p, f, 1.0 / 39916800);
  p = __builtin_fma(p, f, 1.0 / 3628800);
  p = __builtin_fma(p, f, 1.0 / 362880);
  p = __builtin_fma(p, f, 1.0 / 40320);
  p = __builtin_fma(p, f, 1.0 / 5040);
  p = __builtin_fma(p, f, 1.0 / 720);
  p = __builtin_fma(p, f, 1.0 / 120);
  p = __builtin_fma(p, f, 1.0 / 24);
  p = __builtin_fma(p, f, 1.0 / 6);
  p = __builtin_fma(p, f, 0.5);
  p = __builtin_fma(p, f, 1.0);
  p = __builtin_fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

// Order-preserving integer of a float (-0 as +0); 0 for -inf, which no finite
// value has: a masked token.
RLXQ_DEV uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  if (b == 0xff800000u) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
RLXQ_DEV float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr int kSmpThreads = 512;

// What a row asks for, and its largest logit.
struct SmpRow {
  double inv_t, min_w;
  float top;             // the largest logit
  float p, u;
  int k;                 // 0: off
};

RLXQ_DEV float smp_ld(const rlxq_sample_args& a, int64_t row, int i) {
  return a.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.logits)[row * a.V + i])
                : reinterpret_cast<const float*>(a.logits)[row * a.V + i];
}
RLXQ_DEV double smp_w(const SmpRow& r, float v) { return exp_neg(((double)v - (double)r.top) * r.inv_t); }

// The border as one number: key above, falling index below.  An element is
// kept if its own is not smaller.
RLXQ_DEV uint64_t smp_comp(uint32_t key, uint32_t idx) { return (uint64_t)key << 32 | (uint32_t)~idx; }

// Inclusive prefix sums over the workgroup's threads in thread order, and the total.
template <class T>
RLXQ_DEV T smp_scan(T v, T* red, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T o = __shfl_up(v, off, 64);
    if (lane >= off) v += o;
  }
  __syncthreads();
  if (lane == 63) red[wave] = v;
  __syncthreads();
  T before = 0, all = 0;
  for (int w = 0; w < kSmpThreads / 64; w++) {
    if (w < wave) before += red[w];
    all += red[w];
  }
  *total = all;
  return before + v;
}

struct SmpShared {
  uint64_t mass[2048];
  uint32_t count[2048];
  uint64_t r64[16];
  double rd[16];
  uint32_t r32[16];
  uint32_t pick, pick_count;
  uint64_t pick_mass;
  int found, last;
};

// Border among the elements at or ahead of `within`: the one of rank `k` (BY =
// 0, from 1), or the first at which the mass reaches `target` (BY = 1, in fixed
// point).  Three passes over the row narrow its key digit by digit; equal keys
// are told apart by their index.
template <int BY>
RLXQ_DEV uint64_t smp_radix(const rlxq_sample_args& a, const SmpRow& r, int64_t row, uint64_t within, double one,
                            uint64_t need, SmpShared& s, uint64_t* above_mass) {
  const int t = threadIdx.x;
  uint32_t prefix = 0;
  uint64_t above = 0, mass_above = 0;   // ranks or mass ahead of the digit's bin
  int shift = 32;
  for (int bits : {11, 11, 10}) {
    shift -= bits;
    const int bins = 1 << bits;
    for (int i = t; i < bins; i += kSmpThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    for (int i = t; i < a.V; i += kSmpThreads) {
      const float v = smp_ld(a, row, i);
      const uint32_t key = key_of(v);
      if (!key || smp_comp(key, i) < within) continue;
      if (shift + bits < 32 && (key >> (shift + bits)) != (prefix >> (shift + bits))) continue;
      const uint32_t bin = (key >> shift) & (bins - 1);
      atomicAdd(&s.count[bin], 1u);
      atomicAdd((unsigned long long*)&s.mass[bin], (unsigned long long)(smp_w(r, v) * one + 0.5));
    }
    __syncthreads();
    // bins from the top: thread t holds kPer of them, b0 the highest
    constexpr int kPer = 2048 / kSmpThreads;
    const int b0 = bins - 1 - kPer * t;
    uint64_t m = 0, mt;
    uint32_t c = 0, ct;
    for (int j = 0; j < kPer; j++)
      if (b0 - j >= 0) m += s.mass[b0 - j], c += s.count[b0 - j];
    uint64_t mb = mass_above + smp_scan<uint64_t>(m, s.r64, &mt) - m;
    uint64_t cb = above + smp_scan<uint32_t>(c, s.r32, &ct) - c;
    const uint64_t all_c = above + ct;
    for (int j = 0; j < kPer && b0 - j >= 0; j++) {
      const uint64_t mj = s.mass[b0 - j], cj = s.count[b0 - j];
      if (!cj) continue;
      // (the last bin with anything in it ends the search where rounding left the
      // target above the whole mass)
      const bool here = BY == 0 ? cb < need && cb + cj >= need
                                : (mb < need || cb == 0) && (mb + mj >= need || cb + cj == all_c);
      if (here) s.pick = b0 - j, s.pick_mass = mb, s.pick_count = (uint32_t)cb;
      mb += mj, cb += cj;
    }
    __syncthreads();
    prefix |= s.pick << shift;
    mass_above = s.pick_mass;
    above = s.pick_count;
    __syncthreads();
  }
  // equal keys: how many of them, then the index of the last
  const uint64_t each = (uint64_t)(smp_w(r, of_key(prefix)) * one + 0.5);
  uint64_t ties;
  if (BY == 0) ties = need - above;
  else ties = need <= mass_above || !each ? 1 : (need - mass_above + each - 1) / each;
  if (ties < 1) ties = 1;
  const int per = (a.V + kSmpThreads - 1) / kSmpThreads, lo = t * per, hi = lo + per < a.V ? lo + per : a.V;
  uint32_t mine = 0, last = 0;
  for (int i = lo; i < hi; i++) {
    const uint32_t key = key_of(smp_ld(a, row, i));
    if (key == prefix && smp_comp(key, i) >= within) mine++, last = i;
  }
  uint32_t all;
  const uint32_t incl = smp_scan<uint32_t>(mine, s.r32, &all);
  if (ties > all) ties = all;
  if (mine && incl - mine < ties && incl >= ties) {
    uint32_t n = incl - mine;
    for (int i = lo; i < hi && n < ties; i++) {
      const uint32_t key = key_of(smp_ld(a, row, i));
      if (key == prefix && smp_comp(key, i) >= within) n++, last = i;
    }
    s.pick = last;
  }
  __syncthreads();
  const uint32_t idx = s.pick;
  __syncthreads();
  *above_mass = mass_above + ties * each;
  return smp_comp(prefix, idx);
}

// Whether a row with at least one token that is not masked keeps v at or ahead
// of its border.
RLXQ_DEV double smp_kept(const SmpRow& r, uint64_t border, float v, int i) {
  const uint32_t key = key_of(v);
  if (!key || smp_comp(key, i) < border) return 0.0;
  const double w = smp_w(r, v);
  return w >= r.min_w ? w : 0.0;
}

// The token, from what the threads hold in order: m the kept weights of a
// thread's elements, last the last of them (or -1); `before` the kept mass ahead
// of thread 0's, `total` the row's (negative: what the threads hold).  at(c,
// target): the thread's first element whose sum from c on exceeds the target.
template <class F>
RLXQ_DEV void smp_choose(const rlxq_sample_args& a, const SmpRow& r, int64_t row, double m, int last, double before,
                         double total, SmpShared& s, F&& at) {
  double all;
  const double incl = before + smp_scan<double>(m, s.rd, &all);
  if (total < 0.0) total = all;
  const double target = (double)r.u * total;
  if (threadIdx.x == 0) s.found = 0x7fffffff, s.last = -1;
  __syncthreads();
  // (no sum above the target: rounding, or u = 1: the last that is kept)
  if (last >= 0) atomicMax(&s.last, last);
  if (m > 0.0 && incl > target) atomicMin(&s.found, at(incl - m, target));
  __syncthreads();
  if (threadIdx.x == 0) {
    const int tok = s.found == 0x7fffffff ? s.last : s.found;   // (-1: nothing kept, which no row comes to)
    a.tokens[row] = tok;
    if (a.probs) a.probs[row] = tok < 0 ? __builtin_nanf("") : (float)(smp_w(r, smp_ld(a, row, tok)) / total);
  }
}

// The workgroup's best and bad.
RLXQ_DEV void smp_best(uint64_t& best, uint32_t& bad, uint64_t* r64, uint32_t* r32) {
  const int t = threadIdx.x, waves = blockDim.x >> 6;
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    const uint64_t o = __shfl_xor(best, off, 64);
    best = o > best ? o : best;
    bad |= __shfl_xor(bad, off, 64);
  }
  if ((t & 63) == 0) r64[t >> 6] = best, r32[t >> 6] = bad;
  __syncthreads();
  best = 0;
  for (int w = 0; w < waves; w++) {
    best = r64[w] > best ? r64[w] : best;
    bad |= r32[w];
  }
  __syncthreads();
}

// The row's settings.  False: its token is already written (no distribution,
// or the likeliest was asked for).
RLXQ_DEV bool smp_row(const rlxq_sample_args& a, int64_t row, uint64_t best, uint32_t bad, SmpRow& r) {
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  r.u = a.u[row];
  const bool none = bad || !best || T != T || r.u != r.u;
  if (none || !(T > 0.0f)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = none ? -1 : (int32_t)~(uint32_t)best;
      if (a.probs) a.probs[row] = none ? __builtin_nanf("") : 1.0f;
    }
    return false;
  }
  r.top = of_key((uint32_t)(best >> 32));
  r.inv_t = 1.0 / (double)T;
  r.k = a.top_k ? a.top_k[row] : 0;
  r.p = a.top_p ? a.top_p[row] : 1.0f;
  const float q = a.min_p ? a.min_p[row] : 0.0f;
  r.min_w = q > 0.0f ? (q < 1.0f ? (double)q : 1.0) : 0.0;
  return true;
}

// A row by itself: the row read again for every digit of a border.
RLXQ_DEV void smp_scan_row(const rlxq_sample_args& a, const SmpRow& r, int64_t row, SmpShared& s) {
  const int t = threadIdx.x;
  // fixed point: the whole row's mass below 2^62
  const int lg = 32 - __builtin_clz((uint32_t)a.V);
  const double one = (double)(1ull << (62 - lg));
  uint64_t border = 1, mass = 0;   // every element that is not masked
  if (r.k > 0 && r.k < a.V) {
    // (fewer than k that are not masked: all of them)
    uint32_t n = 0, all;
    for (int i = t; i < a.V; i += kSmpThreads) n += key_of(smp_ld(a, row, i)) != 0;
    (void)smp_scan<uint32_t>(n, s.r32, &all);
    __syncthreads();
    if ((uint32_t)r.k < all) border = smp_radix<0>(a, r, row, border, one, (uint64_t)r.k, s, &mass);
  }
  if (r.p < 1.0f) {
    uint64_t m = 0;
    for (int i = t; i < a.V; i += kSmpThreads) {
      const float v = smp_ld(a, row, i);
      const uint32_t key = key_of(v);
      if (key && smp_comp(key, i) >= border) m += (uint64_t)(smp_w(r, v) * one + 0.5);
    }
    (void)smp_scan<uint64_t>(m, s.r64, &mass);
    __syncthreads();
    const double want = r.p > 0.0f ? (double)r.p * (double)mass : 0.0;
    uint64_t need = (uint64_t)want;
    need += (double)need < want;
    border = smp_radix<1>(a, r, row, border, one, need, s, &mass);
  }
  // the kept mass in index order: every thread a run of the row
  const int per = (a.V + kSmpThreads - 1) / kSmpThreads, lo = t * per, hi = lo + per < a.V ? lo + per : a.V;
  double m = 0.0;
  int last = -1;
  for (int i = lo; i < hi; i++) {
    const double w = smp_kept(r, border, smp_ld(a, row, i), i);
    m += w;
    if (w > 0.0) last = i;
  }
  smp_choose(a, r, row, m, last, 0.0, -1.0, s, [&](double c, double target) {
    for (int i = lo; i < last; i++) {
      c += smp_kept(r, border, smp_ld(a, row, i), i);
      if (c > target) return i;
    }
    return last;
  });
}


// ---- two launches: chunk histograms, then a workgroup a row ----------------
//
// The first reads the logits once: each workgroup a chunk of a row, in
// registers, whose weights are taken relative to the chunk's own largest logit
// and summed in fixed point, whole and by bins of l / T.  The bins of all chunks
// lie on one grid, so the second launch adds them up (groups of 32 bins, then the
// 32 of one group), finds the bin that each border falls into, and reads again
// only the chunks that hold anything in those bins; what it finds there is
// listed and settles the borders.  More than the list holds (rows as flat as
// noise): smp_scan_row.

constexpr int kBins = RLXQ_SAMPLE_BINS, kGroups = RLXQ_SAMPLE_GROUPS, kGroup = kBins / kGroups;
constexpr int kHistThreads = RLXQ_SAMPLE_CHUNK / 16;
constexpr int kSmpList = 4096;
constexpr int kSmpChunks = RLXQ_SAMPLE_MAX_VOCAB / RLXQ_SAMPLE_CHUNK + 1;   // (a row may start inside 16 bytes)

// Bin number of v on the row's grid, a whole number that does not fall as v
// rises; the grid's multiple of a group at or above it; bins below one, the last
// one open (and everything in it where l / T has no finite number).
RLXQ_DEV float smp_bin_scale(float T) { return fminf(16.0f / T, 1e30f); }
RLXQ_DEV float smp_bin(float v, float scale) { return floorf(v * scale); }
RLXQ_DEV float smp_anchor(float bin) { return ceilf(bin * (1.0f / kGroup)) * kGroup; }
RLXQ_DEV int smp_below(float anchor, float bin) { return (int)fminf(anchor - bin, (float)(kBins - 1)); }

// The elements of one aligned 16-byte vector of a row: i0 is the index of the
// first, which may lie ahead of the row (its start need not be aligned), unless
// all of it is known to be inside.
template <int BF>
RLXQ_DEV void smp_ld16(const rlxq_sample_args& a, int64_t row, int i0, float* v, bool inside) {
  constexpr int N = BF ? 8 : 4;
  if (inside || (i0 >= 0 && i0 + N <= a.V)) {
    const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.logits) +
                                                    (row * a.V + i0) * (BF ? 2 : 4));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (BF) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      else v[j] = __uint_as_float(w[j]);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; j++) v[j] = i0 + j >= 0 && i0 + j < a.V ? smp_ld(a, row, i0 + j) : -__builtin_inff();
}
// COUNT vectors of a chunk, `step` apart from vector x on: whether the whole
// chunk lies in the row is the same for all threads, and then nothing branches.
template <int BF, int COUNT>
RLXQ_DEV void smp_ld_chunk(const rlxq_sample_args& a, int64_t row, int first, int x, int step, float* v) {
  constexpr int N = BF ? 8 : 4;
  if (first >= 0 && first + RLXQ_SAMPLE_CHUNK <= a.V) {
#pragma unroll
    for (int j = 0; j < COUNT; j++) smp_ld16<BF>(a, row, first + (x + j * step) * N, v + j * N, true);
  } else {
#pragma unroll
    for (int j = 0; j < COUNT; j++) smp_ld16<BF>(a, row, first + (x + j * step) * N, v + j * N, false);
  }
}
// Elements between the 16-byte boundary at or ahead of the row and the row.
template <int BF>
RLXQ_DEV int smp_lead(const rlxq_sample_args& a, int64_t row) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.logits) + (uintptr_t)(row * a.V) * (BF ? 2 : 4);
  return (int)((p & 15) / (BF ? 2 : 4));
}

template <int BF>
RLXQ_DEV void smp_hist(const rlxq_sample_args& a) {
  constexpr int N = BF ? 8 : 4, TH = kHistThreads;
  __shared__ unsigned long long mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double pow2[32];
  __shared__ uint64_t r64[TH / 64];
  __shared__ uint32_t r32[TH / 64];
  __shared__ float rf[TH / 64];
  __shared__ int at;
  const int64_t row = blockIdx.x / a.chunks;
  const int c = (int)(blockIdx.x - row * a.chunks), t = threadIdx.x;
  const int first = c * RLXQ_SAMPLE_CHUNK - smp_lead<BF>(a, row);
  float v[16];
  smp_ld_chunk<BF, 16 / N>(a, row, first, t, TH, v);
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.0f, q = a.min_p ? a.min_p[row] : 0.0f;
  const bool by_k = k > 0 && k < a.V, bins = by_k || p < 1.0f || q > 0.0f;
  for (int i = t; i < kBins; i += TH) mass[i] = 0, count[i] = 0;
  if (t < 32) pow2[t] = 2.0 * exp_neg((t - 32) * (0.6931471805599453 / 32));
  if (t == 0) at = 0x7fffffff;
  float top = -__builtin_inff();
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 16; j++) {
    top = fmaxf(top, v[j]);
    odd |= !(v[j] < __builtin_inff());
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  uint32_t bad = __ballot(odd) != 0;
  if ((t & 63) == 0) rf[t >> 6] = top, r32[t >> 6] = bad;
  __syncthreads();
  for (int w = 0; w < TH / 64; w++) top = fmaxf(top, rf[w]), bad |= r32[w];
  // the lowest index of the largest
  int mine = 0x7fffffff;
#pragma unroll
  for (int j = 15; j >= 0; j--)
    if (v[j] == top) mine = first + ((j / N) * TH + t) * N + j % N;
  if (mine != 0x7fffffff) atomicMin(&at, mine);
  __syncthreads();
  rlxq_sample_chunk* head = a.heads + row * a.chunks + c;
  uint64_t* masses = a.masses + (row * a.chunks + c) * kBins;
  uint16_t* counts = a.counts + (row * a.chunks + c) * kBins;
  const uint64_t best = key_of(top) ? smp_comp(key_of(top), at) : 0;
  if (!(T > 0.0f) || bad || !best) {   // (no weights; no bins are read but those of a chunk that is all masked)
    if (t == 0) head->best = best, head->mass = 0, head->bad = bad, head->count = 0;
    return;
  }
  const float scale = smp_bin_scale(T), anchor = smp_anchor(smp_bin(top, scale));
  // w 2^48 = 2^(n / 32 + 48) 2^(f / 32), n the integer nearest x = 32 (l - top) / (T
  // ln 2), f = x - n: a table by n mod 32, and the Taylor series of the second
  // about 0, whose first term left out is below (ln 2 / 64)^6 / 720 = 3e-15.  n is
  // read off the sum 1.5 2^52 + x.  What is 2^-70 of the top or less, masked
  // tokens among it, counts as that, which rounds to 0.
  constexpr double L = 0.6931471805599453 / 32, kRound = 0x1.8p52;
  const double top64 = (double)top, c32 = 32.0 / (0.6931471805599453 * (double)T);
  const double least = -48.0 * (double)T;
  uint64_t sum = 0;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    uint64_t w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double d = __builtin_fmax((double)v[8 * half + j] - top64, least);
      const double y = __builtin_fma(d, c32, kRound);
      const uint32_t n = (uint32_t)__double_as_longlong(y);
      const double f = __builtin_fma(d, c32, kRound - y);
      double e = __builtin_fma(f, L * L * L * L * L / 120, L * L * L * L / 24);
      e = __builtin_fma(e, f, L * L * L / 6);
      e = __builtin_fma(e, f, L * L / 2);
      e = __builtin_fma(e, f, L);
      e = __builtin_fma(e, f, 1.0);
      const uint64_t b = (uint64_t)__double_as_longlong(pow2[n & 31]);
      const uint32_t hi = (uint32_t)(b >> 32) + ((uint32_t)(((int32_t)n >> 5) + 48) << 20);
      // the integer it rounds to: 2^52 + it, whose low bits it is
      w[j] = (uint64_t)__double_as_longlong(__builtin_fma(e, __hiloint2double((int)hi, (int)(uint32_t)b), 0x1p52)) -
             0x4330000000000000ull;
      sum += w[j];
    }
    if (!(T < 1e36f)) {   // (nothing is that far below the top then: masked tokens by name)
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (v[8 * half + j] == -__builtin_inff()) sum -= w[j], w[j] = 0;
    }
    if (bins) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int d = smp_below(anchor, smp_bin(v[8 * half + j], scale));
        atomicAdd(&mass[d], (unsigned long long)w[j]);
        if (by_k && v[8 * half + j] > -__builtin_inff()) atomicAdd(&count[d], 1u);
      }
    }
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((t & 63) == 0) r64[t >> 6] = sum;
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < TH / 64; w++) sum += r64[w];
    head->best = best, head->mass = sum, head->bad = 0;
  }
  if (!bins) return;
  static_assert(kBins == 2 * TH && kGroup == 32, "a thread takes two bins, 16 threads a group");
  const uint64_t m0 = mass[2 * t], m1 = mass[2 * t + 1];
  const uint32_t n0 = count[2 * t], n1 = count[2 * t + 1];
  reinterpret_cast<ulonglong2*>(masses)[t] = make_ulonglong2(m0, m1);
  if (by_k) reinterpret_cast<uint32_t*>(counts)[t] = n0 | n1 << 16;
  uint64_t gm = m0 + m1;
  uint32_t gn = n0 + n1;
#pragma unroll
  for (int off = 8; off; off >>= 1) gm += __shfl_xor(gm, off, 64), gn += __shfl_xor(gn, off, 64);
  if ((t & 15) == 0) head->group_mass[t >> 4] = gm, head->group_count[t >> 4] = gn;
  if (!by_k) return;
  __syncthreads();
#pragma unroll
  for (int off = 32; off >= 16; off >>= 1) gn += __shfl_xor(gn, off, 64);
  if ((t & 63) == 0) r32[t >> 6] = gn;
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < TH / 64; w++) gn += r32[w];
    head->count = gn;
  }
}

struct SmpPick {
  double scale[kSmpChunks], kept[kSmpChunks];   // chunks: their weights' scale in the row; their kept mass
  unsigned long long add[kSmpChunks];           // kept weights of listed elements, in 2^-50
  int shift[kSmpChunks];                        // groups from the row's top to the chunk's
  uint32_t some[kSmpChunks];                    // which bins of the group that smp_fine took hold something
  uint16_t flagged[kSmpChunks];
  uint8_t flag[kSmpChunks];
  double part[16][32];
  uint32_t part_n[16][32];
  double gcum[kGroups], fcum[kGroup];           // mass down to a group of the row, a bin of one group
  uint32_t gcnt[kGroups], fcnt[kGroup];         // elements
  uint64_t list[kSmpList];
  uint64_t few[64], lo, hi;
  double few_w[64];
  uint32_t n, n_few, n_flag;
  int bin;
  double before, base;
  uint32_t base_n;
};

// The mass and number of elements down to each bin of the row's group j, and
// which chunks hold any of each.
RLXQ_DEV void smp_fine(const rlxq_sample_args& a, int64_t row, int j, bool by_k, double all, uint32_t all_n, SmpPick& g) {
  const int t = threadIdx.x, b = t & 31, slot = t >> 5, C = a.chunks;
  static_assert(kSmpThreads == 512, "32 bins of 16 chunks at a time");
  double m = 0.0;
  uint32_t n = 0;
  __syncthreads();
  for (int c0 = 0; c0 < C; c0 += 64) {   // (four loads on their way)
    uint64_t q[4];
    uint32_t qn[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int c = c0 + 16 * u + slot, jj = c < C ? j - g.shift[c] : -1;
      const int64_t at = (row * C + c) * kBins + jj * kGroup + b;
      q[u] = jj >= 0 ? a.masses[at] : 0;
      qn[u] = jj >= 0 && by_k ? a.counts[at] : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int c = c0 + 16 * u + slot;
      // (the open bin holds what no other says)
      const uint64_t any = __ballot(q[u] != 0 || qn[u] != 0 || (j == kGroups - 1 && b == kGroup - 1));
      if (c < C) {
        if (b == 0) g.some[c] = (uint32_t)(any >> (t & 32));
        m += (double)q[u] * g.scale[c];
        n += qn[u];
      }
    }
  }
  g.part[slot][b] = m;
  g.part_n[slot][b] = n;
  __syncthreads();
  if (t < 32) {
    m = 0.0, n = 0;
    for (int s = 0; s < 16; s++) m += g.part[s][t], n += g.part_n[s][t];
    m *= 0x1p-48;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double om = __shfl_up(m, off, 32);
      const uint32_t on = __shfl_up(n, off, 32);
      if (t >= off) m += om, n += on;
    }
    if (j > 0) m += g.gcum[j - 1], n += g.gcnt[j - 1];
    if (j == kGroups - 1 && t == kGroup - 1) m = m > all ? m : all, n = all_n;
    g.fcum[t] = m;
    g.fcnt[t] = n;
  }
  __syncthreads();
}

// The border among the n listed elements within [lo, hi] (as smp_comp): the one
// of rank `need` (BY 0), or the last whose sum of the elements ahead is below
// `target` (BY 1); base and base_n are what lies ahead of all of them.  *incl:
// the sum down to the border.
template <int BY>
RLXQ_DEV uint64_t smp_select(const SmpRow& r, SmpPick& g, SmpShared& s, int n, uint64_t lo, uint64_t hi, double base,
                             uint32_t base_n, uint32_t need, double target, double* incl) {
  const int t = threadIdx.x;
  auto w_of = [&](uint64_t e) { return smp_w(r, of_key((uint32_t)(e >> 32))); };
  for (;;) {
    __syncthreads();
    if (t == 0) g.n_few = 0, g.lo = ~0ull, g.hi = 0;
    __syncthreads();
    for (int i = t; i < n; i += kSmpThreads) {
      const uint64_t e = g.list[i];
      if (e < lo || e > hi) continue;
      const uint32_t at = atomicAdd(&g.n_few, 1u);
      if (at < 64) g.few[at] = e;
    }
    __syncthreads();
    const uint32_t m = g.n_few;
    if (m <= 64) {   // a wave: every lane's rank, then the sums in order
      if (t < 64) {
        const uint64_t e = t < (int)m ? g.few[t] : 0;
        if (t >= (int)m) g.few[t] = 0;
        __threadfence_block();
        int rank = 0;
#pragma unroll
        for (int i = 0; i < 64; i++) rank += g.few[i] > e;
        const double w = t < (int)m ? w_of(e) : 0.0;
        // (to the lane of its rank: the wave's lanes have all read by now)
        if (t < (int)m) g.few[rank] = e, g.few_w[rank] = w;
        __threadfence_block();
        double c = t < (int)m ? g.few_w[t] : 0.0;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const double o = __shfl_up(c, off, 64);
          if (t >= off) c += o;
        }
        double ahead = __shfl_up(c, 1, 64);
        if (t == 0) ahead = 0.0;
        const bool in = t < (int)m && (BY == 0 ? base_n + t < need : t == 0 || base + ahead < target);
        const uint64_t which = __ballot(in);
        const int last = 63 - __builtin_clzll(which | 1);
        // (nothing listed: as where nothing is kept behind what lies ahead)
        if (t == last) g.lo = m ? g.few[t] : hi, g.base = base + c;
      }
      __syncthreads();
      *incl = g.base;
      const uint64_t border = g.lo;
      __syncthreads();
      return border;
    }
    // 512 bins over the elements' own range
    uint64_t e_lo = ~0ull, e_hi = 0;
    for (int i = t; i < n; i += kSmpThreads) {
      const uint64_t e = g.list[i];
      if (e < lo || e > hi) continue;
      e_lo = e < e_lo ? e : e_lo;
      e_hi = e > e_hi ? e : e_hi;
    }
    atomicMin((unsigned long long*)&g.lo, (unsigned long long)e_lo);
    atomicMax((unsigned long long*)&g.hi, (unsigned long long)e_hi);
    s.mass[t] = 0;
    s.count[t] = 0;
    __syncthreads();
    lo = g.lo, hi = g.hi;
    const int bits = 64 - __builtin_clzll(hi - lo), shift = bits > 9 ? bits - 9 : 0;
    for (int i = t; i < n; i += kSmpThreads) {
      const uint64_t e = g.list[i];
      if (e < lo || e > hi) continue;
      const uint32_t d = (uint32_t)((hi - e) >> shift);
      atomicAdd((unsigned long long*)&s.mass[d], (unsigned long long)(w_of(e) * 0x1p50 + 0.5));
      atomicAdd(&s.count[d], 1u);
    }
    __syncthreads();
    const uint32_t c = s.count[t];
    const double w = (double)s.mass[t] * 0x1p-50;
    double wt;
    uint32_t ct;
    const double ahead = base + smp_scan<double>(w, s.rd, &wt) - w;
    const uint32_t ahead_n = smp_scan<uint32_t>(c, s.r32, &ct) - c;
    const bool in = c && (BY == 0 ? base_n + ahead_n < need : ahead_n == 0 || ahead < target);
    if (t == 0) g.bin = 0;
    __syncthreads();
    if (in) atomicMax(&g.bin, t);   // the last bin that starts ahead of the border
    __syncthreads();
    if (t == g.bin) g.base = ahead, g.base_n = base_n + ahead_n;
    __syncthreads();
    const uint64_t d = (uint64_t)g.bin;
    base = g.base, base_n = g.base_n;
    const uint64_t top = hi - (d << shift), width = (1ull << shift) - 1;
    lo = top - lo > width ? top - width : lo;
    hi = top;
  }
}

template <int BF>
RLXQ_DEV void smp_pick(const rlxq_sample_args& a) {
  constexpr int N = BF ? 8 : 4;
  __shared__ SmpShared s;
  __shared__ SmpPick g;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, C = a.chunks;
  const rlxq_sample_chunk* heads = a.heads + row * C;
  uint64_t best = 0, my_best = 0, my_mass = 0;
  uint32_t bad = 0;
  if (t < C) my_best = heads[t].best, my_mass = heads[t].mass, bad = heads[t].bad;
  best = my_best;
  smp_best(best, bad, s.r64, s.r32);
  SmpRow r;
  if (!smp_row(a, row, best, bad, r)) return;
  const float scale = smp_bin_scale(a.temperature ? a.temperature[row] : 1.0f), anchor = smp_anchor(smp_bin(r.top, scale));
  if (t < C) {
    const float top = of_key((uint32_t)(my_best >> 32));
    g.scale[t] = my_best ? exp_neg(((double)top - (double)r.top) * r.inv_t) : 0.0;
    g.shift[t] = my_best ? (int)fminf((anchor - smp_anchor(smp_bin(top, scale))) * (1.0f / kGroup), (float)kGroups) : kGroups;
    g.kept[t] = (double)my_mass * 0x1p-48 * g.scale[t];
    g.add[t] = 0;
    g.flag[t] = 0;
  }
  const bool by_p = r.p < 1.0f, by_q = r.min_w > 0.0;
  bool by_k = r.k > 0 && r.k < a.V;
  uint64_t border = 1;
  const int lead = smp_lead<BF>(a, row);
  __syncthreads();
  if (by_k || by_p || by_q) {
    // the row's groups: a wave each, a lane a chunk.  (The last is the rest.)
    const int lane = t & 63, wave = t >> 6;
    for (int j = wave; j < kGroups; j += kSmpThreads / 64) {
      double m = 0.0;
      uint32_t n = 0;
      for (int c = lane; c < C; c += 64) {
        const int jj = j - g.shift[c];
        if (j == kGroups - 1) m += g.kept[c], n += heads[c].count;
        else if (jj >= 0) m += (double)heads[c].group_mass[jj] * 0x1p-48 * g.scale[c], n += by_k ? heads[c].group_count[jj] : 0;
      }
#pragma unroll
      for (int off = 32; off; off >>= 1) m += __shfl_xor(m, off, 64), n += __shfl_xor(n, off, 64);
      if (lane == 0) g.gcum[j] = m, g.gcnt[j] = n;
    }
    __syncthreads();
    const double all = g.gcum[kGroups - 1];
    const uint32_t all_n = g.gcnt[kGroups - 1];
    if (t < 16) {
      double m = t < kGroups - 1 ? g.gcum[t] : 0.0;
      uint32_t n = t < kGroups - 1 ? g.gcnt[t] : 0;
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) {
        const double om = __shfl_up(m, off, 16);
        const uint32_t on = __shfl_up(n, off, 16);
        if (t >= off) m += om, n += on;
      }
      if (t == kGroups - 1) m = m > all ? m : all, n = all_n;
      g.gcum[t] = m;
      g.gcnt[t] = n;
    }
    if (t == 0) g.n = 0, g.n_flag = 0;
    __syncthreads();
    by_k = by_k && (uint32_t)r.k < all_n;   // (fewer than k that are not masked: all of them)
    // the first group, and the first bin of fcum's, whose mass or number reaches x
    auto first_of = [](bool reached, int n) {
      const uint64_t b = __ballot(reached) & ((1ull << n) - 1);
      return b ? __builtin_ctzll(b) : n - 1;
    };
    const int bl = lane & (kGroup - 1), gl = lane & (kGroups - 1);
    auto group_of = [&](double x) { return first_of(g.gcum[gl] >= x, kGroups); };
    auto bin_of_mass = [&](double x) { return first_of(g.fcum[bl] >= x, kGroup); };
    auto flag = [&](int lo, int hi) {   // the chunks that hold something in bins lo .. hi of the group
      for (int c = t; c < C; c += kSmpThreads)
        if (g.some[c] & ((2u << (hi - lo)) - 1) << lo) g.flag[c] = 1;
    };
    // bins to look into: K's border's, P's, and about min-p's
    int kg = kGroups;
    if (by_k) kg = first_of(g.gcnt[gl] >= (uint32_t)r.k, kGroups);
    const double p = r.p > 1e-30f ? (double)r.p : 1e-30, under = 1.0 - 1e-12, over = 1.0 + 1e-12;
    int kb = kBins, p_lo = kBins, p_hi = -1, q_lo = kBins, q_hi = -1;
    const int pg = by_p ? group_of(p * (by_k ? (kg ? g.gcum[kg - 1] : 0.0) : all) * under) : kGroups;
    bool q_only = false;
    if (by_q) {
      const float edge = (float)((double)r.top + log(r.min_w) / r.inv_t);
      const int d = smp_below(anchor, smp_bin(edge, scale));
      q_lo = d > 0 ? d - 1 : 0, q_hi = d + 1 < kBins ? d + 1 : kBins - 1;
      q_only = q_hi < kGroup * (pg < kg ? pg : kg);   // min-p ends ahead of K and P
    }
    double k_lo = all, k_hi = all;   // the least and the most that K can weigh
    double k_ahead = 0.0, p_ahead = 0.0;
    uint32_t k_ahead_n = 0;
    if (!q_only) {
      if (by_k) {
        smp_fine(a, row, kg, true, all, all_n, g);
        const int b = first_of(g.fcnt[bl] >= (uint32_t)r.k, kGroup);
        kb = kg * kGroup + b;
        k_ahead = b ? g.fcum[b - 1] : (kg ? g.gcum[kg - 1] : 0.0);
        k_ahead_n = b ? g.fcnt[b - 1] : (kg ? g.gcnt[kg - 1] : 0);
        k_lo = k_ahead, k_hi = g.fcum[b];
        flag(b, b);
      }
      if (by_p) {
        const double lo = p * k_lo * under, hi = p * k_hi * over;
        const int j0 = group_of(lo), j1 = group_of(hi);
        smp_fine(a, row, j0, by_k, all, all_n, g);
        const int b = bin_of_mass(lo);
        p_lo = j0 * kGroup + b;
        p_ahead = b ? g.fcum[b - 1] : (j0 ? g.gcum[j0 - 1] : 0.0);
        int e = j1 > j0 ? kGroup - 1 : bin_of_mass(hi);
        flag(b, e);
        for (int j = j0 + 1; j <= j1; j++) {
          smp_fine(a, row, j, by_k, all, all_n, g);
          e = j < j1 ? kGroup - 1 : bin_of_mass(hi);
          flag(0, e);
        }
        p_hi = j1 * kGroup + e;
      }
    }
    if (!q_only && q_lo > (by_p ? p_hi : kb)) q_lo = kBins, q_hi = -1;   // min-p ends behind them
    if (q_hi >= 0)
      for (int j = q_lo / kGroup; j <= q_hi / kGroup; j++) {
        smp_fine(a, row, j, by_k, all, all_n, g);
        flag(j == q_lo / kGroup ? q_lo % kGroup : 0, j == q_hi / kGroup ? q_hi % kGroup : kGroup - 1);
      }
    const int kp = p_lo < kb ? p_lo : kb;
    const int d_lo = q_lo < kp ? q_lo : kp;   // bins ahead of it are kept whole
    auto bin_at = [&](float v) { return smp_below(anchor, smp_bin(v, scale)); };
    auto wanted = [&](int d) { return d == kb || (d >= p_lo && d <= p_hi) || (d >= q_lo && d <= q_hi); };
    // (an open bin of a chunk below the row's top may hold what falls into a later
    // bin of the row: the row's own last one, for which every chunk is flagged)
    __syncthreads();
    if (t < C && g.flag[t]) g.flagged[atomicAdd(&g.n_flag, 1u)] = (uint16_t)t;
    __syncthreads();
    // (x = l scale of the bins d_first .. d_last, and some more: wanted() decides.  An
    // x past the largest number is in the open bin, and `to` is past it too then.)
    const int d_first = kp < q_lo ? kp : q_lo;
    int d_last = p_hi > q_hi ? p_hi : q_hi;
    if (kb < kBins && kb > d_last) d_last = kb;
    const float slack = 1.0f + fabsf(anchor) * 0x1p-22f;
    const float from = d_last == kBins - 1 ? -__builtin_inff() : anchor - (float)d_last - slack;
    const float to = anchor - (float)d_first + 1.0f + slack;
    constexpr int kPerThread = RLXQ_SAMPLE_CHUNK / kSmpThreads, kAtOnce = 4;
    const int n_flag = (int)g.n_flag;
    for (int f0 = 0; f0 < n_flag; f0 += kAtOnce) {
      float v[kAtOnce][kPerThread];
      int first[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; u++) {
        // (past the last: the last again, whose elements are not taken)
        first[u] = (int)g.flagged[f0 + u < n_flag ? f0 + u : n_flag - 1] * RLXQ_SAMPLE_CHUNK - lead;
        smp_ld_chunk<BF, kPerThread / N>(a, row, first[u], t, kSmpThreads, v[u]);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; u++) {
        if (f0 + u >= n_flag) break;
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < kPerThread; j++) {
          const float x = v[u][j] * scale;
          in |= (!(x < from) && !(x > to)) ? 1u << j : 0u;
        }
        if (!in) continue;
#pragma unroll
        for (int j = 0; j < kPerThread; j++) {
          if (!(in >> j & 1) || v[u][j] == -__builtin_inff() || !wanted(bin_at(v[u][j]))) continue;
          const uint32_t at = atomicAdd(&g.n, 1u);
          if (at < kSmpList) g.list[at] = smp_comp(key_of(v[u][j]), first[u] + ((j / N) * kSmpThreads + t) * N + j % N);
        }
      }
    }
    __syncthreads();
    const int n = (int)g.n;
    if (n > kSmpList) {
      smp_scan_row(a, r, row, s);
      return;
    }
    // the listed elements of bins lo .. hi, as a range of smp_comp
    auto range = [&](int lo, int hi, uint64_t* from, uint64_t* to) {
      __syncthreads();
      if (t == 0) g.lo = ~0ull, g.hi = 0;
      __syncthreads();
      uint64_t f = ~0ull, l = 0;
      for (int i = t; i < n; i += kSmpThreads) {
        const uint64_t e = g.list[i];
        const int d = bin_at(of_key((uint32_t)(e >> 32)));
        if (d < lo || d > hi) continue;
        f = e < f ? e : f;
        l = e > l ? e : l;
      }
      if (l) {
        atomicMin((unsigned long long*)&g.lo, (unsigned long long)f);
        atomicMax((unsigned long long*)&g.hi, (unsigned long long)l);
      }
      __syncthreads();
      *from = g.lo, *to = g.hi;
    };
    if (!q_only && (by_k || by_p)) {
      double mass_k = all;
      uint64_t lo, hi;
      if (by_k) {
        range(kb, kb, &lo, &hi);
        border = smp_select<0>(r, g, s, n, lo, hi, k_ahead, k_ahead_n, (uint32_t)r.k, 0.0, &mass_k);
      }
      if (by_p) {
        range(p_lo, p_hi, &lo, &hi);
        if (lo < border) lo = border;
        // (what is not in K is behind its border)
        double ignored;
        border = smp_select<1>(r, g, s, n, lo, hi, p_ahead, 0, 0, p * mass_k, &ignored);
      }
    }
    // the chunks' kept mass: whole groups and bins, and what is listed (without any
    // border, as where top_k is more than what is not masked, the whole chunk's)
    if (d_lo < kBins) {
      for (int c0 = 0; c0 < C; c0 += 16) {
        const int c = c0 + (t >> 5), b = t & 31, jj = c < C ? d_lo / kGroup - g.shift[c] : -1;
        double m = 0.0;
        if (jj >= 0) {
          if (b < d_lo % kGroup) m = (double)a.masses[(row * C + c) * kBins + jj * kGroup + b];
          if (b < jj) m += (double)heads[c].group_mass[b];
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) m += __shfl_xor(m, off, 32);
        if (c < C && b == 0) g.kept[c] = m * 0x1p-48 * g.scale[c];
      }
      for (int i = t; i < n; i += kSmpThreads) {
        const uint64_t e = g.list[i];
        const float v = of_key((uint32_t)(e >> 32));
        if (e < border || bin_at(v) < d_lo) continue;
        const double w = smp_w(r, v);
        if (w < r.min_w) continue;
        const int idx = (int)~(uint32_t)e;
        atomicAdd(&g.add[(idx + lead) / RLXQ_SAMPLE_CHUNK], (unsigned long long)(w * 0x1p50 + 0.5));
      }
    }
    __syncthreads();
  }
  // the chunk, then the element
  const double m = t < C ? g.kept[t] + (double)g.add[t] * 0x1p-50 : 0.0;
  double total;
  const double incl = smp_scan<double>(m, s.rd, &total);
  const double target = (double)r.u * total;
  if (t == 0) s.found = 0x7fffffff, s.last = -1;
  __syncthreads();
  if (m > 0.0) {
    atomicMax(&s.last, t);
    if (incl > target) atomicMin(&s.found, t);
  }
  __syncthreads();
  const int c = s.found != 0x7fffffff ? s.found : (s.last > 0 ? s.last : 0);
  if (t == c) g.before = incl - m;
  __syncthreads();
  constexpr int kPer = RLXQ_SAMPLE_CHUNK / kSmpThreads;
  const int first = c * RLXQ_SAMPLE_CHUNK - lead;
  float v[kPer];
  double w[kPer], mine = 0.0;
  int last = -1;
  smp_ld_chunk<BF, kPer / N>(a, row, first, t * (kPer / N), 1, v);
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    const int i = first + t * kPer + j;
    w[j] = smp_kept(r, border, v[j], i);
    mine += w[j];
    if (w[j] > 0.0) last = i;
  }
  smp_choose(a, r, row, mine, last, g.before, total, s, [&](double sum, double target) {
    int tok = last;
    bool past = false;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      sum += w[j];
      if (!past && sum > target && w[j] > 0.0) tok = first + t * kPer + j, past = true;
    }
    return tok;
  });
}

}  // namespace rlxq

using namespace rlxq;

// A workgroup a row.
extern "C" __global__ __launch_bounds__(kSmpThreads) void rlxq_sample_scan(rlxq_sample_args a) {
  __shared__ SmpShared s;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x;
  // the largest logit, the lowest index that has it; NaN and +inf
  uint64_t best = 0;
  uint32_t bad = 0;
  for (int i = t; i < a.V; i += kSmpThreads) {
    const float v = smp_ld(a, row, i);
    if (!(v < __builtin_inff())) bad = 1;
    const uint32_t key = key_of(v);
    const uint64_t c = key ? smp_comp(key, i) : 0;
    best = c > best ? c : best;
  }
  smp_best(best, bad, s.r64, s.r32);
  SmpRow r;
  if (smp_row(a, row, best, bad, r)) smp_scan_row(a, r, row, s);
}

extern "C" __global__ __launch_bounds__(kHistThreads) void rlxq_sample_hist_f32(rlxq_sample_args a) { smp_hist<0>(a); }
extern "C" __global__ __launch_bounds__(kHistThreads) void rlxq_sample_hist_bf16(rlxq_sample_args a) { smp_hist<1>(a); }
extern "C" __global__ __launch_bounds__(kSmpThreads) void rlxq_sample_pick_f32(rlxq_sample_args a) { smp_pick<0>(a); }
extern "C" __global__ __launch_bounds__(kSmpThreads) void rlxq_sample_pick_bf16(rlxq_sample_args a) { smp_pick<1>(a); }
