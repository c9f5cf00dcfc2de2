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
// 2e-16.  exp(0) is exactly 1; below 2^-1022 the result has the bits that a
// denormal leaves it, below 2^-1075 it is 0.
RLXQ_DEV double exp_neg(double x) {
  if (x < -746.0) return 0.0;
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
  float temperature, p, q, u;
  int k;                 // 0: off
};

RLXQ_DEV float smp_ld(const rlxq_sample_args& a, int64_t row, int i) {
  return a.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(a.logits)[row * a.V + i])
                : reinterpret_cast<const float*>(a.logits)[row * a.V + i];
}
RLXQ_DEV double smp_w(const SmpRow& r, float v) { return exp_neg(((double)v - (double)r.top) * r.inv_t); }

// What the token's sum has to exceed: u times the kept mass, or (u from 1 up) what
// no sum does, so that the last kept token is taken whatever the sums round to.
RLXQ_DEV double smp_target(const SmpRow& r, double total) { return r.u < 1.0f ? (double)r.u * total : __builtin_inf(); }

// The border as one number: key above, falling index below.  An element is
// kept if its own is not smaller.
RLXQ_DEV uint64_t smp_comp(uint32_t key, uint32_t idx) { return (uint64_t)key << 32 | (uint32_t)~idx; }

// Sums over the workgroup's threads in thread order: down to the thread, ahead of it
// (summed by itself: the difference would lose it beside a large v), and of all.
template <class T>
RLXQ_DEV T smp_scan(T v, T* red, T* ahead, T* total) {
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
  const T o = __shfl_up(v, 1, 64);
  *ahead = lane ? before + o : before;
  return before + v;
}

struct SmpShared {
  uint64_t mass[kSmpThreads + 8];
  uint32_t count[kSmpThreads];
  uint64_t r64[16];
  double rd[16];
  uint32_t r32[16];
  int found, last, first_past[8], last_some[8];
};

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
  double all, ahead;
  const double incl = before + smp_scan<double>(m, s.rd, &ahead, &all);
  if (total < 0.0) total = all;
  const double target = smp_target(r, total);
  // the first thread whose sum exceeds the target, else (rounding, or u from 1 up) the
  // last that keeps anything
  const int t = threadIdx.x, wave = t >> 6;
  const uint64_t some = __ballot(last >= 0), past = __ballot(m > 0.0 && incl > target);
  if ((t & 63) == 0) {
    s.first_past[wave] = past ? t + __builtin_ctzll(past) : -1;
    s.last_some[wave] = some ? t + 63 - __builtin_clzll(some) : -1;
  }
  __syncthreads();
  int who = -1, end = -1;
  for (int w = kSmpThreads / 64 - 1; w >= 0; w--) {
    if (s.first_past[w] >= 0) who = s.first_past[w];
    if (end < 0) end = s.last_some[w];
  }
  if (who < 0 && end < 0) {   // (nothing kept, which no row comes to)
    if (t == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = __builtin_nanf("");
    }
  } else if (t == (who >= 0 ? who : end)) {
    const int tok = who >= 0 ? at(before + ahead, target) : last;
    a.tokens[row] = tok;
    if (a.probs) a.probs[row] = (float)(smp_w(r, smp_ld(a, row, tok)) / total);
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

// The row's settings; temperature is not positive where the likeliest is asked for.
RLXQ_DEV void smp_settings(const rlxq_sample_args& a, int64_t row, SmpRow& r) {
  r.temperature = a.temperature ? a.temperature[row] : 1.0f;
  r.u = a.u[row];
  r.k = a.top_k ? a.top_k[row] : 0;
  r.p = a.top_p ? a.top_p[row] : 1.0f;
  r.q = a.min_p ? a.min_p[row] : 0.0f;
}
// The row's largest logit is known.  False: its token is already written (no
// distribution, or the likeliest was asked for).
RLXQ_DEV bool smp_row(const rlxq_sample_args& a, int64_t row, uint64_t best, uint32_t bad, SmpRow& r) {
  const bool none = bad || !best || r.temperature != r.temperature || r.u != r.u;
  if (none || !(r.temperature > 0.0f)) {
    if (threadIdx.x == 0) {
      a.tokens[row] = none ? -1 : (int32_t)~(uint32_t)best;
      if (a.probs) a.probs[row] = none ? __builtin_nanf("") : 1.0f;
    }
    return false;
  }
  r.top = of_key((uint32_t)(best >> 32));
  r.inv_t = 1.0 / (double)r.temperature;
  r.min_w = r.q > 0.0f ? (r.q < 1.0f ? (double)r.q : 1.0) : 0.0;
  return true;
}

// ---- two launches: chunk histograms, then a workgroup a row ----------------
//
// The first reads the logits once: each workgroup a chunk of a row, in
// registers, whose weights are taken relative to the chunk's own largest logit
// and summed, in f64 where the row has no border, else by bins of l / T in fixed
// point.  The bins of all chunks lie on one grid, so the second launch adds them up (groups of 32 bins, then the
// 32 of one group), finds the bin that each border falls into, and reads again
// only the chunks that hold anything in those bins; what it finds there is
// listed and settles the borders.  Where that is more than the list holds (rows as
// flat as noise), the flagged chunks are gone through once more, which narrows the
// border to what can be listed, and again for the kept mass.
//
// What bounds it: the first launch the vector unit and the loads' latency (256
// rows of 128000 bf16, a quarter of them with borders: 47 us, 30 instructions an
// element, half of the time issuing; 64 of 151936 f32, most of them with borders: 25,
// 23 of them with one step for all bins; 512 threads a chunk took a sixth more, and
// held to fewer registers it spilled); the
// second a row's chain of dependent steps on one CU: 19 us for one row of 151936
// with top-k 50; a row with min-p and 42 pieces 22 (settings and heads 3, groups and
// bins 6, the pieces 6, their list, the border and the token 7); up to 50 where a
// wide top-p reads the whole row again at a CU's 20 GB/s.  1024 threads were 8%
// faster there and 10% slower for one row; more of its loads ahead changed nothing.

constexpr int kBins = RLXQ_SAMPLE_BINS, kGroups = RLXQ_SAMPLE_GROUPS, kGroup = kBins / kGroups;
constexpr int kHistThreads = RLXQ_SAMPLE_CHUNK / 16, kHistWaves = kHistThreads / 64;
constexpr int kSmpList = 8192;
constexpr int kSmpSort = 512;   // kept elements that are sorted as a whole
constexpr int kSmpChunks = RLXQ_SAMPLE_MAX_VOCAB / RLXQ_SAMPLE_CHUNK + 1;   // (a row may start inside 16 bytes)

// Bin number of v on the row's grid, a whole number that does not fall as v
// rises; the grid's multiple of a group at or above it; bins below one, the last
// one open (and everything in it where l / T has no finite number).
RLXQ_DEV float smp_bin_scale(float T) { return fminf(16.0f / T, 1e30f); }
RLXQ_DEV float smp_bin(float v, float scale) { return floorf(v * scale); }
RLXQ_DEV float smp_anchor(float bin) { return ceilf(bin * (1.0f / kGroup)) * kGroup; }
RLXQ_DEV int smp_below(float anchor, float bin) { return (int)fminf(anchor - bin, (float)(kBins - 1)); }

// Bin d of a chunk is summed in steps of 2^-(48 + s) of the chunk's largest weight,
// s = d fine / 256 cut to a whole number: 23 / 256 is a little less than the 1 /
// (16 ln 2) binary digits that weights fall by from bin to bin.  So each of a bin's
// 4096 at most stays below 2^52 steps (up to 31 bins lie between the anchor and the
// top, nine more are rounding) and has 46 bits or more, in all bins but the last.
// Where l / T is past 2^23 the bins' numbers round to more than that: 2^-48 in all.
RLXQ_DEV int smp_fine_steps(float anchor) { return fabsf(anchor) < 0x1p27f ? 23 : 0; }
RLXQ_DEV double smp_bin_mass(uint64_t m, int d, int fine) { return __builtin_ldexp((double)m, -(d * fine >> 8)); }

// The elements of 16 bytes.
template <int BF>
RLXQ_DEV void smp_unpack(const uint4& q, float* v) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (BF) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    else v[j] = __uint_as_float(w[j]);
  }
}

// The elements of one aligned 16-byte vector of a row: i0 is the index of the
// first, which may lie ahead of the row (its start need not be aligned), unless
// all of it is known to be inside.
template <int BF>
RLXQ_DEV void smp_ld16(const rlxq_sample_args& a, int64_t row, int i0, float* v, bool inside) {
  constexpr int N = BF ? 8 : 4;
  if (inside || (i0 >= 0 && i0 + N <= a.V)) {
    smp_unpack<BF>(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.logits) + (row * a.V + i0) * (BF ? 2 : 4)),
                   v);
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

// One chunk of smp_hist, its elements in v.
template <int BF>
RLXQ_DEV void smp_hist_chunk(const rlxq_sample_args& a, int64_t row, int c, int first, const float* v, float T, bool by_k,
                             bool bins, unsigned long long* mass, uint32_t* count, const double* pow2, double* rd,
                             uint32_t* r32, float* rf, int* at) {
  constexpr int N = BF ? 8 : 4, TH = kHistThreads, kPiece = RLXQ_SAMPLE_CHUNK / kHistWaves;
  const int t = threadIdx.x;
  for (int i = t; i < kBins; i += TH) mass[i] = 0, count[i] = 0;
  if (t == 0) *at = 0x7fffffff;
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
  rlxq_sample_chunk* head = a.heads + row * a.chunks + c;
  if ((t & 63) == 0) rf[t >> 6] = head->tops[t >> 6] = top, r32[t >> 6] = bad;
  __syncthreads();
  for (int w = 0; w < TH / 64; w++) top = fmaxf(top, rf[w]), bad |= r32[w];
  if (rf[t >> 6] == top) {   // the lowest index of the largest
    int mine = 0x7fffffff;
#pragma unroll
    for (int j = 15; j >= 0; j--)
      if (v[j] == top) mine = first + (t >> 6) * kPiece + ((j / N) * 64 + (t & 63)) * N + j % N;
    if (mine != 0x7fffffff) atomicMin(at, mine);
  }
  __syncthreads();
  uint64_t* masses = a.masses + (row * a.chunks + c) * kBins;
  uint16_t* counts = a.counts + (row * a.chunks + c) * kBins;
  const uint64_t best = key_of(top) ? smp_comp(key_of(top), *at) : 0;
  if (!(T > 0.0f) || bad || !best) {   // (no weights; no bins are read but those of a chunk that is all masked)
    if (t == 0) head->best = best, head->mass = 0, head->bad = bad, head->count = 0;
    return;
  }
  const float scale = smp_bin_scale(T), anchor = smp_anchor(smp_bin(top, scale));
  const int fine = smp_fine_steps(anchor);
  // w 2^48 = 2^(n / 32 + 48) 2^(f / 32), n the integer nearest x = 32 (l - top) / (T
  // ln 2), f = x - n: a table by n mod 32 (its entries times 2^48), and the Taylor
  // series of the second about 0, whose first term left out is below (ln 2 / 64)^6 /
  // 720 = 3e-15.  n is read off the sum 1.5 2^52 + x.  What is e^-600 of the top or
  // less, masked tokens among it, counts as that, which rounds to 0 in every bin and
  // beside the top.
  constexpr double L = 0.6931471805599453 / 32, kRound = 0x1.8p52;
  const double top64 = (double)top, c32 = 32.0 / (0.6931471805599453 * (double)T);
  const double least = -600.0 * (double)T;
  const bool wide = !(T < 1e36f);   // (nothing is that far below the top then: masked tokens by name)
  double sum = 0.0;
#pragma unroll
  for (int half = 0; half < 2; half++) {
    double e[8], f2[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const double d = __builtin_fmax((double)v[8 * half + j] - top64, least);
      const double y = __builtin_fma(d, c32, kRound);
      const uint32_t n = (uint32_t)__double_as_longlong(y);
      const double f = __builtin_fma(d, c32, kRound - y);
      e[j] = __builtin_fma(f, L * L * L * L * L / 120, L * L * L * L / 24);
      e[j] = __builtin_fma(e[j], f, L * L * L / 6);
      e[j] = __builtin_fma(e[j], f, L * L / 2);
      e[j] = __builtin_fma(e[j], f, L);
      e[j] = __builtin_fma(e[j], f, 1.0);
      const uint2 b = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(pow2) + (n << 3 & 0xf8));
      f2[j] = __hiloint2double((int)(b.y + ((n & ~31u) << 15)), (int)b.x);   // (an exponent of 1071 - 866 at least)
    }
    if (wide) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (v[8 * half + j] == -__builtin_inff()) e[j] = f2[j] = 0.0;
    }
    if (bins) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int d = smp_below(anchor, smp_bin(v[8 * half + j], scale));
        const double f = __hiloint2double(__double2hiint(f2[j]) + ((d * fine & ~255) << 12), __double2loint(f2[j]));
        const uint64_t w = (uint64_t)__double_as_longlong(__builtin_fma(e[j], f, 0x1p52)) & 0xfffffffffffffull;
        atomicAdd(&mass[d], (unsigned long long)w);
        if (by_k && v[8 * half + j] > -__builtin_inff()) atomicAdd(&count[d], 1u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) sum = __builtin_fma(e[j], f2[j], sum);
    }
  }
  if (!bins) {
#pragma unroll
    for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if ((t & 63) == 0) rd[t >> 6] = sum;
    __syncthreads();
    if (t == 0) {
      for (int w = 1; w < TH / 64; w++) sum += rd[w];
      head->best = best, head->mass = sum, head->bad = 0;
    }
    return;
  }
  __syncthreads();
  static_assert(kBins == 2 * TH && kGroup == 32, "a thread takes two bins, 16 threads a group");
  const uint64_t m0 = mass[2 * t], m1 = mass[2 * t + 1];
  const uint32_t n0 = count[2 * t], n1 = count[2 * t + 1];
  reinterpret_cast<ulonglong2*>(masses)[t] = make_ulonglong2(m0, m1);
  if (by_k) reinterpret_cast<uint32_t*>(counts)[t] = n0 | n1 << 16;
  double gm = smp_bin_mass(m0, 2 * t, fine) + smp_bin_mass(m1, 2 * t + 1, fine);
  uint32_t gn = n0 + n1;
#pragma unroll
  for (int off = 8; off; off >>= 1) gm += __shfl_xor(gm, off, 64), gn += __shfl_xor(gn, off, 64);
  if ((t & 15) == 0) head->group_mass[t >> 4] = gm, head->group_count[t >> 4] = gn;
#pragma unroll
  for (int off = 32; off >= 16; off >>= 1) gm += __shfl_xor(gm, off, 64), gn += __shfl_xor(gn, off, 64);
  if ((t & 63) == 0) rd[t >> 6] = gm, r32[t >> 6] = gn;
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < TH / 64; w++) gm += rd[w], gn += r32[w];
    head->best = best, head->mass = gm, head->bad = 0, head->count = gn;
  }
}

template <int BF>
RLXQ_DEV void smp_hist(const rlxq_sample_args& a) {
  constexpr int N = BF ? 8 : 4, TH = kHistThreads;
  __shared__ unsigned long long mass[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double pow2[32];
  __shared__ double rd[TH / 64];
  __shared__ uint32_t r32[TH / 64];
  __shared__ float rf[TH / 64];
  __shared__ int at;
  // a.per chunks of one row, one after the other
  const int runs = (a.chunks + a.per - 1) / a.per, t = threadIdx.x;
  const int64_t row = blockIdx.x / runs;
  const int c0 = (int)(blockIdx.x - row * runs) * a.per, c1 = c0 + a.per < a.chunks ? c0 + a.per : a.chunks;
  const int lead = smp_lead<BF>(a, row);
  // (a wave's elements: kPiece neighbouring ones)
  constexpr int kPiece = RLXQ_SAMPLE_CHUNK / kHistWaves;
  uint4 raw[16 / N];   // a chunk that lies in the row as a whole, on its way
  auto inside = [&](int first) { return first >= 0 && first + RLXQ_SAMPLE_CHUNK <= a.V; };
  auto fetch = [&](int first) {
#pragma unroll
    for (int j = 0; j < 16 / N; j++)
      raw[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.logits) +
                                               (row * a.V + first + (t >> 6) * kPiece + (j * 64 + (t & 63)) * N) * (BF ? 2 : 4));
  };
  if (inside(c0 * RLXQ_SAMPLE_CHUNK - lead)) fetch(c0 * RLXQ_SAMPLE_CHUNK - lead);
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.0f, q = a.min_p ? a.min_p[row] : 0.0f;
  const bool by_k = k > 0 && k < a.V, bins = by_k || p < 1.0f || q > 0.0f;
  if (t < 32) pow2[t] = 0x1p49 * exp_neg((t - 32) * (0.6931471805599453 / 32));
#pragma unroll 1
  for (int c = c0; c < c1; c++) {
    const int first = c * RLXQ_SAMPLE_CHUNK - lead;
    float v[16];
    if (inside(first)) {
#pragma unroll
      for (int j = 0; j < 16 / N; j++) smp_unpack<BF>(raw[j], v + j * N);
    } else {
#pragma unroll
      for (int j = 0; j < 16 / N; j++) smp_ld16<BF>(a, row, first + (t >> 6) * kPiece + (j * 64 + (t & 63)) * N, v + j * N, false);
    }
    if (c + 1 < c1 && inside(first + RLXQ_SAMPLE_CHUNK)) fetch(first + RLXQ_SAMPLE_CHUNK);
    if (c > c0) __syncthreads();   // (the last one's LDS is read)
    smp_hist_chunk<BF>(a, row, c, first, v, T, by_k, bins, mass, count, pow2, rd, r32, rf, &at);
  }
}

struct SmpPick {
  double scale[kSmpChunks], kept[kSmpChunks];   // chunks: their weights' scale in the row; their kept mass
  unsigned long long add[kSmpChunks];           // kept weights of listed elements, in 2^-51 of the chunk's top
  double gmass[kSmpChunks][kGroups];            // the chunks' groups, as the first launch left them
  uint32_t gnum[kSmpChunks][kGroups];
  int shift[kSmpChunks];                        // groups from the row's top to the chunk's
  int fine[kSmpChunks];                         // its bins' steps
  float top[kSmpChunks];                        // its largest logit
  uint32_t some[kSmpChunks];                    // which bins of the group that smp_fine took hold something
  uint16_t flagged[kSmpChunks * kHistWaves];    // pieces to read again
  float tops[kSmpChunks][kHistWaves];           // their largest logits
  uint8_t flag[kSmpChunks];
  double part[16][32];
  uint32_t part_n[16][32];
  double gcum[kGroups], fcum[kGroup];           // mass down to a group of the row, a bin of one group
  uint32_t gcnt[kGroups], fcnt[kGroup];         // elements
  uint64_t list[kSmpList];
  uint64_t few[64], lo, hi;
  double few_w[64], sorted_w[kSmpSort];
  uint32_t n, n_few, n_flag;
  int bin;
  double before, base;
  uint32_t base_n, bin_n;
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
        m += smp_bin_mass(q[u], (j - g.shift[c]) * kGroup + b, g.fine[c]) * g.scale[c];
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

// f of every element of the flagged chunks that is not masked, a thread's in
// order of their index.
template <int BF, class F>
RLXQ_DEV void smp_each(const rlxq_sample_args& a, int64_t row, int lead, const SmpPick& g, F&& f) {
  constexpr int N = BF ? 8 : 4, PER = RLXQ_SAMPLE_CHUNK / kSmpThreads;
  const int x = threadIdx.x * (PER / N);
  float v[PER], next[PER];   // (the next chunk is on its way)
  smp_ld_chunk<BF, PER / N>(a, row, -lead, x, 1, next);
#pragma unroll 1
  for (int c = 0; c < a.chunks; c++) {
#pragma unroll
    for (int j = 0; j < PER; j++) v[j] = next[j];
    const int first = c * RLXQ_SAMPLE_CHUNK - lead;
    if (c + 1 < a.chunks) smp_ld_chunk<BF, PER / N>(a, row, first + RLXQ_SAMPLE_CHUNK, x, 1, next);
    if (!g.flag[c]) continue;
#pragma unroll
    for (int j = 0; j < PER; j++)
      if (v[j] > -__builtin_inff()) f(smp_comp(key_of(v[j]), first + threadIdx.x * PER + j));
  }
}

// The border among the listed elements of bins b_lo .. b_hi that are not smaller
// than `lo` (as smp_comp), n of them, or (n above kSmpList) among those that
// `each` goes through: by_rank the one of rank `need`, else the last whose sum
// of the elements ahead is below `target`; base and base_n are what lies
// ahead of all of them.  *incl: the sum down to the border.  Bins over the range
// of what is left narrow it until a wave can sort it.  Their sums are fixed point,
// in steps of 2^-42 (2^-50 of a list's) of the weight at the range's upper end: at
// most 2^20 elements, so that they are off by 2^-23 of that weight at most,
// however small it is beside the row's largest.
template <class B, class E>
RLXQ_DEV uint64_t smp_select(bool by_rank, const SmpRow& r, SmpPick& g, SmpShared& s, int n, E&& each, B&& bin_at, int b_lo, int b_hi, uint64_t lo,
                             uint64_t hi, double base, uint32_t base_n, uint32_t need, double target, double* incl) {
  const int t = threadIdx.x, lane = t & 63;
  auto w_of = [&](uint64_t e) { return smp_w(r, of_key((uint32_t)(e >> 32))); };
  auto within = [&](uint64_t e) {
    if (e < lo || e > hi) return false;
    const int d = bin_at(of_key((uint32_t)(e >> 32)));
    return d >= b_lo && d <= b_hi;
  };
  uint32_t left = (uint32_t)n;   // at most so many
  bool listed = n <= kSmpList;
  for (bool first = true;; first = false) {
    __syncthreads();
    if (t == 0) g.n_few = 0, g.lo = ~0ull, g.hi = 0, g.bin = 0;
    s.mass[t] = 0;
    s.count[t] = 0;
    __syncthreads();
    if (!listed && left <= kSmpList) {
      each([&](uint64_t e) {
        if (within(e)) g.list[atomicAdd(&g.n_few, 1u)] = e;
      });
      __syncthreads();
      n = (int)g.n_few;
      listed = true;
      __syncthreads();
      if (t == 0) g.n_few = 0;
      __syncthreads();
    }
    if (left <= 64) {
      for (int i = t; i < n; i += kSmpThreads)
        if (within(g.list[i])) g.few[atomicAdd(&g.n_few, 1u)] = g.list[i];
      __syncthreads();
      const int m = (int)g.n_few;
      if (t < 64) {   // a wave: every lane's rank, then the sums in order
        const uint64_t e = t < m ? g.few[t] : 0;
        if (t >= m) g.few[t] = 0;
        __threadfence_block();
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < 64; i++) rank += g.few[i] > e;
        const double w = t < m ? w_of(e) : 0.0;
        // (to the lane of its rank: the wave's lanes have all read by now)
        if (t < m) g.few[rank] = e, g.few_w[rank] = w;
        __threadfence_block();
        double c = t < m ? g.few_w[t] : 0.0;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const double o = __shfl_up(c, off, 64);
          if (t >= off) c += o;
        }
        double ahead = __shfl_up(c, 1, 64);
        if (t == 0) ahead = 0.0;
        const bool in = t < m && (by_rank ? base_n + t < need : t == 0 || base + ahead < target);
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
    if (!first) {   // the elements' own range
      uint64_t e_lo = ~0ull, e_hi = 0;
      auto range = [&](uint64_t e) {
        if (!within(e)) return;
        e_lo = e < e_lo ? e : e_lo;
        e_hi = e > e_hi ? e : e_hi;
      };
      if (listed)
        for (int i = t; i < n; i += kSmpThreads) range(g.list[i]);
      else
        each(range);
#pragma unroll
      for (int off = 32; off; off >>= 1) {
        const uint64_t ol = __shfl_xor(e_lo, off, 64), oh = __shfl_xor(e_hi, off, 64);
        e_lo = ol < e_lo ? ol : e_lo;
        e_hi = oh > e_hi ? oh : e_hi;
      }
      if (lane == 0) {
        atomicMin((unsigned long long*)&g.lo, (unsigned long long)e_lo);
        atomicMax((unsigned long long*)&g.hi, (unsigned long long)e_hi);
      }
      __syncthreads();
      lo = g.lo, hi = g.hi;
    }
    const int bits = hi > lo ? 64 - __builtin_clzll(hi - lo) : 1, shift = bits > 9 ? bits - 9 : 0;
    // (kSmpList, or a whole row, of weights up to 1 at most 2^63)
    const float end = of_key((uint32_t)(hi >> 32));
    const double one = listed ? 0x1p50 : 0x1p42, unit = smp_w(r, end) / one;
    auto narrow = [&](uint64_t e) {
      if (!within(e)) return;
      const uint32_t d = (uint32_t)((hi - e) >> shift);
      const double w = exp_neg(((double)of_key((uint32_t)(e >> 32)) - (double)end) * r.inv_t);
      atomicAdd((unsigned long long*)&s.mass[d], (unsigned long long)(w * one + 0.5));
      atomicAdd(&s.count[d], 1u);
    };
    if (listed)
      for (int i = t; i < n; i += kSmpThreads) narrow(g.list[i]);
    else
      each(narrow);
    __syncthreads();
    const uint32_t c = s.count[t];
    const double w = (double)s.mass[t] * unit;
    double ahead, wt;
    uint32_t ahead_n, ct;
    smp_scan<double>(w, s.rd, &ahead, &wt);
    smp_scan<uint32_t>(c, s.r32, &ahead_n, &ct);
    ahead += base;
    const bool in = c && (by_rank ? base_n + ahead_n < need : ahead_n == 0 || ahead < target);
    // the last bin that starts ahead of the border
    const uint64_t which = __ballot(in);
    if (lane == 0 && which) atomicMax(&g.bin, t + 63 - __builtin_clzll(which));
    __syncthreads();
    if (t == g.bin) g.base = ahead, g.base_n = base_n + ahead_n, g.bin_n = c;
    __syncthreads();
    const uint64_t d = (uint64_t)g.bin;
    base = g.base, base_n = g.base_n, left = g.bin_n;
    const uint64_t top = hi - (d << shift), width = (1ull << shift) - 1;
    lo = top - lo > width ? top - width : lo;
    hi = top;
  }
}

// A row whose n listed elements (at most kSmpSort) are everything down to a bin
// behind K's border: sorted as a whole, the borders follow from prefix sums, and
// the token from the kept ones sorted by index.
RLXQ_DEV void smp_small(const rlxq_sample_args& a, const SmpRow& r, int64_t row, int n, SmpPick& g, SmpShared& s) {
  static_assert(kSmpSort == kSmpThreads, "an element a thread");
  const int t = threadIdx.x;
  const uint64_t e = t < n ? g.list[t] : 0;
  const double w = t < n ? smp_w(r, of_key((uint32_t)(e >> 32))) : 0.0;
  if (t >= n) g.list[t] = 0;   // (up to a multiple of 8)
  __syncthreads();
  auto rank_of = [&](const uint64_t* v, uint64_t x, int count) {   // elements of v that are larger
    int rank = 0;
    for (int i = 0; i < count; i += 8) {
#pragma unroll
      for (int j = 0; j < 8; j++) rank += v[i + j] > x;
    }
    return rank;
  };
  const int rank = rank_of(g.list, e, n);
  if (t < n) g.sorted_w[rank] = w;
  __syncthreads();
  const int k = r.k < n ? r.k : n;
  const double mine = t < k ? g.sorted_w[t] : 0.0;
  double ahead, mass_k;
  smp_scan<double>(mine, s.rd, &ahead, &mass_k);
  const double target = r.p < 1.0f ? (r.p > 0.0f ? (double)r.p * mass_k : 0.0) : __builtin_inf();
  // of K's in order: what starts ahead of P's border and is not below min-p
  const bool keep = t < k && (t == 0 || (ahead < target && mine >= r.min_w));
  const uint64_t which = __ballot(keep);
  if ((t & 63) == 0) s.r32[t >> 6] = (uint32_t)__popcll(which);
  __syncthreads();
  int m = 0;
  for (int i = 0; i < kSmpThreads / 64; i++) m += (int)s.r32[i];
  // by index: the kept ones' places
  const bool mine_kept = t < n && rank < m;
  const uint32_t idx = ~(uint32_t)e;
  uint64_t* by_index = s.mass;   // (falling, as rank_of counts)
  if (mine_kept) by_index[rank] = (uint64_t)(uint32_t)~idx + 1;
  if (t >= m && t < m + 8) by_index[t] = 0;
  __syncthreads();
  if (mine_kept) {
    const int at = rank_of(by_index, (uint64_t)(uint32_t)~idx + 1, m);
    g.sorted_w[at] = w;
    g.list[at] = (uint64_t)idx;
  }
  __syncthreads();
  const double kw = t < m ? g.sorted_w[t] : 0.0;
  smp_choose(a, r, row, kw, kw > 0.0 ? (int)g.list[t] : -1, 0.0, -1.0, s, [&](double, double) { return (int)g.list[t]; });
}

template <int BF>
RLXQ_DEV void smp_pick(const rlxq_sample_args& a) {
  constexpr int N = BF ? 8 : 4;
  __shared__ SmpShared s;
  __shared__ SmpPick g;
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, C = a.chunks, lane = t & 63, wave = t >> 6;
  const rlxq_sample_chunk* heads = a.heads + row * C;
  uint64_t best = 0, my_best = 0;
  double my_mass = 0.0;
  uint32_t bad = 0;
  if (t < C) my_best = heads[t].best, my_mass = heads[t].mass, bad = heads[t].bad;
  SmpRow r;
  smp_settings(a, row, r);
  const bool by_p = r.p < 1.0f, by_q = r.q > 0.0f;
  bool by_k = r.k > 0 && r.k < a.V;
  const bool borders = by_k || by_p || by_q;
  if (borders)   // (not written for the likeliest, nor read)
    for (int i = t; i < C * kGroups; i += kSmpThreads) {
      g.gmass[i / kGroups][i % kGroups] = heads[i / kGroups].group_mass[i % kGroups];
      g.gnum[i / kGroups][i % kGroups] = heads[i / kGroups].group_count[i % kGroups];
      if (i % kGroups < kHistWaves) g.tops[i / kGroups][i % kGroups] = heads[i / kGroups].tops[i % kGroups];
    }
  best = my_best;
  smp_best(best, bad, s.r64, s.r32);
  if (!smp_row(a, row, best, bad, r)) return;
  const float scale = smp_bin_scale(r.temperature), anchor = smp_anchor(smp_bin(r.top, scale));
  if (t < C) {
    const float top = of_key((uint32_t)(my_best >> 32));
    g.scale[t] = my_best ? exp_neg(((double)top - (double)r.top) * r.inv_t) : 0.0;
    const float mine = smp_anchor(smp_bin(top, scale));
    g.shift[t] = my_best ? (int)fminf((anchor - mine) * (1.0f / kGroup), (float)kGroups) : kGroups;
    g.fine[t] = smp_fine_steps(mine);
    g.top[t] = top;
    g.kept[t] = my_mass * 0x1p-48 * g.scale[t];
    g.add[t] = 0;
    g.flag[t] = 0;
  }
  if (t == 0) g.n = 0, g.n_flag = 0;
  uint64_t border = 1;
  const int lead = smp_lead<BF>(a, row);
  __syncthreads();
  if (borders) {
    // the row's groups: a wave each, a lane a chunk.  (The last is the rest.)
    for (int j = wave; j < kGroups; j += kSmpThreads / 64) {
      double m = 0.0;
      uint32_t n = 0;
      for (int c = lane; c < C; c += 64) {
        const int jj = j - g.shift[c];
        if (j == kGroups - 1) m += g.kept[c], n += by_k ? heads[c].count : 0;
        else if (jj >= 0) m += g.gmass[c][jj] * 0x1p-48 * g.scale[c], n += g.gnum[c][jj];
      }
#pragma unroll
      for (int off = 32; off; off >>= 1) m += __shfl_xor(m, off, 64), n += __shfl_xor(n, off, 64);
      if (lane == 0) g.gcum[j] = m, g.gcnt[j] = n;
    }
    __syncthreads();
    const double all = g.gcum[kGroups - 1];
    const uint32_t all_n = g.gcnt[kGroups - 1];
    __syncthreads();
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
    // bins to look into: K's border's, P's, and about min-p's
    const int kg = by_k ? first_of(g.gcnt[gl] >= (uint32_t)r.k, kGroups) : kGroups;
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
    bool small = false;   // K is little enough to be listed and sorted as a whole
    int kind = 0, j = kg, j0 = kg, j1 = by_k && !q_only ? kg : -1;   // K's group; P's groups; min-p's
#pragma unroll 1
    for (;;) {
      double lo = 0.0, hi = 0.0;
      if (kind == 0 && j > j1) {
        kind = 1, j = 0, j1 = -1;
        if (by_p && !q_only && !small) {
          lo = p * k_lo * under, hi = p * k_hi * over;
          j = j0 = group_of(lo), j1 = group_of(hi);
        }
      }
      if (kind == 1 && j > j1) {
        kind = 2, j = 0, j1 = -1;
        if (small || (!q_only && q_lo > (by_p ? p_hi : kb))) q_lo = kBins, q_hi = -1;   // min-p ends behind them
        if (q_hi >= 0) j = j0 = q_lo / kGroup, j1 = q_hi / kGroup;
      }
      if (j > j1) break;
      smp_fine(a, row, j, by_k, all, all_n, g);
      int from = 0, to = kGroup - 1;   // bins of the group whose chunks are read again
      if (kind == 0) {
        const int b = first_of(g.fcnt[bl] >= (uint32_t)r.k, kGroup);
        kb = kg * kGroup + b;
        k_ahead = b ? g.fcum[b - 1] : (kg ? g.gcum[kg - 1] : 0.0);
        k_ahead_n = b ? g.fcnt[b - 1] : (kg ? g.gcnt[kg - 1] : 0);
        k_lo = k_ahead, k_hi = g.fcum[b];
        small = g.fcnt[b] <= kSmpSort;
        from = small ? 0 : b, to = b;
        // (everything ahead of K's group too)
        if (small && t < C && g.shift[t] < kg) g.flag[t] = 1;
      } else if (kind == 1) {
        lo = p * k_lo * under, hi = p * k_hi * over;
        if (j == j0) {
          from = bin_of_mass(lo);
          p_lo = j * kGroup + from;
          p_ahead = from ? g.fcum[from - 1] : (j ? g.gcum[j - 1] : 0.0);
        }
        if (j == j1) to = bin_of_mass(hi);
        p_hi = j * kGroup + to;
      } else {
        if (j == j0) from = q_lo % kGroup;
        if (j == j1) to = q_hi % kGroup;
      }
      for (int c = t; c < C; c += kSmpThreads)   // the chunks that hold something there
        if (g.some[c] & ((2u << (to - from)) - 1) << from) g.flag[c] = 1;
      j++;
    }
    const int kp = p_lo < kb ? p_lo : kb;
    const int d_lo = q_lo < kp ? q_lo : kp;   // bins ahead of it are kept whole
    auto bin_at = [&](float v) { return smp_below(anchor, smp_bin(v, scale)); };
    // pieces (what a wave of the first launch held) to read again: of a flagged
    // chunk, and high enough for the last bin wanted
    const int d_first = small ? 0 : d_lo;
    int d_last = p_hi > q_hi ? p_hi : q_hi;
    if (kb < kBins && kb > d_last) d_last = kb;
    __syncthreads();
    for (int i = t; i < C * kHistWaves; i += kSmpThreads) {
      const int c = i / kHistWaves;
      const bool take = g.flag[c] && (d_last == kBins - 1 || bin_at(g.tops[c][i % kHistWaves]) <= d_last);
      const uint64_t which = __ballot(take);
      uint32_t at = 0;
      if (which && (int)__builtin_ctzll(which) == lane) at = atomicAdd(&g.n_flag, (uint32_t)__popcll(which));
      if (which) at = __shfl(at, __builtin_ctzll(which), 64);
      if (take) g.flagged[at + __popcll(which & ((1ull << lane) - 1))] = (uint16_t)i;
    }
    __syncthreads();
    // wanted: bins 0 .. kb, or kb, p_lo .. p_hi and q_lo .. q_hi.  One range of them is
    // from <= l scale < to, exactly, where no rounding is in the way.
    const float k0 = small ? 0.0f : (float)kb, k1 = (float)kb, p0 = (float)p_lo, p1 = (float)p_hi, q0 = (float)q_lo,
                q1 = (float)q_hi;
    const float from = anchor - (float)d_last, to = anchor - (float)d_first + 1.0f;
    const bool exact = fabsf(anchor) < 0x1p20f && d_last < kBins - 1 && (small || (!by_k && !by_p) || q_only ||
                                                                       ((kb == kBins || !by_p) && q_hi < 0));
    constexpr int kPiece = RLXQ_SAMPLE_CHUNK / kHistWaves, kPieceLane = kPiece / 64;
    const int n_flag = (int)g.n_flag;
    // (a wave's pieces are the same for its lanes; the next one that lies in the row
    // as a whole is on its way, as it is in memory)
    auto first_at = [&](int f) {
      const int i = __builtin_amdgcn_readfirstlane((int)g.flagged[f]);
      return i / kHistWaves * RLXQ_SAMPLE_CHUNK - lead + i % kHistWaves * kPiece;
    };
    auto inside = [&](int first) { return first >= 0 && first + kPiece <= a.V; };
    const int w0 = __builtin_amdgcn_readfirstlane(wave);
    constexpr int kVecs = kPieceLane / N;
    uint4 raw[kVecs];
    auto fetch = [&](int first) {
#pragma unroll
      for (int j = 0; j < kVecs; j++)
        raw[j] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.logits) +
                                                 (row * a.V + first + (j * 64 + lane) * N) * (BF ? 2 : 4));
    };
    int next = 0;
    if (w0 < n_flag) {
      next = first_at(w0);
      if (inside(next)) fetch(next);
    }
#pragma unroll 1
    for (int f = w0; f < n_flag; f += kSmpThreads / 64) {
      const int here = next;
      float v[kPieceLane];
      if (inside(here)) {
#pragma unroll
        for (int j = 0; j < kVecs; j++) smp_unpack<BF>(raw[j], v + j * N);
      } else {
#pragma unroll
        for (int j = 0; j < kVecs; j++) smp_ld16<BF>(a, row, here + (j * 64 + lane) * N, v + j * N, false);
      }
      if (f + kSmpThreads / 64 < n_flag) {
        next = first_at(f + kSmpThreads / 64);
        if (inside(next)) fetch(next);
      }
      // (no short circuits: a branch an element costs more than the comparisons)
      uint64_t hit[kPieceLane];
      uint32_t hits = 0;
      if (exact) {
#pragma unroll
        for (int i = 0; i < kPieceLane; i++) {
          const float x = v[i] * scale;
          hit[i] = __ballot(x >= from) & __ballot(x < to);
          hits += (uint32_t)__popcll(hit[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPieceLane; i++) {
          const float d = fminf(anchor - smp_bin(v[i], scale), (float)(kBins - 1));
          hit[i] = ((__ballot(d >= k0) & __ballot(d <= k1)) | (__ballot(d >= p0) & __ballot(d <= p1)) |
                    (__ballot(d >= q0) & __ballot(d <= q1))) & __ballot(v[i] != -__builtin_inff());
          hits += (uint32_t)__popcll(hit[i]);
        }
      }
      if (!hits) continue;
      // a place in the list for all of the wave's at once
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&g.n, hits);
      at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
      for (int i = 0; i < kPieceLane; i++) {
        if (!hit[i]) continue;
        const uint32_t mine = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(hit[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit[i], 0));
        if ((bool)(hit[i] >> lane & 1) & (mine < kSmpList))
          g.list[mine] = smp_comp(key_of(v[i]), here + ((i / N) * 64 + lane) * N + i % N);
        at += (uint32_t)__popcll(hit[i]);
      }
    }
    __syncthreads();
    const int n = (int)g.n;
    auto each = [&](auto&& f) { smp_each<BF>(a, row, lead, g, f); };
    if (small) {
      smp_small(a, r, row, n, g, s);
      return;
    }
    if (!q_only && (by_k || by_p)) {
      // (the bins' range in smp_comp, or more: the bins' numbers decide)
      constexpr float kMost = 3.402823466e38f;
      auto lowest = [&](int d) {
        float x = (anchor - (float)(d + 1)) / scale;
        x -= fabsf(x) * 0x1p-20f;
        return d >= kBins - 1 ? 1ull : smp_comp(key_of(x > -kMost ? x : -kMost), 0xffffffffu);
      };
      auto highest = [&](int d) {
        float x = (anchor - (float)(d - 2)) / scale;
        x += fabsf(x) * 0x1p-20f;
        x = x < kMost ? x : kMost;
        return smp_comp(key_of(x < r.top ? x : r.top), 0);
      };
      double mass_k = all;
#pragma unroll 1
      for (int by = by_k ? 0 : 1; by < (by_p ? 2 : 1); by++) {   // K's border, then P's
        // (what is not in K is behind its border)
        const int b0 = by ? p_lo : kb, b1 = by ? p_hi : kb;
        uint64_t lo = lowest(b1);
        lo = lo > border ? lo : border;
        double incl;
        border = smp_select(by == 0, r, g, s, n, each, bin_at, b0, b1, lo, highest(b0), by ? p_ahead : k_ahead, by ? 0 : k_ahead_n,
                            (uint32_t)r.k, p * mass_k, &incl);
        mass_k = incl;
      }
    }
    // the chunks' kept mass: whole groups and bins, and what is listed (without any
    // border, as where top_k is more than what is not masked, the whole chunk's)
    if (d_lo < kBins) {
      for (int c0 = 0; c0 < C; c0 += 16) {
        const int c = c0 + (t >> 5), b = t & 31, jj = c < C ? d_lo / kGroup - g.shift[c] : -1;
        double m = 0.0;
        if (jj >= 0) {
          if (b < d_lo % kGroup) m = smp_bin_mass(a.masses[(row * C + c) * kBins + jj * kGroup + b], jj * kGroup + b, g.fine[c]);
          if (b < jj) m += g.gmass[c][b];
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) m += __shfl_xor(m, off, 32);
        if (c < C && b == 0) g.kept[c] = m * 0x1p-48 * g.scale[c];
      }
      auto add = [&](uint64_t e) {
        const float x = of_key((uint32_t)(e >> 32));
        if (e < border || bin_at(x) < d_lo) return;
        if (by_q && smp_w(r, x) < r.min_w) return;
        // (beside the chunk's largest: 4096 of up to 2^51)
        const int c = ((int)~(uint32_t)e + lead) / RLXQ_SAMPLE_CHUNK;
        atomicAdd(&g.add[c], (unsigned long long)(exp_neg(((double)x - (double)g.top[c]) * r.inv_t) * 0x1p51 + 0.5));
      };
      if (n <= kSmpList)
        for (int i = t; i < n; i += kSmpThreads) add(g.list[i]);
      else
        each(add);
    }
    __syncthreads();
  }
  // the chunk, then the element
  const double m = t < C ? g.kept[t] + (double)g.add[t] * 0x1p-51 * g.scale[t] : 0.0;
  double ahead, total;
  const double incl = smp_scan<double>(m, s.rd, &ahead, &total);
  const double target = smp_target(r, total);
  if (t == 0) s.found = 0x7fffffff, s.last = -1;
  __syncthreads();
  const uint64_t some = __ballot(m > 0.0), past = __ballot(m > 0.0 && incl > target);
  if (lane == 0 && some) atomicMax(&s.last, t + 63 - __builtin_clzll(some));
  if (lane == 0 && past) atomicMin(&s.found, t + __builtin_ctzll(past));
  __syncthreads();
  const int c = s.found != 0x7fffffff ? s.found : (s.last > 0 ? s.last : 0);
  if (t == c) g.before = ahead;
  __syncthreads();
  constexpr int kPer = RLXQ_SAMPLE_CHUNK / kSmpThreads;
  const int first = c * RLXQ_SAMPLE_CHUNK - lead;
  float v[kPer];
  smp_ld_chunk<BF, kPer / N>(a, row, first, t * (kPer / N), 1, v);
  float* mine = reinterpret_cast<float*>(g.list) + t;   // (its elements, kSmpThreads apart; nothing listed is read any more)
#pragma unroll
  for (int j = 0; j < kPer; j++) mine[j * kSmpThreads] = v[j];
  double kept = 0.0;
  int last = -1;
#pragma unroll 4
  for (int j = 0; j < kPer; j++) {
    const double w = smp_kept(r, border, mine[j * kSmpThreads], first + t * kPer + j);
    kept += w;
    if (w > 0.0) last = first + t * kPer + j;
  }
  smp_choose(a, r, row, kept, last, g.before, total, s, [&](double sum, double goal) {
    for (int j = 0; j < kPer; j++) {
      const int i = first + t * kPer + j;
      if (i == last) break;
      const double w = smp_kept(r, border, mine[j * kSmpThreads], i);
      sum += w;
      if (sum > goal && w > 0.0) return i;
    }
    return last;
  });
}

}  // namespace rlxq

using namespace rlxq;

extern "C" __global__ __launch_bounds__(kHistThreads, 4) void rlxq_sample_hist_f32(rlxq_sample_args a) { smp_hist<0>(a); }
extern "C" __global__ __launch_bounds__(kHistThreads, 4) void rlxq_sample_hist_bf16(rlxq_sample_args a) { smp_hist<1>(a); }
extern "C" __global__ __launch_bounds__(kSmpThreads) void rlxq_sample_pick_f32(rlxq_sample_args a) { smp_pick<0>(a); }
extern "C" __global__ __launch_bounds__(kSmpThreads) void rlxq_sample_pick_bf16(rlxq_sample_args a) { smp_pick<1>(a); }
