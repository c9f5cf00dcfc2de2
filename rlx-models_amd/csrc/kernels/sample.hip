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

constexpr int kSmpThreads = 1024;

// What a row asks for, and its largest logit.
struct SmpRow {
  double inv_t;
  float top;             // the largest logit
  float p, q, u;
  int k;                 // 0: off
  bool greedy;
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
  int found;
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
    // bins from the top: thread t holds bins bins - 1 - 2t and the one below
    uint64_t m0 = 0, m1 = 0;
    uint32_t c0 = 0, c1 = 0;
    const int b0 = bins - 1 - 2 * t, b1 = b0 - 1;
    if (b0 >= 0) m0 = s.mass[b0], c0 = s.count[b0];
    if (b1 >= 0) m1 = s.mass[b1], c1 = s.count[b1];
    uint64_t mt;
    uint32_t ct;
    const uint64_t mi = smp_scan<uint64_t>(m0 + m1, s.r64, &mt);
    const uint32_t ci = smp_scan<uint32_t>(c0 + c1, s.r32, &ct);
    // the last bin with anything in it ends the search where rounding left the
    // target above the whole mass
    const uint64_t mb = mass_above + mi - m0 - m1;
    const uint64_t cb = above + ci - c0 - c1;
    auto crosses = [&](uint64_t before_m, uint64_t m, uint64_t before_c, uint64_t c, uint64_t all_c) {
      if (!c) return false;
      if (BY == 0) return before_c < need && before_c + c >= need;
      const bool first = before_m < need || before_c == 0;
      return first && (before_m + m >= need || before_c + c == all_c);
    };
    const uint64_t all_c = above + ct;
    if (crosses(mb, m0, cb, c0, all_c)) s.pick = b0, s.pick_mass = mb, s.pick_count = (uint32_t)cb;
    if (crosses(mb + m0, m1, cb + c0, c1, all_c)) s.pick = b1, s.pick_mass = mb + m0, s.pick_count = (uint32_t)(cb + c0);
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

// Smallest key whose weight reaches q (0 < q <= 1), as a border ahead of every
// index: the weight does not fall with the key.
RLXQ_DEV uint64_t smp_min_p(const SmpRow& r) {
  const double q = r.q < 1.0f ? (double)r.q : 1.0;
  uint32_t hi = key_of(r.top), lo = 0;   // weight(hi) = 1 >= q; weight(lo) counts as below
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (smp_w(r, of_key(mid)) >= q) hi = mid;
    else lo = mid;
  }
  return smp_comp(hi, 0xffffffffu);
}

}  // namespace rlxq

using namespace rlxq;

// A workgroup a row, the row read again for every digit.
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
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    const uint64_t o = __shfl_xor(best, off, 64);
    best = o > best ? o : best;
    bad |= __shfl_xor(bad, off, 64);
  }
  if ((t & 63) == 0) s.r64[t >> 6] = best, s.r32[t >> 6] = bad;
  __syncthreads();
  best = 0;
  for (int w = 0; w < kSmpThreads / 64; w++) {
    best = s.r64[w] > best ? s.r64[w] : best;
    bad |= s.r32[w];
  }
  __syncthreads();
  SmpRow r;
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  r.u = a.u[row];
  if (bad || !best || T != T || r.u != r.u) {
    if (t == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = __builtin_nanf("");
    }
    return;
  }
  r.top = of_key((uint32_t)(best >> 32));
  r.greedy = !(T > 0.0f);
  if (r.greedy) {
    if (t == 0) {
      a.tokens[row] = (int32_t)~(uint32_t)best;
      if (a.probs) a.probs[row] = 1.0f;
    }
    return;
  }
  r.inv_t = 1.0 / (double)T;
  r.k = a.top_k ? a.top_k[row] : 0;
  r.p = a.top_p ? a.top_p[row] : 1.0f;
  r.q = a.min_p ? a.min_p[row] : 0.0f;
  // fixed point: the whole row's mass below 2^62
  const int lg = 32 - __builtin_clz((uint32_t)a.V);
  const double one = (double)(1ull << (62 - lg));
  uint64_t border = 1, mass = 0;   // every element that is not masked
  auto mass_of = [&](uint64_t from) {
    uint64_t m = 0;
    for (int i = t; i < a.V; i += kSmpThreads) {
      const float v = smp_ld(a, row, i);
      const uint32_t key = key_of(v);
      if (key && smp_comp(key, i) >= from) m += (uint64_t)(smp_w(r, v) * one + 0.5);
    }
    uint64_t all;
    (void)smp_scan<uint64_t>(m, s.r64, &all);
    __syncthreads();
    return all;
  };
  if (r.k > 0 && r.k < a.V) {
    // (fewer than k that are not masked: all of them)
    uint32_t n = 0, all;
    for (int i = t; i < a.V; i += kSmpThreads) n += key_of(smp_ld(a, row, i)) != 0;
    (void)smp_scan<uint32_t>(n, s.r32, &all);
    __syncthreads();
    if ((uint32_t)r.k < all) border = smp_radix<0>(a, r, row, border, one, (uint64_t)r.k, s, &mass);
  }
  if (r.p < 1.0f) {
    mass = mass_of(border);
    const double want = r.p > 0.0f ? (double)r.p * (double)mass : 0.0;
    uint64_t need = (uint64_t)want;
    need += (double)need < want;
    border = smp_radix<1>(a, r, row, border, one, need, s, &mass);
  }
  if (r.q > 0.0f) {
    const uint64_t m = smp_min_p(r);
    border = m > border ? m : border;
  }
  // the kept mass in index order: every thread a run of the row
  const int per = (a.V + kSmpThreads - 1) / kSmpThreads, lo = t * per, hi = lo + per < a.V ? lo + per : a.V;
  auto weight = [&](int i) {
    const float v = smp_ld(a, row, i);
    const uint32_t key = key_of(v);
    return key && smp_comp(key, i) >= border ? smp_w(r, v) : 0.0;
  };
  double m = 0.0, total;
  int last = -1;
  for (int i = lo; i < hi; i++) {
    const double w = weight(i);
    m += w;
    if (w > 0.0) last = i;
  }
  const double incl = smp_scan<double>(m, s.rd, &total);
  const double target = (double)r.u * total;
  if (t == 0) s.found = 0x7fffffff, s.pick = 0;
  __syncthreads();
  if (last >= 0) atomicMax((int*)&s.pick, last);
  if (m > 0.0 && incl > target) {
    double c = incl - m;
    for (int i = lo; i < hi; i++) {
      const double w = weight(i);
      c += w;
      if (w > 0.0 && c > target) {
        atomicMin(&s.found, i);
        break;
      }
    }
  }
  __syncthreads();
  if (t == 0) {
    const int tok = s.found == 0x7fffffff ? (int)s.pick : s.found;
    a.tokens[row] = tok;
    if (a.probs) a.probs[row] = (float)(weight(tok) / total);
  }
}
