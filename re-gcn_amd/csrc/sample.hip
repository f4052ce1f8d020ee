// Sampling ids from scores with temperature, top-k, top-p and min-p, from given random numbers.
//
// For a row s of N scores (NaN and -inf are never taken), in the order "larger score first, ties by
// lower index":
//   w_i = exp((s_i - max s) / T)
//   kept: the first k;  of those the shortest prefix whose weights reach p times their sum;  w_i >= m
//   id(u) = the lowest i whose running sum (by index) of kept weights exceeds u * (sum of kept weights)
// T <= 0 takes the first of the order.  A row without a score to take gives -1.
//
// Weights are whole numbers: round(w 2^S) with 2^S N <= 2^63 (S <= 51), from a 64-bit exp.  Their sums are
// exact in any order, so histograms by atomics, partial sums and prefix sums agree bit for bit.  What the rounding
// loses is at most N 2^-(S+1) of the largest weight: 2^-37 at 2,048 scores, 2^-33 at 32,768, 2^-24 at 2^20, 2^-16 at 2^24, where
// a weight below 2^-40 (28 T under the largest) is 0.
//
// No sort.  Each of k and p asks for the place in the order where a running sum (of ones, of weights) reaches
// a target: a histogram over 2048 bins of the scores finds the bin, whose few members then add up the members
// before them.  A bin that holds too many (ties, scores far from each other) is cut into bins again, twice in a
// row held in LDS; then a radix descent over the scores' bits as ordered keys goes on from it, and one over the
// indices of equal scores.  So a kept set is {score > c} and {score = c, index <= i}.  (3080 x 23033, k = 50 or p = 0.9:
// 0.20 and 0.32 ms; two different scores 0.7 and 0.8; scores a million T apart 0.6 and 0.25.  16 x 1,000,000: 0.08 and
// 0.16 ms, and 1.3 to 1.9 where the descent reads the row, by one workgroup.)
//
// k_sample: a workgroup takes a row of up to 32768 scores, which stay in its LDS (one read of them; in
// registers, the compiler spilled them around the exponentials).  What bounds it is the issue of vector
// instructions, about 90 per score with top_p: 30 for its exponential (a second one for the scores it keeps), the
// rest for loads, bins and sums.  3080 x 23033, p = 0.9: 319 us again and again on one input, 349 on inputs that change, whose
// 284 MB would take 60.
// k_spread_*: longer rows are cut into segments of 8192 scores, a workgroup each, in launches that pass
// histograms, the bin's members and the segments' sums through a workspace.
#include "elem.h"
#include "regcn_internal.h"

namespace regcn {
namespace {

constexpr int HBITS = 11, HBINS = 1 << HBITS;
constexpr int ROW_MAX = 32768;  // scores of a row held in LDS
constexpr int LIST = 256;       // members of a bin that are put in order one against the other
constexpr int SEG = 8192, SEG_THR = 512;
constexpr int MAX_COLS = 1 << 24;
// A launch has fewer than 2^32 threads along a dimension: rows (up to 1024 threads each) and draws (SEG_THR) of one.
constexpr int LAUNCH_ROWS = 1 << 21, LAUNCH_DRAWS = 1 << 22;
constexpr int MAX_DRAWS = 1 << 30;
constexpr uint32_t ALL = 0xffffffffu;
constexpr int NO_TIE = 0x7fffffff;
constexpr float LOWEST = -3.402823466e+38f;

// Constants of scaled_exp, as kernel arguments: in scalar registers each is an operand of its fma (as literals
// the compiler copies every one into vector registers first, a third of the instructions).
struct ExpConsts {
  double log2e, round, ln2_hi, ln2_lo, p[11];  // p: 1 / 12!, ..., 1 / 2!
};

struct RowArgs {
  const void* score;
  int64_t ld;
  int32_t rows, cols, draws, u_wide;
  const void* u;
  double temperature, top_p, min_p;
  int32_t top_k, shift;  // shift: S
  const void *temperature_v, *top_p_v, *min_p_v;
  const int32_t* top_k_v;
  int32_t rows_wide;  // which of the three are doubles: bits 0, 1, 2
  int64_t* ids;
  float* logp;
  ExpConsts c;
};

struct Limits {
  double inv_t, top_p, min_w;  // min_w: min_p 2^S
  uint32_t top_k;              // ALL: off
  int shift;
  // set once the row's largest score is known
  float top;
  bool ties_only;  // an infinite score, or a temperature whose inverse is: weight only on the largest
};

__device__ __forceinline__ double row_value(const void* v, int wide, int row, double all) {
  return !v ? all : wide ? ((const double*)v)[row] : (double)((const float*)v)[row];
}

__device__ __forceinline__ Limits row_limits(const RowArgs& a, int row) {
  Limits l;
  const double t = row_value(a.temperature_v, a.rows_wide & 1, row, a.temperature);
  const int k = a.top_k_v ? a.top_k_v[row] : a.top_k;
  const double m = row_value(a.min_p_v, a.rows_wide & 4, row, a.min_p);
  l.top_p = row_value(a.top_p_v, a.rows_wide & 2, row, a.top_p);
  l.min_w = m > 0 ? __builtin_ldexp(m < 1.0 ? m : 1.0, a.shift) : 0.0;
  l.top_k = k > 0 && k < a.cols ? (uint32_t)k : ALL;
  l.inv_t = 1.0 / t;
  if (!(t > 0)) {  // greedy
    l.inv_t = 1.0;
    l.top_k = 1;
  }
  l.shift = a.shift;
  return l;
}

__device__ __forceinline__ void set_top(Limits& l, float top) {
  l.top = top;
  l.ties_only = !(fabsf(top) < __builtin_inff() && l.inv_t < __builtin_inf());
}

// A score as the rest of this file sees it: -0 as 0, NaN as -inf (never taken).
__device__ __forceinline__ float canonical(float s) { return s > -__builtin_inff() ? s + 0.f : -__builtin_inff(); }

// Whole numbers in the order of the scores, above 0.
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t b = __float_as_uint(s);
  return b ^ ((int32_t)b < 0 ? ALL : 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t k) { return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : ALL)); }

// exp(x) 2^S for x = (s - top) / T <= 0.  exp(x) = 2^n p(r), r = x - n ln 2 in two parts, |r| <= ln 2 / 2;
// p is the Taylor polynomial of degree 12 (remainder below 2^-52 of p).  n comes out of the low bits of
// x / ln 2 + 1.5 2^52 and goes into the exponent of p by an integer add (n + S >= -1010: still normal).
__device__ __forceinline__ double scaled_exp(float s, const Limits& l, const ExpConsts& c) {
  const double x = fmax(((double)s - (double)l.top) * l.inv_t, -700.0);
  const double t = fma(x, c.log2e, c.round);
  const double n = t - c.round;
  double r = fma(n, c.ln2_hi, x);
  r = fma(n, c.ln2_lo, r);
  double p = fma(c.p[0], r, c.p[1]);
#pragma unroll
  for (int j = 2; j < 11; ++j) p = fma(p, r, c.p[j]);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int e = (int)(uint32_t)__double_as_longlong(t) + l.shift;
  return __hiloint2double(__double2hiint(p) + (e << 20), __double2loint(p));
}

// To the nearest whole number: adding 2^52 to a number up to 2^51 leaves it in the low bits.
__device__ __forceinline__ uint64_t whole(double v) { return __double_as_longlong(v + 0x1p52) & ((1ull << 52) - 1); }

__device__ __forceinline__ uint64_t weight(float s, const Limits& l, const ExpConsts& c) {
  if (l.ties_only) return s == l.top ? 1ull << l.shift : 0;
  return whole(scaled_exp(s, l, c));
}

// A place in the order: everything with a larger score, and of its own score the indices up to idx.  Every
// score that may be taken: {LOWEST, NO_TIE}.
struct Cut {
  float s;
  int idx;
  __device__ bool keeps(float x, int i) const { return x > s || (x == s && i <= idx); }
  // The shorter of two kept sets, of which `from` holds this one: a cut found among from's knows nothing of the
  // equal scores that from leaves out.
  __device__ Cut within(const Cut& from) const { return {s, s == from.s && from.idx < idx ? from.idx : idx}; }
};

// The weights of VE consecutive scores, 0 where a limit leaves one out.  No branch a score: the exponentials
// run together, and where no lane keeps one they are passed over.
template <int VE>
__device__ __forceinline__ void kept_weights(const float* s, int i0, const Cut& cut, const Limits& l, const ExpConsts& c,
                                             uint64_t (&w)[VE]) {
  bool keep[VE], some = false;
  if (cut.idx == NO_TIE) {
#pragma unroll
    for (int e = 0; e < VE; ++e) some |= keep[e] = s[e] >= cut.s;
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) some |= keep[e] = cut.keeps(s[e], i0 + e);
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) w[e] = 0;
  if (!some) return;
  if (l.ties_only) {
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = keep[e] && s[e] == l.top ? 1ull << l.shift : 0;
    return;
  }
  if (l.min_w > 0) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const double v = scaled_exp(s[e], l, c);
      w[e] = whole(keep[e] && v >= l.min_w ? v : 0.0);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) w[e] = whole(keep[e] ? scaled_exp(s[e], l, c) : 0.0);
}

// ------------------------------------------------------------------------------- sums over lanes
template <int CTRL, int ROWS, bool ZERO>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, ZERO);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, ZERO);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int l) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
// Inclusive prefix over the wave: shifts within rows of 16 lanes, then row totals broadcast to the rows after.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  v += dpp64<0x111, 0xF, true>(v);  // row_shr:1, 2, 4, 8 (0 shifted in)
  v += dpp64<0x112, 0xF, true>(v);
  v += dpp64<0x114, 0xF, true>(v);
  v += dpp64<0x118, 0xF, true>(v);
  v += dpp64<0x142, 0xA, false>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp64<0x143, 0xC, false>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}

template <int THR>
struct Shared {
  uint64_t hist[HBINS];  // later: the threads' running sums
  uint64_t wave[16];
  uint64_t above, sum, value[LIST];
  uint2 list[LIST];  // {score, index}
  uint32_t bin, count, kmax, kmin_inv, lo_inv, hi;
  Cut cut;
};

// Exclusive prefix of v over the workgroup's threads; *total: the sum.  Two barriers.
template <int THR>
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t* wave, uint64_t* total) {
  constexpr int W = THR / WAVE;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t inc = wave_scan64(v);
  __syncthreads();  // wave[] may still be read from the call before
  if (lane == 63) wave[w] = inc;
  __syncthreads();
  const uint64_t sums = wave_scan64(lane < W ? wave[lane & (W - 1)] : 0);
  *total = readlane64(sums, W - 1);
  const uint64_t base = w ? readlane64(sums, __builtin_amdgcn_readfirstlane(w - 1 < 0 ? 0 : w - 1)) : 0;
  return base + inc - v;
}

// ------------------------------------------------------------------------------ places in the order
// The bin of hist in which the running sum, `above` before bin 0, reaches the target: into sh.bin, with the
// sum before it in sh.above and its own in sh.sum (1 <= target - above <= the histogram's total).  target_of
// gives the target from the total; it is returned.
template <int THR, typename Target>
__device__ __forceinline__ uint64_t find_bin(Shared<THR>& sh, const uint64_t* hist, uint64_t above, Target target_of) {
  constexpr int PER = HBINS / THR;
  uint64_t own = 0, total, h[PER];
#pragma unroll
  for (int b = 0; b < PER; ++b) own += h[b] = hist[threadIdx.x * PER + b];
  uint64_t before = above + block_scan64<THR>(own, sh.wave, &total);
  const uint64_t target = target_of(total);
  if (before < target && before + own >= target) {  // one thread's
#pragma unroll
    for (int b = 0; b < PER; ++b) {
      if (before < target && before + h[b] >= target) {
        sh.above = before;
        sh.bin = threadIdx.x * PER + b;
        sh.sum = h[b];
      }
      before += h[b];
    }
  }
  __syncthreads();
  return target;
}

__device__ __forceinline__ uint64_t count_target(const Limits& l, uint64_t total) { return min((uint64_t)l.top_k, total); }
__device__ __forceinline__ uint64_t weight_target(const Limits& l, uint64_t total) {
  const double t = ceil(l.top_p * (double)total);
  return t < 1.0 ? (uint64_t)1 : min(total, (uint64_t)t);
}

// Bins of the scores on a linear scale from the largest down, over at most 44 T (weights below exp(-44) are
// none); the last bin is open.  fp32: monotone, which is all that a bin has to be.
__device__ __forceinline__ uint32_t value_bin(float s, float top, float per) {
  return (uint32_t)fminf((top - s) * per, (float)(HBINS - 1));
}
__device__ __forceinline__ float bins_per(float smin, const Limits& l) {
  return (float)HBINS / fminf(l.top - smin, (float)(44.0 / l.inv_t));
}
__device__ __forceinline__ bool bins_work(float per, const Limits& l) { return per > 0.f && per < 1e30f && !l.ties_only; }

// The scores that bins are made of: from the largest, of bin 0, down to the smallest.
struct Bins {
  float top, low, per;
};

// The bin of each of VE scores receives its one or its weight.
template <bool WEIGHTS, int VE>
__device__ __forceinline__ void add_to_bins(uint64_t* hist, const float* s, int i0, const Cut& from, const Bins& b,
                                            const Limits& l, const ExpConsts& c) {
  uint64_t w[VE];
  if (WEIGHTS) {
    kept_weights<VE>(s, i0, from, l, c, w);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = 1;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (w[e] && s[e] >= b.low && s[e] <= b.top)
      atomicAdd((unsigned long long*)&hist[value_bin(s[e], b.top, b.per)], (unsigned long long)w[e]);
}

// The members of a bin among VE scores: f(score, index).
template <int VE, typename F>
__device__ __forceinline__ void members(const float* s, int i0, const Cut& from, uint32_t bin, const Bins& b, F f) {
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (value_bin(s[e], b.top, b.per) == bin && s[e] >= b.low && s[e] <= b.top && from.keeps(s[e], i0 + e)) f(s[e], i0 + e);
}

// The cut among the `count` <= LIST members in sh.list, `above` before them.
template <bool WEIGHTS, int THR>
__device__ __forceinline__ Cut order_list(Shared<THR>& sh, int count, uint64_t above, uint64_t target, const Limits& l,
                                          const ExpConsts& c) {
  uint2 me = make_uint2(0, 0);
  uint64_t own = 0, before = above;
  if ((int)threadIdx.x < count) {
    me = sh.list[threadIdx.x];
    own = WEIGHTS ? weight(__uint_as_float(me.x), l, c) : 1;
    sh.value[threadIdx.x] = own;
  }
  __syncthreads();
  if ((int)threadIdx.x < count) {
    const float s = __uint_as_float(me.x);
    bool last = true;  // of its score
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const uint2 o = sh.list[j];
      const float x = __uint_as_float(o.x);
      before += x > s || (x == s && o.y < me.y) ? sh.value[j] : 0;
      last &= !(x == s && o.y > me.y);
    }
    if (before < target && before + own >= target) sh.cut = Cut{s, last ? NO_TIE : (int)me.y};  // one thread's
  }
  __syncthreads();
  const Cut cut = sh.cut;
  __syncthreads();  // sh may be written again
  return cut;
}

// Radix descent in decreasing order of keys in [lo, hi]: the key at which the running sum of values, `above`
// before hi, reaches the target.  each(f) calls f(key, value functor).
struct Place {
  uint32_t key;
  uint64_t above, sum, target;  // sums before the key, of the key
};
template <int THR, typename Each, typename Target>
__device__ Place descend(Shared<THR>& sh, uint32_t lo, uint32_t hi, uint64_t above, Each each, Target target_of) {
  uint64_t target = 0;
  for (bool first = true;; first = false) {
    const uint32_t range = hi - lo;
    const int bits = range ? 32 - __builtin_clz(range) : 0;
    const int shift = bits > HBITS ? bits - HBITS : 0;
    for (int b = threadIdx.x; b < HBINS; b += THR) sh.hist[b] = 0;
    __syncthreads();
    each([&](uint32_t k, auto value) {
      if (k >= lo && k <= hi) atomicAdd((unsigned long long*)&sh.hist[(hi - k) >> shift], (unsigned long long)value());
    });
    __syncthreads();
    target = find_bin<THR>(sh, sh.hist, above, [&](uint64_t total) { return first ? target_of(total) : target; });
    above = sh.above;
    const uint32_t top = hi - (sh.bin << shift), low = (1u << shift) - 1;
    lo = max(lo, top >= low ? top - low : 0);
    hi = top;
    if (shift == 0) break;
  }
  const Place p{hi, above, sh.sum, target};
  __syncthreads();  // sh may be written again
  return p;
}

// The cut by descent, over the scores that src.each(f(score, index)) gives (all of them taken).
template <bool WEIGHTS, int THR, typename Source, typename Target>
__device__ Cut descend_cut(const Source& src, Shared<THR>& sh, uint32_t kmin, uint32_t kmax, uint64_t above, int cols,
                           const Limits& l, const ExpConsts& c, Target target_of) {
  const Place p = descend<THR>(
      sh, kmin, kmax, above,
      [&](auto f) {
        src.each([&](float s, int) { f(key_of(s), [&] { return WEIGHTS ? weight(s, l, c) : (uint64_t)1; }); });
      },
      target_of);
  // one score left: its elements each add the same; the lowest indices are kept
  const float s = score_of(p.key);
  const uint64_t one = WEIGHTS ? weight(s, l, c) : 1;
  const uint64_t need = one ? (p.target - p.above + one - 1) / one : 1, have = one ? p.sum / one : 1;
  if (need >= have) return Cut{s, NO_TIE};
  const Place q = descend<THR>(
      sh, ALL - (uint32_t)(cols - 1), ALL, 0,
      [&](auto f) {
        src.each([&](float x, int i) {
          if (x == s) f(ALL - (uint32_t)i, [] { return (uint64_t)1; });
        });
      },
      [&](uint64_t) { return need; });
  return Cut{s, (int)(ALL - q.key)};
}

// ------------------------------------------------------------------------------------- draws
// The number in [0, sum) that the drawn u stands for; NaN and negative u: 0.
__device__ __forceinline__ uint64_t draw_at(const RowArgs& a, int64_t at, uint64_t sum) {
  const double u = a.u_wide ? ((const double*)a.u)[at] : (double)((const float*)a.u)[at];
  const double x = u > 0.0 ? u * (double)sum : 0.0;
  return x < (double)sum ? min((uint64_t)x, sum - 1) : sum - 1;
}
__device__ __forceinline__ void store_draw(const RowArgs& a, int64_t at, int id, float s, uint64_t sum, const Limits& l) {
  a.ids[at] = id;
  if (a.logp) {
    const double log_sum = log(__builtin_ldexp((double)sum, -l.shift));  // a sum of one weight 1: exactly 0
    a.logp[at] = (float)((s == l.top ? 0.0 : ((double)s - (double)l.top) * l.inv_t) - log_sum);
  }
}
__device__ __forceinline__ void store_none(const RowArgs& a, int64_t at) {
  a.ids[at] = -1;
  if (a.logp) a.logp[at] = -__builtin_inff();
}

// VE scores from p (m of them within the row), -inf past it.
template <typename T>
__device__ __forceinline__ void load_scores(float (&s)[Piece<T>::VE], const T* p, int m) {
  constexpr int VE = Piece<T>::VE;
  if (m > 0) load_piece<T>(s, p, m);
#pragma unroll
  for (int e = 0; e < VE; ++e) s[e] = e < m ? canonical(s[e]) : -__builtin_inff();
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor(v, o));
  return v;
}

// ----------------------------------------------------------------------------- a row a workgroup
// The row in LDS, a multiple of 4 THR scores (-inf past its end): piece q of thread t is the 4 scores from
// (q THR + t) 4 on.
template <int THR>
struct LdsRow {
  const float* s;
  int pieces;
  template <typename F>
  __device__ __forceinline__ void each4(F f) const {
    for (int q = 0; q < pieces; ++q) {
      const int i0 = (q * THR + (int)threadIdx.x) * 4;
      const f4 v = *reinterpret_cast<const f4*>(s + i0);
      const float x[4] = {v.x, v.y, v.z, v.w};
      f(x, i0);
    }
  }
  // The same over this thread's consecutive scores.
  template <typename F>
  __device__ __forceinline__ void own4(F f) const {
    for (int q = 0; q < pieces; ++q) {
      const int i0 = ((int)threadIdx.x * pieces + q) * 4;
      const f4 v = *reinterpret_cast<const f4*>(s + i0);
      const float x[4] = {v.x, v.y, v.z, v.w};
      f(x, i0);
    }
  }
  // Weights of what a cut keeps of them: where that is up to a quarter of the wave's scores (as the first four of each lane's
  // consecutive ones tell), each lane takes its own one after the other; else all the wave's, four at a time.
  // (3080 x 23033 on one input: p = 0.9 346 -> 320 us, k = 500 and p = 0.9 390 -> 343 by the sums and -> 304 by the bins; p = 0.999
  // 348 -> 356, and 384 without the second way.)
  __device__ __forceinline__ bool few(const Cut& cut) const {
    if (!(cut.s > LOWEST)) return false;
    const int i0 = (int)threadIdx.x * pieces * 4;
    int n = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) n += __popcll(__ballot(cut.keeps(s[i0 + e], i0 + e)));
    return n <= WAVE;
  }
  template <typename F>
  __device__ __forceinline__ void each_kept(const Cut& cut, F f) const {
    const int begin = (int)threadIdx.x * pieces * 4;
    uint32_t kept = 0;  // pieces <= 8
    own4([&](const float* x, int i0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) kept |= (uint32_t)cut.keeps(x[e], i0 + e) << (i0 - begin + e);
    });
    for (; kept; kept &= kept - 1) {
      const int i = begin + __builtin_ctz(kept);
      f(s[i], i);
    }
  }
};

// Those of a row that a cut keeps.
template <typename Row>
struct Among {
  const Row& row;
  Cut from;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    row.each4([&](const float* x, int i0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x[e] >= LOWEST && from.keeps(x[e], i0 + e)) f(x[e], i0 + e);
    });
  }
};

template <bool WEIGHTS, int THR, typename Target>
__device__ Cut find_cut(const LdsRow<THR>& row, Shared<THR>& sh, uint32_t kmin, int cols, const Cut from, const Limits& l,
                        const ExpConsts& c, Target target_of) {
  uint64_t above = 0, target = 0;
  uint32_t kmax = key_of(l.top);
  Bins bins{l.top, score_of(kmin), bins_per(score_of(kmin), l)};
  // a bin with too many members becomes bins itself, twice
  for (int round = 0; round < 3 && kmin < kmax && bins_work(bins.per, l); ++round) {
    for (int b = threadIdx.x; b < HBINS; b += THR) sh.hist[b] = 0;
    if (threadIdx.x == 0) sh.count = sh.lo_inv = sh.hi = 0;
    __syncthreads();
    const auto add = [&](const float* x, int i0) { add_to_bins<WEIGHTS, 4>(sh.hist, x, i0, from, bins, l, c); };
    if (!WEIGHTS || !(from.s > LOWEST))
      row.each4(add);
    else if (row.few(from))  // a wave's choice: both ways take the threads' consecutive scores
      row.each_kept(from, [&](float s, int i) { add_to_bins<WEIGHTS, 1>(sh.hist, &s, i, from, bins, l, c); });
    else
      row.own4(add);
    __syncthreads();
    target = find_bin<THR>(sh, sh.hist, above, [&](uint64_t total) { return round ? target : target_of(total); });
    above = sh.above;
    const uint32_t bin = sh.bin;
    uint32_t lo_inv = 0, hi = 0;
    row.each4([&](const float* x, int i0) {
      members<4>(x, i0, from, bin, bins, [&](float s, int i) {
        const uint32_t at = atomicAdd(&sh.count, 1u);
        if (at < LIST) sh.list[at] = make_uint2(__float_as_uint(s), (uint32_t)i);
        lo_inv = max(lo_inv, ALL - key_of(s));
        hi = max(hi, key_of(s));
      });
    });
    if (hi) {
      atomicMax(&sh.lo_inv, lo_inv);
      atomicMax(&sh.hi, hi);
    }
    __syncthreads();
    const int count = (int)sh.count;
    if (count <= LIST) return order_list<WEIGHTS>(sh, count, above, target, l, c).within(from);
    kmin = ALL - sh.lo_inv;
    kmax = sh.hi;
    bins = Bins{score_of(kmax), score_of(kmin), (float)HBINS / (score_of(kmax) - score_of(kmin))};
    __syncthreads();
  }
  return descend_cut<WEIGHTS>(Among<LdsRow<THR>>{row, from}, sh, kmin, kmax, above, cols, l, c,
                              [&](uint64_t total) { return target ? target : target_of(total); })
      .within(from);
}

template <typename T, int THR, int MAX>
__global__ __launch_bounds__(THR) void k_sample(RowArgs a) {
  constexpr int VE = Piece<T>::VE, WAVES = THR / WAVE, MOST = MAX / (THR * VE) + (MAX % (THR * VE) != 0);
  __shared__ __align__(16) float score[MAX];
  __shared__ Shared<THR> sh;
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const LdsRow<THR> row{score, (a.cols + THR * 4 - 1) / (THR * 4)};
  Limits lim = row_limits(a, r);

  // the row into LDS, all its loads under way at once (a loop over bounds-checked pieces waits for each)
  const T* p = (const T*)a.score + (int64_t)r * a.ld;
  typename Piece<T>::vec raw[MOST];
#pragma unroll
  for (int q = 0; q < MOST; ++q) {
    const int i0 = (q * THR + (int)threadIdx.x) * VE;
    if (i0 + VE <= a.cols) raw[q] = *reinterpret_cast<const typename Piece<T>::uvec*>(p + i0);
  }
  if (threadIdx.x == 0) sh.kmax = sh.kmin_inv = 0;
  float smax = -__builtin_inff(), smin = __builtin_inff();
#pragma unroll
  for (int q = 0; q < MOST; ++q) {
    const int i0 = (q * THR + (int)threadIdx.x) * VE;
    if (i0 >= row.pieces * THR * 4) continue;
    float x[VE];
    if (i0 + VE <= a.cols) {
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = canonical(to_f32<T>(raw[q][e]));
    } else {
      load_scores<T>(x, p + i0, a.cols - i0);
    }
#pragma unroll
    for (int e = 0; e < VE; e += 4) *reinterpret_cast<f4*>(score + i0 + e) = f4{x[e], x[e + 1], x[e + 2], x[e + 3]};
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      smax = fmaxf(smax, x[e]);
      smin = fminf(smin, x[e] >= LOWEST ? x[e] : smin);
    }
  }
  __syncthreads();
  {  // keys of the extremes; 0: nothing to take
    const bool any = smax >= LOWEST;
    const uint32_t hi = wave_max(any ? key_of(smax) : 0), lo = wave_max(any ? ALL - key_of(smin) : 0);
    if (lane == 0 && hi) {
      atomicMax(&sh.kmax, hi);
      atomicMax(&sh.kmin_inv, lo);
    }
  }
  __syncthreads();
  const uint32_t kmax = sh.kmax, kmin = ALL - sh.kmin_inv;
  if (kmax == 0) {
    for (int d = threadIdx.x; d < a.draws; d += THR) store_none(a, (int64_t)r * a.draws + d);
    return;
  }
  set_top(lim, score_of(kmax));

  Cut cut{LOWEST, NO_TIE};
  const double min_w = lim.min_w;
  lim.min_w = 0;  // min_p looks at what the other two leave
  if (lim.top_k != ALL)
    cut = find_cut<false>(row, sh, kmin, a.cols, cut, lim, a.c, [&](uint64_t total) { return count_target(lim, total); });
  if (lim.top_p < 1.0)
    cut = find_cut<true>(row, sh, kmin, a.cols, cut, lim, a.c, [&](uint64_t total) { return weight_target(lim, total); });
  lim.min_w = min_w;

  // kept weight up to the end of each thread's `mine` consecutive scores
  const int mine = row.pieces * 4;
  static_assert(MAX / THR <= 32, "a bit for each of a thread's scores");
  uint64_t own = 0, sum;
  if (row.few(cut)) {
    row.each_kept(cut, [&](float s, int i) {
      uint64_t wt[1];
      kept_weights<1>(&s, i, cut, lim, a.c, wt);
      own += wt[0];
    });
  } else {
    row.own4([&](const float* x, int i0) {
      uint64_t wt[4];
      kept_weights<4>(x, i0, cut, lim, a.c, wt);
      own += (wt[0] + wt[1]) + (wt[2] + wt[3]);
    });
  }
  uint64_t* run = sh.hist;
  const uint64_t before = block_scan64<THR>(own, sh.wave, &sum);
  run[threadIdx.x] = before + own;
  __syncthreads();

  // a wave a draw: the first thread whose running sum exceeds the number, then the score among its own
  for (int d = w; d < a.draws; d += WAVES) {
    const int64_t at = (int64_t)r * a.draws + d;
    const uint64_t t = draw_at(a, at, sum);
    const int g = __builtin_ctzll(__ballot(run[lane * WAVES + WAVES - 1] > t));
    const int th = g * WAVES + __builtin_ctzll(__ballot(lane < WAVES && run[g * WAVES + (lane & (WAVES - 1))] > t));
    uint64_t upto = th ? run[th - 1] : 0;
    const int i = th * mine + lane;
    const float s = lane < mine ? score[i] : -__builtin_inff();
    uint64_t wt[1];
    kept_weights<1>(&s, i, cut, lim, a.c, wt);
    upto += wave_scan64(wt[0]);
    if (lane == (int)__builtin_ctzll(__ballot(upto > t))) store_draw(a, at, i, s, sum, lim);
  }
}

template <typename T, int THR, int MAX>
int launch(const RowArgs& a, hipStream_t st) {
  static_assert(MAX % (THR * 4) == 0 && MAX / THR <= WAVE, "whole pieces, at most a wave of scores a thread");
  k_sample<T, THR, MAX><<<a.rows, THR, 0, st>>>(a);
  return check_launch("sample");
}

// ------------------------------------------------------------------------- a row's segments
// Members of a bin in a list: the row's share of the workspace.
struct Member {
  float s;
  int idx;
};

// What the launches over a row's segments leave for each other.
struct RowState {
  uint64_t hist[2][HBINS];  // ones, weights
  uint64_t above[2], target[2];
  uint32_t kmax, kmin_inv, count[2], lo_inv[2], hi[2], ready[2];  // ready: the bin was looked for
  Cut cut[2];
};

struct Spread {
  RowArgs a;
  RowState* state;
  uint64_t* seg_sum;  // rows x segs
  Member* list;       // rows x cap
  int segs, cap, draw0;
  int per;  // segments a workgroup of the range, histogram and member launches
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Spread& p, int r) {
  return (const T*)p.a.score + (int64_t)r * p.a.ld;
}

// f(scores, first index) for the segment's pieces.
template <typename T, int THR, typename F>
__device__ __forceinline__ void each_piece(const T* row, int cols, int begin, int end, F f) {
  constexpr int VE = Piece<T>::VE;
  for (int i0 = begin + (int)threadIdx.x * VE; i0 < end; i0 += THR * VE) {
    float x[VE];
    load_scores<T>(x, row + i0, cols - i0);
    f(x, i0);
  }
}

__global__ __launch_bounds__(256) void k_spread_clear(Spread p) {
  uint64_t* q = (uint64_t*)p.state;
  const int64_t n = (int64_t)p.a.rows * sizeof(RowState) / 8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) q[i] = 0;
}

template <typename T>
__global__ __launch_bounds__(SEG_THR) void k_spread_range(Spread p) {
  __shared__ uint32_t ends[2];
  const int r = blockIdx.y, begin = blockIdx.x * p.per * SEG;
  uint32_t hi = 0, lo = 0;
  if (threadIdx.x < 2) ends[threadIdx.x] = 0;
  each_piece<T, SEG_THR>(row_of<T>(p, r), p.a.cols, begin, min(begin + p.per * SEG, p.a.cols), [&](const float* x, int) {
#pragma unroll
    for (int e = 0; e < Piece<T>::VE; ++e)
      if (x[e] >= LOWEST) {
        hi = max(hi, key_of(x[e]));
        lo = max(lo, ALL - key_of(x[e]));
      }
  });
  hi = wave_max(hi);
  lo = wave_max(lo);
  __syncthreads();
  if ((threadIdx.x & 63) == 0 && hi) {
    atomicMax(&ends[0], hi);
    atomicMax(&ends[1], lo);
  }
  __syncthreads();
  if (threadIdx.x == 0 && ends[0]) {
    atomicMax(&p.state[r].kmax, ends[0]);
    atomicMax(&p.state[r].kmin_inv, ends[1]);
  }
}

// The row's limits with its largest score; false: nothing to take, or this limit is off.
template <bool WEIGHTS>
__device__ __forceinline__ bool spread_limits(const Spread& p, int r, Limits& l, float& per) {
  const RowState& s = p.state[r];
  if (s.kmax == 0) return false;
  l = row_limits(p.a, r);
  set_top(l, score_of(s.kmax));
  l.min_w = 0;
  per = bins_per(score_of(ALL - s.kmin_inv), l);
  return WEIGHTS ? l.top_p < 1.0 : l.top_k != ALL;
}
__device__ __forceinline__ Cut cut_k(const Spread& p, int r, const Limits& l) {
  return l.top_k != ALL ? p.state[r].cut[0] : Cut{LOWEST, NO_TIE};
}

template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(SEG_THR) void k_spread_hist(Spread p) {
  __shared__ uint64_t hist[HBINS];
  const int r = blockIdx.y, begin = blockIdx.x * p.per * SEG;
  Limits l;
  float per;
  if (!spread_limits<WEIGHTS>(p, r, l, per) || !bins_work(per, l)) return;
  const Cut from = WEIGHTS ? cut_k(p, r, l) : Cut{LOWEST, NO_TIE};
  for (int b = threadIdx.x; b < HBINS; b += SEG_THR) hist[b] = 0;
  __syncthreads();
  each_piece<T, SEG_THR>(row_of<T>(p, r), p.a.cols, begin, min(begin + p.per * SEG, p.a.cols), [&](const float* x, int i0) {
    add_to_bins<WEIGHTS, Piece<T>::VE>(hist, x, i0, from, Bins{l.top, LOWEST, per}, l, p.a.c);
  });
  __syncthreads();
  for (int b = threadIdx.x; b < HBINS; b += SEG_THR)
    if (hist[b]) atomicAdd((unsigned long long*)&p.state[r].hist[WEIGHTS][b], (unsigned long long)hist[b]);
}

// The bin's members into the row's list.
template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(SEG_THR) void k_spread_members(Spread p) {
  __shared__ Shared<SEG_THR> sh;
  const int r = blockIdx.y, begin = blockIdx.x * p.per * SEG;
  Limits l;
  float per;
  if (!spread_limits<WEIGHTS>(p, r, l, per) || !bins_work(per, l)) return;
  const Cut from = WEIGHTS ? cut_k(p, r, l) : Cut{LOWEST, NO_TIE};
  RowState& st = p.state[r];
  const uint64_t target = find_bin<SEG_THR>(sh, st.hist[WEIGHTS], 0, [&](uint64_t total) {
    return WEIGHTS ? weight_target(l, total) : count_target(l, total);
  });
  const uint32_t bin = sh.bin;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    st.above[WEIGHTS] = sh.above;
    st.target[WEIGHTS] = target;
    st.ready[WEIGHTS] = 1;
  }
  each_piece<T, SEG_THR>(row_of<T>(p, r), p.a.cols, begin, min(begin + p.per * SEG, p.a.cols), [&](const float* x, int i0) {
    members<Piece<T>::VE>(x, i0, from, bin, Bins{l.top, LOWEST, per}, [&](float s, int i) {
      const uint32_t at = atomicAdd(&st.count[WEIGHTS], 1u);
      if (at < (uint32_t)p.cap) p.list[(int64_t)r * p.cap + at] = Member{s, i};
      atomicMax(&st.lo_inv[WEIGHTS], ALL - key_of(s));
      atomicMax(&st.hi[WEIGHTS], key_of(s));
    });
  });
}

// Members, or the whole row where they were too many for the list or there are no bins, as a source of a descent.
struct ListSource {
  const Member* m;
  int n;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x; i < n; i += 1024) f(m[i].s, m[i].idx);
  }
};
template <typename T>
struct RowSource {
  const T* row;
  int cols;
  Cut from;
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each_piece<T, 1024>(row, cols, 0, cols, [&](const float* x, int i0) {
#pragma unroll
      for (int e = 0; e < Piece<T>::VE; ++e)
        if (x[e] >= LOWEST && from.keeps(x[e], i0 + e)) f(x[e], i0 + e);
    });
  }
};

// The cut of a row from its bin's members.
template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(1024) void k_spread_cut(Spread p) {
  __shared__ Shared<1024> sh;
  const int r = blockIdx.x;
  Limits l;
  float per;
  if (!spread_limits<WEIGHTS>(p, r, l, per)) return;
  const Cut from = WEIGHTS ? cut_k(p, r, l) : Cut{LOWEST, NO_TIE};
  RowState& st = p.state[r];
  const bool ready = st.ready[WEIGHTS];
  const int count = (int)st.count[WEIGHTS];
  const Member* m = p.list + (int64_t)r * p.cap;
  const auto target_of = [&](uint64_t total) {
    return ready ? st.target[WEIGHTS] : WEIGHTS ? weight_target(l, total) : count_target(l, total);
  };
  Cut cut;
  if (ready && count <= LIST) {
    if ((int)threadIdx.x < count) sh.list[threadIdx.x] = make_uint2(__float_as_uint(m[threadIdx.x].s), (uint32_t)m[threadIdx.x].idx);
    __syncthreads();
    cut = order_list<WEIGHTS>(sh, count, st.above[WEIGHTS], st.target[WEIGHTS], l, p.a.c);
  } else if (ready && count <= p.cap) {
    cut = descend_cut<WEIGHTS>(ListSource{m, count}, sh, ALL - st.lo_inv[WEIGHTS], st.hi[WEIGHTS], st.above[WEIGHTS],
                               p.a.cols, l, p.a.c, target_of);
  } else {
    const RowSource<T> all{row_of<T>(p, r), p.a.cols, from};
    const uint32_t lo = ready ? ALL - st.lo_inv[WEIGHTS] : ALL - st.kmin_inv, hi = ready ? st.hi[WEIGHTS] : st.kmax;
    cut = descend_cut<WEIGHTS>(all, sh, lo, hi, ready ? st.above[WEIGHTS] : 0, p.a.cols, l, p.a.c, target_of);
  }
  if (threadIdx.x == 0) st.cut[WEIGHTS] = cut.within(from);
}

// The row's last cut and its limits, min_p among them.
__device__ __forceinline__ Cut last_cut(const Spread& p, int r, Limits& l) {
  l = row_limits(p.a, r);
  set_top(l, score_of(p.state[r].kmax));
  return l.top_p < 1.0 ? p.state[r].cut[1] : cut_k(p, r, l);
}

template <typename T>
__global__ __launch_bounds__(SEG_THR) void k_spread_sums(Spread p) {
  constexpr int VE = Piece<T>::VE;
  __shared__ uint64_t wave[16];
  const int r = blockIdx.y, begin = blockIdx.x * SEG;
  uint64_t own = 0, total = 0;
  if (p.state[r].kmax) {
    Limits l;
    const Cut cut = last_cut(p, r, l);
    each_piece<T, SEG_THR>(row_of<T>(p, r), p.a.cols, begin, min(begin + SEG, p.a.cols), [&](const float* x, int i0) {
      uint64_t w[VE];
      kept_weights<VE>(x, i0, cut, l, p.a.c, w);
#pragma unroll
      for (int e = 0; e < VE; ++e) own += w[e];
    });
  }
  block_scan64<SEG_THR>(own, wave, &total);
  if (threadIdx.x == 0) p.seg_sum[(int64_t)r * p.segs + blockIdx.x] = total;
}

// A workgroup a draw: the segment that passes the number, then the score in it.
template <typename T>
__global__ __launch_bounds__(SEG_THR) void k_spread_draw(Spread p) {
  constexpr int VE = Piece<T>::VE;
  __shared__ uint64_t wave[16];
  __shared__ uint64_t found_run;
  __shared__ int found;
  const int r = blockIdx.y;
  const int64_t at = (int64_t)r * p.a.draws + p.draw0 + blockIdx.x;
  if (p.state[r].kmax == 0) {
    if (threadIdx.x == 0) store_none(p.a, at);
    return;
  }
  Limits l;
  const Cut cut = last_cut(p, r, l);
  const uint64_t* seg = p.seg_sum + (int64_t)r * p.segs;
  uint64_t sum = 0, total;
  for (int g0 = 0; g0 < p.segs; g0 += SEG_THR) {
    block_scan64<SEG_THR>(g0 + (int)threadIdx.x < p.segs ? seg[g0 + threadIdx.x] : 0, wave, &total);
    sum += total;
  }
  const uint64_t t = draw_at(p.a, at, sum);
  uint64_t run = 0;
  for (int g0 = 0; g0 < p.segs; g0 += SEG_THR) {
    const int g = g0 + (int)threadIdx.x;
    const uint64_t v = g < p.segs ? seg[g] : 0;
    const uint64_t before = run + block_scan64<SEG_THR>(v, wave, &total);
    if (before <= t && before + v > t) {  // one thread's, once
      found = g;
      found_run = before;
    }
    run += total;
  }
  __syncthreads();
  run = found_run;
  const int begin = found * SEG;
  const T* row = row_of<T>(p, r);
  for (int i00 = begin; i00 < begin + SEG; i00 += SEG_THR * VE) {
    const int i0 = i00 + (int)threadIdx.x * VE;
    float x[VE];
    uint64_t w[VE], own = 0;
    load_scores<T>(x, row + i0, p.a.cols - i0);
    kept_weights<VE>(x, i0, cut, l, p.a.c, w);
#pragma unroll
    for (int e = 0; e < VE; ++e) own += w[e];
    uint64_t before = run + block_scan64<SEG_THR>(own, wave, &total);
    if (before <= t && before + own > t) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (before <= t && before + w[e] > t) store_draw(p.a, at, i0 + e, x[e], sum, l);
        before += w[e];
      }
    }
    run += total;
    if (run > t) break;
  }
}

int64_t round256(int64_t b) { return (b + 255) / 256 * 256; }

// Room for an eighth of the row in the list of a bin's members.
int list_cap(int cols) { return cols / 8 + 1024; }

// Rows that share a set of launches: a workspace of about 256 MB, and within the grid's second dimension.
int rows_at_once(int cols) {
  const int64_t row = sizeof(RowState) + (cols + SEG - 1) / SEG * 8 + list_cap(cols) * (int64_t)sizeof(Member);
  return (int)std::max<int64_t>(1, std::min<int64_t>(32768, (256 << 20) / row));
}

template <typename T, bool WEIGHTS>
void launch_cut(const Spread& p, hipStream_t st) {
  const dim3 grid((p.segs + p.per - 1) / p.per, p.a.rows);
  k_spread_hist<T, WEIGHTS><<<grid, SEG_THR, 0, st>>>(p);
  k_spread_members<T, WEIGHTS><<<grid, SEG_THR, 0, st>>>(p);
  k_spread_cut<T, WEIGHTS><<<p.a.rows, 1024, 0, st>>>(p);
}

template <typename T>
int launch_spread(const RowArgs& a, void* ws, hipStream_t st) {
  Spread p{};
  p.a = a;
  p.segs = (a.cols + SEG - 1) / SEG;
  p.cap = list_cap(a.cols);
  // every workgroup adds its histogram to the row's by atomics on the same 2048 words: no more of them than
  // fill the card twice (16 x 1 M: 53 us with a segment each, 20 with 4)
  p.per = (int)std::max<int64_t>(1, std::min<int64_t>(16, (int64_t)a.rows * p.segs / 512));
  char* w = (char*)ws;
  p.state = (RowState*)w;
  w += round256((int64_t)a.rows * sizeof(RowState));
  p.seg_sum = (uint64_t*)w;
  w += round256((int64_t)a.rows * p.segs * 8);
  p.list = (Member*)w;
  const int64_t words = (int64_t)a.rows * sizeof(RowState) / 8;
  k_spread_clear<<<(int)std::min<int64_t>((words + 255) / 256, 2048), 256, 0, st>>>(p);
  const dim3 grid(p.segs, a.rows);
  k_spread_range<T><<<dim3((p.segs + p.per - 1) / p.per, a.rows), SEG_THR, 0, st>>>(p);
  if (a.top_k_v || (a.top_k > 0 && a.top_k < a.cols) || a.temperature_v || !(a.temperature > 0)) launch_cut<T, false>(p, st);
  if (a.top_p_v || a.top_p < 1.0) launch_cut<T, true>(p, st);
  k_spread_sums<T><<<grid, SEG_THR, 0, st>>>(p);
  for (; p.draw0 < a.draws; p.draw0 += LAUNCH_DRAWS)
    k_spread_draw<T><<<dim3(std::min(a.draws - p.draw0, LAUNCH_DRAWS), a.rows), SEG_THR, 0, st>>>(p);
  return check_launch("sample");
}

template <typename T>
int launch_rows(const RowArgs& a, void* ws, hipStream_t st) {
  // As few threads as leave a CU several rows: without the first tier 3080 x 1,000 takes 48 us for 36, without the second
  // 3080 x 7,128 165 for 90; the third, a row a CU like the last, gains 1.5 % (3080 x 12,000, 109.4 us and 107.6).
  if (a.cols <= 2048) return launch<T, 256, 2048>(a, st);
  if (a.cols <= 8192) return launch<T, 512, 8192>(a, st);
  if (a.cols <= 16384) return launch<T, 1024, 16384>(a, st);
  if (a.cols <= ROW_MAX) return launch<T, 1024, ROW_MAX>(a, st);
  return launch_spread<T>(a, ws, st);
}

template <typename T>
int dispatch(const RowArgs& a, void* ws, hipStream_t st) {
  RowArgs part = a;
  const auto from = [&](const void* v, int wide, int64_t r0) { return v ? (const char*)v + r0 * (wide ? 8 : 4) : nullptr; };
  const int most = a.cols <= ROW_MAX ? LAUNCH_ROWS : rows_at_once(a.cols);
  for (int64_t r0 = 0; r0 < a.rows; r0 += most) {
    part.rows = (int)std::min<int64_t>(most, a.rows - r0);
    part.score = (const T*)a.score + r0 * a.ld;
    part.u = (const char*)a.u + r0 * a.draws * (a.u_wide ? 8 : 4);
    part.ids = a.ids + r0 * a.draws;
    part.logp = a.logp ? a.logp + r0 * a.draws : nullptr;
    part.temperature_v = from(a.temperature_v, a.rows_wide & 1, r0);
    part.top_k_v = a.top_k_v ? a.top_k_v + r0 : nullptr;
    part.top_p_v = from(a.top_p_v, a.rows_wide & 2, r0);
    part.min_p_v = from(a.min_p_v, a.rows_wide & 4, r0);
    if (int rc = launch_rows<T>(part, ws, st)) return rc;
  }
  return 0;
}

}  // namespace

int64_t sample_ws_bytes(int rows, int cols, int) {
  if (rows <= 0 || cols <= ROW_MAX || cols > MAX_COLS) return 0;
  const int64_t r = std::min(rows, rows_at_once(cols)), segs = (cols + SEG - 1) / SEG;
  return round256(r * sizeof(RowState)) + round256(r * segs * 8) + round256(r * list_cap(cols) * (int64_t)sizeof(Member));
}

int sample(const regcn_sample_desc& d, hipStream_t st) {
  if (d.rows < 0 || d.cols < 0 || d.draws < 0) return set_error(REGCN_EINVAL, "sample: negative size");
  if (d.dtype < REGCN_F32 || d.dtype > REGCN_F16) return set_error(REGCN_EINVAL, "sample: bad element type %d", d.dtype);
  if (d.cols > MAX_COLS) return set_error(REGCN_ENOTSUP, "sample: rows of up to %d scores", MAX_COLS);
  if (d.draws > MAX_DRAWS) return set_error(REGCN_ENOTSUP, "sample: up to %d draws a row", MAX_DRAWS);
  if (!d.ids || !d.u || (d.cols > 0 && !d.score)) return set_error(REGCN_EINVAL, "sample: null score, u or ids");
  if (d.rows > 1 && d.ld < d.cols) return set_error(REGCN_EINVAL, "sample: row stride %lld below cols=%d", (long long)d.ld, d.cols);
  if (d.rows == 0 || d.draws == 0) return 0;
  const int64_t need = sample_ws_bytes(d.rows, d.cols, d.dtype);
  if (need && (!d.workspace || (int64_t)d.ws_bytes < need))
    return set_error(REGCN_EINVAL, "sample: workspace of %zu bytes, needs %lld", d.ws_bytes, (long long)need);
  RowArgs a{};
  a.score = d.score;
  a.ld = d.ld;
  a.rows = d.rows;
  a.cols = d.cols;
  a.draws = d.draws;
  a.u = d.u;
  a.u_wide = d.u_wide;
  a.temperature = d.temperature;
  a.top_k = d.top_k;
  a.top_p = d.top_p;
  a.min_p = d.min_p;
  a.temperature_v = d.temperature_rows;
  a.top_k_v = d.top_k_rows;
  a.top_p_v = d.top_p_rows;
  a.min_p_v = d.min_p_rows;
  a.rows_wide = d.rows_wide;
  a.ids = d.ids;
  a.logp = d.logp;
  a.c.log2e = 1.4426950408889634074;
  a.c.round = 0x1.8p52;
  // ln 2 = 0.693147180559945309417232121458...: its first 32 bits, whose products with a whole number below 2^21 are
  // exact, and what is left of it
  a.c.ln2_hi = -2977044471.0 / 4294967296.0;
  a.c.ln2_lo = -1.908214929270587816e-10;
  double f = 1.0;
  for (int j = 2; j <= 12; ++j) a.c.p[12 - j] = 1.0 / (f *= j);
  int bits = 0;
  while ((1ll << bits) < d.cols) ++bits;
  a.shift = std::min(51, 63 - bits);
  if (d.dtype == REGCN_F32) return dispatch<float>(a, d.workspace, st);
  if (d.dtype == REGCN_BF16) return dispatch<__bf16>(a, d.workspace, st);
  return dispatch<_Float16>(a, d.workspace, st);
}

}  // namespace regcn
