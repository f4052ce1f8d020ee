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
// exact in any order, so histograms by atomics, partial sums and prefix sums agree bit for bit.
//
// No sort.  Scores become 32-bit keys of the same order.  Each of k and p asks for the place in the order
// where a running sum (of ones, of weights) reaches a target: a radix descent over the keys finds the
// key (histograms of 11 bits; a round after the first touches the elements of one bin only), and where several
// elements share that key, a descent over their indices finds the last one kept.  So a kept set is
// {key > K} and {key = K, index <= I}.
//
// k_sample: a workgroup takes a row.  Up to 32768 scores stay in its LDS as keys (one read of the scores;
// in registers, the compiler spilled them around the 64-bit exponentials); longer rows are read again in each
// pass.
// Few long rows: several workgroups take a row's segments, in launches that pass histograms, the members of
// the bin in question and segment sums through a workspace (k_spread_*).
#include "elem.h"
#include "regcn_internal.h"

namespace regcn {
namespace {

constexpr int HBITS = 11, HBINS = 1 << HBITS;
constexpr int ROW_KEYS = 32768;  // scores of a row held in LDS
constexpr uint32_t ALL = 0xffffffffu;
constexpr int LIST = 256;        // members of a bin that are put in order one against the other
constexpr int CHUNKS = 4096;  // running sums of kept weights kept in LDS, at most
constexpr int MAX_COLS = 1 << 24;

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
  const float *temperature_v, *top_p_v, *min_p_v;
  const int32_t* top_k_v;
  int64_t* ids;
  float* logp;
  ExpConsts c;
};

struct Limits {
  double inv_t, top_p, min_w;  // min_w: min_p 2^S
  uint32_t top_k;              // ALL: off
  int shift;
  // set once the row's largest score is known
  uint32_t kmax;
  double top;
  bool ties_only;  // an infinite score, or a temperature whose inverse is: weight only on the largest
  ExpConsts c;
};

__device__ __forceinline__ Limits row_limits(const RowArgs& a, int row) {
  Limits l;
  const double t = a.temperature_v ? (double)a.temperature_v[row] : a.temperature;
  const int k = a.top_k_v ? a.top_k_v[row] : a.top_k;
  l.top_p = a.top_p_v ? (double)a.top_p_v[row] : a.top_p;
  l.min_w = __builtin_ldexp(a.min_p_v ? (double)a.min_p_v[row] : a.min_p, a.shift);
  l.top_k = k > 0 && k < a.cols ? (uint32_t)k : ALL;
  l.inv_t = 1.0 / t;
  if (!(t > 0)) {  // greedy
    l.inv_t = 1.0;
    l.top_k = 1;
  }
  l.shift = a.shift;
  l.c = a.c;
  return l;
}

// 0: never taken; otherwise increasing with the score, -0 and 0 alike.
__device__ __forceinline__ uint32_t score_key(float s) {
  const uint32_t b = __float_as_uint(s + 0.f);
  const uint32_t k = b ^ ((int32_t)b < 0 ? ALL : 0x80000000u);
  return s > -__builtin_inff() ? k : 0u;  // false for NaN
}
__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : ALL)); }

__device__ __forceinline__ void set_top(Limits& l, uint32_t kmax) {
  l.kmax = kmax;
  l.top = (double)key_score(kmax);
  l.ties_only = !(fabs(l.top) < __builtin_inf() && l.inv_t < __builtin_inf());
}

// exp(x) 2^S for x = (s - top) / T <= 0.  exp(x) = 2^n p(r), r = x - n ln 2 in two parts, |r| <= ln 2 / 2;
// p is the Taylor polynomial of degree 12 (remainder below 2^-52 of p).  n comes out of the low bits of
// x / ln 2 + 1.5 2^52 and goes into the exponent of p by an integer add (n + S >= -1010: still normal): the
// conversions, rounding and ldexp instructions run at a quarter of the rate of the rest.
__device__ __forceinline__ double scaled_exp(uint32_t key, const Limits& l) {
  const double x = fmax(((double)key_score(key) - l.top) * l.inv_t, -700.0);
  const double t = fma(x, l.c.log2e, l.c.round);
  const double n = t - l.c.round;
  double r = fma(n, l.c.ln2_hi, x);
  r = fma(n, l.c.ln2_lo, r);
  double p = fma(l.c.p[0], r, l.c.p[1]);
#pragma unroll
  for (int j = 2; j < 11; ++j) p = fma(p, r, l.c.p[j]);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int e = (int)(uint32_t)__double_as_longlong(t) + l.shift;
  return __hiloint2double(__double2hiint(p) + (e << 20), __double2loint(p));
}

// To the nearest whole number: adding 2^52 to a number up to 2^51 leaves it in the low bits.
__device__ __forceinline__ uint64_t whole(double v) { return __double_as_longlong(v + 0x1p52) & ((1ull << 52) - 1); }

__device__ __forceinline__ uint64_t weight(uint32_t key, const Limits& l) {
  if (l.ties_only) return key == l.kmax ? 1ull << l.shift : 0;
  return whole(scaled_exp(key, l));
}

// A place in the order: everything with a larger key, and of its own key the indices up to idx.
struct Cut {
  uint32_t key;
  int idx;
  __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= idx); }
};

// The weights of a piece's elements, 0 where a limit leaves one out.  No branch an element: the exponentials
// of the piece run together, and pieces without an element kept by any lane are passed over.
template <int VE>
__device__ __forceinline__ void kept_weights(const uint32_t* k, int i0, const Cut& cut, const Limits& l, uint64_t (&w)[VE]) {
  bool keep[VE], some = false;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    keep[e] = k[e] && cut.keeps(k[e], i0 + e);
    some |= keep[e];
    w[e] = 0;
  }
  if (!some) return;
  if (l.ties_only) {
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = keep[e] && k[e] == l.kmax ? 1ull << l.shift : 0;
    return;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const double v = scaled_exp(k[e], l);
    w[e] = keep[e] && (v >= l.min_w || k[e] == l.kmax) ? whole(v) : 0;
  }
}

// Sum over the wave, in every lane: two halves by DPP within rows of 16 lanes, the four rows by readlane.
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#define REGCN_STEP(ctrl)                                                                                       \
  v += (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, ctrl, 0xF, 0xF, false) |            \
       (uint64_t)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), ctrl, 0xF, 0xF, false) << 32
  REGCN_STEP(0xB1);   // quad_perm [1,0,3,2]
  REGCN_STEP(0x4E);   // quad_perm [2,3,0,1]
  REGCN_STEP(0x124);  // row_ror:4
  REGCN_STEP(0x128);  // row_ror:8
#undef REGCN_STEP
  uint64_t s = 0;
#pragma unroll
  for (int row = 0; row < 4; ++row)
    s += (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 16 * row) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 16 * row) << 32;
  return s;
}

template <int THR>
struct Shared {
  uint64_t hist[HBINS];
  uint64_t wave[THR / WAVE];
  uint32_t kmax[THR / WAVE], kmin[THR / WAVE];
  uint64_t above, sum;
  uint32_t bin, count, lo, hi;
  uint2 list[LIST];      // {key, index}
  uint64_t value[LIST];
  Cut cut;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
  const uint32_t lo = __shfl_up((uint32_t)v, o), hi = __shfl_up((uint32_t)(v >> 32), o);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int l) {
  const uint32_t lo = __shfl((uint32_t)v, l), hi = __shfl((uint32_t)(v >> 32), l);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const uint64_t y = shfl_up64(v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Exclusive prefix of v over the workgroup's threads; *total: the sum.
template <int THR>
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t* wave, uint64_t* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t inc = wave_scan64(v);
  __syncthreads();  // wave[] may still be read from the call before
  if (lane == 63) wave[w] = inc;
  __syncthreads();
  uint64_t base = 0, sum = 0;
#pragma unroll
  for (int u = 0; u < THR / WAVE; ++u) {
    const uint64_t x = wave[u];
    base += u < w ? x : 0;
    sum += x;
  }
  *total = sum;
  return base + inc - v;
}

// The row as this workgroup sees it: piece q of thread t holds the VE scores from (q THR + t) VE on.  With
// KEYS > 0 it is read once, into `keys` (LDS); otherwise again in each pass.
template <typename T, int THR, int KEYS>
struct Row {
  static constexpr int VE = KEYS > 0 ? 4 : Piece<T>::VE;
  const T* p;
  uint32_t* keys;
  int n, pieces;  // pieces a thread

  template <int N>
  __device__ __forceinline__ void load(int i0, uint32_t (&k)[N]) const {
    static_assert(N == Piece<T>::VE, "a piece of the type");
    float x[N];
    const int m = n - i0;
    if (m > 0) load_piece<T>(x, p + i0, m);
#pragma unroll
    for (int e = 0; e < N; ++e) k[e] = e < m ? score_key(x[e]) : 0u;
  }
  // the keys from i0 (a multiple of VE) on; 0 past the row's end
  __device__ __forceinline__ void read_at(int i0, uint32_t (&k)[VE]) const {
    if constexpr (KEYS > 0) {
      const uint4 v = i0 < KEYS ? *reinterpret_cast<const uint4*>(keys + i0) : make_uint4(0, 0, 0, 0);
      k[0] = v.x, k[1] = v.y, k[2] = v.z, k[3] = v.w;
    } else {
      load(i0, k);
    }
  }
  // Also the largest and smallest key (0, ALL: none) of this thread's.
  __device__ __forceinline__ void init(const T* row, int cols, uint32_t* lds, uint32_t& kmax, uint32_t& kmin) {
    kmax = 0;
    kmin = ALL;
    p = row;
    n = cols;
    keys = lds;
    pieces = (cols + THR * VE - 1) / (THR * VE);
    if constexpr (KEYS > 0) {
      // all the row's loads under way at once: a loop over bounds-checked pieces waits for each
      constexpr int PV = Piece<T>::VE, MOST = (KEYS + THR * PV - 1) / (THR * PV);
      typedef typename Piece<T>::vec vec;
      typedef typename Piece<T>::uvec uvec;
      vec x[MOST];
#pragma unroll
      for (int q = 0; q < MOST; ++q) {
        const int i0 = (q * THR + (int)threadIdx.x) * PV;
        if (i0 + PV <= n) x[q] = *reinterpret_cast<const uvec*>(p + i0);
      }
#pragma unroll
      for (int q = 0; q < MOST; ++q) {
        const int i0 = (q * THR + (int)threadIdx.x) * PV;
        if (i0 >= pieces * THR * VE) continue;
        uint32_t k[PV];
        if (i0 + PV <= n) {
#pragma unroll
          for (int e = 0; e < PV; ++e) k[e] = score_key(to_f32<T>(x[q][e]));
        } else {
          load(i0, k);
        }
#pragma unroll
        for (int e = 0; e < PV; ++e) {
          kmax = max(kmax, k[e]);
          kmin = min(kmin, k[e] ? k[e] : ALL);
        }
#pragma unroll
        for (int e = 0; e < PV; e += 4)
          *reinterpret_cast<uint4*>(keys + i0 + e) = make_uint4(k[e], k[e + 1], k[e + 2], k[e + 3]);
      }
    } else {
      pieces_of([&](int, int, const uint32_t* k) {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          kmax = max(kmax, k[e]);
          kmin = min(kmin, k[e] ? k[e] : ALL);
        }
      });
    }
  }
  // f(q, first index, keys of the piece) for every piece
  template <typename F>
  __device__ __forceinline__ void pieces_of(F f) const {
    for (int q = 0; q < pieces; ++q) {
      uint32_t k[VE];
      const int i0 = (q * THR + (int)threadIdx.x) * VE;
      read_at(i0, k);
      f(q, i0, k);
    }
  }
};

// The bin of sh.hist in which the running sum, `above` before bin 0, reaches the target: into sh.bin, with the
// sum before it in sh.above and its own in sh.sum (1 <= target - above <= the histogram's total).  target_of
// gives the target from the total.
template <int THR, int BINS, typename Target>
__device__ __forceinline__ uint64_t find_bin(Shared<THR>& sh, const uint64_t* hist, uint64_t above, Target target_of) {
  constexpr int PER = BINS / THR;
  uint64_t own = 0, total, h[PER];
#pragma unroll
  for (int b = 0; b < PER; ++b) own += h[b] = hist[threadIdx.x * PER + b];
  uint64_t before = above + block_scan64<THR>(own, sh.wave, &total);
  const uint64_t target = target_of(total);
#pragma unroll
  for (int b = 0; b < PER; ++b) {
    if (before < target && before + h[b] >= target) {  // one thread's
      sh.above = before;
      sh.bin = threadIdx.x * PER + b;
      sh.sum = h[b];
    }
    before += h[b];
  }
  __syncthreads();
  return target;
}

struct Place {
  uint32_t key;
  uint64_t above, sum, target;  // sums before the key, of the key
};

// Radix descent in decreasing order of keys in [lo, hi]: the key at which the running sum of values, `above`
// before hi, reaches the target.  each(f, lo, hi) calls f(key, value) for the elements with a key in [lo, hi].
template <int THR, typename Each, typename Target>
__device__ Place descend(Shared<THR>& sh, uint32_t lo, uint32_t hi, uint64_t above, Each each, Target target_of) {
  uint64_t target = 0;
  for (bool first = true;; first = false) {
    const uint32_t range = hi - lo;
    const int bits = range ? 32 - __builtin_clz(range) : 0;
    const int shift = bits > HBITS ? bits - HBITS : 0;
    for (int b = threadIdx.x; b < HBINS; b += THR) sh.hist[b] = 0;
    __syncthreads();
    each([&](uint32_t k, uint64_t value) {
      if (value) atomicAdd((unsigned long long*)&sh.hist[(hi - k) >> shift], (unsigned long long)value);
    }, lo, hi);
    __syncthreads();
    const uint64_t t = find_bin<THR, HBINS>(sh, sh.hist, above, [&](uint64_t total) { return first ? target_of(total) : target; });
    target = t;
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

// The bin of a key's score on a linear scale from the largest score down (fp32: monotone, which is all that a
// bin has to be); the last bin is open.
__device__ __forceinline__ uint32_t value_bin(uint32_t key, float top, float per) {
  return (uint32_t)fminf((top - key_score(key)) * per, (float)(HBINS - 1));
}

// The cut at which a running sum over the order reaches the target, among the elements that `from` keeps: of
// ones (WEIGHTS false) or of weights.  First over 2048 bins of the scores' range, at most 44 T of it (weights
// below exp(-44) are none): the bin in question then rarely has over LIST members, and each of those adds up
// the members before it.  Otherwise, and for infinite scores, a descent over the keys.
template <bool WEIGHTS, int THR, typename R, typename Target>
__device__ Cut find_cut(const R& row, Shared<THR>& sh, uint32_t kmin, uint32_t kmax, int cols, const Cut& from,
                        const Limits& lim, Target target_of) {
  constexpr int VE = R::VE;
  uint64_t above = 0, target = 0;
  const float top = key_score(kmax), span = fminf(top - key_score(kmin), (float)(44.0 / lim.inv_t));
  const float per = (float)HBINS / span;
  if (per > 0.f && per < 1e30f && !lim.ties_only) {
    for (int b = threadIdx.x; b < HBINS; b += THR) sh.hist[b] = 0;
    if (threadIdx.x == 0) {
      sh.count = 0;
      sh.lo = ALL;
      sh.hi = 0;
    }
    __syncthreads();
    row.pieces_of([&](int, int i0, const uint32_t* k) {
      uint64_t w[VE];
      if (WEIGHTS) {
        kept_weights<VE>(k, i0, from, lim, w);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) w[e] = k[e] != 0;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (w[e]) atomicAdd((unsigned long long*)&sh.hist[value_bin(k[e], top, per)], (unsigned long long)w[e]);
    });
    __syncthreads();
    target = find_bin<THR, HBINS>(sh, sh.hist, 0, target_of);
    above = sh.above;
    const uint32_t bin = sh.bin;
    row.pieces_of([&](int, int i0, const uint32_t* k) {
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (k[e] && value_bin(k[e], top, per) == bin && from.keeps(k[e], i0 + e)) {
          const uint32_t at = atomicAdd(&sh.count, 1u);
          if (at < LIST) sh.list[at] = make_uint2(k[e], (uint32_t)(i0 + e));
          atomicMin(&sh.lo, k[e]);
          atomicMax(&sh.hi, k[e]);
        }
    });
    __syncthreads();
    const int count = (int)sh.count;
    if (count <= LIST) {
      uint2 me = make_uint2(0, 0);
      uint64_t own = 0, before = above;
      if ((int)threadIdx.x < count) {
        me = sh.list[threadIdx.x];
        own = WEIGHTS ? weight(me.x, lim) : 1;
        sh.value[threadIdx.x] = own;
      }
      __syncthreads();
      if ((int)threadIdx.x < count) {
#pragma unroll 4
        for (int j = 0; j < count; ++j) {
          const uint2 o = sh.list[j];
          before += o.x > me.x || (o.x == me.x && o.y < me.y) ? sh.value[j] : 0;
        }
        if (before < target && before + own >= target) sh.cut = Cut{me.x, (int)me.y};  // one thread's
      }
      __syncthreads();
      const Cut cut = sh.cut;
      __syncthreads();  // sh may be written again
      return cut;
    }
    kmin = sh.lo;
    kmax = sh.hi;
    __syncthreads();
  }
  const Place p = descend<THR>(
      sh, kmin, kmax, above,
      [&](auto f, uint32_t lo, uint32_t hi) {
        row.pieces_of([&](int, int i0, const uint32_t* k) {
          uint64_t w[VE];
          if (WEIGHTS) {
            uint32_t in[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) in[e] = k[e] >= lo && k[e] <= hi ? k[e] : 0;
            kept_weights<VE>(in, i0, from, lim, w);
          } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) w[e] = k[e] && k[e] >= lo && k[e] <= hi;
          }
#pragma unroll
          for (int e = 0; e < VE; ++e) f(k[e], w[e]);
        });
      },
      [&](uint64_t total) { return target ? target : target_of(total); });
  // one key left: its elements each add the same; the lowest indices are kept
  const uint64_t one = WEIGHTS ? weight(p.key, lim) : 1;
  const uint64_t need = one ? (p.target - p.above + one - 1) / one : 1, have = one ? p.sum / one : 1;
  if (need >= have) return Cut{p.key, 0x7fffffff};
  const Place q = descend<THR>(
      sh, ALL - (uint32_t)(cols - 1), ALL, 0,
      [&](auto f, uint32_t lo, uint32_t hi) {
        row.pieces_of([&](int, int i0, const uint32_t* k) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const uint32_t at = ALL - (uint32_t)(i0 + e);
            f(at, k[e] == p.key && from.keeps(k[e], i0 + e) && at >= lo && at <= hi);
          }
        });
      },
      [&](uint64_t) { return need; });
  return Cut{p.key, (int)(ALL - q.key)};
}

__device__ __forceinline__ uint64_t count_target(const Limits& l, uint64_t total) { return min((uint64_t)l.top_k, total); }
__device__ __forceinline__ uint64_t weight_target(const Limits& l, uint64_t total) {
  const double t = ceil(l.top_p * (double)total);
  return t < 1.0 ? (uint64_t)1 : min(total, (uint64_t)t);
}

// The number in [0, sum) that the drawn u stands for; NaN and negative u: 0.
__device__ __forceinline__ uint64_t draw_at(const RowArgs& a, int64_t at, uint64_t sum) {
  const double u = a.u_wide ? ((const double*)a.u)[at] : (double)((const float*)a.u)[at];
  const double x = u > 0.0 ? u * (double)sum : 0.0;
  return x < (double)sum ? min((uint64_t)x, sum - 1) : sum - 1;
}
__device__ __forceinline__ double log_of_sum(uint64_t sum, const Limits& l) {
  return log((double)sum) - (double)l.shift * 0.69314718055994530942;
}
__device__ __forceinline__ void store_draw(const RowArgs& a, int64_t at, int id, uint32_t key, const Limits& l, double log_sum) {
  a.ids[at] = id;
  if (a.logp) a.logp[at] = (float)((key == l.kmax ? 0.0 : ((double)key_score(key) - l.top) * l.inv_t) - log_sum);
}
__device__ __forceinline__ void store_none(const RowArgs& a, int64_t at) {
  a.ids[at] = -1;
  if (a.logp) a.logp[at] = -__builtin_inff();
}

// Largest and smallest key (0, ALL: none) over the workgroup; a barrier.
template <int THR>
__device__ __forceinline__ void block_minmax(Shared<THR>& sh, uint32_t& kmax, uint32_t& kmin) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    kmax = max(kmax, __shfl_xor(kmax, o));
    kmin = min(kmin, __shfl_xor(kmin, o));
  }
  if ((threadIdx.x & 63) == 0) {
    sh.kmax[threadIdx.x >> 6] = kmax;
    sh.kmin[threadIdx.x >> 6] = kmin;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < THR / WAVE; ++u) {
    kmax = max(kmax, sh.kmax[u]);
    kmin = min(kmin, sh.kmin[u]);
  }
}

template <typename T, int THR, int KEYS>
__global__ __launch_bounds__(THR) void k_sample(RowArgs a) {
  constexpr int VE = Row<T, THR, KEYS>::VE, WAVES = THR / WAVE;
  __shared__ __align__(16) uint32_t keys[KEYS > 0 ? KEYS : 4];
  const int subs = (a.cols + WAVE * VE - 1) / (WAVE * VE);  // a wave's pieces: WAVE * VE consecutive scores
  const int group = (subs + CHUNKS - 1) / CHUNKS, chunks = (subs + group - 1) / group;
  __shared__ Shared<THR> sh;
  extern __shared__ uint64_t chunk[];  // running kept weight after each chunk of `group` waves' pieces
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  Limits lim = row_limits(a, r);
  Row<T, THR, KEYS> row;
  uint32_t kmax, kmin;
  row.init((const T*)a.score + (int64_t)r * a.ld, a.cols, keys, kmax, kmin);
  block_minmax(sh, kmax, kmin);
  if (kmax == 0) {  // nothing to take
    for (int d = threadIdx.x; d < a.draws; d += THR) store_none(a, (int64_t)r * a.draws + d);
    return;
  }
  set_top(lim, kmax);

  Cut cut{0, 0x7fffffff};
  const double min_w = lim.min_w;
  lim.min_w = 0;  // min_p looks at what the other two leave
  if (lim.top_k != ALL)
    cut = find_cut<false, THR>(row, sh, kmin, kmax, a.cols, cut, lim, [&](uint64_t total) { return count_target(lim, total); });
  if (lim.top_p < 1.0)
    cut = find_cut<true, THR>(row, sh, max(kmin, cut.key), kmax, a.cols, Cut(cut), lim,
                              [&](uint64_t total) { return weight_target(lim, total); });
  lim.min_w = min_w;

  // running sums of the kept weights over chunks of consecutive scores
  for (int c = threadIdx.x; c < chunks; c += THR) chunk[c] = 0;
  __syncthreads();
  row.pieces_of([&](int q, int i0, const uint32_t* k) {
    uint64_t wt[VE], s = 0;
    kept_weights<VE>(k, i0, cut, lim, wt);
#pragma unroll
    for (int e = 0; e < VE; ++e) s += wt[e];
    s = wave_sum64(s);
    const int sub = q * WAVES + w;
    if (lane == 0 && sub < subs) atomicAdd((unsigned long long*)&chunk[sub / group], (unsigned long long)s);
  });
  __syncthreads();
  uint64_t sum = 0;
  for (int c0 = 0; c0 < chunks; c0 += THR) {
    const int c = c0 + threadIdx.x;
    const uint64_t v = c < chunks ? chunk[c] : 0;
    uint64_t total;
    const uint64_t before = sum + block_scan64<THR>(v, sh.wave, &total);
    if (c < chunks) chunk[c] = before + v;
    sum += total;
  }
  __syncthreads();

  // a wave a draw: the first chunk whose running sum exceeds u * sum, then the score within it
  const double log_sum = a.logp ? log_of_sum(sum, lim) : 0.0;
  for (int d = w; d < a.draws; d += WAVES) {
    const int64_t at = (int64_t)r * a.draws + d;
    const uint64_t t = draw_at(a, at, sum);
    int lo = 0, hi = chunks - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (chunk[mid] > t) hi = mid;
      else lo = mid + 1;
    }
    uint64_t run = lo ? chunk[lo - 1] : 0, wt[VE];
    uint32_t k[VE];
    int i0, who;
    for (int sub = lo * group;; ++sub) {  // the chunk's pieces in order; one of them passes t
      i0 = (sub * WAVE + lane) * VE;
      uint64_t own = 0;
      row.read_at(i0, k);
      kept_weights<VE>(k, i0, cut, lim, wt);
#pragma unroll
      for (int e = 0; e < VE; ++e) own += wt[e];
      const uint64_t end = run + wave_scan64(own);
      const uint64_t past = __ballot(end > t);
      if (past || sub + 1 >= min(subs, (lo + 1) * group)) {
        who = past ? __builtin_ctzll(past) : WAVE - 1;
        run = end - own;
        break;
      }
      run = shfl64(end, WAVE - 1);
    }
    if (lane == who) {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (run <= t && run + wt[e] > t) store_draw(a, at, i0 + e, k[e], lim, log_sum);
        run += wt[e];
      }
    }
  }
}

template <typename T, int THR, int KEYS>
int launch(const RowArgs& a, hipStream_t st) {
  constexpr int piece = WAVE * Row<T, THR, KEYS>::VE;
  const size_t lds = (size_t)std::min((a.cols + piece - 1) / piece, CHUNKS) * 8;
  k_sample<T, THR, KEYS><<<a.rows, THR, lds, st>>>(a);
  return check_launch("sample");
}

template <typename T>
int dispatch(const RowArgs& a, hipStream_t st) {
  if (a.cols <= 2048) return launch<T, 256, 2048>(a, st);
  if (a.cols <= 8192) return launch<T, 512, 8192>(a, st);
  if (a.cols <= 16384) return launch<T, 1024, 16384>(a, st);
  if (a.cols <= 24576) return launch<T, 1024, 24576>(a, st);
  if (a.cols <= ROW_KEYS) return launch<T, 1024, ROW_KEYS>(a, st);
  return launch<T, 1024, 0>(a, st);
}

}  // namespace

int64_t sample_ws_bytes(int, int, int) { return 0; }

int sample(const regcn_sample_desc& d, hipStream_t st) {
  if (d.rows < 0 || d.cols < 0 || d.draws < 0) return set_error(REGCN_EINVAL, "sample: negative size");
  if (d.dtype < REGCN_F32 || d.dtype > REGCN_F16) return set_error(REGCN_EINVAL, "sample: bad element type %d", d.dtype);
  if (d.cols > MAX_COLS) return set_error(REGCN_ENOTSUP, "sample: rows of up to %d scores", MAX_COLS);
  if (!d.ids || !d.u || (d.cols > 0 && !d.score)) return set_error(REGCN_EINVAL, "sample: null score, u or ids");
  if (d.rows > 1 && d.ld < d.cols) return set_error(REGCN_EINVAL, "sample: row stride %lld below cols=%d", (long long)d.ld, d.cols);
  if (d.rows == 0 || d.draws == 0) return 0;
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
  a.ids = d.ids;
  a.logp = d.logp;
  a.c.log2e = 1.4426950408889634074;
  a.c.round = 0x1.8p52;
  a.c.ln2_hi = -6.93147180369123816490e-01;
  a.c.ln2_lo = -1.90821492927058770002e-10;
  double f = 1.0;
  for (int j = 2; j <= 12; ++j) a.c.p[12 - j] = 1.0 / (f *= j);
  int bits = 0;
  while ((1ll << bits) < d.cols) ++bits;
  a.shift = std::min(51, 63 - bits);
  if (d.dtype == REGCN_F32) return dispatch<float>(a, st);
  if (d.dtype == REGCN_BF16) return dispatch<__bf16>(a, st);
  return dispatch<_Float16>(a, st);
}

}  // namespace regcn
