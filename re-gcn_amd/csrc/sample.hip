// Sampling ids from scores with temperature, top-k, top-p and min-p, from given random numbers.
//
// For a row s of N scores (NaN and -inf are never taken), in the order "larger score first, ties by
// lower index":
//   w_i = exp((s_i - max s) / T)
//   kept: the first k;  of those the shortest prefix whose weights reach p times their sum;  w_i >= m
//   id(u) = the lowest i whose running sum (by index) of kept weights exceeds u * (sum of kept weights)
// T <= 0 takes the first of the order.  A row without a score to take gives -1.
//
// Weights are whole numbers: round(w 2^S) with 2^S N <= 2^63 (S <= 52), from a 64-bit exp.  Their sums are
// exact in any order, so histograms by atomics, partial sums and prefix sums agree bit for bit.
//
// No sort.  Scores become 32-bit keys of the same order.  Each of k and p asks for the place in the order
// where a running sum (of ones, of weights) reaches a target: a radix descent over the keys finds the
// key (histograms of 11 bits; a round after the first touches the elements of one bin only), and where several
// elements share that key, how many of them, lowest indices first.  So a kept set is {key > K} and
// {key = K, index <= I}.
//
// A workgroup takes a row.  Up to 32768 scores stay in its registers as keys (one read of the scores);
// longer rows are read again in each pass, from the caches where they fit.
#include "elem.h"
#include "regcn_internal.h"

namespace regcn {
namespace {

constexpr int HBITS = 11, HBINS = 1 << HBITS;
constexpr int MAX_KEYS = 32;  // keys a thread holds
constexpr uint32_t ALL = 0xffffffffu;
constexpr int CHUNKS = 4096;  // running sums of kept weights kept in LDS, at most
constexpr int MAX_COLS = 1 << 24;

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
};

struct Limits {
  double inv_t, top_p, min_p;
  uint32_t top_k;  // ALL: off
  int shift;
};

__device__ __forceinline__ Limits row_limits(const RowArgs& a, int row) {
  Limits l;
  const double t = a.temperature_v ? (double)a.temperature_v[row] : a.temperature;
  const int k = a.top_k_v ? a.top_k_v[row] : a.top_k;
  l.top_p = a.top_p_v ? (double)a.top_p_v[row] : a.top_p;
  l.min_p = a.min_p_v ? (double)a.min_p_v[row] : a.min_p;
  l.top_k = k > 0 && k < a.cols ? (uint32_t)k : ALL;
  l.inv_t = 1.0 / t;
  if (!(t > 0)) {  // greedy
    l.inv_t = 1.0;
    l.top_k = 1;
  }
  l.shift = a.shift;
  return l;
}

// 0: never taken; otherwise increasing with the score, -0 and 0 alike.
__device__ __forceinline__ uint32_t score_key(float s) {
  const uint32_t b = __float_as_uint(s + 0.f);
  const uint32_t k = b ^ ((int32_t)b < 0 ? ALL : 0x80000000u);
  return s > -__builtin_inff() ? k : 0u;  // false for NaN
}
__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : ALL)); }

// round(exp(x) 2^S) for x = (s - top) / T <= 0, and exp(x) itself.  exp(x) = 2^n p(r), r = x - n ln 2 in
// two parts, |r| <= ln 2 / 2; p is the Taylor polynomial of degree 13 (remainder below 2^-57).
__device__ __forceinline__ uint64_t weight(uint32_t key, float top, const Limits& l, double* value = nullptr) {
  const float s = key_score(key);
  double x = s == top ? 0.0 : ((double)s - (double)top) * l.inv_t;
  x = x > -700.0 ? x : -700.0;
  const double n = __builtin_rint(x * 1.4426950408889634074);
  double r = fma(n, -6.93147180369123816490e-01, x);
  r = fma(n, -1.90821492927058770002e-10, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int e = (int)n;
  if (value) *value = __builtin_ldexp(p, e);
  // p's 53-bit number, shifted so that its last bit is 2^-S, to nearest
  const uint64_t bits = __double_as_longlong(p);
  const uint64_t m = (bits & ((1ull << 52) - 1)) | (1ull << 52);
  const int sh = 52 - ((int)(bits >> 52) - 1023) - e - l.shift;  // >= -1 (p in [0.7, 1.42), e <= 0)
  if (sh <= 0) return m << -sh;
  return sh > 54 ? 0 : (m + (1ull << (sh - 1))) >> sh;
}

// A place in the order: everything with a larger key, and of its own key the indices up to idx.
struct Cut {
  uint32_t key;
  int idx;
  __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= idx); }
};

template <int THR>
struct Shared {
  uint64_t hist[HBINS];
  uint64_t wave[THR / WAVE];
  uint32_t kmax[THR / WAVE], kmin[THR / WAVE];
  uint64_t above, tie;
  uint32_t bin;
  int idx;
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

// The row as this workgroup sees it: piece q of thread t holds the VE scores from (q THR + t) VE on.
template <typename T, int THR, int NP>  // NP: pieces in registers, 0: read again each time
struct Row {
  static constexpr int VE = Piece<T>::VE;
  const T* p;
  int n, pieces;  // pieces a thread
  uint32_t keys[NP > 0 ? NP : 1][VE];

  __device__ __forceinline__ void read(int q, uint32_t (&k)[VE]) const {
    const int i0 = (q * THR + threadIdx.x) * VE;
    float x[VE];
    const int m = n - i0;
    if (m > 0) load_piece<T>(x, p + i0, m);
#pragma unroll
    for (int e = 0; e < VE; ++e) k[e] = e < m ? score_key(x[e]) : 0u;
  }
  __device__ __forceinline__ void init(const T* row, int cols) {
    p = row;
    n = cols;
    pieces = (cols + THR * VE - 1) / (THR * VE);
    if (NP > 0) {
#pragma unroll
      for (int q = 0; q < NP; ++q) read(q, keys[q]);
    }
  }
  // f(q, first index, keys of the piece) for every piece
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if (NP > 0) {
#pragma unroll
      for (int q = 0; q < NP; ++q) f(q, (q * THR + (int)threadIdx.x) * VE, keys[q]);
    } else {
      for (int q = 0; q < pieces; ++q) {
        uint32_t k[VE];
        read(q, k);
        f(q, (q * THR + (int)threadIdx.x) * VE, k);
      }
    }
  }
};

// The cut where the running sum of `value` over the order first reaches the target, among the elements that
// `in` admits: an element is kept when the sum before it is below the target.  target_of(total) gives the
// target once the total is known (after the first histogram).
template <typename R, int THR, typename In, typename Value, typename Target>
__device__ Cut find_cut(const R& row, Shared<THR>& sh, uint32_t kmin, uint32_t kmax, In in, Value value, Target target_of) {
  constexpr int PER = HBINS / THR;
  uint32_t lo = kmin, hi = kmax;  // the keys still in question
  uint64_t above = 0, target = 0;
  bool first = true;
  for (;;) {
    const uint32_t range = hi - lo;
    const int bits = range ? 32 - __builtin_clz(range) : 0;
    const int shift = bits > HBITS ? bits - HBITS : 0;
    for (int b = threadIdx.x; b < HBINS; b += THR) sh.hist[b] = 0;
    __syncthreads();
    row.each([&](int, int i0, const uint32_t* k) {
#pragma unroll
      for (int e = 0; e < R::VE; ++e)
        if (k[e] >= lo && k[e] <= hi && k[e] && in(k[e], i0 + e))
          atomicAdd((unsigned long long*)&sh.hist[(hi - k[e]) >> shift], (unsigned long long)value(k[e]));
    });
    __syncthreads();
    uint64_t own = 0, total;
    uint64_t h[PER];
#pragma unroll
    for (int b = 0; b < PER; ++b) own += h[b] = sh.hist[threadIdx.x * PER + b];
    uint64_t before = above + block_scan64<THR>(own, sh.wave, &total);
    if (first) target = target_of(total);
    first = false;
    // the bin in which the sum reaches the target: exactly one thread finds it (the target is at most the total)
#pragma unroll
    for (int b = 0; b < PER; ++b) {
      if (before < target && before + h[b] >= target) {
        sh.above = before;
        sh.bin = threadIdx.x * PER + b;
        sh.tie = h[b];
      }
      before += h[b];
    }
    __syncthreads();
    above = sh.above;
    const uint32_t top = hi - (sh.bin << shift);
    const uint32_t low = (1u << shift) - 1;
    lo = max(lo, top >= low ? top - low : 0);
    hi = top;
    if (shift == 0) break;
  }
  // one key left: its elements each add the same; the lowest indices are kept
  const uint64_t one = value(hi), need = one ? (target - above + one - 1) / one : 1, have = one ? sh.tie / one : 1;
  Cut cut{hi, 0x7fffffff};
  if (need < have) {
    uint64_t seen = 0;
    if (threadIdx.x == 0) sh.idx = 0x7fffffff;
    for (int q = 0; q < row.pieces; ++q) {  // THR * VE elements at a time, in index order
      int mine = 0;
      uint32_t k[R::VE];
      const int i0 = (q * THR + (int)threadIdx.x) * R::VE;
      row.read(q, k);
#pragma unroll
      for (int e = 0; e < R::VE; ++e) mine += k[e] == hi && in(k[e], i0 + e);
      uint64_t total;
      uint64_t at = seen + block_scan64<THR>((uint64_t)mine, sh.wave, &total);
#pragma unroll
      for (int e = 0; e < R::VE; ++e)
        if (k[e] == hi && in(k[e], i0 + e) && ++at == need) sh.idx = i0 + e;
      seen += total;
      if (seen >= need) break;
    }
    __syncthreads();
    cut.idx = sh.idx;
  }
  __syncthreads();  // hist and the rest may be written again
  return cut;
}

template <typename T, int THR, int NP>
__global__ __launch_bounds__(THR) void k_sample(RowArgs a) {
  constexpr int VE = Piece<T>::VE, WAVES = THR / WAVE;
  const int subs = (a.cols + WAVE * VE - 1) / (WAVE * VE);  // a wave's pieces: WAVE * VE consecutive scores
  const int group = (subs + CHUNKS - 1) / CHUNKS, chunks = (subs + group - 1) / group;
  __shared__ Shared<THR> sh;
  extern __shared__ uint64_t chunk[];  // running kept weight after each chunk of `group` waves' pieces
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const Limits lim = row_limits(a, r);
  Row<T, THR, NP> row;
  row.init((const T*)a.score + (int64_t)r * a.ld, a.cols);

  uint32_t kmax = 0, kmin = ALL;
  row.each([&](int, int, const uint32_t* k) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      kmax = max(kmax, k[e]);
      kmin = min(kmin, k[e] ? k[e] : ALL);
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    kmax = max(kmax, __shfl_xor(kmax, o));
    kmin = min(kmin, __shfl_xor(kmin, o));
  }
  if (lane == 0) {
    sh.kmax[w] = kmax;
    sh.kmin[w] = kmin;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < WAVES; ++u) {
    kmax = max(kmax, sh.kmax[u]);
    kmin = min(kmin, sh.kmin[u]);
  }
  if (kmax == 0) {  // nothing to take
    for (int d = threadIdx.x; d < a.draws; d += THR) {
      a.ids[(int64_t)r * a.draws + d] = -1;
      if (a.logp) a.logp[(int64_t)r * a.draws + d] = -__builtin_inff();
    }
    return;
  }
  const float top = key_score(kmax);

  Cut cut{0, 0x7fffffff};
  if (lim.top_k != ALL)
    cut = find_cut<Row<T, THR, NP>, THR>(
        row, sh, kmin, kmax, [](uint32_t, int) { return true; }, [](uint32_t) { return (uint64_t)1; },
        [&](uint64_t total) { return min((uint64_t)lim.top_k, total); });
  if (lim.top_p < 1.0) {
    const Cut first = cut;
    cut = find_cut<Row<T, THR, NP>, THR>(
        row, sh, max(kmin, first.key), kmax, [&](uint32_t k, int i) { return first.keeps(k, i); },
        [&](uint32_t k) { return weight(k, top, lim); },
        [&](uint64_t total) {
          const double t = ceil(lim.top_p * (double)total);
          return t < 1.0 ? (uint64_t)1 : min(total, (uint64_t)t);
        });
  }

  // running sums of the kept weights over chunks of consecutive scores
  const auto kept = [&](uint32_t k, int i) -> uint64_t {
    if (!k || !cut.keeps(k, i)) return 0;
    if (lim.min_p > 0) {
      double v;
      const uint64_t x = weight(k, top, lim, &v);
      return v >= lim.min_p || k == kmax ? x : 0;
    }
    return weight(k, top, lim);
  };
  for (int c = threadIdx.x; c < chunks; c += THR) chunk[c] = 0;
  __syncthreads();
  row.each([&](int q, int i0, const uint32_t* k) {
    uint64_t s = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) s += kept(k[e], i0 + e);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint32_t lo = __shfl_xor((uint32_t)s, o), hi = __shfl_xor((uint32_t)(s >> 32), o);
      s += (uint64_t)hi << 32 | lo;
    }
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
  const double log_sum = a.logp ? log((double)sum) - (double)lim.shift * 0.69314718055994530942 : 0.0;
  for (int d = w; d < a.draws; d += WAVES) {
    const int64_t at = (int64_t)r * a.draws + d;
    const double u = a.u_wide ? ((const double*)a.u)[at] : (double)((const float*)a.u)[at];
    const double x = u > 0.0 ? u * (double)sum : 0.0;  // NaN: 0
    const uint64_t t = x < (double)sum ? min((uint64_t)x, sum - 1) : sum - 1;
    int lo = 0, hi = chunks - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (chunk[mid] > t) hi = mid;
      else lo = mid + 1;
    }
    uint64_t run = lo ? chunk[lo - 1] : 0;
    float s[VE];
    uint64_t wt[VE];
    int i0, who;
    for (int sub = lo * group;; ++sub) {  // the chunk's pieces in order; one of them passes t
      i0 = (sub * WAVE + lane) * VE;
      const int m = a.cols - i0;
      uint64_t own = 0;
      if (m > 0) load_piece<T>(s, row.p + i0, m);
#pragma unroll
      for (int e = 0; e < VE; ++e) own += wt[e] = e < m ? kept(score_key(s[e]), i0 + e) : 0;
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
      int id = -1;
      float sc = top;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        run += wt[e];
        if (id < 0 && run > t) {
          id = i0 + e;
          sc = s[e];
        }
      }
      a.ids[at] = id;
      if (a.logp) a.logp[at] = (float)((sc == top ? 0.0 : ((double)sc - (double)top) * lim.inv_t) - log_sum);
    }
  }
}

template <typename T, int THR, int NP>
int launch(const RowArgs& a, hipStream_t st) {
  const size_t lds = (size_t)std::min((a.cols + WAVE * Piece<T>::VE - 1) / (WAVE * Piece<T>::VE) + 1, CHUNKS) * 8;
  k_sample<T, THR, NP><<<a.rows, THR, lds, st>>>(a);
  return check_launch("sample");
}

template <typename T>
int dispatch(const RowArgs& a, hipStream_t st) {
  constexpr int VE = Piece<T>::VE;
  if (a.cols <= 256 * MAX_KEYS / 4) return launch<T, 256, 8 / VE>(a, st);
  const int np = (a.cols + 1024 * VE - 1) / (1024 * VE);
  if (np <= 8 / VE) return launch<T, 1024, 8 / VE>(a, st);
  if (np <= 16 / VE) return launch<T, 1024, 16 / VE>(a, st);
  if (np <= 24 / VE) return launch<T, 1024, 24 / VE>(a, st);
  if (np <= 32 / VE) return launch<T, 1024, 32 / VE>(a, st);
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
  int bits = 0;
  while ((1ll << bits) < d.cols) ++bits;
  a.shift = std::min(52, 63 - bits);
  if (d.dtype == REGCN_F32) return dispatch<float>(a, st);
  if (d.dtype == REGCN_BF16) return dispatch<__bf16>(a, st);
  return dispatch<_Float16>(a, st);
}

}  // namespace regcn
