// Embedding lookup with scaling and its gradient by sorted tokens.
//
//   out[i, :]   = s * table[idx[i], :]
//   dtable[v, :] = s * sum over the tokens i with idx[i] = v, in ascending i, of g[i, :]
//
// An index outside [0, V) reads nothing: its output row is NaN and it joins no gradient row.
// Tokens of `pad` join no gradient row either.
//
// Both directions are bound by memory: the forward reads and writes n rows, the gradient reads
// n rows of g and writes all V rows of dtable once (zeros included; no clearing pass).
//
// The gradient first sorts the tokens by index (stable), so that each row's tokens are one run of
// sorted positions, then sums the runs in a fixed order: no atomics, the same bits on every call.
//   * up to RANK_MAX tokens one launch ranks each token by counting the keys before it;
//   * more take least-significant-digit radix passes of 10 bits (two launches a pass).
// A run of any length is summed over a tree of fan 16 and five levels on the sorted positions (k_partials: nodes whose
// tokens all belong to one row); the row's thread adds the at most 15 tokens or nodes at each end of each level (30 at the
// level where a run ends) and, at the last, one node for every 65,536 tokens of the run.  Sums are fp32; a 16-bit type is
// rounded once, at the store.
#include "elem.h"
#include "regcn_internal.h"

namespace regcn {
namespace {

constexpr int RANK_MAX = 8192;     // tokens ranked by counting (their keys in 32 KB of LDS; two workgroups a CU)
constexpr int FAN = 16, LEVELS = 5;  // the tree of partial sums: 16, 256, 4096, 65536 tokens a node
constexpr int RADIX_BITS = 10, BINS = 1 << RADIX_BITS;
constexpr int MAX_TILES = 256;     // radix tiles (a workgroup each)
constexpr int SORT_THR = 1024, SORT_WAVES = SORT_THR / WAVE;
constexpr int ROW_THR = 256;
// Outputs above half of the card's L2s (8 x 4 MB) are stored past them: nothing of them is left there for
// a reader anyway, and the rows being read stay (a 33 MB lookup: 15.5 -> 10.2 us, a 210 MB one 82 -> 68 us,
// a 268 MB gradient 75 -> 59 us).  Smaller ones stay cached for the kernel that reads them next.
constexpr int64_t STREAM_BYTES = 16 << 20;
constexpr int MAX_ROWS = 512;      // rows a workgroup of k_row_grads
constexpr int DEAL = 32;           // workgroups that share out their rows
constexpr int GRID_Y = 65535;      // most workgroups along a launch's second dimension
constexpr int SLICE = 16;          // 16-byte pieces of the columns a workgroup of k_partials takes

struct Tokens {
  const void* idx;
  int wide;      // idx is int64
  int64_t n, V, pad;
};

// The sort key: the row, or V for a token without one.
__device__ __forceinline__ uint32_t token_key(const Tokens& t, int64_t i) {
  const int64_t v = t.wide ? ((const int64_t*)t.idx)[i] : (int64_t)((const int32_t*)t.idx)[i];
  return (uint32_t)(v < 0 || v >= t.V || v == t.pad ? t.V : v);
}

// ------------------------------------------------------------------------------------ forward
template <typename T>
__global__ __launch_bounds__(ROW_THR) void k_lookup(const T* __restrict__ table, int64_t ld, Tokens t, int d,
                                                    float scale, bool stream_out, T* __restrict__ out) {
  constexpr int VE = Piece<T>::VE;
  const int C = (d + VE - 1) / VE;
  const int64_t total = t.n * C;
  for (int64_t it = (int64_t)blockIdx.x * ROW_THR + threadIdx.x; it < total; it += (int64_t)gridDim.x * ROW_THR) {
    const int64_t i = total <= 0x7fffffff ? (int64_t)((uint32_t)it / (uint32_t)C) : it / C;
    const int c0 = (int)(it - i * C) * VE;
    const int m = d - c0;
    const int64_t v = t.wide ? ((const int64_t*)t.idx)[i] : (int64_t)((const int32_t*)t.idx)[i];
    float x[VE];
    if (v >= 0 && v < t.V) {
      load_piece<T>(x, table + v * ld + c0, m);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) x[e] = __builtin_nanf("");
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] *= scale;
    store_piece<T>(out + i * d + c0, x, m, stream_out);
  }
}

// --------------------------------------------------------------------------------------- sort
// Runs of every row cleared: {first, end} = {0, 0}.
__device__ __forceinline__ void clear_runs(int2* runs, int64_t V) {
  for (int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; v < V; v += (int64_t)gridDim.x * blockDim.x)
    runs[v] = make_int2(0, 0);
}

// One launch for n <= RANK_MAX: a workgroup ranks 64 tokens, each of its 16 waves counting a
// sixteenth of the keys: rank = #{key_j < key} + #{j < i, key_j = key}.  n^2 compares spread over
// the card: 7.5 us at 3,080 tokens, 10.9 at 4,999, 14.4 at 8,192 and 25 at 16,384, where two radix passes take 28
// and grow with n only.
__global__ __launch_bounds__(SORT_THR) void k_rank(Tokens t, int32_t* __restrict__ perm, uint32_t* __restrict__ skey,
                                                   int2* __restrict__ runs) {
  __shared__ __align__(16) uint32_t keys[RANK_MAX];
  __shared__ int part[SORT_WAVES][WAVE];
  clear_runs(runs, t.V);
  const int n = (int)t.n, i0 = blockIdx.x * WAVE;
  if (i0 >= n) return;
  const int npad = (n + 255) & ~255;  // whole uint4 per wave stripe; the padding never counts
  for (int j = threadIdx.x; j < npad; j += SORT_THR) keys[j] = j < n ? token_key(t, j) : 0xffffffffu;
  __syncthreads();
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int i = i0 + lane;
  const uint32_t k = keys[min(i, n - 1)];
  const int per = npad / SORT_WAVES;  // a multiple of 16
  const int j0 = w * per, j1 = j0 + per;
  int cnt = 0;
  // keys of the lower positions count when <= k, those of the higher ones when < k; the 64
  // positions around i0 are told apart one by one
  const int lo = min(j1, i0), hi = max(j0, i0 + WAVE);
#pragma unroll 8
  for (int j = j0; j < lo; j += 4) {
    const uint4 q = *(const uint4*)(keys + j);
    cnt += (q.x <= k) + (q.y <= k) + (q.z <= k) + (q.w <= k);
  }
#pragma unroll 4
  for (int j = max(j0, i0); j < min(j1, i0 + WAVE); j += 4) {
    const uint4 q = *(const uint4*)(keys + j);
    cnt += (q.x < k + (j < i)) + (q.y < k + (j + 1 < i)) + (q.z < k + (j + 2 < i)) + (q.w < k + (j + 3 < i));
  }
#pragma unroll 8
  for (int j = hi; j < j1; j += 4) {
    const uint4 q = *(const uint4*)(keys + j);
    cnt += (q.x < k) + (q.y < k) + (q.z < k) + (q.w < k);
  }
  part[w][lane] = cnt;
  __syncthreads();
  if (w == 0 && i < n) {
    int r = 0;
#pragma unroll
    for (int u = 0; u < SORT_WAVES; ++u) r += part[u][lane];
    perm[r] = i;
    skey[r] = k;
  }
}

// Radix pass, first half: hist[tile][bin] of the pass's digit.
__global__ __launch_bounds__(SORT_THR) void k_hist(Tokens t, const uint32_t* __restrict__ key_in, int shift, int64_t tile,
                                                   uint32_t* __restrict__ hist, int2* __restrict__ runs) {
  __shared__ uint32_t h[BINS];
  if (runs) clear_runs(runs, t.V);
  for (int b = threadIdx.x; b < BINS; b += SORT_THR) h[b] = 0;
  __syncthreads();
  const int64_t p0 = (int64_t)blockIdx.x * tile, p1 = min(p0 + tile, t.n);
  for (int64_t p = p0 + threadIdx.x; p < p1; p += SORT_THR) {
    const uint32_t k = key_in ? key_in[p] : token_key(t, p);
    atomicAdd(&h[(k >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < BINS; b += SORT_THR) hist[(int64_t)blockIdx.x * BINS + b] = h[b];
}

// Second half: each workgroup finds where its tile's bins begin from the whole histogram, then
// places its tokens in order (stable): a wave ranks 64 consecutive tokens at a time by matching
// digits across its lanes, the waves of a 1024-token step in wave order.
__global__ __launch_bounds__(SORT_THR) void k_scatter(Tokens t, const uint32_t* __restrict__ key_in,
                                                      const int32_t* __restrict__ val_in, int shift, int64_t tile,
                                                      const uint32_t* __restrict__ hist, uint32_t* __restrict__ key_out,
                                                      int32_t* __restrict__ val_out) {
  __shared__ uint32_t base[BINS];                  // where the next token of a bin goes
  __shared__ uint16_t wcnt[SORT_WAVES][BINS];      // a step's tokens per wave and bin
  __shared__ uint32_t wsum[SORT_WAVES];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int tiles = gridDim.x, me = blockIdx.x;
  static_assert(BINS == SORT_THR, "a thread per bin");
  uint32_t before = 0, total = 0;
#pragma unroll 32
  for (int s = 0; s < tiles; ++s) {
    const uint32_t c = hist[(int64_t)s * BINS + tid];
    before += s < me ? c : 0;
    total += c;
  }
  // exclusive scan of the totals over the bins
  uint32_t x = total;
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const uint32_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) wsum[w] = x;
  __syncthreads();
  uint32_t wbase = 0;
  for (int u = 0; u < w; ++u) wbase += wsum[u];
  base[tid] = wbase + x - total + before;
  const int64_t p0 = (int64_t)me * tile, p1 = min(p0 + tile, t.n);
  for (int64_t s = p0; s < p1; s += SORT_THR) {
    for (int u = 0; u < SORT_WAVES; ++u) wcnt[u][tid] = 0;
    __syncthreads();
    const int64_t p = s + tid;
    const bool ok = p < p1;
    uint32_t k = 0, dig = 0;
    int32_t val = 0;
    if (ok) {
      k = key_in ? key_in[p] : token_key(t, p);
      val = val_in ? val_in[p] : (int32_t)p;
      dig = (k >> shift) & (BINS - 1);
    }
    uint64_t same = __ballot(ok);
#pragma unroll
    for (int b = 0; b < RADIX_BITS; ++b) {
      const uint64_t m = __ballot((dig >> b) & 1);
      same &= (dig >> b) & 1 ? m : ~m;
    }
    const uint32_t in_wave = __popcll(same & ((1ull << lane) - 1));
    if (ok && in_wave == 0) wcnt[w][dig] = (uint16_t)__popcll(same);
    __syncthreads();
    if (ok) {
      uint32_t r = base[dig] + in_wave;
      for (int u = 0; u < w; ++u) r += wcnt[u][dig];
      key_out[r] = k;
      val_out[r] = val;
    }
    __syncthreads();
    uint32_t add = 0;
    for (int u = 0; u < SORT_WAVES; ++u) add += wcnt[u][tid];
    base[tid] += add;
    __syncthreads();
  }
}

// --------------------------------------------------------------------------------------- sums
// acc += the row pieces row(0) .. row(cnt - 1) in order, up to eight loads in flight.
template <typename T, typename Row>
__device__ __forceinline__ void add_rows(float (&acc)[Piece<T>::VE], int m, int cnt, Row row) {
  constexpr int VE = Piece<T>::VE, U = 8;
  int j = 0;
  for (; j + U <= cnt; j += U) {
    float x[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) load_piece<T>(x[u], row(j + u), m);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] += x[u][e];
  }
  for (; j < cnt; j += 2) {
    float x[2][VE];
    load_piece<T>(x[0], row(j), m);
    load_piece<T>(x[1], row(min(j + 1, cnt - 1)), m);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      acc[e] += x[0][e];
      acc[e] = j + 1 < cnt ? acc[e] + x[1][e] : acc[e];
    }
  }
}

// The same over cnt fp32 partial rows dp apart.
template <int VE>
__device__ __forceinline__ void add_partials(float (&acc)[VE], const float* __restrict__ part, int64_t dp, int cnt) {
#pragma unroll
  for (int h = 0; h < VE / 4; ++h) {
    float a[4] = {acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]};
    add_rows<float>(a, 4, cnt, [&](int j) { return part + j * dp + 4 * h; });
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[4 * h + e] = a[e];
  }
}

template <int VE>
__device__ __forceinline__ void store_partial(float* __restrict__ part, const float (&acc)[VE]) {
  f4* q = reinterpret_cast<f4*>(part);
#pragma unroll
  for (int h = 0; h < VE / 4; ++h) q[h] = f4{acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]};
}

// Partial sums: level 0 is the sorted tokens; a node of level l + 1 is the sum of FAN nodes of level l
// and exists where all its tokens belong to one row.
struct Levels {
  float* part[LEVELS];  // [1..]: nodes of dp floats
};

// Two levels in one launch, a workgroup per FAN * FAN nodes of level `lo`: the sums of FAN nodes each
// (level lo + 1), then, where the whole workgroup's tokens belong to one row, of those (lo + 2).
// Level 0 also writes the ends of the runs that lie in its tokens.
template <typename T, int LO>
__global__ __launch_bounds__(ROW_THR) void k_partials(const T* __restrict__ g, const int32_t* __restrict__ perm,
                                                      const uint32_t* __restrict__ skey, int64_t n, int64_t V, int d,
                                                      int64_t dp, int per, int slice0, int2* __restrict__ runs, Levels lv) {
  constexpr int VE = Piece<T>::VE;
  constexpr int64_t NODE = LO == 0 ? FAN : (int64_t)FAN * FAN * FAN;  // tokens of a node of level LO + 1
  const int64_t p0 = (int64_t)blockIdx.x * NODE * FAN;
  __shared__ int32_t tok[LO == 0 ? FAN * FAN : 1];
  __shared__ int full[FAN];
  if (LO == 0) {  // (every column slice writes the same runs)
    static_assert(LO != 0 || ROW_THR == FAN * FAN, "a thread per token");
    const int64_t p = p0 + threadIdx.x;
    if (p < n) {
      const uint32_t k = skey[p];
      tok[threadIdx.x] = perm[p];
      if (k < V) {
        if (p == 0 || skey[p - 1] != k) runs[k].x = (int)p;
        if (p == n - 1 || skey[p + 1] != k) runs[k].y = (int)p + 1;
      }
    }
  }
  if (threadIdx.x < FAN) {
    const int64_t q = p0 + threadIdx.x * NODE;
    full[threadIdx.x] = q + NODE <= n && skey[q] < V && skey[q] == skey[q + NODE - 1];
  }
  __syncthreads();
  const int slice = (slice0 + blockIdx.y) * per;  // this workgroup's `per` pieces of the columns
  const int C = min((int)(dp / VE) - slice, per);
  const int64_t node0 = (int64_t)blockIdx.x * FAN;
  const int b = threadIdx.x / SLICE, c0 = (slice + threadIdx.x % SLICE) * VE;
  static_assert(FAN * SLICE == ROW_THR, "a thread per node and piece");
  if (full[b] && (int)(threadIdx.x % SLICE) < C) {
    float acc[VE] = {};
    if (LO == 0)
      add_rows<T>(acc, d - c0, FAN, [&](int j) { return g + (int64_t)tok[b * FAN + j] * d + c0; });
    else
      add_partials<VE>(acc, lv.part[LO] + (node0 + b) * FAN * dp + c0, dp, FAN);
    store_partial<VE>(lv.part[LO + 1] + (node0 + b) * dp + c0, acc);
  }
  if (p0 + NODE * FAN > n || skey[p0] >= V || skey[p0] != skey[p0 + NODE * FAN - 1]) return;
  __syncthreads();  // all FAN nodes of level LO + 1 exist and are written
  if ((int)threadIdx.x < C) {
    float acc[VE] = {};
    add_partials<VE>(acc, lv.part[LO + 1] + node0 * dp + c0, dp, FAN);
    store_partial<VE>(lv.part[LO + 2] + (int64_t)blockIdx.x * dp + c0, acc);
  }
}

// Every row of dtable, once: s times the sum of its run of sorted tokens, taken as the run's ends at
// each level and the nodes between them; zero for a row without tokens.  Frequent
// rows often lie side by side, and a wave sums its rows one after the other: so every DEAL workgroups share out
// their rows in groups of 2^grp, a wave's pieces and, where the output goes past the caches, whole 128-byte lines
// (50,000 x 512 bf16, 8,192 tokens of Zipf exponent 1.2: 90 us with a workgroup's rows in one piece, 50 dealt; without
// whole lines a 1,000,000 x 200 fp32 gradient took 361 us for 322).
template <typename T>
__global__ __launch_bounds__(ROW_THR) void k_row_grads(const T* __restrict__ g, const int32_t* __restrict__ perm,
                                                       const int2* __restrict__ runs, Levels lv, int64_t V, int d,
                                                       int64_t dp, int rows, int grp, float scale, bool stream_out,
                                                       T* __restrict__ out) {
  constexpr int VE = Piece<T>::VE;
  const int C = (d + VE - 1) / VE;
  const int64_t first = ((int64_t)(blockIdx.x / DEAL) * DEAL * (rows >> grp) + blockIdx.x % DEAL) << grp;
  const auto row_of = [&](int r) { return first + ((r >> grp) * DEAL << grp) + (r & ((1 << grp) - 1)); };
  __shared__ int2 lrun[MAX_ROWS];  // one wait for all the rows' runs, then stores without loads for empty rows
  for (int r = threadIdx.x; r < rows; r += ROW_THR) {
    const int64_t v = row_of(r);
    if (v < V) lrun[r] = runs[v];
  }
  __syncthreads();
  for (int it = threadIdx.x; it < rows * C; it += ROW_THR) {
    const int r = (int)((uint32_t)it / (uint32_t)C);
    const int c0 = (it - r * C) * VE, m = d - c0;
    const int64_t v = row_of(r);
    if (v >= V) continue;
    const int2 run = lrun[r];
    float acc[VE] = {};
    if (run.x < run.y) {
      int lo = run.x, hi = run.y;
#pragma unroll
      for (int l = 0; l < LEVELS; ++l) {
        const auto add = [&](int a, int b) {
          if (l == 0)
            add_rows<T>(acc, m, b - a, [&](int j) { return g + (int64_t)perm[a + j] * d + c0; });
          else
            add_partials<VE>(acc, lv.part[l] + a * dp + c0, dp, b - a);
        };
        const int up = lo / FAN + (lo % FAN != 0), dn = hi / FAN;
        if (l == LEVELS - 1 || up >= dn) {
          add(lo, hi);
          break;
        }
        add(lo, up * FAN);
        add(dn * FAN, hi);
        lo = up;
        hi = dn;
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) acc[e] *= scale;
    }
    store_piece<T>(out + v * d + c0, acc, m, stream_out);
  }
}

// --------------------------------------------------------------------------------------- host
int elem_size(int dtype) { return dtype == REGCN_F32 ? 4 : 2; }

struct GradWs {
  int2* runs;
  uint32_t* key[2];
  int32_t* val[2];
  uint32_t* hist;
  Levels lv;
  int64_t dp, bytes;
};

// The workspace's parts (ws null: sizes only).  16-byte pieces of 2-byte elements are the widest,
// so the partial rows are rounded up to 8 columns.
GradWs grad_ws(int64_t n, int64_t V, int d, void* ws) {
  GradWs w{};
  char* p = (char*)ws;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    char* q = p ? p + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return q;
  };
  w.dp = ((int64_t)d + 7) / 8 * 8;
  w.runs = (int2*)take(V * 8);
  for (int k = 0; k < 2; ++k) {
    const bool need = k == 0 || n > RANK_MAX;
    w.key[k] = (uint32_t*)take(need ? n * 4 : 0);
    w.val[k] = (int32_t*)take(need ? n * 4 : 0);
  }
  w.hist = (uint32_t*)take(n > RANK_MAX ? (int64_t)MAX_TILES * BINS * 4 : 0);
  for (int l = 1; l < LEVELS; ++l) w.lv.part[l] = (float*)take((n >> (4 * l)) * w.dp * 4);
  w.bytes = at;
  return w;
}

int check_common(const char* what, const void* idx, int64_t n, int64_t V, int d, int dtype) {
  if (d <= 0 || n < 0 || V < 0) return set_error(REGCN_EINVAL, "%s: bad size (n=%lld V=%lld d=%d)", what, (long long)n, (long long)V, d);
  if (n > 0x7fffffff - 1024 || V >= 0x7fffffff || d > 0x7fffffff - 1024) return set_error(REGCN_ENOTSUP, "%s: n, V and d below 2^31 - 1023", what);
  if (dtype < REGCN_F32 || dtype > REGCN_F16) return set_error(REGCN_EINVAL, "%s: bad element type %d", what, dtype);
  if (n > 0 && !idx) return set_error(REGCN_EINVAL, "%s: null index", what);
  return 0;
}

template <typename T>
int launch_lookup(const void* table, int64_t ld, const Tokens& t, int d, float scale, void* out, hipStream_t st) {
  const int64_t total = t.n * ((d + Piece<T>::VE - 1) / Piece<T>::VE);
  const int64_t wgs = (total + ROW_THR - 1) / ROW_THR;
  k_lookup<T><<<(int)std::min<int64_t>(wgs, 1 << 20), ROW_THR, 0, st>>>((const T*)table, ld, t, d, scale,
                                                                       t.n * d * (int64_t)sizeof(T) > STREAM_BYTES, (T*)out);
  return check_launch("embedding lookup");
}

template <typename T>
int launch_grad(const void* g, const Tokens& t, int d, float scale, void* out, const GradWs& w, hipStream_t st) {
  constexpr int VE = Piece<T>::VE;
  const int64_t n = t.n, V = t.V;
  const int clear_wgs = (int)std::min<int64_t>((V + 4 * SORT_THR - 1) / (4 * SORT_THR), 1024);
  int side = 0;  // which of the key / val pairs holds the sorted tokens
  if (n <= RANK_MAX) {
    const int wgs = std::max((int)((n + WAVE - 1) / WAVE), clear_wgs);
    if (wgs > 0)
      k_rank<<<wgs, SORT_THR, 0, st>>>(t, w.val[0], w.key[0], w.runs);
  } else {
    int bits = 0;
    while (V >> bits) ++bits;  // the key V itself included
    const int passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
    int64_t tile = (n + MAX_TILES - 1) / MAX_TILES;
    tile = std::max<int64_t>((tile + SORT_THR - 1) / SORT_THR * SORT_THR, 2 * SORT_THR);
    const int tiles = (int)((n + tile - 1) / tile);
    for (int p = 0; p < passes; ++p) {
      const uint32_t* ki = p ? w.key[side] : nullptr;
      const int32_t* vi = p ? w.val[side] : nullptr;
      const int to = p ? 1 - side : 0;
      k_hist<<<tiles, SORT_THR, 0, st>>>(t, ki, p * RADIX_BITS, tile, w.hist, p ? nullptr : w.runs);
      k_scatter<<<tiles, SORT_THR, 0, st>>>(t, ki, vi, p * RADIX_BITS, tile, w.hist, w.key[to], w.val[to]);
      side = to;
    }
  }
  if (int rc = check_launch("embedding gradient sort")) return rc;
  const uint32_t* skey = w.key[side];
  const int32_t* perm = w.val[side];
  static_assert(FAN == 16, "levels by shifts of 4");
  const int slices = (int)((w.dp / VE + SLICE - 1) / SLICE);
  const int per = ((int)(w.dp / VE) + slices - 1) / slices;
  for (int y0 = 0; n > 0 && y0 < slices; y0 += GRID_Y) {  // (one launch each up to a row of 4 M fp32)
    const int ys = std::min(slices - y0, GRID_Y);
    k_partials<T, 0><<<dim3((int)((n + FAN * FAN - 1) / (FAN * FAN)), ys), ROW_THR, 0, st>>>((const T*)g, perm, skey, n, V, d, w.dp, per,
                                                                                             y0, w.runs, w.lv);
    if (n >> 12)
      k_partials<T, 2><<<dim3((int)((n + 65535) / 65536), ys), ROW_THR, 0, st>>>((const T*)g, perm, skey, n, V, d, w.dp, per, y0, w.runs,
                                                                                  w.lv);
  }
  const int C = (d + VE - 1) / VE;
  // rows a workgroup: enough for its 256 threads, up to 2048 pieces while that leaves 2048 workgroups
  const int64_t want = std::min<int64_t>(2048, std::max<int64_t>(ROW_THR, V * C / 2048));
  const bool stream_out = V * d * (int64_t)sizeof(T) > STREAM_BYTES;
  int grp = 0, lines = 0;  // at most 6: rows <= MAX_ROWS
  while (C << grp < WAVE) ++grp;
  while (((d * (int64_t)sizeof(T)) << lines) % 128) ++lines;
  if (stream_out && (int64_t)C << lines <= 4096) grp = std::max(grp, lines);
  const int rows = std::max(1, std::min(MAX_ROWS, (int)(want / C)) >> grp) << grp;
  const int64_t dealt = (int64_t)DEAL * rows;
  k_row_grads<T><<<(int)((V + dealt - 1) / dealt * DEAL), ROW_THR, 0, st>>>((const T*)g, perm, w.runs, w.lv, V, d, w.dp, rows,
                                                                           grp, scale, stream_out, (T*)out);
  return check_launch("embedding gradient");
}

}  // namespace

int64_t embedding_grad_ws_bytes(int64_t n, int64_t V, int d) {
  if (n < 0 || V < 0 || d <= 0) return 0;
  return grad_ws(n, V, d, nullptr).bytes;
}

int embedding(const void* table, int64_t ld, const void* idx, int wide, int64_t n, int64_t V, int d, int dtype, float scale,
              void* out, hipStream_t st) {
  if (int rc = check_common("embedding", idx, n, V, d, dtype)) return rc;
  if (n == 0) return 0;
  if ((V > 0 && !table) || !out) return set_error(REGCN_EINVAL, "embedding: null table or output");
  if (V > 1 && ld < d) return set_error(REGCN_EINVAL, "embedding: row stride %lld below d=%d", (long long)ld, d);
  const Tokens t{idx, wide != 0, n, V, -1};
  if (dtype == REGCN_F32) return launch_lookup<float>(table, ld, t, d, scale, out, st);
  if (dtype == REGCN_BF16) return launch_lookup<__bf16>(table, ld, t, d, scale, out, st);
  return launch_lookup<_Float16>(table, ld, t, d, scale, out, st);
}

int embedding_grad(const void* g, const void* idx, int wide, int64_t n, int64_t V, int d, int64_t pad, int dtype,
                   float scale, void* out, void* ws, size_t ws_bytes, hipStream_t st) {
  if (int rc = check_common("embedding gradient", idx, n, V, d, dtype)) return rc;
  if (V == 0) return 0;
  if ((n > 0 && !g) || !out) return set_error(REGCN_EINVAL, "embedding gradient: null gradient or output");
  const GradWs w = grad_ws(n, V, d, ws);
  if (!ws || ws_bytes < (size_t)w.bytes)
    return set_error(REGCN_EINVAL, "embedding gradient: workspace of %zu bytes, needs %lld", ws_bytes, (long long)w.bytes);
  const Tokens t{idx, wide != 0, n, V, pad < 0 ? -1 : pad};
  if (dtype == REGCN_F32) return launch_grad<float>(g, t, d, scale, out, w, st);
  if (dtype == REGCN_BF16) return launch_grad<__bf16>(g, t, d, scale, out, w, st);
  return launch_grad<_Float16>(g, t, d, scale, out, w, st);
}

}  // namespace regcn
