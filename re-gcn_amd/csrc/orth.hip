// Orthogonalising matrices by Newton-Schulz products (the step of the Muon optimiser):
//
//   X = G / (|G|_F + eps)              G transposed where it has more rows than columns: m <= n
//   repeat: A = X X^T;  B = b A + c A A;  X = a X + B X
//
// Every product is C = P Q^T with both operands stored row by row along k: A = X (X)^T,
// A A = A (A)^T since A is symmetric, and B X = B (X^T)^T with X^T kept beside X.
//
// Precision.  The products' errors are amplified by a^steps along small singular directions, so they
// are made as exact as fp32 products, on the fp16 matrix cores: an fp32 number x is held as two fp16
// numbers, x = hi + lo / 2048 with hi = fp16(x) and lo = fp16(2048 (x - hi)) (22 bits and a sign, to
// 2^-36 in absolute terms), and
//   P Q^T = hi hi^T + (hi lo^T + lo hi^T) / 2048      (lo lo^T is below 2^-24 of the product)
// in two fp32 accumulators.  Three fp16 products at 8 times the fp32 matrix rate.  X, A and B stay within
// fp16's range (|X| <= 1 at the start; the binding refuses coefficients whose iteration leaves [-4, 4]).
//
// Layout of an operand: rows of 8-element groups, each group 8 hi then 8 lo halves: a tile's k-step of
// 32 is one 128-byte line of a row.  Rows and columns are padded to the tile with zeros, which
// stay zero through every product, so the inner loop has no bounds.
//
// Up to MAXM matrices go through one set of launches (their descriptors travel as kernel arguments):
// norm, split, then three products a step; a workgroup finds its matrix by its index.
#include "elem.h"
#include "regcn_internal.h"

namespace regcn {
namespace {

constexpr int MAXM = 32;      // matrices in a set of launches
constexpr int THR = 256;      // four waves, 2 x 2 over the tile
constexpr int KSTEP = 32;     // k of a stage: a 128-byte line of each row
constexpr int NORM_WGS = 1024;  // most partial sums of a norm
constexpr float LO = 2048.f;  // scale of the low halves

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct Mat {
  const void* g;
  void* out;
  char* ws;
  int32_t m, n;     // m <= n
  int32_t trans;    // G holds X^T
  int32_t dtype;
  int32_t splits;   // of k in A = X X^T
};

struct Job {
  Mat mat[MAXM];
  int32_t start[MAXM + 1];  // first workgroup of each matrix
  int32_t count, side, last;
  float a, b, c, eps;
};

__host__ __device__ inline int pad_to(int v, int t) { return (v + t - 1) / t * t; }

// Where a matrix's operands lie in its workspace.
template <int T>
struct Parts {
  int mp, np;
  int64_t xt[2], x, A, B, norm, split, bytes;
  __host__ __device__ Parts(const Mat& q) {
    mp = pad_to(q.m, T);
    np = pad_to(q.n, T);
    const int64_t xb = (int64_t)mp * np * 4, ab = (int64_t)mp * mp * 4, nt = mp / T;
    xt[0] = 0;
    xt[1] = xb;
    x = 2 * xb;
    A = 3 * xb;
    B = A + ab;
    norm = B + ab;
    split = norm + NORM_WGS * 8;
    bytes = split + (q.splits > 1 ? q.splits * (nt * (nt + 1) / 2) * T * T * 4 : 0);
  }
};

// This workgroup's matrix; wg becomes its index within it.
__device__ __forceinline__ int find_mat(const Job& j, int& wg) {
  // one load a lane and a ballot: a loop over the starts would wait for each in turn
  const int lane = threadIdx.x & 63;
  const int q = __popcll(__ballot(lane < j.count && wg >= j.start[lane + 1]));
  wg -= j.start[q];
  return q;
}

// Tile t of the upper triangle of nt x nt tiles, row by row.
__device__ __forceinline__ void triangle(int t, int nt, int& i, int& j) {
  i = 0;
  while (t >= nt - i) t -= nt - i++;
  j = i + t;
}

// ------------------------------------------------------------------------------------ prologue
template <typename T>
__device__ double sum_squares(const T* __restrict__ g, int64_t count, int part, int parts) {
  constexpr int VE = Piece<T>::VE;
  const int64_t pieces = (count + VE - 1) / VE;
  double s = 0;
  for (int64_t p = (int64_t)part * THR + threadIdx.x; p < pieces; p += (int64_t)parts * THR) {
    float x[VE];
    load_piece<T>(x, g + p * VE, (int)min((int64_t)VE, count - p * VE));
#pragma unroll
    for (int e = 0; e < VE; ++e) s += (double)x[e] * x[e];
  }
  return s;
}

__host__ __device__ inline int norm_parts(int64_t count) {
  return (int)(count < 8192 ? 1 : count / 8192 < NORM_WGS ? count / 8192 : NORM_WGS);
}

// Partial sums of squares in 64 bits (squares of any finite fp32 number neither over- nor underflow).
template <int T>
__global__ __launch_bounds__(THR) void k_norm(Job job) {
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const int64_t count = (int64_t)q.m * q.n;
  const int parts = norm_parts(count);
  double s = q.dtype == REGCN_F32    ? sum_squares((const float*)q.g, count, wg, parts)
             : q.dtype == REGCN_BF16 ? sum_squares((const __bf16*)q.g, count, wg, parts)
                                     : sum_squares((const _Float16*)q.g, count, wg, parts);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  __shared__ double ws[THR / WAVE];
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) ((double*)(q.ws + Parts<T>(q).norm))[wg] = (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

// 8 numbers as a group: 8 hi, 8 lo.
__device__ __forceinline__ void store_group(char* p, const float (&v)[8]) {
  h8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = (_Float16)v[e];
    lo[e] = (_Float16)((v[e] - (float)hi[e]) * LO);
  }
  reinterpret_cast<h8*>(p)[0] = hi;
  reinterpret_cast<h8*>(p)[1] = lo;
}

__device__ __forceinline__ void load_group(float (&v)[8], const char* p) {
  const h8 hi = reinterpret_cast<const h8*>(p)[0], lo = reinterpret_cast<const h8*>(p)[1];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)hi[e] + (float)lo[e] * (1.f / LO);
}

// X and X^T from G: a 64 x 64 tile of X through LDS.
template <int T>
__global__ __launch_bounds__(THR) void k_split(Job job) {
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<T> w(q);
  __shared__ float tile[64][65];
  const int lane = threadIdx.x & 63;
  // every wave sums the partial norms in the same order
  const double* part = (const double*)(q.ws + w.norm);
  const int parts = norm_parts((int64_t)q.m * q.n);
  double s = 0;
#pragma unroll 16
  for (int p = lane; p < parts; p += WAVE) s += part[p];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  const float den = (float)sqrt(s) + job.eps;
  const int nt = w.np / 64, i0 = wg / nt * 64, j0 = wg % nt * 64;
  const int rows = q.trans ? q.n : q.m, cols = q.trans ? q.m : q.n;  // as stored
  const int r0 = q.trans ? j0 : i0, c0 = q.trans ? i0 : j0;
  for (int r = threadIdx.x >> 6; r < 64; r += THR / WAVE) {
    float v = 0.f;
    if (r0 + r < rows && c0 + lane < cols) {
      const int64_t at = (int64_t)(r0 + r) * cols + c0 + lane;
      v = q.dtype == REGCN_F32    ? ((const float*)q.g)[at]
          : q.dtype == REGCN_BF16 ? (float)((const __bf16*)q.g)[at]
                                  : (float)((const _Float16*)q.g)[at];
      v /= den;
    }
    tile[q.trans ? lane : r][q.trans ? r : lane] = v;
  }
  __syncthreads();
  char* X = q.ws + w.x + (int64_t)i0 * w.np * 4 + j0 * 4;
  char* XT = q.ws + w.xt[0] + (int64_t)j0 * w.mp * 4 + i0 * 4;
  for (int it = threadIdx.x; it < 512; it += THR) {
    const int r = it >> 3, g = it & 7;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r][8 * g + e];
    store_group(X + (int64_t)r * w.np * 4 + g * 32, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[8 * g + e][r];
    store_group(XT + (int64_t)r * w.mp * 4 + g * 32, v);
  }
}

// ------------------------------------------------------------------------------------ products
// LDS of a stage: T rows of P, then T rows of Q, 128 bytes each.  The 16-byte piece p of row r lies
// at p ^ ((r >> 1) & 7): the 16 rows that a quarter-wave of a fragment read covers then fall into the 16
// different 16-byte slots of the 64 banks.
__device__ __forceinline__ int swizzle(int row, int piece) { return row * 128 + ((piece ^ ((row >> 1) & 7)) << 4); }

// C tile (T x T) of P Q^T over `steps` k-steps, added up in fp32 as main + cross / 2048 and left in LDS
// as [T][T + 1] floats.  p, q: the tile's first rows; ld: bytes of a row.
template <int T, int STAGES>
__device__ __forceinline__ void product(const char* __restrict__ p, const char* __restrict__ q, int64_t ld, int steps,
                                        char* lds) {
  constexpr int W = T / 2, F = W / 32;          // a wave's square of the tile, in 32 x 32 fragments
  constexpr int LOADS = 2 * T / 8 / 4;          // 8-row loads of a stage and wave
  constexpr int STAGE = 2 * T * 128;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const char* src[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int row = (w * LOADS + u) * 8 + (lane >> 3);
    const char* base = row < T ? p + row * ld : q + (int64_t)(row - T) * ld;
    src[u] = base + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  const auto load = [&](int k, int stage) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
      __builtin_amdgcn_global_load_lds((const void*)(src[u] + (int64_t)k * 128),
                                       (__attribute__((address_space(3))) void*)(lds + stage * STAGE + (w * LOADS + u) * 1024),
                                       16, 0, 0);
  };
  f16v main[F][F] = {}, cross[F][F] = {};
  const int r32 = lane & 31, half = lane >> 5;
  const int wr = (w >> 1) * W, wc = T + (w & 1) * W;
  // stage s is loaded STAGES - 1 steps ahead; one barrier a step: a stage is overwritten only after the
  // barrier that follows its last reads
  for (int s = 0; s < STAGES - 1 && s < steps; ++s) load(s, s);
  for (int k = 0; k < steps; ++k) {
    // this wave's loads of stage k have landed (at most the STAGES - 2 younger stages' are under way)
    if (STAGES == 3 && k + 1 < steps) {
      if (LOADS == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (k + STAGES - 1 < steps) load(k + STAGES - 1, (k + STAGES - 1) % STAGES);
    const char* st = lds + k % STAGES * STAGE;
#pragma unroll
    for (int kk = 0; kk < KSTEP / 16; ++kk) {
      const int g = 2 * (half + 2 * kk);  // piece of the hi halves of this lane's 8 k
      h8 ah[F], al[F], bh[F], bl[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        ah[f] = *reinterpret_cast<const h8*>(st + swizzle(wr + 32 * f + r32, g));
        al[f] = *reinterpret_cast<const h8*>(st + swizzle(wr + 32 * f + r32, g + 1));
        bh[f] = *reinterpret_cast<const h8*>(st + swizzle(wc + 32 * f + r32, g));
        bl[f] = *reinterpret_cast<const h8*>(st + swizzle(wc + 32 * f + r32, g + 1));
      }
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
          main[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], main[i][j], 0, 0, 0);
          cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], cross[i][j], 0, 0, 0);
          cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], cross[i][j], 0, 0, 0);
        }
    }
  }
  __syncthreads();  // the stages are read: their LDS becomes the tile
  float* c = (float*)lds;
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        c[((w >> 1) * W + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3)) * (T + 1) + (w & 1) * W + 32 * j + r32] =
            main[i][j][r] + cross[i][j][r] * (1.f / LO);
  __syncthreads();
}

// The tile in LDS becomes alpha * old + beta * tile (old: the same tile of an operand; null: absent),
// stored as operand rows at `dst` and, transposed, at `dst_t` (null: not stored), both at the tile's corner.
template <int T>
__device__ __forceinline__ void finish(float* c, const char* old, float alpha, float beta, char* dst, char* dst_t,
                                       int64_t ld, int64_t ld_t) {
  constexpr int G = T / 8;
  for (int it = threadIdx.x; it < T * G; it += blockDim.x) {
    const int r = it / G, g = it % G;
    float v[8], x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c[r * (T + 1) + 8 * g + e];
    if (old) {
      load_group(x, old + r * ld + g * 32);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = fmaf(alpha, x[e], beta * v[e]);
        c[r * (T + 1) + 8 * g + e] = v[e];
      }
    }
    if (dst) store_group(dst + r * ld + g * 32, v);
  }
  if (!dst_t) return;
  __syncthreads();
  for (int it = threadIdx.x; it < T * G; it += blockDim.x) {
    const int col = it / 64 * 16 % T + (it & 15), g = it / 64 * 16 / T * 4 + (it >> 4 & 3);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c[(8 * g + e) * (T + 1) + col];
    store_group(dst_t + col * ld_t + g * 32, v);
  }
}

template <typename E>
__device__ __forceinline__ void store8(E* p, const float (&v)[8], int m) {
  constexpr int VE = Piece<E>::VE;
#pragma unroll
  for (int h = 0; h < 8 / VE; ++h) {
    float x[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] = v[h * VE + e];
    store_piece<E>(p + h * VE, x, m - h * VE);
  }
}

__device__ __forceinline__ void store_out(const Mat& q, int64_t at, const float (&v)[8], int m) {
  if (m <= 0) return;
  if (q.dtype == REGCN_F32) store8((float*)q.out + at, v, m);
  else if (q.dtype == REGCN_BF16) store8((__bf16*)q.out + at, v, m);
  else store8((_Float16*)q.out + at, v, m);
}

// The last step's tile into the result, in G's type and orientation.
template <int T>
__device__ __forceinline__ void finish_out(const Mat& q, float* c, const char* old, float alpha, int64_t ld, int i0, int j0) {
  constexpr int G = T / 8;
  for (int it = threadIdx.x; it < T * G; it += blockDim.x) {
    const int r = it / G, g = it % G;
    float v[8], x[8];
    load_group(x, old + r * ld + g * 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = fmaf(alpha, x[e], c[r * (T + 1) + 8 * g + e]);
      c[r * (T + 1) + 8 * g + e] = v[e];
    }
    if (!q.trans && i0 + r < q.m) store_out(q, (int64_t)(i0 + r) * q.n + j0 + 8 * g, v, q.n - j0 - 8 * g);
  }
  if (!q.trans) return;
  __syncthreads();
  for (int it = threadIdx.x; it < T * G; it += blockDim.x) {
    const int col = it / 64 * 16 % T + (it & 15), g = it / 64 * 16 / T * 4 + (it >> 4 & 3);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c[(8 * g + e) * (T + 1) + col];
    if (j0 + col < q.n) store_out(q, (int64_t)(j0 + col) * q.m + i0 + 8 * g, v, q.m - i0 - 8 * g);
  }
}

template <int T>
constexpr int stages() { return T == 64 ? 3 : 2; }
template <int T>
constexpr int lds_bytes() {
  constexpr int a = stages<T>() * 2 * T * 128, b = T * (T + 1) * 4;
  return a > b ? a : b;
}

// A = X X^T, upper triangle of tiles, both halves stored; or one of `splits` pieces of k of a tile.
template <int T>
__global__ __launch_bounds__(THR, 2) void k_gram(Job job) {
  __shared__ __align__(16) char lds[lds_bytes<T>()];
  int wg = blockIdx.x, i, j;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<T> w(q);
  const int nt = w.mp / T, tri = nt * (nt + 1) / 2;
  const int s = wg / tri, t = wg % tri;
  triangle(t, nt, i, j);
  const int64_t ld = (int64_t)w.np * 4;
  const char* X = q.ws + w.x;
  const int all = w.np / KSTEP, k0 = (int)((int64_t)all * s / q.splits), k1 = (int)((int64_t)all * (s + 1) / q.splits);
  product<T, stages<T>()>(X + (int64_t)i * T * ld + k0 * 128, X + (int64_t)j * T * ld + k0 * 128, ld, k1 - k0, lds);
  float* c = (float*)lds;
  if (q.splits > 1) {
    float* part = (float*)(q.ws + w.split) + ((int64_t)s * tri + t) * T * T;
    for (int it = threadIdx.x; it < T * T; it += THR) part[it] = c[it / T * (T + 1) + it % T];
    return;
  }
  const int64_t la = (int64_t)w.mp * 4;
  char* A = q.ws + w.A;
  finish<T>(c, nullptr, 0.f, 1.f, A + i * T * la + j * T * 4, i == j ? nullptr : A + j * T * la + i * T * 4, la, la);
}

// The pieces of k of a tile added up in order: a thread per 4 columns, its pieces' loads under way together.
template <int T>
__global__ __launch_bounds__(T * T / 4 < 1024 ? T * T / 4 : 1024) void k_gram_sum(Job job) {
  __shared__ __align__(16) float c[T * (T + 1)];
  int wg = blockIdx.x, i, j;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<T> w(q);
  const int nt = w.mp / T, tri = nt * (nt + 1) / 2;
  triangle(wg, nt, i, j);
  const f4* part = (const f4*)(q.ws + w.split) + (int64_t)wg * (T * T / 4);
  for (int it = threadIdx.x; it < T * T / 4; it += blockDim.x) {
    f4 v = part[it];
#pragma unroll 8
    for (int s = 1; s < q.splits; ++s) v += part[(int64_t)s * tri * (T * T / 4) + it];
    const int at = it * 4 / T * (T + 1) + it * 4 % T;
#pragma unroll
    for (int e = 0; e < 4; ++e) c[at + e] = v[e];
  }
  __syncthreads();
  const int64_t la = (int64_t)w.mp * 4;
  char* A = q.ws + w.A;
  finish<T>(c, nullptr, 0.f, 1.f, A + i * T * la + j * T * 4, i == j ? nullptr : A + j * T * la + i * T * 4, la, la);
}

// B = b A + c A A, upper triangle of tiles, both halves stored.
template <int T>
__global__ __launch_bounds__(THR, 2) void k_poly(Job job) {
  __shared__ __align__(16) char lds[lds_bytes<T>()];
  int wg = blockIdx.x, i, j;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<T> w(q);
  triangle(wg, w.mp / T, i, j);
  const int64_t la = (int64_t)w.mp * 4;
  const char* A = q.ws + w.A;
  char* B = q.ws + w.B;
  product<T, stages<T>()>(A + i * T * la, A + j * T * la, la, w.mp / KSTEP, lds);
  finish<T>((float*)lds, A + i * T * la + j * T * 4, job.b, job.c, B + i * T * la + j * T * 4,
            i == j ? nullptr : B + j * T * la + i * T * 4, la, la);
}

// X = a X + B X: X in place (a tile is read by its own workgroup only), X^T into its other copy; the last
// step writes the result instead.
template <int T>
__global__ __launch_bounds__(THR, 2) void k_update(Job job) {
  __shared__ __align__(16) char lds[lds_bytes<T>()];
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<T> w(q);
  const int mt = w.mp / T, i = wg % mt, j = wg / mt;
  const int64_t la = (int64_t)w.mp * 4, lx = (int64_t)w.np * 4;
  product<T, stages<T>()>(q.ws + w.B + i * T * la, q.ws + w.xt[job.side] + j * T * la, la, w.mp / KSTEP, lds);
  char* X = q.ws + w.x + i * T * lx + (int64_t)j * T * 4;
  if (job.last)
    finish_out<T>(q, (float*)lds, X, job.a, lx, i * T, j * T);
  else
    finish<T>((float*)lds, X, job.a, 1.f, X, q.ws + w.xt[1 - job.side] + j * T * la + (int64_t)i * T * 4, lx, la);
}

// ---------------------------------------------------------------------------------------- host
// Tiles of 128 fill the card from 192 tiles of X on; below that tiles of 64 give four times the workgroups.
bool wide_tiles(const Mat& q) { return (int64_t)((q.m + 127) / 128) * ((q.n + 127) / 128) >= 192; }

int tile_of(const Mat& q) { return wide_tiles(q) ? 128 : 64; }

// Pieces of k in X X^T: enough for about 512 workgroups, each of at least 24 k-steps (about 6 us: the
// second launch that adds them up costs 4).
int gram_splits(const Mat& q) {
  const int t = tile_of(q), nt = (q.m + t - 1) / t, tri = nt * (nt + 1) / 2, steps = pad_to(q.n, t) / KSTEP;
  return std::max(1, std::min({512 / tri, steps / 24, 32}));
}

template <typename F>
int layout(Job& job, F wgs_of) {
  job.start[0] = 0;
  for (int q = 0; q < job.count; ++q) job.start[q + 1] = job.start[q] + wgs_of(job.mat[q]);
  return job.start[job.count];
}

template <int T>
int run_set(Job& job, int steps, hipStream_t st) {
  int n = layout(job, [](const Mat& q) { return norm_parts((int64_t)q.m * q.n); });
  k_norm<T><<<n, THR, 0, st>>>(job);
  n = layout(job, [](const Mat& q) { return pad_to(q.m, T) / 64 * (pad_to(q.n, T) / 64); });
  k_split<T><<<n, THR, 0, st>>>(job);
  const auto tri = [](const Mat& q) { const int nt = pad_to(q.m, T) / T; return nt * (nt + 1) / 2; };
  for (int s = 0; s < steps; ++s) {
    n = layout(job, [&](const Mat& q) { return tri(q) * q.splits; });
    k_gram<T><<<n, THR, 0, st>>>(job);
    n = layout(job, [&](const Mat& q) { return q.splits > 1 ? tri(q) : 0; });
    if (n) k_gram_sum<T><<<n, std::min(1024, T * T / 4), 0, st>>>(job);
    n = layout(job, tri);
    k_poly<T><<<n, THR, 0, st>>>(job);
    n = layout(job, [](const Mat& q) { return pad_to(q.m, T) / T * (pad_to(q.n, T) / T); });
    job.side = s & 1;
    job.last = s == steps - 1;
    k_update<T><<<n, THR, 0, st>>>(job);
  }
  return check_launch("orthogonalize");
}

int64_t mat_bytes(const Mat& q) {
  const int64_t b = wide_tiles(q) ? Parts<128>(q).bytes : Parts<64>(q).bytes;
  return (b + 255) / 256 * 256;
}

// A valid descriptor as a Mat.
int to_mat(const regcn_matrix& d, Mat& q) {
  if (d.rows <= 0 || d.cols <= 0) return set_error(REGCN_EINVAL, "orthogonalize: bad size %lld x %lld", (long long)d.rows, (long long)d.cols);
  if (d.rows > (1 << 20) || d.cols > (1 << 20)) return set_error(REGCN_ENOTSUP, "orthogonalize: sides up to 2^20");
  if (d.dtype < REGCN_F32 || d.dtype > REGCN_F16) return set_error(REGCN_EINVAL, "orthogonalize: bad element type %d", d.dtype);
  q = Mat{};
  q.g = d.x;
  q.out = d.out;
  q.trans = d.rows > d.cols;
  q.m = (int)std::min(d.rows, d.cols);
  q.n = (int)std::max(d.rows, d.cols);
  q.dtype = d.dtype;
  if ((int64_t)q.m * q.n > (1ll << 40)) return set_error(REGCN_ENOTSUP, "orthogonalize: up to 2^40 elements");
  q.splits = gram_splits(q);
  return 0;
}

// Matrices in sets: one tile size, at most MAXM.
template <typename F>
int for_sets(const regcn_matrix* mats, int count, F run) {
  for (int wide = 0; wide < 2; ++wide) {
    Job job{};
    for (int k = 0; k < count; ++k) {
      Mat q;
      if (int rc = to_mat(mats[k], q)) return rc;
      if (wide_tiles(q) == (bool)wide) job.mat[job.count++] = q;
      if (job.count == MAXM || (k == count - 1 && job.count)) {
        if (int rc = run(job, wide)) return rc;
        job = Job{};
      }
    }
  }
  return 0;
}

}  // namespace

int64_t orthogonalize_ws_bytes(const regcn_matrix* mats, int count) {
  if (!mats || count <= 0) return 0;
  int64_t most = 0;
  if (for_sets(mats, count, [&](Job& job, int) {
        int64_t b = 0;
        for (int q = 0; q < job.count; ++q) b += mat_bytes(job.mat[q]);
        most = std::max(most, b);
        return 0;
      }))
    return 0;
  return most;
}

int orthogonalize(const regcn_matrix* mats, int count, int steps, float a, float b, float c, float eps, void* ws,
                  size_t ws_bytes, hipStream_t st) {
  if (!mats || count < 0) return set_error(REGCN_EINVAL, "orthogonalize: null matrices");
  if (steps < 1 || steps > 1000) return set_error(REGCN_EINVAL, "orthogonalize: 1 to 1000 steps (got %d)", steps);
  if (count == 0) return 0;
  for (int k = 0; k < count; ++k) {
    Mat q;
    if (int rc = to_mat(mats[k], q)) return rc;
    if (!mats[k].x || !mats[k].out) return set_error(REGCN_EINVAL, "orthogonalize: null matrix %d", k);
  }
  const int64_t need = orthogonalize_ws_bytes(mats, count);
  if (!ws || (int64_t)ws_bytes < need)
    return set_error(REGCN_EINVAL, "orthogonalize: workspace of %zu bytes, needs %lld", ws_bytes, (long long)need);
  return for_sets(mats, count, [&](Job& job, int wide) {
    char* p = (char*)ws;
    for (int q = 0; q < job.count; ++q) {
      job.mat[q].ws = p;
      p += mat_bytes(job.mat[q]);
    }
    job.a = a;
    job.b = b;
    job.c = c;
    job.eps = eps;
    return wide ? run_set<128>(job, steps, st) : run_set<64>(job, steps, st);
  });
}

}  // namespace regcn
