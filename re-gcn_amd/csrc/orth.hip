// Orthogonalising matrices by Newton-Schulz products (the step of the Muon optimiser):
//
//   X = G / (|G|_F + eps)              G transposed where it has more rows than columns: m <= n
//   repeat: A = X X^T;  B = b A + c A A;  X = a X + B X
//
// Every product is C = P Q^T with both operands stored row by row along k: A = X (X)^T,
// A A = A (A)^T since A is symmetric, and B X = B (X^T)^T with X^T kept beside X.
//
// Precision.  The products' errors are amplified by a^steps along small singular directions, so they
// are made as exact as fp32 products, on the fp16 matrix cores: an fp32 number is held as two fp16
// numbers, x 2^E = hi + lo, hi and lo the roundings of x 2^E and of what is left (22 bits and a sign; 2^-37
// in absolute terms for X), and
//   P Q^T = hi hi^T + hi lo^T + lo hi^T      (lo lo^T is below 2^-24 of the product)
// in one fp32 accumulator: three fp16 products, each at 16 times the fp32 matrix rate.  The matrix cores take
// subnormal halves as they are.  E is 12 for X and A and 11 for B: the binding refuses coefficients whose
// iteration leaves |s| <= 2 or |b s^2 + c s^4| <= 16, so nothing passes 2^15.
//
// Matrices of up to 64 rows (or columns) stay in fp32 and use the fp32 matrix instruction: their few singular values
// leave little to average errors out, and 3 x 30 in halves was off by 1 to 4.5e-6 of its norm after five steps where
// fp32 is by 0.3 to 1.4e-6; from 100 x 200 on halves are the closer ones (200 x 200: 1.2e-6, 1.6e-6).  Their
// products are short, so it costs little: 3 x 30 71 -> 75 us, 64 x 1024 107 -> 136, 64 x 10000 139 -> 148.
//
// What the halves do not keep: X's 2^-37 is absolute, so a row of G that is 1e-4, 1e-5 or 1e-6 of the others is off by 4e-6,
// 4e-5, 4e-4 of itself (fp32: 3e-7), at any number of steps.  Of the whole matrix that is nothing until the small
// rows have grown by a^steps: the halves' error, modelled in 64 bits over rows of 1 to 1e-8, is 0.3 to 0.7 of fp32's up to 8
// steps, 4 times it at 10, 40 at 12.  So more than 8 steps take fp32 operands, and a caller may ask for them (REGCN_FULL_FP32): 8 steps of 200 x 200
// then take 214 us for 164, of 1333 x 777 576 for 341, of 4096 x 4096 16.9 ms for 6.0.
//
// Layout of an operand: rows of 8-element groups, each group 8 hi then 8 lo halves (or 8 fp32): a tile's k-step of
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
constexpr int FP32_ROWS = 64;  // of matrices that stay in fp32
constexpr int SPLIT_STEPS = 8;  // most steps of operands in halves
constexpr int THR = 256;
constexpr int KSTEP = 32;     // k of a stage: a 128-byte line of each row
constexpr int NORM_WGS = 1024;  // most partial sums of a norm
constexpr float EX = 4096.f, EB = 2048.f;  // 2^E of X and A, of B

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct Mat {
  const void* g;
  void* out;
  char* ws;
  int32_t m, n;     // m <= n
  int32_t trans;    // G holds X^T
  int32_t dtype;
  struct Cut {
    int32_t full, splits;  // whole tiles, pieces of k of the others
  } gram, poly;
  int32_t sym;      // tile of the symmetric products
  int32_t fp32;     // operands held in fp32: tiles of 64
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
  int64_t xb, x, A, B, norm, split, bytes;
  // X^T's two copies (no array: indexed by an argument it would lie in scratch memory)
  __host__ __device__ int64_t xt(int side) const { return side ? xb : 0; }
  __host__ __device__ Parts(const Mat& q) {
    mp = pad_to(q.m, T);
    np = pad_to(q.n, T);
    xb = (int64_t)mp * np * 4;
    const int64_t ab = (int64_t)mp * mp * 4;
    x = 2 * xb;
    A = 3 * xb;
    B = A + ab;
    norm = B + ab;
    split = norm + NORM_WGS * 8;
    const int64_t st = q.sym, nt = mp / st, tri = nt * (nt + 1) / 2;  // the symmetric products' tiles
    const auto cut = [&](const Mat::Cut& c) { return c.splits > 1 ? (tri - c.full) * c.splits * st * st * 4 : 0; };
    bytes = split + (cut(q.gram) > cut(q.poly) ? cut(q.gram) : cut(q.poly));
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

// The workgroups of one XCD (every eighth) take consecutive indices of n, so that what neighbours read in common comes
// into its L2 once.  Two of 200 x 10000, five steps: 309 -> 251 us (279 by the update alone, 279 by the pieces of k
// alone); 1000 x 16000 1,193 -> 1,078; 1024 x 4096 420 -> 397.
__device__ __forceinline__ int by_xcd(int wg, int n) {
  const int x = wg & 7, q = n >> 3, r = n & 7;
  return x * q + min(x, r) + (wg >> 3);
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

// 8 numbers as a group: 8 hi, 8 lo, or 8 fp32.
__device__ __forceinline__ void store_group(char* p, const float (&v)[8], bool fp32) {
  if (fp32) {
    reinterpret_cast<f4*>(p)[0] = f4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f4*>(p)[1] = f4{v[4], v[5], v[6], v[7]};
    return;
  }
  h8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = (_Float16)v[e];
    lo[e] = (_Float16)(v[e] - (float)hi[e]);
  }
  reinterpret_cast<h8*>(p)[0] = hi;
  reinterpret_cast<h8*>(p)[1] = lo;
}

__device__ __forceinline__ void load_group(float (&v)[8], const char* p, bool fp32) {
  if (fp32) {
    const f4 a = reinterpret_cast<const f4*>(p)[0], b = reinterpret_cast<const f4*>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
    return;
  }
  const h8 hi = reinterpret_cast<const h8*>(p)[0], lo = reinterpret_cast<const h8*>(p)[1];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)hi[e] + (float)lo[e];
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
  const double inv = 1.0 / (sqrt(s) + (double)job.eps);  // in 64 bits: the norm of finite numbers may pass the fp32 range
  const int nt = w.np / 64, i0 = wg / nt * 64, j0 = wg % nt * 64;
  const int rows = q.trans ? q.n : q.m, cols = q.trans ? q.m : q.n;  // as stored
  const int r0 = q.trans ? j0 : i0, c0 = q.trans ? i0 : j0;
  constexpr int PER = 64 / (THR / WAVE);  // this wave's rows, their loads under way together
  float v[PER];
  const auto read = [&](const auto* g) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + (threadIdx.x >> 6) + u * (THR / WAVE), c = c0 + lane;
      v[u] = r < rows && c < cols ? (float)g[(int64_t)r * cols + c] : 0.f;
    }
  };
  if (q.dtype == REGCN_F32) read((const float*)q.g);
  else if (q.dtype == REGCN_BF16) read((const __bf16*)q.g);
  else read((const _Float16*)q.g);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = (threadIdx.x >> 6) + u * (THR / WAVE);
    tile[q.trans ? lane : r][q.trans ? r : lane] = (float)(v[u] * inv) * EX;
  }
  __syncthreads();
  char* X = q.ws + w.x + (int64_t)i0 * w.np * 4 + j0 * 4;
  char* XT = q.ws + w.xt(0) + (int64_t)j0 * w.mp * 4 + i0 * 4;
  for (int it = threadIdx.x; it < 512; it += THR) {
    const int r = it >> 3, g = it & 7;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r][8 * g + e];
    store_group(X + (int64_t)r * w.np * 4 + g * 32, v, T == 64 && q.fp32);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[8 * g + e][r];
    store_group(XT + (int64_t)r * w.mp * 4 + g * 32, v, T == 64 && q.fp32);
  }
}

// ------------------------------------------------------------------------------------ products
// LDS of a stage: T rows of P, then T rows of Q, 128 bytes each.  The 16-byte piece p of row r lies
// at p ^ ((r >> 1) & 7): the 16 rows that a quarter-wave of a fragment read covers then fall into the 16
// different 16-byte slots of the 64 banks.
__device__ __forceinline__ int swizzle(int row, int piece) { return row * 128 + ((piece ^ ((row >> 1) & 7)) << 4); }

// Shape of a tile: T x T by R x C waves, each FR x FC fragments of 32 x 32.
template <int T_>
struct Shape {
  static constexpr int T = T_;
  static constexpr int R = 2, C = T == 256 ? 4 : 2, WAVES = R * C, THREADS = 64 * WAVES;
  static constexpr int FR = T / R / 32, FC = T / C / 32;
  static constexpr int STAGE = 2 * T * 128, STAGES = T == 64 ? 3 : 2;
  static constexpr int LOADS = 2 * T / 8 / WAVES;  // 8-row loads of a stage and wave
  // what is finished at a time: SUB x SUB of the tile, [SUB][SUB + 1] floats in LDS, one per 256 threads
  static constexpr int SUB = T < 128 ? T : 128, SUBS = THREADS / THR;
  static constexpr int LDS = STAGES * STAGE > SUBS * SUB * (SUB + 1) * 4 ? STAGES * STAGE : SUBS * SUB * (SUB + 1) * 4;
};

// 16 bytes a lane from base + voff + soff to LDS, lane l's at dst + 16 l.
__device__ __forceinline__ void load_lds(char* base, int voff, int soff, char* dst) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, (short)0, -1, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, soff, 0, 0);
}

// P Q^T over `steps` k-steps into this wave's fragments.  p, q: the tile's first rows; ld: bytes of a row.
// The stages hold 256 rows of T = 128 twice (two workgroups a CU) or 512 rows of T = 256 (one of 8 waves).
// T = 256 halves what a product reads (L2 to LDS) and, with fragments of 128 x 64 a wave, cuts the LDS reads to
// three quarters.
//
// Two half steps of 16 k alternate, each with fragments of its own: while the matrix cores work on one half's,
// the other's are read, and in the second half the next stage's first.  The barrier stands between
// the halves: behind it every wave has read all of stage k, whose place the loads of stage k + STAGES take, and
// stage k + 1 has landed.  So neither an LDS read nor a load is waited for right after its issue.
//
// FP32: the operands hold fp32 numbers and each of the 8 k of a group is a product of its own, two groups at a time.
template <typename S, bool FP32>
__device__ __forceinline__ void product(const char* __restrict__ p, const char* __restrict__ q, int64_t ld, int steps,
                                        char* lds, f16v (&acc)[S::FR][S::FC]) {
  constexpr int T = S::T;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the first half of the waves loads P's rows, the other Q's: 32-bit offsets from a buffer resource
  const bool of_p = w < S::WAVES / 2;
  const uint64_t from = (uint64_t)(of_p ? p : q);  // in scalar registers: a resource in vector ones is looped over
  char* const base = (char*)((uint64_t)__builtin_amdgcn_readfirstlane((int)(from >> 32)) << 32 |
                             (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)from));
  int voff[S::LOADS];
#pragma unroll
  for (int u = 0; u < S::LOADS; ++u) {
    const int row = (w % (S::WAVES / 2) * S::LOADS + u) * 8 + (lane >> 3);
    voff[u] = (int)(row * ld) + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  const auto load = [&](int k, int stage) {
#pragma unroll
    for (int u = 0; u < S::LOADS; ++u) load_lds(base, voff[u], k * 128, lds + stage * S::STAGE + (w * S::LOADS + u) * 1024);
  };
#pragma unroll
  for (int i = 0; i < S::FR; ++i)
#pragma unroll
    for (int j = 0; j < S::FC; ++j) acc[i][j] = f16v{};
  const int r32 = lane & 31, half = lane >> 5;
  const int wr = w / S::C * (T / S::R) + r32, wc = T + w % S::C * (T / S::C) + r32;
  struct Half {
    h8 ah[S::FR], al[S::FR], bh[S::FC], bl[S::FC];
  };
  const auto read = [&](Half& f, const char* st, int kk) {
    const int g = 2 * (half + 2 * kk);  // piece of the hi halves of this lane's 8 k
#pragma unroll
    for (int i = 0; i < S::FC; ++i) f.bh[i] = *reinterpret_cast<const h8*>(st + swizzle(wc, g) + i * 4096);
#pragma unroll
    for (int i = 0; i < S::FR; ++i) f.ah[i] = *reinterpret_cast<const h8*>(st + swizzle(wr, g) + i * 4096);
#pragma unroll
    for (int i = 0; i < S::FC; ++i) f.bl[i] = *reinterpret_cast<const h8*>(st + swizzle(wc, g + 1) + i * 4096);
#pragma unroll
    for (int i = 0; i < S::FR; ++i) f.al[i] = *reinterpret_cast<const h8*>(st + swizzle(wr, g + 1) + i * 4096);
  };
  const auto multiply = [&](const Half& f) {
    if constexpr (FP32) {
      static_assert(S::FR == 1 && S::FC == 1, "one fragment of 32 x 32 a wave");
      const f4 a0 = __builtin_bit_cast(f4, f.ah[0]), a1 = __builtin_bit_cast(f4, f.al[0]);
      const f4 b0 = __builtin_bit_cast(f4, f.bh[0]), b1 = __builtin_bit_cast(f4, f.bl[0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a0[e], b0[e], acc[0][0], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a1[e], b1[e], acc[0][0], 0, 0, 0);
      return;
    }
#pragma unroll
    for (int i = 0; i < S::FR; ++i)
#pragma unroll
      for (int j = 0; j < S::FC; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < S::FR; ++i)
#pragma unroll
      for (int j = 0; j < S::FC; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bl[j], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < S::FR; ++i)
#pragma unroll
      for (int j = 0; j < S::FC; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[i], f.bh[j], acc[i][j], 0, 0, 0);
  };
  // All but the loads of the STAGES - 2 younger stages have landed, for every wave.  No branch in the loop: past
  // the last stage it is loaded again, into a place that nobody reads.
  static_assert(S::STAGES == 2 || (S::STAGES == 3 && S::LOADS == 4), "the wait counts a stage's loads");
  const auto wait = [&] {
    if (S::STAGES == 3) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  const int last = steps - 1;
  for (int s = 0; s < S::STAGES - 1; ++s) load(min(s, last), s);
  wait();
  load(min(S::STAGES - 1, last), S::STAGES - 1);
  Half even, odd;
  read(even, lds, 0);
  // reads, loads and products interleaved one by one, so that the matrix cores never wait for a run of issues
  constexpr int NM = (FP32 ? 8 : 3) * S::FR * S::FC, NR = 2 * (S::FR + S::FC), NL = S::LOADS;
  int at = 0, next = S::STAGE;  // stage k, stage k + 1
  for (int k = 0; k < last; ++k) {
    read(odd, lds + at, 1);
    multiply(even);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);      // LDS read
      __builtin_amdgcn_sched_group_barrier(0x8, NM / NR, 0);  // product
    }
    __builtin_amdgcn_sched_barrier(0);
    wait();
    read(even, lds + next, 0);
    load(min(k + S::STAGES, last), at / S::STAGE);
    multiply(odd);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);  // load
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    at = next;
    next = next == (S::STAGES - 1) * S::STAGE ? 0 : next + S::STAGE;
  }
  read(odd, lds + at, 1);
  multiply(even);
  multiply(odd);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the loads past the end, before the stages become the tile
}

// The same in the matrix's own form.
template <typename S>
__device__ __forceinline__ void product_of(bool fp32, const char* __restrict__ p, const char* __restrict__ q, int64_t ld,
                                           int steps, char* lds, f16v (&acc)[S::FR][S::FC]) {
  if constexpr (S::T == 64) {
    if (fp32) return product<S, true>(p, q, ld, steps, lds, acc);
  }
  product<S, false>(p, q, ld, steps, lds, acc);
}

// The tile through LDS in parts: f(c, i, j, thread) for each SUB x SUB part at row i, column j of the tile, its
// products (times `unscale`) in c, by 256 threads.
template <typename S, typename F>
__device__ __forceinline__ void parts_of(const f16v (&acc)[S::FR][S::FC], float unscale, char* lds, F f) {
  constexpr int SUB = S::SUB, WT = S::T / S::C;  // columns of a wave
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r32 = lane & 31, half = lane >> 5;
  constexpr int ROWS = S::T / SUB, COLS = S::T / SUB;  // parts; a row of parts at a time
  static_assert(S::SUBS == COLS && (ROWS == 1 || S::T / S::R == SUB), "a row of parts is a row of waves, and fits");
#pragma unroll
  for (int pr = 0; pr < ROWS; ++pr) {
    __syncthreads();  // the stages, or the parts before, are read
    if (ROWS == 1 || w / S::C == pr) {
      const int row0 = ROWS == 1 ? w / S::C * (S::T / S::R) : 0, col0 = w % S::C * WT;
      float* c = (float*)lds + col0 / SUB * (SUB * (SUB + 1)) + row0 * (SUB + 1) + col0 % SUB;
#pragma unroll
      for (int i = 0; i < S::FR; ++i)
#pragma unroll
        for (int j = 0; j < S::FC; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            c[(32 * i + 8 * (r >> 2) + 4 * half + (r & 3)) * (SUB + 1) + 32 * j + r32] = acc[i][j][r] * unscale;
    }
    __syncthreads();
    const int part = threadIdx.x / THR;
    f((float*)lds + part * (SUB * (SUB + 1)), pr * SUB, part * SUB, (int)threadIdx.x % THR);
  }
}

// The RW x CL part of a tile in LDS becomes alpha * old + beta * part (old: the same of an operand; null: absent),
// stored as operand rows at `dst` and, transposed, at `dst_t` (null: not stored), both at the part's corner.
// One barrier of the workgroup.
template <int RW, int CL>
__device__ __forceinline__ void finish(bool fp32, float* c, const char* old, float alpha, float beta, char* dst, char* dst_t,
                                       int64_t ld, int64_t ld_t, int thread, int threads) {
  constexpr int G = CL / 8, LD = CL + 1;
  for (int it = thread; it < RW * G; it += threads) {
    const int r = it / G, g = it % G;
    float v[8], x[8];
    if (old) load_group(x, old + r * ld + g * 32, fp32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = beta * c[r * LD + 8 * g + e];
      if (old) v[e] = fmaf(alpha, x[e], v[e]);
      c[r * LD + 8 * g + e] = v[e];
    }
    if (dst) store_group(dst + r * ld + g * 32, v, fp32);
  }
  __syncthreads();
  if (!dst_t) return;
  static_assert(RW % 32 == 0 && CL % 16 == 0, "a wave takes 16 columns of 32 rows");
  for (int it = thread; it < RW * G; it += threads) {
    const int col = it / 64 * 16 % CL + (it & 15), g = it / 64 * 16 / CL * 4 + (it >> 4 & 3);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c[(8 * g + e) * LD + col];
    store_group(dst_t + col * ld_t + g * 32, v, fp32);
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

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t at, const float (&v)[8], int m) {
  if (m <= 0) return;
  if (dtype == REGCN_F32) store8((float*)out + at, v, m);
  else if (dtype == REGCN_BF16) store8((__bf16*)out + at, v, m);
  else store8((_Float16*)out + at, v, m);
}

// The last step's tile into the result, in G's type and orientation.
template <int T>
__device__ __forceinline__ void finish_out(bool fp32, void* out, int dtype, bool trans, int m, int n, float* c, const char* old,
                                           float alpha, int64_t ld, int i0, int j0, int thread) {
  constexpr int G = T / 8;
  for (int it = thread; it < T * G; it += THR) {
    const int r = it / G, g = it % G;
    float v[8], x[8];
    load_group(x, old + r * ld + g * 32, fp32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = fmaf(alpha, x[e], c[r * (T + 1) + 8 * g + e]) * (1.f / EX);
      c[r * (T + 1) + 8 * g + e] = v[e];
    }
    if (!trans && i0 + r < m) store_out(out, dtype, (int64_t)(i0 + r) * n + j0 + 8 * g, v, n - j0 - 8 * g);
  }
  __syncthreads();
  if (!trans) return;
  for (int it = thread; it < T * G; it += THR) {
    const int col = it / 64 * 16 % T + (it & 15), g = it / 64 * 16 / T * 4 + (it >> 4 & 3);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c[(8 * g + e) * (T + 1) + col];
    if (j0 + col < n) store_out(out, dtype, (int64_t)(j0 + col) * m + i0 + 8 * g, v, m - i0 - 8 * g);
  }
}

// Where a workgroup of a symmetric product stands: tile (i, j) of the upper triangle, piece s of k.  The
// first `full` tiles are whole; the others are cut into `splits` pieces of k each, so that a last round of few
// tiles (or a matrix of few) still fills the card.
struct Piece2 {
  int i, j, t, s;  // t: of the cut tiles, -1: whole
};
__device__ __forceinline__ Piece2 symmetric_piece(int wg, int nt, int full, int splits, bool wide) {
  Piece2 p{0, 0, -1, 0};
  const int cut = nt * (nt + 1) / 2 - full;
  // whole tiles: not where 128-wide ones fill the card less than once (2900 x 2900: 1,935 -> 1,995 us; else 1300 x 1300
  // 317 -> 311, 4096 x 4096 3,854 -> 3,795)
  int t = wide && full < 512 ? wg : by_xcd(wg, full);
  if (wg >= full) {
    const int at = by_xcd(wg - full, cut * splits);
    p.t = at % cut;
    p.s = at / cut;
    t = full + p.t;
    if (splits == 1) p.t = -1;
  }
  triangle(t, nt, p.i, p.j);
  return p;
}

// alpha old + beta P P^T of one tile of the upper triangle, both halves stored; or one piece of k of it, stored as
// fp32 partial sums.
template <typename S>
__device__ __forceinline__ void symmetric(bool fp32, const Piece2& at, int splits, const char* P, int64_t ld, int steps, const char* old,
                                          float alpha, float beta, char* out, int64_t la, float* part, int64_t cut,
                                          char* lds) {
  constexpr int T = S::T;
  static_assert(S::SUB == T, "one part");
  const int k0 = at.t < 0 ? 0 : (int)((int64_t)steps * at.s / splits);
  const int k1 = at.t < 0 ? steps : (int)((int64_t)steps * (at.s + 1) / splits);
  f16v acc[S::FR][S::FC];
  product_of<S>(fp32, P + (int64_t)at.i * T * ld + k0 * 128, P + (int64_t)at.j * T * ld + k0 * 128, ld, k1 - k0, lds, acc);
  parts_of<S>(acc, 1.f, lds, [&](float* c, int, int, int thread) {
    if (at.t >= 0) {
      float* to = part + (at.s * cut + at.t) * T * T;
      for (int it = thread; it < T * T; it += THR) to[it] = c[it / T * (T + 1) + it % T];
      return;
    }
    finish<T, T>(fp32, c, old ? old + at.i * T * la + at.j * T * 4 : nullptr, alpha, beta, out + at.i * T * la + at.j * T * 4,
              at.i == at.j ? nullptr : out + at.j * T * la + at.i * T * 4, la, la, thread, THR);
  });
}

// The pieces of k of a cut tile added up in order, then as above: a workgroup a strip of 32 rows, a thread per 4
// columns, its pieces' loads under way together.
constexpr int STRIP = 32;
template <int T>
__device__ __forceinline__ void symmetric_sum(bool fp32, int wg, int nt, int full, int splits, const float* part, const char* old,
                                              float alpha, float beta, char* out, int64_t la, float* c) {
  int i, j;
  const int t = wg / (T / STRIP), r0 = wg % (T / STRIP) * STRIP;
  triangle(full + t, nt, i, j);
  const int64_t cut = nt * (nt + 1) / 2 - full;
  const f4* from = (const f4*)part + (int64_t)t * (T * T / 4) + r0 * (T / 4);
  for (int it = threadIdx.x; it < STRIP * T / 4; it += THR) {
    f4 v = from[it];
#pragma unroll 8
    for (int s = 1; s < splits; ++s) v += from[s * cut * (T * T / 4) + it];
    const int to = it * 4 / T * (T + 1) + it * 4 % T;
#pragma unroll
    for (int e = 0; e < 4; ++e) c[to + e] = v[e];
  }
  __syncthreads();
  const int64_t at = (int64_t)(i * T + r0) * la + j * T * 4;
  finish<STRIP, T>(fp32, c, old ? old + at : nullptr, alpha, beta, out + at,
                   i == j ? nullptr : out + j * T * la + (i * T + r0) * 4, la, la, threadIdx.x, THR);
}

// A = X X^T.  PAD: what the operands are padded to.
template <int PAD, int T>
__global__ __launch_bounds__(THR, 2) void k_gram(Job job) {
  typedef Shape<T> S;
  __shared__ __align__(16) char lds[S::LDS];
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<PAD> w(q);
  const int nt = w.mp / T;
  symmetric<S>(PAD == 64 && q.fp32, symmetric_piece(wg, nt, q.gram.full, q.gram.splits, T == 128), q.gram.splits, q.ws + w.x, (int64_t)w.np * 4,
               w.np / KSTEP, nullptr, 0.f, 1.f / EX, q.ws + w.A, (int64_t)w.mp * 4, (float*)(q.ws + w.split),
               nt * (nt + 1) / 2 - q.gram.full, lds);
}
template <int PAD, int T>
__global__ __launch_bounds__(THR) void k_gram_sum(Job job) {
  __shared__ __align__(16) float c[STRIP * (T + 1)];
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<PAD> w(q);
  symmetric_sum<T>(PAD == 64 && q.fp32, wg, w.mp / T, q.gram.full, q.gram.splits, (const float*)(q.ws + w.split), nullptr, 0.f, 1.f / EX,
                   q.ws + w.A, (int64_t)w.mp * 4, c);
}

// B = b A + c A A.
template <int PAD, int T>
__global__ __launch_bounds__(THR, 2) void k_poly(Job job) {
  typedef Shape<T> S;
  __shared__ __align__(16) char lds[S::LDS];
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<PAD> w(q);
  const int nt = w.mp / T;
  const char* A = q.ws + w.A;
  symmetric<S>(PAD == 64 && q.fp32, symmetric_piece(wg, nt, q.poly.full, q.poly.splits, T == 128), q.poly.splits, A, (int64_t)w.mp * 4,
               w.mp / KSTEP, A, job.b * (EB / EX), job.c * (EB / EX / EX), q.ws + w.B, (int64_t)w.mp * 4, (float*)(q.ws + w.split),
               nt * (nt + 1) / 2 - q.poly.full, lds);
}
template <int PAD, int T>
__global__ __launch_bounds__(THR) void k_poly_sum(Job job) {
  __shared__ __align__(16) float c[STRIP * (T + 1)];
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<PAD> w(q);
  symmetric_sum<T>(PAD == 64 && q.fp32, wg, w.mp / T, q.poly.full, q.poly.splits, (const float*)(q.ws + w.split), q.ws + w.A,
                   job.b * (EB / EX), job.c * (EB / EX / EX), q.ws + w.B, (int64_t)w.mp * 4, c);
}

// X = a X + B X: X in place (a tile is read by its own workgroup only), X^T into its other copy; the last
// step writes the result instead.
template <int T>
__global__ __launch_bounds__(Shape<T>::THREADS, 2) void k_update(Job job) {
  typedef Shape<T> S;
  constexpr int SUB = S::SUB;
  __shared__ __align__(16) char lds[S::LDS];
  int wg = blockIdx.x;
  const Mat& q = job.mat[find_mat(job, wg)];
  const Parts<T> w(q);
  char* const ws = q.ws;
  void* const result = q.out;
  const int m = q.m, n = q.n, dtype = q.dtype;
  const bool trans = q.trans, fp32 = T == 64 && q.fp32;
  const int mt = w.mp / T;
  wg = by_xcd(wg, mt * (w.np / T));
  const int i0 = wg % mt * T, j0 = wg / mt * T;
  const int64_t la = (int64_t)w.mp * 4, lx = (int64_t)w.np * 4;
  f16v acc[S::FR][S::FC];
  product_of<S>(fp32, ws + w.B + i0 * la, ws + w.xt(job.side) + j0 * la, la, w.mp / KSTEP, lds, acc);
  parts_of<S>(acc, 1.f / EB, lds, [&](float* c, int pi, int pj, int thread) {
    const int i = i0 + pi, j = j0 + pj;
    char* X = ws + w.x + i * lx + (int64_t)j * 4;
    if (job.last)
      finish_out<SUB>(fp32, result, dtype, trans, m, n, c, X, job.a, lx, i, j, thread);
    else
      finish<SUB, SUB>(fp32, c, X, job.a, 1.f, X, ws + w.xt(1 - job.side) + j * la + (int64_t)i * 4, lx, la, thread, THR);
  });
}

// ---------------------------------------------------------------------------------------- host
// The tile of X: 256 from 136 of those on, 128 from 192 of those on, else 64, and none that fewer rows than half of it
// would fill.  Measured, five steps: 64 x 40000 542 us in tiles of 256, 232 in 64; 128 x 40000 545, and 264 in 128; 2048 x 4096,
// 128 tiles of 256, 1,125 us in tiles of 128 and 1,266 of 256; 2900 x 2900, 144 tiles, 2,012 and 1,888; 1536 x 1536,
// 144 tiles of 128, 589 us and 447 in 64; 2048 x 4096, 512 tiles, 1,125 and 1,229.
int tile_of(const Mat& q) {
  if (q.fp32) return 64;
  const auto tiles = [&](int t) { return q.m > t / 2 ? (int64_t)((q.m + t - 1) / t) * ((q.n + t - 1) / t) : 0; };
  return tiles(256) >= 136 ? 256 : tiles(128) >= 192 ? 128 : 64;
}

// The tile of the symmetric products, at most 128 (256 would leave half of the CUs idle at 4096): where X's is 128,
// 64 up to 192 tiles of 128 (1024 x 4096, 36 tiles: 531 us in tiles of 128, 413 in 64; 2900 x 2900, 276: 2,012, 2,332).
int sym_tile_of(const Mat& q, int tile) {
  const int64_t nt = (q.m + 127) / 128;
  return tile == 64 || (tile == 128 && nt * (nt + 1) / 2 <= 192) ? 64 : 128;
}

// Which tiles of a symmetric product over `steps` k-steps are cut along k.  Fewer than half of what the card
// holds (two workgroups a CU): cut into pieces of at least 24 k-steps (about 6 us; the second launch that adds them
// up costs 4), 12 in fp32.  More: a last round that fills less than half of it is cut (4096: 16 of 528 tiles; 280 -> 220 us).
Mat::Cut cut_of(int tri, int steps, bool fp32) {
  const int slots = 512, rest = tri % slots;
  const int full = tri - rest;
  if (rest == 0 || rest > slots / 2) return {tri, 1};
  const int splits = full ? std::min({slots / rest, steps / 8, 8}) : std::min({slots / rest, steps / (fp32 ? 12 : 24), fp32 ? 64 : 32});
  if (splits < 2) return {tri, 1};
  return {full, splits};
}

template <typename F>
int layout(Job& job, F wgs_of) {
  job.start[0] = 0;
  for (int q = 0; q < job.count; ++q) job.start[q + 1] = job.start[q] + wgs_of(job.mat[q]);
  return job.start[job.count];
}

template <int T, int ST>
int run_set(Job& job, int steps, hipStream_t st) {
  int n = layout(job, [](const Mat& q) { return norm_parts((int64_t)q.m * q.n); });
  k_norm<T><<<n, THR, 0, st>>>(job);
  n = layout(job, [](const Mat& q) { return pad_to(q.m, T) / 64 * (pad_to(q.n, T) / 64); });
  k_split<T><<<n, THR, 0, st>>>(job);
  const auto tri = [](const Mat& q) { const int nt = pad_to(q.m, T) / ST; return nt * (nt + 1) / 2; };
  const auto wgs = [&](const Mat& q, const Mat::Cut& c) { return c.full + (tri(q) - c.full) * c.splits; };
  const auto sums = [&](const Mat& q, const Mat::Cut& c) { return c.splits > 1 ? (tri(q) - c.full) * (ST / STRIP) : 0; };
  for (int s = 0; s < steps; ++s) {
    n = layout(job, [&](const Mat& q) { return wgs(q, q.gram); });
    k_gram<T, ST><<<n, THR, 0, st>>>(job);
    n = layout(job, [&](const Mat& q) { return sums(q, q.gram); });
    if (n) k_gram_sum<T, ST><<<n, THR, 0, st>>>(job);
    n = layout(job, [&](const Mat& q) { return wgs(q, q.poly); });
    k_poly<T, ST><<<n, THR, 0, st>>>(job);
    n = layout(job, [&](const Mat& q) { return sums(q, q.poly); });
    if (n) k_poly_sum<T, ST><<<n, THR, 0, st>>>(job);
    n = layout(job, [](const Mat& q) { return pad_to(q.m, T) / T * (pad_to(q.n, T) / T); });
    job.side = s & 1;
    job.last = s == steps - 1;
    k_update<T><<<n, Shape<T>::THREADS, 0, st>>>(job);
  }
  return check_launch("orthogonalize");
}

int64_t mat_bytes(const Mat& q) {
  const int t = tile_of(q);
  const int64_t b = t == 256 ? Parts<256>(q).bytes : t == 128 ? Parts<128>(q).bytes : Parts<64>(q).bytes;
  return (b + 255) / 256 * 256;
}

// A valid descriptor as a Mat.
int to_mat(const regcn_matrix& d, Mat& q) {
  if (d.rows <= 0 || d.cols <= 0) return set_error(REGCN_EINVAL, "orthogonalize: bad size %lld x %lld", (long long)d.rows, (long long)d.cols);
  if (d.rows > (1 << 20) || d.cols > (1 << 20)) return set_error(REGCN_ENOTSUP, "orthogonalize: sides up to 2^20");
  const int dtype = d.dtype & ~REGCN_FULL_FP32;
  if (dtype < REGCN_F32 || dtype > REGCN_F16) return set_error(REGCN_EINVAL, "orthogonalize: bad element type %d", d.dtype);
  q = Mat{};
  q.g = d.x;
  q.out = d.out;
  q.trans = d.rows > d.cols;
  q.m = (int)std::min(d.rows, d.cols);
  q.n = (int)std::max(d.rows, d.cols);
  q.dtype = dtype;
  q.fp32 = q.m <= FP32_ROWS || (d.dtype & REGCN_FULL_FP32) != 0;
  if ((int64_t)q.m * q.n > (1ll << 40)) return set_error(REGCN_ENOTSUP, "orthogonalize: up to 2^40 elements");
  const int t = tile_of(q), st = q.sym = sym_tile_of(q, t), nt = pad_to(q.m, t) / st, tri = nt * (nt + 1) / 2;
  q.gram = cut_of(tri, pad_to(q.n, t) / KSTEP, q.fp32);
  q.poly = cut_of(tri, pad_to(q.m, t) / KSTEP, q.fp32);
  return 0;
}

// Matrices in sets: one pair of tile sizes, at most MAXM.
template <typename F>
int for_sets(const regcn_matrix* mats, int count, F run) {
  constexpr int sets[4][2] = {{64, 64}, {128, 64}, {128, 128}, {256, 128}};
  for (const auto& set : sets) {
    Job job{};
    for (int k = 0; k < count; ++k) {
      Mat q;
      if (int rc = to_mat(mats[k], q)) return rc;
      if (tile_of(q) == set[0] && q.sym == set[1]) job.mat[job.count++] = q;
      if (job.count == MAXM || (k == count - 1 && job.count)) {
        if (int rc = run(job, set[0])) return rc;
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
    if (steps > SPLIT_STEPS && !q.fp32)
      return set_error(REGCN_ENOTSUP, "orthogonalize: more than %d steps take REGCN_FULL_FP32 (matrix %d)", SPLIT_STEPS, k);
    if (!mats[k].x || !mats[k].out) return set_error(REGCN_EINVAL, "orthogonalize: null matrix %d", k);
  }
  const int64_t need = orthogonalize_ws_bytes(mats, count);
  if (!ws || (int64_t)ws_bytes < need)
    return set_error(REGCN_EINVAL, "orthogonalize: workspace of %zu bytes, needs %lld", ws_bytes, (long long)need);
  return for_sets(mats, count, [&](Job& job, int tile) {
    char* p = (char*)ws;
    for (int q = 0; q < job.count; ++q) {
      job.mat[q].ws = p;
      p += mat_bytes(job.mat[q]);
    }
    job.a = a;
    job.b = b;
    job.c = c;
    job.eps = eps;
    if (tile == 256) return run_set<256, 128>(job, steps, st);
    if (tile == 128) return job.mat[0].sym == 64 ? run_set<128, 64>(job, steps, st) : run_set<128, 128>(job, steps, st);
    return run_set<64, 64>(job, steps, st);
  });
}

}  // namespace regcn
