// Element types of the operators that take fp32, bf16 or fp16 tensors (lookup.hip, orth.hip,
// sample.hip): conversion to and from fp32 and 16-byte pieces of rows that need not be aligned
// beyond their element.
#pragma once
#include "common.h"

namespace regcn {

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }
// One rounding to nearest even; NaN stays NaN (v_cvt_pk_bf16_f32 / v_cvt_f16_f32).
template <typename T>
__device__ __forceinline__ T from_f32(float v) { return (T)v; }

// 16 bytes of a row: VE elements.  gfx950 reads and writes 16 bytes at any element-aligned
// address, so odd row widths keep wide accesses.
template <typename T>
struct Piece {
  static constexpr int VE = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(VE)));
  typedef vec uvec __attribute__((aligned(sizeof(T))));
};

// o[0..VE) = p[0..m) (the rest 0).
template <typename T>
__device__ __forceinline__ void load_piece(float (&o)[Piece<T>::VE], const T* __restrict__ p, int m) {
  constexpr int VE = Piece<T>::VE;
  if (m >= VE) {
    const typename Piece<T>::vec v = *reinterpret_cast<const typename Piece<T>::uvec*>(p);
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = to_f32<T>(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) o[e] = e < m ? to_f32<T>(p[e]) : 0.f;
  }
}

// p[0..m) = o; `stream`: past the caches (an output larger than they hold).
template <typename T>
__device__ __forceinline__ void store_piece(T* __restrict__ p, const float (&o)[Piece<T>::VE], int m, bool stream = false) {
  constexpr int VE = Piece<T>::VE;
  if (m >= VE) {
    typename Piece<T>::vec v;
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = from_f32<T>(o[e]);
    if (stream)
      __builtin_nontemporal_store((typename Piece<T>::uvec)v, reinterpret_cast<typename Piece<T>::uvec*>(p));
    else
      *reinterpret_cast<typename Piece<T>::uvec*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e < m) p[e] = from_f32<T>(o[e]);
  }
}

}  // namespace regcn
