// Rows of activations in 32 or 16 bits: their types, and eight values of one in and out.
#pragma once
#include "common.h"

namespace spx {

// ------------------------------------------------------------------ 16-bit and 32-bit rows
struct RowF32 { typedef float E; };
struct RowF16 { typedef _Float16 E; };
struct RowBF16 { typedef uint16_t E; };

__device__ __forceinline__ float row_get(RowF32, float v) { return v; }
__device__ __forceinline__ float row_get(RowF16, _Float16 v) { return (float)v; }
__device__ __forceinline__ float row_get(RowBF16, uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float row_put(RowF32, float v) { return v; }
__device__ __forceinline__ _Float16 row_put(RowF16, float v) { return (_Float16)v; }
__device__ __forceinline__ uint16_t bf16_rne(float v) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 64);  // NaN stays one
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
__device__ __forceinline__ uint16_t row_put(RowBF16, float v) { return bf16_rne(v); }

// Eight values of a row. VEC: rows lie at multiples of 16 bytes.
template <class R, bool VEC>
__device__ __forceinline__ void get8(const typename R::E *src, float *x) {
  alignas(16) typename R::E e[8];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; i++) ((uint4 *)e)[i] = ((const uint4 *)src)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = src[j];
  }
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = row_get(R{}, e[j]);
}
template <class R, bool VEC>
__device__ __forceinline__ void put8(typename R::E *dst, const float *x) {
  alignas(16) typename R::E e[8];
#pragma unroll
  for (int j = 0; j < 8; j++) e[j] = row_put(R{}, x[j]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; i++) ((uint4 *)dst)[i] = ((const uint4 *)e)[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) dst[j] = e[j];
  }
}

// The same by a flag that is one for the launch; N values out.
template <class R>
__device__ __forceinline__ void get8_if(bool vec, const typename R::E *src, float *x) {
  if (vec) get8<R, true>(src, x);
  else get8<R, false>(src, x);
}
template <class R, int N>
__device__ __forceinline__ void put_if(bool vec, typename R::E *dst, const float *x) {
  typedef typename R::E E;
  alignas(16) E e[N];
#pragma unroll
  for (int i = 0; i < N; i++) e[i] = row_put(R{}, x[i]);
  if (vec) {
    if constexpr (sizeof(e) == 8) *(uint2 *)dst = *(const uint2 *)e;
    else
#pragma unroll
      for (int i = 0; i < (int)sizeof(e) / 16; i++) ((uint4 *)dst)[i] = ((const uint4 *)e)[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) dst[i] = e[i];
  }
}

}  // namespace spx
