// Rows of bf16, fp16 or fp32 read and written as fp32, 16 bytes per lane at any element alignment (gfx950 loads and
// stores them unaligned); the vector that crosses the end of a row goes element by element.
#pragma once
#include "common.h"

typedef _Float16 f16;

enum { IO_BF16 = 0, IO_F16 = 1, IO_F32 = 2 };  // element types at the C entry points

template <typename T>
struct RowVec {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// A 16-byte vector held as it is stored.  (As a vector of 16-bit elements the compiler may give every element a register
// of its own.)
typedef unsigned row_u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ row_u32x4 row_raw(const T* at) {
  return __builtin_bit_cast(row_u32x4, *(const typename RowVec<T>::V*)at);
}
template <typename T>
__device__ __forceinline__ float row_element(const row_u32x4& v, int j) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(v[j]);
  } else if constexpr (__is_same(T, bf16)) {
    return __uint_as_float(j & 1 ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16);
  } else {
    typedef f16 H __attribute__((ext_vector_type(2)));
    const unsigned w = v[j >> 1];  // (by value: a vector's element has no address to cast at)
    const H h = __builtin_bit_cast(H, w);
    return (float)h[j & 1];
  }
}
// The compiler would convert a vector once and keep the fp32 copies; after this it converts again.
__device__ __forceinline__ void row_forget(row_u32x4& v) { asm volatile("" : "+v"(v)); }

// VEC (a multiple of the 16-byte vector) consecutive elements from column `col` of a row of C as fp32; zeros behind
// the end
template <typename T, int VEC>
__device__ __forceinline__ void row_load(const T* __restrict__ row, int col, int C, float (&v)[VEC]) {
  constexpr int N = RowVec<T>::N;
  static_assert(VEC % N == 0, "whole vectors");
  if (col + VEC <= C) {
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
      const typename RowVec<T>::V w = *(const typename RowVec<T>::V*)(row + col + i);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = (float)w[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = col + j < C ? (float)row[col + j] : 0.f;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void row_store(T* __restrict__ row, int col, int C, const float (&v)[VEC]) {
  constexpr int N = RowVec<T>::N;
  static_assert(VEC % N == 0, "whole vectors");
  if (col + VEC <= C) {
#pragma unroll
    for (int i = 0; i < VEC; i += N) {
      typename RowVec<T>::V w;
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = (T)v[i + j];
      *(typename RowVec<T>::V*)(row + col + i) = w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (col + j < C) row[col + j] = (T)v[j];
  }
}
