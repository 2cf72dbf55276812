// Rows of float, bfloat16 or float16 read and written in 16-byte vectors at any element alignment; lane sums.
#pragma once
#include "common.h"

// element types of the operators that take more than float (the dtype argument of their entry points)
#define MM_F32 0
#define MM_BF16 1
#define MM_F16 2

// CALL with T_ as the element type of a dtype argument.
#define MM_DISPATCH(dtype, CALL)                     \
  do {                                               \
    if ((dtype) == MM_F32) { using T_ = float; CALL; }      \
    else if ((dtype) == MM_BF16) { using T_ = __bf16; CALL; } \
    else { using T_ = _Float16; CALL; }               \
  } while (0)

// 16 bytes of T, known to be aligned to one element only
template <typename T>
struct MMVec {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// v[0 .. N) = p[c .. c + N), zeros from column D on (a row's last vector may be cut)
template <typename T>
__device__ __forceinline__ void mm_load_vec(const T* __restrict__ p, int c, int D, float* v) {
  constexpr int N = MMVec<T>::N;
  if (c + N <= D) {
    const typename MMVec<T>::type x = *(const typename MMVec<T>::type*)(p + c);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < D ? (float)p[c + i] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void mm_store_vec(T* __restrict__ p, int c, int D, const float* v) {
  constexpr int N = MMVec<T>::N;
  if (c + N <= D) {
    typename MMVec<T>::type x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    *(typename MMVec<T>::type*)(p + c) = x;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < D) p[c + i] = (T)v[i];
  }
}

// four values, likewise
template <typename T>
__device__ __forceinline__ void mm_store4(T* __restrict__ p, int c, int N, const float* v) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (c + 4 <= N) {
    *(vec*)(p + c) = vec{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c + q < N) p[c + q] = (T)v[q];
  }
}

template <typename T>
__device__ __forceinline__ void mm_load4(const T* __restrict__ p, int c, int N, float* v) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (c + 4 <= N) {
    const vec x = *(const vec*)(p + c);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = (float)x[q];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = c + q < N ? (float)p[c + q] : 0.f;
  }
}

// The value of the lane at xor distance W / 2, ..., combined by op over groups of W lanes (a power of two up to 64):
// every lane of a group ends with the same bits.  Distances below 16 are DPP moves inside a row of 16 lanes.
template <int W, typename F>
__device__ __forceinline__ float mm_lanes(float v, F op) {
  if constexpr (W >= 2) v = op(v, mm_dpp<0xB1>(v));
  if constexpr (W >= 4) v = op(v, mm_dpp<0x4E>(v));
  if constexpr (W >= 8) v = op(v, mm_dpp<0x141>(v));
  if constexpr (W >= 16) v = op(v, mm_dpp<0x140>(v));
  if constexpr (W >= 32) v = op(v, __shfl_xor(v, 16));
  if constexpr (W >= 64) v = op(v, __shfl_xor(v, 32));
  return v;
}

template <int W>
__device__ __forceinline__ float mm_lanes_sum(float v) {
  return mm_lanes<W>(v, [](float a, float b) { return a + b; });
}

template <int W>
__device__ __forceinline__ float mm_lanes_max(float v) {
  return mm_lanes<W>(v, [](float a, float b) { return fmaxf(a, b); });
}
