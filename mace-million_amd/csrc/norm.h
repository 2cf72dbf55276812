// What the norms share (norm.hip, groupnorm.hip).
#pragma once
#include "rowvec.h"

namespace mm {
// dw[c] = sum over the n_part rows of part [2][n_part][D] (db: of its second half), in a fixed order; dw, db of out_dtype,
// each nullable
void sum_partials(const float* part, int n_part, int D, int out_dtype, void* dw, void* db, hipStream_t stream);
}  // namespace mm

// v[0 .. N) = the parameters of columns c .., p of T or float, nullable (`none` then)
template <typename T>
__device__ __forceinline__ void mm_norm_param(const void* p, int pdtype_f32, float none, int c, int D, float* v) {
  constexpr int N = MMVec<T>::N;
  if (!p) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = none;
  } else if (pdtype_f32) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c + i < D ? ((const float*)p)[c + i] : 0.f;
  } else {
    mm_load_vec((const T*)p, c, D, v);
  }
}
