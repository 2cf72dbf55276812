// Newton-Schulz orthogonalisation of a batch of matrices:
//     X = M / (|M| + eps),  steps times:  A = X X^T,  X <- a X + (b A + c A A) X     (on the shorter side of M)
// Each step drives the singular values of X towards 1 by the odd polynomial a s + b s^3 + c s^5.  Bound by the matrix
// cores: with m <= n the sides, 2 m^2 n + 2 m^3 + 2 m^2 n operations a step.
//
// X is carried in fp32 and a X is added in fp32: small singular values, which grow by a in every step, keep its bits.
// The products take float16 operands, scaled by powers of two (X and A by 2^12, B = b A + c A A by 2^10) into the middle
// of its range: one plane for bfloat16 matrices (2^-11 of an operand, against 2^-8 of the result's own rounding), two
// planes and three products (2^-22) for float and float16.  Entries of X, A and W (of the small matrices, below) have
// to stay below 16, of B below 64: the norm of M bounds X and A by 1 at first, and the usual coefficients keep all of
// them below 3; what passes becomes infinite or NaN.  Norms are summed in 64 bits, so that neither large nor tiny
// values leave the range.
#include "nt.h"

#include <utility>

#define MM_ORTHO_PARTS 1024   // partial sums of a matrix's norm, at most
#define MM_ORTHO_X 4096.f     // scales of the operands
#define MM_ORTHO_A 4096.f
#define MM_ORTHO_B 1024.f

template <typename T>
struct MMOrthoType {
  static constexpr int P = sizeof(T) == 2 && !__is_same(T, _Float16) ? 1 : 3, PLANES = P == 1 ? 1 : 2;
};

typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));

template <int PLANES>
__device__ __forceinline__ void mm_ortho_put4(_Float16* __restrict__ p, long plane, const float* v) {
  halfx4 h[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[0][i] = (_Float16)v[i];
    h[1][i] = (_Float16)(v[i] - (float)h[0][i]);
  }
#pragma unroll
  for (int q = 0; q < PLANES; ++q) *(halfx4*)(p + q * plane) = h[q];
}

// sums of squares of parts of matrix blockIdx.y
template <typename T>
__global__ void __launch_bounds__(256)
mm_ortho_norm_kernel(const T* __restrict__ m, long size, double* __restrict__ part) {
  constexpr int N = MMVec<T>::N;
  __shared__ double s[4];
  const T* __restrict__ p = m + (long)blockIdx.y * size;
  const long nv = (size + N - 1) / N;
  double t = 0.;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < nv; i += (long)gridDim.x * 256) {
    const long at = i * N;
    float v[N];
    mm_load_vec(p + at, 0, (int)min((long)N, size - at), v);
#pragma unroll
    for (int j = 0; j < N; ++j) t = fma((double)v[j], (double)v[j], t);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) part[(long)blockIdx.y * gridDim.x + blockIdx.x] = s[0] + s[1] + s[2] + s[3];
}

struct MMOrtho {
  const void* m;
  void* out;
  double* part;
  float* x;                       // [batch][rows][cols]
  // planes of [batch]: X [rows][ldu], X^T [cols][ldv], A and B [side][lda]; the one that a step multiplies (X^T if rows
  // <= cols, else X) is written to `next` meanwhile
  _Float16 *u, *v, *a, *b, *next;
  float* sums;                    // [splits][batch][side][lda] of A's parts, where the longer side is split
  int splits;
  long ldu, ldv, lda, pu, pv, pa;   // pu, pv, pa: distance of planes
  int batch, rows, cols, side, parts;
  float ca, cb, cc, eps;
};

// 64 x 64 values a workgroup: X = M / (|M| + eps) and its planes; out (no steps): X itself
template <typename T>
__global__ void __launch_bounds__(256) mm_ortho_start_kernel(MMOrtho a, int steps) {
  constexpr int PLANES = MMOrthoType<T>::PLANES;
  __shared__ float s[64][65];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, e = blockIdx.z;
  const int q = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
  __shared__ double s_norm[4];
  double norm = 0.;
  for (int i = threadIdx.x; i < a.parts; i += 256) norm += a.part[(long)e * a.parts + i];
#pragma unroll
  for (int d = 32; d; d >>= 1) norm += __shfl_xor(norm, d);
  if ((threadIdx.x & 63) == 0) s_norm[threadIdx.x >> 6] = norm;
  __syncthreads();
  norm = s_norm[0] + s_norm[1] + s_norm[2] + s_norm[3];
  const double by = 1. / (sqrt(norm) + (double)a.eps);
  const long size = (long)a.rows * a.cols;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + q + 16 * k;
    float v[4] = {};
    if (r < a.rows) {
      mm_load4((const T*)a.m + e * size + (long)r * a.cols, c0 + c, a.cols, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = v[i] == 0.f ? v[i] : (float)((double)v[i] * by);   // no norm: zeros stay
      if (!steps) {
        mm_store4((T*)a.out + e * size + (long)r * a.cols, c0 + c, a.cols, v);
      } else {
        mm_store4(a.x + e * size + (long)r * a.cols, c0 + c, a.cols, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= MM_ORTHO_X;
        mm_ortho_put4<PLANES>(a.u + ((long)e * a.rows + r) * a.ldu + c0 + c, a.pu, v);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[q + 16 * k][c + i] = v[i];
  }
  if (!steps) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int col = c0 + q + 16 * k;
    if (col >= a.cols) continue;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = s[c + i][q + 16 * k];
    mm_ortho_put4<PLANES>(a.v + ((long)e * a.cols + col) * a.ldv + r0 + c, a.pv, v);
  }
}

// one value, as mm_ortho_put4
__device__ __forceinline__ void mm_ortho_put1(_Float16* p, long plane, float v) {
  const _Float16 h = (_Float16)v;
  p[0] = h;
  p[plane] = (_Float16)(v - (float)h);
}

// out = f acc as planes, rows (or, transposed, columns) of it: one plane through LDS in whole lines, two from the
// registers (their tiles are small, and LDS would take two barriers for each plane).  HALF: of a tile on the diagonal,
// what lies on and below it (transposed: what lies below it).
template <int PLANES, bool HALF = false, typename Nt>
__device__ __forceinline__ void mm_ortho_tiles(const Nt& t, uint4* lds, _Float16* out, long ld, long plane, int rows,
                                               int cols, float f) {
  if constexpr (PLANES == 1) {
    mm_nt_store(t, (_Float16*)lds, out, ld, rows, cols, [&](int i, int j) { return t.acc[i][j] * f; });
  } else {
#pragma unroll
    for (int j = 0; j < Nt::FM; ++j)
#pragma unroll
      for (int i = 0; i < Nt::FN; ++i) {
        const floatx4 v = t.acc[i][j] * f;
        const int m = t.row(j), n = t.col(i);
        _Float16* const p = out + (long)m * ld + n;
        if (m >= rows || n >= cols) continue;
        if (!HALF || n + 3 <= m) {
          mm_ortho_put4<2>(p, plane, (const float*)&v);
        } else {
#pragma unroll
          for (int q = 0; q < 3; ++q)
            if (n + q <= m) mm_ortho_put1(p + q, plane, v[q]);
        }
      }
  }
}

template <int PLANES, bool HALF = false, typename Nt>
__device__ __forceinline__ void mm_ortho_tiles_transposed(const Nt& t, uint4* lds, _Float16* out, long ld, long plane,
                                                          int rows, int cols, float f) {
  if constexpr (PLANES == 1) {
    mm_nt_store_transposed(t, (_Float16*)lds, out, ld, rows, cols, [&](int i, int j) { return t.acc[i][j] * f; });
  } else {
#pragma unroll
    for (int j = 0; j < Nt::FM; ++j)
#pragma unroll
      for (int i = 0; i < Nt::FN; ++i) {
        const int m = t.row(j) & ~3, n = t.col(i) + (t.lane & 3);
        const floatx4 v = t.acc[i][j] * f;
        _Float16 h[4], l[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          h[q] = (_Float16)v[q];
          l[q] = (_Float16)(v[q] - (float)h[q]);
        }
        mm_quad_transpose(h);
        mm_quad_transpose(l);
        if (m >= rows || n >= cols) continue;
        _Float16* const p = out + (long)n * ld + m;
        if (!HALF || m > n) {
          *(halfx4*)p = halfx4{h[0], h[1], h[2], h[3]};
          *(halfx4*)(p + plane) = halfx4{l[0], l[1], l[2], l[3]};
        } else {
#pragma unroll
          for (int q = 1; q < 4; ++q)
            if (m + q > n) {
              p[q] = h[q];
              p[plane + q] = l[q];
            }
        }
      }
  }
}

// 4096 x 8192 bfloat16: 214 us for A (640 TFLOP/s of the half that is computed), 122 for B: 136 tiles on 256 CUs.
// A = X X^T (WHAT 0) or B = b A + c A A (1): planes [side][lda], zeros past the last column.  Both are symmetric: tiles
// below the diagonal are written twice, those above are not computed.  Two planes' products (high x low, low x high) come
// in the other order above the diagonal, so there a tile on it is written twice as well: a result then has the same bits
// whatever the tiles, which the number of matrices decides.
template <int P, int WHAT, typename Nt>
__global__ void __launch_bounds__(Nt::TH, Nt::PER_CU) mm_ortho_square_kernel(MMOrtho a, int tiles) {
  constexpr int PLANES = P == 1 ? 1 : 2;
  extern __shared__ uint4 mm_ortho_lds[];
  int e, tm, tn, split = 0;
  if (!mm_nt_lower(blockIdx.x, WHAT ? a.batch : a.batch * a.splits, tiles, &e, &tm, &tn)) return;
  if (WHAT == 0) {
    split = e / a.batch;
    e -= split * a.batch;
  }
  MMNtOperand<_Float16> x;
  int k;
  if constexpr (WHAT == 1) {
    x = {a.a + (long)e * a.side * a.lda, a.lda, a.pa, a.side};
    k = (int)(a.lda / MM_NT_K);
  } else if (a.rows <= a.cols) {
    x = {a.u + (long)e * a.rows * a.ldu, a.ldu, a.pu, a.side};
    k = (int)(a.ldu / MM_NT_K);
  } else {
    x = {a.v + (long)e * a.cols * a.ldv, a.ldv, a.pv, a.side};
    k = (int)(a.ldv / MM_NT_K);
  }
  const int m0 = tm * Nt::BM, n0 = tn * Nt::BN;
  Nt t;
  if (WHAT == 0 && a.splits > 1) {   // a part of the sums, of the lower tiles alone
    t.run(x, m0, x, n0, (int)((long)k * split / a.splits), (int)((long)k * (split + 1) / a.splits), mm_ortho_lds);
    float* sums = a.sums + ((long)split * a.batch + e) * a.side * a.lda;
#pragma unroll
    for (int j = 0; j < Nt::FM; ++j)
#pragma unroll
      for (int i = 0; i < Nt::FN; ++i) {
        const int m = m0 + t.row(j), n = n0 + t.col(i);
        if (m < a.side && n < a.lda) *(floatx4*)(sums + (long)m * a.lda + n) = t.acc[i][j];
      }
    return;
  }
  t.run(x, m0, x, n0, 0, k, mm_ortho_lds);
  _Float16* out = (WHAT ? a.b : a.a) + (long)e * a.side * a.lda;
  const _Float16* in = a.a + (long)e * a.side * a.lda;
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j) {
    const int m = m0 + t.row(j);
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i) {
      const int n = n0 + t.col(i);
      floatx4 v = {};
      if (m < a.side && n < a.side) {
        if constexpr (WHAT == 0) {
          v = t.acc[i][j] * (MM_ORTHO_A / (MM_ORTHO_X * MM_ORTHO_X));
        } else {
          const halfx4 h = *(const halfx4*)(in + (long)m * a.lda + n);
          const halfx4 l = *(const halfx4*)(in + (PLANES == 2 ? a.pa : 0) + (long)m * a.lda + n);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float old = (float)h[q] + (PLANES == 2 ? (float)l[q] : 0.f);
            v[q] = a.cb * (MM_ORTHO_B / MM_ORTHO_A) * old
                 + a.cc * (MM_ORTHO_B / (MM_ORTHO_A * MM_ORTHO_A)) * t.acc[i][j][q];
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = n + q < a.side ? v[q] : 0.f;
      }
      t.acc[i][j] = v;
    }
  }
  const int left = (int)a.lda - n0, low = (int)a.lda - m0;   // columns with their zeros
  if (PLANES > 1 && tm == tn) {
    mm_ortho_tiles<PLANES, true>(t, mm_ortho_lds, out + (long)m0 * a.lda + n0, a.lda, a.pa, a.side - m0, left, 1.f);
    mm_ortho_tiles_transposed<PLANES, true>(t, mm_ortho_lds, out + (long)n0 * a.lda + m0, a.lda, a.pa, low, a.side - n0,
                                            1.f);
    return;
  }
  mm_ortho_tiles<PLANES>(t, mm_ortho_lds, out + (long)m0 * a.lda + n0, a.lda, a.pa, a.side - m0, left, 1.f);
  if (tm != tn)
    mm_ortho_tiles_transposed<PLANES>(t, mm_ortho_lds, out + (long)n0 * a.lda + m0, a.lda, a.pa, low, a.side - n0, 1.f);
}

// A from its parts: the values on and below the diagonal summed and written twice, zeros past the last column; one
// thread for 4 columns of a row.
template <int PLANES>
__global__ void __launch_bounds__(256) mm_ortho_join_kernel(MMOrtho a) {
  const int nv = (int)(a.lda / 4);
  const int one = a.side * nv, e = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;   // one: at most 192 x 48
  if (i >= one) return;
  const int m = i / nv, n = (i - m * nv) * 4;
  floatx4 v = {};
  const float* p = a.sums + (long)e * a.side * a.lda;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = n + q < a.side ? n + q : 0;
      const float u = c <= m ? p[(long)m * a.lda + c] : p[(long)c * a.lda + m];
      v[q] += n + q < a.side ? u : 0.f;
    }
    p += (long)a.batch * a.side * a.lda;
  }
  v *= MM_ORTHO_A / (MM_ORTHO_X * MM_ORTHO_X);
  mm_ortho_put4<PLANES>(a.a + ((long)e * a.side + m) * a.lda + n, a.pa, (const float*)&v);
}

// 4096 x 8192 bfloat16: 350 us, 785 TFLOP/s; the epilogue moves 16 bytes a value (X in fp32, both planes of halves).
// X <- a X + B X (rows <= cols) or a X + X B; the last step writes out alone.  Other workgroups still read the operand
// of X's planes: its new values go to a.next.
template <typename T, typename Nt>
__global__ void __launch_bounds__(Nt::TH, Nt::PER_CU)
mm_ortho_step_kernel(MMOrtho a, int tiles_m, int tiles_n, int last) {
  constexpr int PLANES = MMOrthoType<T>::PLANES;
  extern __shared__ uint4 mm_ortho_lds[];
  int e, tm, tn;
  if (!mm_nt_tile(blockIdx.x, a.batch, tiles_m, tiles_n, &e, &tm, &tn)) return;
  const MMNtOperand<_Float16> b{a.b + (long)e * a.side * a.lda, a.lda, a.pa, a.side};
  const bool wide = a.rows <= a.cols;
  _Float16 *u = wide ? a.u : a.next, *vt = wide ? a.next : a.v;
  const int m0 = tm * Nt::BM, n0 = tn * Nt::BN;
  Nt t;
  if (wide) {
    const MMNtOperand<_Float16> x{a.v + (long)e * a.cols * a.ldv, a.ldv, a.pv, a.cols};
    t.run(b, m0, x, n0, 0, (int)(a.lda / MM_NT_K), mm_ortho_lds);
  } else {
    const MMNtOperand<_Float16> x{a.u + (long)e * a.rows * a.ldu, a.ldu, a.pu, a.rows};
    t.run(x, m0, b, n0, 0, (int)(a.lda / MM_NT_K), mm_ortho_lds);
  }
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j) {
    const int m = m0 + t.row(j);
    const long row = ((long)e * a.rows + m) * a.cols;
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i) {
      const int n = n0 + t.col(i);
      floatx4 v = {};   // zeros past the last row and column
      if (m < a.rows && n < a.cols) {
        mm_load4(a.x + row, n, a.cols, (float*)&v);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          v[q] = n + q < a.cols ? fmaf(t.acc[i][j][q], 1.f / (MM_ORTHO_B * MM_ORTHO_X), a.ca * v[q]) : 0.f;
        if (last) mm_store4((T*)a.out + row, n, a.cols, (const float*)&v);
        else mm_store4(a.x + row, n, a.cols, (const float*)&v);
      }
      t.acc[i][j] = v;
    }
  }
  if (last) return;
  mm_ortho_tiles<PLANES>(t, mm_ortho_lds, u + ((long)e * a.rows + m0) * a.ldu + n0, a.ldu, a.pu, a.rows - m0,
                         (int)a.ldu - n0, MM_ORTHO_X);
  mm_ortho_tiles_transposed<PLANES>(t, mm_ortho_lds, vt + ((long)e * a.cols + n0) * a.ldv + m0, a.ldv, a.pv,
                                    (int)a.ldv - m0, a.cols - n0, MM_ORTHO_X);
}

// ------------------------------------------------------------------------------------------------ small matrices
// All steps of a small matrix in one workgroup and one launch: a wave holds RT times 16 rows of X (its shorter side) in
// fp32 registers, and LDS the planes of X, then those of W.  A step:
//     A = X X^T: a wave's rows of A, which as they come out of the matrix cores are operands of the next two products
//     W = b X + c (A X), which takes X's place in LDS;  X <- a X + A W, which takes it back
// so that neither A nor B is stored (B X = A (b X + c A X)).  The order of an operand along the summed index is free as
// long as both operands agree: 32 values are taken as k = 16 (e / 4) + 4 g + e % 4, the order in which a lane has its
// results.  W has the scale of X (of a singular value s it makes b s + c s^3: where X stays below 2, W stays below 16
// with the usual coefficients).  Bound by LDS (an operand read from it meets 16 rows only) and barriers: float, 128 x
// 128 45 us for five steps, 89 of 201 x 137 123 - 138.
struct MMOrthoSmall {
  const void* m;
  void* out;
  int rows, cols, side, other, steps;   // side <= other: of X
  float eps, c[3 * 16];                 // a, b, c of at most 16 steps
};

template <typename T, int WAVES, int RT, int NT, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) mm_ortho_small_kernel(MMOrthoSmall a) {
  // units of 16 bytes of a row: an odd number, so that any 8 consecutive rows lie in different banks
  constexpr int PLANES = MMOrthoType<T>::PLANES, P = MMOrthoType<T>::P, MT = WAVES * RT, MS = MT / 2;
  constexpr int KS = (NT + 1) / 2, UNITS = 4 * KS + 1;   // stages of 32 columns
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef short s4 __attribute__((ext_vector_type(4)));
  extern __shared__ uint4 mm_ortho_lds[];
  __shared__ double s_norm[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, g = lane >> 4;
  // All tiles take part (rows past the last one are zeros), so that no branch stands between the reads and the products
  // (128 x 128 float: 9.4 -> 7.9 us a step) - but for ten waves and two planes, whose 168 registers a branch relieves
  // (89 of 201 x 137: 305 -> 137 us).
  constexpr bool GUARD = NT == 13 && PLANES == 2;
  const int mt = GUARD ? (a.side + 15) / 16 : MT, ms = GUARD ? (a.side + 31) / 32 : MS;
  constexpr int plane = MS * 32 * UNITS;   // units of a plane
  const bool work = !GUARD || wave * RT < mt;
  const bool wide = a.rows <= a.cols;
  auto row = [&](int t) { return 16 * (wave * RT + t) + i16; };
  const size_t size = (size_t)a.rows * a.cols, base = blockIdx.x * size;
  floatx4 x[RT][NT], acc[RT][NT > MT ? NT : MT];
  double norm = 0.;
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int n = 16 * i + 4 * g, r = row(t);
      floatx4 v = {};
      if (r < a.side && wide) {
        mm_load4((const T*)a.m + base + (size_t)r * a.cols, n, a.cols, (float*)&v);
      } else if (r < a.side) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < a.other) v[q] = (float)((const T*)a.m)[base + (size_t)(n + q) * a.cols + r];
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) norm = fma((double)v[q], (double)v[q], norm);
      x[t][i] = v;
    }
#pragma unroll
  for (int d = 32; d; d >>= 1) norm += __shfl_xor(norm, d);
  if (lane == 0) s_norm[wave] = norm;
  __syncthreads();
  norm = 0.;
  for (int w = 0; w < WAVES; ++w) norm += s_norm[w];
  const double by = 1. / (sqrt(norm) + (double)a.eps);
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v = x[t][i][q];
        x[t][i][q] = v == 0.f ? v : (float)((double)v * by);   // no norm: zeros
      }

  _Float16* const tile = (_Float16*)mm_ortho_lds;
  auto put = [&](floatx4 r, int t, int i) {   // 4 values of tile i of this lane's row of t
    r *= MM_ORTHO_X;
    _Float16* const at = tile + 8 * (row(t) * UNITS + 2 * i) + 4 * g;
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      halfx4 h;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        h[q] = (_Float16)r[q];
        r[q] -= (float)h[q];
      }
      *(halfx4*)(at + 8 * p * plane) = h;
    }
  };
  // operand of 16 rows r0 .., values 32 s + 8 g ..
  const _Float16* const at_row = tile + 8 * (i16 * UNITS + g);
  auto read_rows = [&](half8 (&v)[PLANES], int r0, int s) {
#pragma unroll
    for (int p = 0; p < PLANES; ++p) v[p] = *(const half8*)(at_row + 8 * (p * plane + r0 * UNITS + 4 * s));
  };
  // operand of 16 columns 16 i .., rows 32 s + 16 (e / 4) + 4 g + e % 4: transposing reads
  const _Float16* const at_col = tile + 8 * ((4 * g + (i16 >> 2)) * UNITS + (i16 >> 1 & 1)) + 4 * (i16 & 1);
  auto read_cols = [&](half8 (&v)[PLANES], int i, int s) {
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      s4 h[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
        h[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s4*)(at_col + 8 * (p * plane + (32 * s + 16 * b) * UNITS + 2 * i)));
      v[p] = __builtin_bit_cast(half8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  // c[t][i] += the products of operand u with the rows' operands v[t], by passes, so that no product waits for another
  auto mma = [&](auto& c, int i, const half8 (&u)[PLANES], const half8 (&v)[RT][PLANES]) {
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int t = 0; t < RT; ++t)
        c[t][i] =
            __builtin_amdgcn_mfma_f32_16x16x32_f16(u[mm_nt_first<P>(q)], v[t][mm_nt_second<P>(q)], c[t][i], 0, 0, 0);
  };

  auto put_all = [&](const auto& v) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < NT; ++i) put(v[t][i], t, i);
  };

  if constexpr (NT % 2 == 1) {   // the rest of the last stage, never written again
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
        if (g < 2) mm_ortho_lds[p * plane + row(t) * UNITS + 2 * NT + g] = uint4{0, 0, 0, 0};
  }
  put_all(x);
  __syncthreads();
  for (int step = 0; step < a.steps; ++step) {
    const float ca = a.c[3 * step], cb = a.c[3 * step + 1], cc = a.c[3 * step + 2];
    half8 fa[RT][MS][PLANES];
    if (work) {   // A: this wave's rows
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[t][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int s = 0; s < KS; ++s) {
        half8 v[RT][PLANES], u[AHEAD + 1][PLANES];
#pragma unroll
        for (int t = 0; t < RT; ++t) read_rows(v[t], 16 * (wave * RT + t), s);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) read_rows(u[i], 16 * i, s);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (i + AHEAD < MT && (!GUARD || i + AHEAD < mt))
            read_rows(u[(i + AHEAD) % (AHEAD + 1)], 16 * (i + AHEAD), s);
          __builtin_amdgcn_sched_barrier(0);
          if (!GUARD || i < mt) mma(acc, i, u[i % (AHEAD + 1)], v);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int s = 0; s < MS; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v = acc[t][2 * s + e / 4][e % 4] * (MM_ORTHO_A / (MM_ORTHO_X * MM_ORTHO_X));
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              const _Float16 h = (_Float16)v;
              fa[t][s][p][e] = h;
              v -= (float)h;
            }
          }
    }
    auto product = [&]() {   // acc = this wave's rows of A times what is in LDS, in units of both scales
      half8 u[AHEAD + 1][PLANES];
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) read_cols(u[s], 0, s);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < MS; ++s) {
          constexpr int SEQ = AHEAD + 1;
          const int q = i * MS + s;   // of the sequence of operands, read AHEAD before their products
          if (s + AHEAD < MS) {
            if (!GUARD || s + AHEAD < ms) read_cols(u[(q + AHEAD) % SEQ], i, s + AHEAD);
          } else if (i + 1 < NT) {
            read_cols(u[(q + AHEAD) % SEQ], i + 1, s + AHEAD - MS);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (!GUARD || s < ms) {
            half8 v[RT][PLANES];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
              for (int p = 0; p < PLANES; ++p) v[t][p] = fa[t][s][p];
            mma(acc, i, u[q % SEQ], v);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    constexpr float UNIT = 1.f / (MM_ORTHO_A * MM_ORTHO_X);
    if (work) {
      product();
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          acc[t][i] = cb * x[t][i] + cc * UNIT * acc[t][i];
          x[t][i] *= ca;
        }
    }
    __syncthreads();   // everyone is done with X
    if (work) put_all(acc);
    __syncthreads();
    if (work) {
      product();
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < NT; ++i) x[t][i] += UNIT * acc[t][i];
    }
    if (step + 1 == a.steps) break;
    __syncthreads();
    if (work) put_all(x);
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = row(t);
    if (r >= a.side) break;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int n = 16 * i + 4 * g;
      if (wide) {
        mm_store4((T*)a.out + base + (size_t)r * a.cols, n, a.cols, (const float*)&x[t][i]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < a.other) ((T*)a.out)[base + (size_t)(n + q) * a.cols + r] = (T)x[t][i][q];
      }
    }
  }
}

namespace {
constexpr long MAX_SIDE = 65536;

long div_up(long a, long b) { return (a + b - 1) / b; }

struct Space {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t n) {
    T* p = base ? (T*)(base + used) : nullptr;
    used += (n * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

size_t space(MMOrtho* a, int dtype, char* base) {
  Space p{base};
  const int planes = dtype == MM_BF16 ? 1 : 2;
  a->side = a->rows < a->cols ? a->rows : a->cols;
  a->ldu = mm_up(a->cols, MM_NT_K);
  a->ldv = mm_up(a->rows, MM_NT_K);
  a->lda = mm_up(a->side, MM_NT_K);
  a->pu = (long)a->batch * a->rows * a->ldu;
  a->pv = (long)a->batch * a->cols * a->ldv;
  a->pa = (long)a->batch * a->side * a->lda;
  const long parts = div_up((long)a->rows * a->cols, 256 * 32);   // the same whatever the batch: so are its sums' bits
  a->parts = (int)(parts < MM_ORTHO_PARTS ? parts : MM_ORTHO_PARTS);
  a->part = p.take<double>((size_t)a->batch * a->parts);
  a->x = p.take<float>((size_t)a->batch * a->rows * a->cols);
  a->u = p.take<_Float16>(planes * a->pu);
  a->v = p.take<_Float16>(planes * a->pv);
  a->a = p.take<_Float16>(planes * a->pa);
  a->b = p.take<_Float16>(planes * a->pa);
  a->next = p.take<_Float16>(planes * (a->rows <= a->cols ? a->pv : a->pu));
  // A long side is summed in parts of 512 values or more where A has few tiles.  The rule looks at the matrix alone,
  // so that its result does not depend on how many stand beside it.  (Five steps, us in 1 | 4 | 8 parts: 192 x 4096
  // float 348 | 189 | 196, bfloat16 237 | 140 | 157, 64 of the float ones 2369 | 1974 | 2104; 192 x 16,384 float 1074
  // | 411 | 339; 192 x 768 in one part 148, in two 138; 256 x 4096, not split, 359 | 209 | 211.)
  const long other = a->rows < a->cols ? a->cols : a->rows;
  a->splits = a->side <= 192 && other >= 1024 ? (int)(other / 512 < 8 ? other / 512 : 8) : 1;
  a->sums = a->splits > 1 ? p.take<float>(a->splits * a->pa) : nullptr;
  return p.used;
}

template <auto KERNEL, typename Nt, typename... A>
bool launch(const MMOrtho& a, long workgroups, hipStream_t stream, A... rest) {
  if (!lds_granted<KERNEL>(Nt::LDS)) return false;
  hipLaunchKernelGGL(KERNEL, dim3((unsigned)workgroups), dim3(Nt::TH), Nt::LDS, stream, a, rest...);
  return true;
}

template <int P, int WHAT, typename Nt>
bool square(const MMOrtho& a, hipStream_t stream) {
  const int t = (int)div_up(a.side, Nt::BM);
  const long batch = WHAT ? a.batch : (long)a.batch * a.splits;
  if (!launch<mm_ortho_square_kernel<P, WHAT, Nt>, Nt>(a, batch * t * (t + 1) / 2, stream, t)) return false;
  if (WHAT == 0 && a.splits > 1)
    hipLaunchKernelGGL((mm_ortho_join_kernel<P == 1 ? 1 : 2>), dim3((unsigned)div_up(a.side * a.lda / 4, 256), a.batch),
                       dim3(256), 0, stream, a);
  return true;
}

template <typename T, typename Nt>
bool step(const MMOrtho& a, int last, hipStream_t stream) {
  const int tm = (int)div_up(a.rows, Nt::BM), tn = (int)div_up(a.cols, Nt::BN);
  return launch<mm_ortho_step_kernel<T, Nt>, Nt>(a, (long)a.batch * tm * tn, stream, tm, tn, last);
}

template <typename T, int WAVES, int RT, int NT, int AHEAD>
bool small(const MMOrthoSmall& a, int batch, int lds, hipStream_t stream) {
  if (!lds_granted<mm_ortho_small_kernel<T, WAVES, RT, NT, AHEAD>>(lds)) return false;
  hipLaunchKernelGGL((mm_ortho_small_kernel<T, WAVES, RT, NT, AHEAD>), dim3(batch), dim3(64 * WAVES), lds, stream, a);
  return true;
}

// rows, tiles of columns and LDS of the workgroup that holds a matrix (rows 0: none does).  Five float steps, us held
// | by tiles: one of 128 x 128 44 | 98, of 128 x 256 106 | 107, of 160 x 208 122 | 117; 89 of 201 x 137 122 | 301, of
// 160 x 208 127 | 312; 300 of 128 x 256 255 | 457.  bfloat16: one of 160 x 208 56 | 90, 300 of them 120 | 364.  Larger
// shapes were not built, as a single float one gains nothing already (by tiles 89 of 176 x 176 258, of 160 x 256 311).
struct Held { int rows, nt, lds; };
Held held(long rows, long cols, int dtype, int steps) {
  const long side = rows < cols ? rows : cols, other = rows < cols ? cols : rows;
  Held h{0, 0, 0};
  if (steps > 16) return h;
  if (side <= 64 && other <= 64) h = Held{64, 4, 0};
  else if (side <= 64 && other <= 256) h = Held{64, 16, 0};
  else if (side <= 128 && other <= 128) h = Held{128, 8, 0};
  else if (side <= 128 && other <= 256) h = Held{128, 16, 0};
  else if (side <= 160 && other <= 208) h = Held{160, 13, 0};
  h.lds = h.rows * ((h.nt + 1) / 2 * 4 + 1) * 16 * (dtype == MM_BF16 ? 1 : 2);
  return h;
}

template <typename T>
int orthogonalize_small(const MMOrtho& o, int steps, const float* c, const Held& h, hipStream_t stream) {
  MMOrthoSmall a{o.m, o.out, o.rows, o.cols, o.side, o.rows < o.cols ? o.cols : o.rows, steps, o.eps, {}};
  for (int i = 0; i < 3 * steps; ++i) a.c[i] = c[i];
  bool ok;
  if (h.nt == 4) ok = small<T, 4, 1, 4, 2>(a, o.batch, h.lds, stream);
  else if (h.rows == 64) ok = small<T, 4, 1, 16, 2>(a, o.batch, h.lds, stream);
  else if (h.nt == 8) ok = small<T, 8, 1, 8, 2>(a, o.batch, h.lds, stream);
  else if (h.nt == 16) ok = small<T, 8, 1, 16, 2>(a, o.batch, h.lds, stream);
  else ok = small<T, 10, 1, 13, 1>(a, o.batch, h.lds, stream);
  return ok ? mm::launch_status("mm_orthogonalize") : MM_ELAUNCH;
}

template <typename T>
int orthogonalize(MMOrtho a, int steps, const float* c, hipStream_t stream) {
  constexpr int P = MMOrthoType<T>::P;
  typedef MMNtBig<_Float16, P> Big;
  typedef MMNt<_Float16, P, 128, 128, 2, 2> Mid;
  typedef MMNt<_Float16, P, 64, 64, 2, 2> Low;
  hipLaunchKernelGGL(mm_ortho_norm_kernel<T>, dim3(a.parts, a.batch), dim3(256), 0, stream, (const T*)a.m,
                     (long)a.rows * a.cols, a.part);
  hipLaunchKernelGGL(mm_ortho_start_kernel<T>, dim3((unsigned)div_up(a.rows, 64), (unsigned)div_up(a.cols, 64), a.batch),
                     dim3(256), 0, stream, a, steps);
  auto lower = [&](long n) { return a.batch * div_up(a.side, n) * (div_up(a.side, n) + 1) / 2; };
  auto all = [&](long n) { return a.batch * div_up(a.rows, n) * div_up(a.cols, n); };
  const int sq = mm_tile_side(P, lower(256) * a.splits, lower(128) * a.splits, lower(64) * a.splits);
  const int st = mm_tile_side(P, all(256), all(128), all(64));
  bool ok = true;
  for (int i = 0; i < steps && ok; ++i, c += 3) {
    a.ca = c[0];
    a.cb = c[1];
    a.cc = c[2];
    if (sq == 256) ok = square<P, 0, Big>(a, stream) && square<P, 1, Big>(a, stream);
    else if (sq == 128) ok = square<P, 0, Mid>(a, stream) && square<P, 1, Mid>(a, stream);
    else ok = square<P, 0, Low>(a, stream) && square<P, 1, Low>(a, stream);
    const int last = i + 1 == steps;
    if (st == 256) ok = ok && step<T, Big>(a, last, stream);
    else if (st == 128) ok = ok && step<T, Mid>(a, last, stream);
    else ok = ok && step<T, Low>(a, last, stream);
    std::swap(a.next, a.rows <= a.cols ? a.v : a.u);
  }
  return ok ? mm::launch_status("mm_orthogonalize") : MM_ELAUNCH;
}

int check(const char* name, long batch, long rows, long cols, int dtype) {
  if (dtype < MM_F32 || dtype > MM_F16 || batch < 0 || rows <= 0 || cols <= 0) {
    mm::set_error(std::string(name) + ": bad sizes or dtype");
    return MM_EINVAL;
  }
  if (rows > MAX_SIDE || cols > MAX_SIDE || batch > 65535 ||
      batch * div_up(rows, 64) * div_up(cols, 64) * 256 >= 4294967296L) {
    mm::set_error(std::string(name) + ": sizes beyond the launches' limits");
    return MM_ERANGE;
  }
  return MM_OK;
}

// Matrices taken at once.  Up to 240 MB of workspace, so that their planes stay in the last cache (256 MB) between the
// products, and a number whose tiles fill their rounds (64 bfloat16 matrices of 1024 x 1024: 64 at once 2900 us, 16 2910,
// 14 2540).
int part_of(MMOrtho a, long batch, int dtype) {
  a.batch = 1;
  const long fits = 251658240L / (long)space(&a, dtype, nullptr), most = fits < 1 ? 1 : fits < batch ? fits : batch;
  const int P = dtype == MM_BF16 ? 1 : 3;
  auto lower = [&](long p, long n) { return p * div_up(a.side, n) * (div_up(a.side, n) + 1) / 2; };
  auto all = [&](long p, long n) { return p * div_up(a.rows, n) * div_up(a.cols, n); };
  long best = most;
  double least = 1e300;
  for (long p = most; p >= 1 && 2 * p >= most; --p) {
    double time = 2. * mm_tile_time(P, lower(p, 256), lower(p, 128), lower(p, 64))
                + mm_tile_time(P, all(p, 256), all(p, 128), all(p, 64));
    time *= (double)div_up(batch, p);
    if (time < least) {
      least = time;
      best = p;
    }
  }
  return (int)best;
}
}  // namespace

extern "C" int mm_orthogonalize_workspace(long batch, long rows, long cols, int dtype, size_t* bytes) {
  const int rc = check("mm_orthogonalize_workspace", batch, rows, cols, dtype);
  if (rc != MM_OK) return rc;
  MM_CHECK_ARG(bytes, "no result");
  MMOrtho a{};
  a.rows = (int)rows;
  a.cols = (int)cols;
  a.batch = batch ? part_of(a, batch, dtype) : 0;
  *bytes = batch ? space(&a, dtype, nullptr) : 0;
  return MM_OK;
}

extern "C" int mm_orthogonalize_workspace_steps(long batch, long rows, long cols, int dtype, int steps, size_t* bytes) {
  const int rc = check("mm_orthogonalize_workspace_steps", batch, rows, cols, dtype);
  if (rc != MM_OK) return rc;
  MM_CHECK_ARG(steps >= 0 && bytes, "bad steps or no result");
  if (batch == 0 || !held(rows, cols, dtype, steps).rows)
    return mm_orthogonalize_workspace(batch, rows, cols, dtype, bytes);
  *bytes = 256;   // not touched
  return MM_OK;
}

extern "C" int mm_orthogonalize(const void* m, int dtype, long batch, long rows, long cols, int steps,
                                const float* coefficients, float eps, void* out, void* workspace, hipStream_t stream) {
  const int rc = check("mm_orthogonalize", batch, rows, cols, dtype);
  if (rc != MM_OK) return rc;
  MM_CHECK_ARG(steps >= 0 && (steps == 0 || coefficients) && eps >= 0.f, "bad steps, coefficients or eps");
  if (batch == 0) return MM_OK;
  MM_CHECK_ARG(m && out && workspace, "null pointer");
  MMOrtho a{};
  a.eps = eps;
  a.rows = (int)rows;
  a.cols = (int)cols;
  a.side = (int)(rows < cols ? rows : cols);
  const Held h = held(rows, cols, dtype, steps);
  const long part = h.rows ? batch : part_of(a, batch, dtype), size = rows * cols * (dtype == MM_F32 ? 4 : 2);
  for (long i = 0; i < batch; i += part) {
    a.m = (const char*)m + i * size;
    a.out = (char*)out + i * size;
    a.batch = (int)(batch - i < part ? batch - i : part);
    int done = MM_OK;
    if (h.rows) {
      MM_DISPATCH(dtype, done = orthogonalize_small<T_>(a, steps, coefficients, h, stream));
    } else {
      space(&a, dtype, (char*)workspace);
      MM_DISPATCH(dtype, done = orthogonalize<T_>(a, steps, coefficients, stream));
    }
    if (done != MM_OK) return done;
  }
  return MM_OK;
}
