// Tiles of C = A B^T with both operands rows of 16-bit values along the summed index:
//     C[m, n] = sum over the passes (i, j) and k of A_i[m, k] B_j[n, k]
// P = 1: one plane each.  P = 3: two planes (float16 high and low parts, 22 bits), the three products without low x
// low.  P = 6: three bfloat16 planes of float, the six products with i + j <= 2.  Rows are 16-byte aligned, their length
// a multiple of 64 values, zeros past the summed index.  Rows past the last one of an operand are read as the last one
// and give results that nobody stores.
#pragma once
#include "tile.h"

#define MM_NT_K 64   // values of the summed index of a stage

template <typename H>
struct MMNtOperand {
  const H* p;
  long ld, plane;   // distances of rows and planes
  int rows;
};

// planes of pass q
template <int P>
__device__ __forceinline__ int mm_nt_first(int q) {
  return P == 1 ? 0 : P == 3 ? (q == 0 ? 1 : 0) : (q == 0 ? 2 : q == 1 || q == 3 ? 1 : 0);
}
template <int P>
__device__ __forceinline__ int mm_nt_second(int q) {
  return P == 1 ? 0 : P == 3 ? (q == 1 ? 1 : 0) : (q == 2 ? 2 : q == 1 || q == 4 ? 1 : 0);
}

// A workgroup's tile of BM rows of A by BN rows of B, WM x WN waves; lane's results acc[i][j][q]: row m = wm + 16 j +
// (lane & 15) of the tile, column n = wn + 16 i + 4 (lane >> 4) + q.
template <typename H, int P, int BM, int BN, int WM, int WN>
struct MMNt {
  static constexpr int TH = 64 * WM * WN, UA = BM * 8 / TH, UB = BN * 8 / TH;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int LDS = 2 * (BM + BN) * 8 * 16;   // bytes
  floatx4 acc[FN][FM];
  int wm, wn, lane;

  __device__ __forceinline__ MMNt() {
    const int wave = threadIdx.x >> 6;
    lane = threadIdx.x & 63;
    wm = (wave % WM) * (BM / WM);
    wn = (wave / WM) * (BN / WN);
  }
  __device__ __forceinline__ int row(int j) const { return wm + 16 * j + (lane & 15); }
  __device__ __forceinline__ int col(int i) const { return wn + 16 * i + 4 * (lane >> 4); }

  // stages k0 .. k1 - 1 (of 64 values) of every pass; the LDS is free afterwards
  __device__ __forceinline__ void run(const MMNtOperand<H>& a, int m0, const MMNtOperand<H>& b, int n0, int k0, int k1,
                                      uint4* lds) {
    uint4 *As = lds, *Bs = lds + 2 * BM * 8;
    const int tid = threadIdx.x, ka = ((tid & 7) ^ (tid >> 3 & 7)) * 8;
    const H *pa[UA], *pb[UB];
#pragma unroll
    for (int j = 0; j < UA; ++j) pa[j] = a.p + (long)min(m0 + ((tid + TH * j) >> 3), a.rows - 1) * a.ld + ka;
#pragma unroll
    for (int j = 0; j < UB; ++j) pb[j] = b.p + (long)min(n0 + ((tid + TH * j) >> 3), b.rows - 1) * b.ld + ka;
    MMStage<H, TH, UA, true> sa;
    MMStage<H, TH, UB, true> sb;
    auto load = [&](int k, int q, int buf) {
      const long oa = mm_nt_first<P>(q) * a.plane + (long)k * MM_NT_K;
      const long ob = mm_nt_second<P>(q) * b.plane + (long)k * MM_NT_K;
#pragma unroll
      for (int j = 0; j < UA; ++j) sa.load(As + buf * BM * 8, j, pa[j] + oa, 8);
#pragma unroll
      for (int j = 0; j < UB; ++j) sb.load(Bs + buf * BN * 8, j, pb[j] + ob, 8);
    };
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (k0 >= k1) return;
    load(k0, 0, 0);
    mm_stage_done();
    int buf = 0, k = k0, q = 0;
    while (k < k1) {
      if (++q == P) {
        q = 0;
        ++k;
      }
      if (k < k1) load(k, q, buf ^ 1);
      const uint4 *A = As + buf * BM * 8, *B = Bs + buf * BN * 8;
      mm_products<H, FN, FM, 2>(
          acc, [&](int s, int i) { return mm_read_kc<H>(B, wn + 16 * i, s, lane); },
          [&](int s, int j) { return mm_read_kc<H>(A, wm + 16 * j, s, lane); });
      mm_stage_done();
      buf ^= 1;
    }
  }
};

// Tile of workgroup b among `batch` times tiles_m x tiles_n: consecutive numbers on one XCD (workgroups are dealt out to
// the 8 XCDs in turn), in bands of 8 tiles of rows, so that neighbours share operands in that XCD's L2.  False: none.
__device__ __forceinline__ bool mm_nt_tile(int b, int batch, int tiles_m, int tiles_n, int* e, int* tm, int* tn) {
  const int one = tiles_m * tiles_n, all = batch * one;
  if (b >= all) return false;
  const int share = all / 8, rest = all % 8, x = b % 8;
  int at = x * share + min(x, rest) + b / 8;
  *e = at / one;
  at -= *e * one;
  const int band = at / (8 * tiles_n), high = min(8, tiles_m - 8 * band), r = at - band * 8 * tiles_n;
  *tm = 8 * band + r % high;
  *tn = r / high;
  return true;
}

__host__ __device__ inline long mm_up(long n, long size) { return (n + size - 1) / size * size; }
