// Products of rows with the weight blocks of their experts:
//   mm_expert_rows     out[s, m] = in[s / k, m] @ W[e]  (or @ W[e]^T): fp32 rows in slot order
//   mm_expert_combine  y[t, m] = sum_j gate rows[t k + j, m];  mm_expert_combine_bwd  dx and dgates from the rows of dy
//   mm_expert_joined   one or two choices of a row joined before they are written
//   mm_expert_few      few rows straight through their blocks
#include "experts.h"

// ------------------------------------------------------------------------------------------------ rows
// A workgroup: a tile of BM rows of one expert by BN columns, its WM x WN waves with BM / WM x BN / WN each, two
// stages in LDS: the next stage is on its way while this one is multiplied.  The weights are the first operand, so
// that a lane ends with 4 consecutive columns of a row.  TRANS: W[e] is [N][K], else [K][N].  Bound by the products
// and, for large tiles, by the fp32 rows they write at the same time: 65,536 bfloat16 rows 1024 -> 1024, 64 experts: 256
// us (537 TFLOP/s; 213 us TRANS, whose weights need no transposing reads), of which 268 MB of rows take about 76.
template <typename T, bool TRANS, bool DMA, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) mm_expert_rows_kernel(MMRows a, int tiles_n) {
  constexpr int TH = 64 * WM * WN, BK = MM_TILE_K<T>, N = MMVec<T>::N, UPR = BN / N, KS = BK / 32;
  constexpr int UA = BM * 8 / TH, UB = BN * 8 / TH, FM = BM / WM / 16, FN = BN / WN / 16;
  extern __shared__ uint4 mm_lds[];
  uint4 *As = mm_lds, *Bs = As + 2 * BM * 8;             // [2][BM * 8], [2][BN * 8]
  long* s_out = (long*)(Bs + 2 * BN * 8);                // [BM]
  int part, number;
  const MMTile t = mm_expert_tile(a.offsets, a.E, a.offsets[a.E], a.M, BM, tiles_n, blockIdx.x, &part, &number);
  if (t.e < 0) return;
  const int n0 = part * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* __restrict__ W = (const T*)a.W + (size_t)t.e * a.K * a.N;
  const int* __restrict__ list = a.order + a.offsets[t.e];
  if (tid < BM) {
    const int r = t.row0 + min(tid, t.rows - 1), p = r / a.M, m = r - p * a.M;
    s_out[tid] = ((long)list[p] * a.M + m) * a.N;
  }
  // sources of this thread's units: row pu / 8 of the tile, unit (pu & 7) ^ (row & 7)
  const T *pa[UA], *pb[UB];
  int kb[UB], nb[UB];   // B: TRANS: columns n0 + row, k as A's; else k row and values left in that row
  const int ka = ((tid & 7) ^ (tid >> 3 & 7)) * N;
#pragma unroll
  for (int j = 0; j < UA; ++j) {
    const int row = (tid + TH * j) >> 3;
    const int r = t.row0 + min(row, t.rows - 1), p = r / a.M, m = r - p * a.M;
    pa[j] = (const T*)a.in + (long)(list[p] / a.k) * a.st + m * a.sm + ka;
  }
#pragma unroll
  for (int j = 0; j < UB; ++j) {
    const int pu = tid + TH * j;
    if constexpr (TRANS) {
      const int n = n0 + (pu >> 3);
      nb[j] = n < a.N;
      kb[j] = ka;
      pb[j] = W + (size_t)min(n, a.N - 1) * a.K + ka;
    } else {
      const int q = pu / UPR, u = (pu % UPR) ^ mm_nc_swizzle<T, UPR>(q);
      kb[j] = q;
      nb[j] = a.N - n0 - u * N;
      pb[j] = W + (size_t)q * a.N + n0 + u * N;
    }
  }
  MMStage<T, TH, UA, DMA> sa;
  MMStage<T, TH, UB, DMA> sb;
  auto load = [&](int k0, int buf) {
#pragma unroll
    for (int j = 0; j < UA; ++j) sa.load(As + buf * BM * 8, j, pa[j] + k0, a.K - k0 - ka);
#pragma unroll
    for (int j = 0; j < UB; ++j) {
      if constexpr (TRANS) sb.load(Bs + buf * BN * 8, j, pb[j] + k0, nb[j] ? a.K - k0 - kb[j] : 0);
      else sb.load(Bs + buf * BN * 8, j, pb[j] + (size_t)k0 * a.N, k0 + kb[j] < a.K ? nb[j] : 0);
    }
  };
  auto put = [&](int buf) {
    sa.put(As + buf * BM * 8);
    sb.put(Bs + buf * BN * 8);
  };
  floatx4 acc[FN][FM] = {};
  const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
  load(0, 0);
  put(0);
  mm_stage_done();
  int buf = 0;
  for (int k0 = 0; k0 < a.K; k0 += BK) {
    const bool more = k0 + BK < a.K;
    if (more) load(k0 + BK, buf ^ 1);
    const uint4 *A = As + buf * BM * 8, *B = Bs + buf * BN * 8;
    mm_products<T, FN, FM, KS>(
        acc,
        [&](int s, int i) {
          if constexpr (TRANS) return mm_read_kc<T>(B, wn + 16 * i, s, lane);
          else return mm_read_nc<T, UPR>(B, wn + 16 * i, s, lane);
        },
        [&](int s, int j) { return mm_read_kc<T>(A, wm + 16 * j, s, lane); });
    if (more) put(buf ^ 1);
    mm_stage_done();
    buf ^= 1;
  }
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int m = wm + 16 * j + (lane & 15);
    if (m >= t.rows) continue;
    float* __restrict__ o = a.out + s_out[m];
#pragma unroll
    for (int i = 0; i < FN; ++i) mm_store_vec(o, n0 + wn + 16 * i + 4 * (lane >> 4), a.N, (const float*)&acc[i][j]);
  }
}

// ------------------------------------------------------------------------------------------------ joined rows
// All k <= 2 choices of a row in one workgroup: rows sorted by the set of their experts (the plan of the slots for k =
// 1, of the pairs for k = 2) share both blocks, so that the products of a row are joined in registers and written
// once, in its type, where the path through slots writes k fp32 rows and reads them again.  Rows without an expert are
// written as zeros.  DG (k = 1): with the rows of dy and W[e]^T, also dgates[t] = sum over m of <x[t, m], (dy W^T)[t,
// m]>; a tile holds whole rows t (all M components) and all columns.
struct MMJoined {
  const void *in, *W, *x;
  const float* gates;
  const int *experts, *offsets, *order;   // offsets [buckets]: where each set's rows begin
  void* out;
  float* dgates;
  long st, sm, xt, xm;
  int T, M, K, N, E, buckets;
};

template <typename T, bool TRANS, bool DMA, int J, bool DG, int BM>
__global__ void __launch_bounds__(256, 2) mm_expert_joined_kernel(MMJoined a, int tiles_n) {
  constexpr int BN = 128, WM = 2, WN = 2, TH = 256, BK = MM_TILE_K<T>, N = MMVec<T>::N, UPR = BN / N;
  constexpr int KS = BK / 32, UA = BM * 8 / TH, UB = BN * 8 / TH, FM = BM / WM / 16, FN = BN / WN / 16;
  __shared__ uint4 As[2 * BM * 8], Bs[2 * BN * 8];
  __shared__ long s_out[BM], s_x[DG ? BM : 1];
  __shared__ float s_g[J][BM], s_dg[DG ? WN : 1][BM];
  int part, number;
  const int rows_of_tile = BM / a.M * a.M;
  const MMTile t = mm_expert_tile(a.offsets, a.buckets, a.T, a.M, rows_of_tile, tiles_n, blockIdx.x, &part, &number);
  if (t.e < 0) return;
  const int n0 = part * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int e[J];   // this set's experts, a.E: none
  if constexpr (J == 1) {
    e[0] = t.e;
  } else {
    int lo = 0, rest = t.e;
    while (rest >= a.E + 1 - lo) rest -= a.E + 1 - lo++;
    e[0] = lo;
    e[1] = lo + rest;
  }
  const int* __restrict__ list = a.order + a.offsets[t.e];
  if (tid < BM) {
    const int r = t.row0 + min(tid, t.rows - 1), p = r / a.M, m = r - p * a.M, tok = list[p];
    s_out[tid] = ((long)tok * a.M + m) * a.N;
    if constexpr (DG) s_x[tid] = tok * a.xt + m * a.xm;
    if constexpr (J == 1) {
      s_g[0][tid] = a.gates ? a.gates[tok] : 1.f;
    } else {
      const int first = a.experts[2 * (long)tok], swap = ((unsigned)first < (unsigned)a.E ? first : a.E) != e[0];
      s_g[0][tid] = a.gates ? a.gates[2 * (long)tok + swap] : 1.f;
      s_g[1][tid] = a.gates ? a.gates[2 * (long)tok + (1 - swap)] : 1.f;
    }
  }
  const int ka = ((tid & 7) ^ (tid >> 3 & 7)) * N;
  const T *pa[UA];
  int kb[UB], nb[UB];
  long ob[UB];
#pragma unroll
  for (int j = 0; j < UA; ++j) {
    const int row = (tid + TH * j) >> 3;
    const int r = t.row0 + min(row, t.rows - 1), p = r / a.M, m = r - p * a.M;
    pa[j] = (const T*)a.in + (long)list[p] * a.st + m * a.sm + ka;
  }
#pragma unroll
  for (int j = 0; j < UB; ++j) {
    const int pu = tid + TH * j;
    if constexpr (TRANS) {
      const int n = n0 + (pu >> 3);
      nb[j] = n < a.N;
      kb[j] = ka;
      ob[j] = (long)min(n, a.N - 1) * a.K + ka;
    } else {
      const int q = pu / UPR, u = (pu % UPR) ^ mm_nc_swizzle<T, UPR>(q);
      kb[j] = q;
      nb[j] = a.N - n0 - u * N;
      ob[j] = (long)q * a.N + n0 + u * N;
    }
  }
  MMStage<T, TH, UA, DMA> sa;
  MMStage<T, TH, UB, DMA> sb;
  auto load = [&](int c, int k0, int buf) {
    const T* __restrict__ W = (const T*)a.W + (size_t)e[c] * a.K * a.N;
#pragma unroll
    for (int j = 0; j < UA; ++j) sa.load(As + buf * BM * 8, j, pa[j] + k0, a.K - k0 - ka);
#pragma unroll
    for (int j = 0; j < UB; ++j) {
      if constexpr (TRANS) sb.load(Bs + buf * BN * 8, j, W + ob[j] + k0, nb[j] ? a.K - k0 - kb[j] : 0);
      else sb.load(Bs + buf * BN * 8, j, W + ob[j] + (size_t)k0 * a.N, k0 + kb[j] < a.K ? nb[j] : 0);
    }
  };
  auto put = [&](int buf) {
    sa.put(As + buf * BM * 8);
    sb.put(Bs + buf * BN * 8);
  };
  // The gates: on each choice's products, in sums of their own, or on the rows' values as they become operands (two
  // choices of float, whose planes leave no registers for the sums: one more rounding of 2^-24, and gate x value must
  // stay below what rounds to infinity in bfloat16).
  constexpr bool SCALED = sizeof(T) == 4 && J == 2, SUM = !SCALED;
  floatx4 acc[FN][FM] = {}, sum[SUM ? FN : 1][SUM ? FM : 1] = {};
  const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
  int buf = 0;
  if (e[0] < a.E) {   // the choices without an expert are the last ones
    load(0, 0, 0);
    put(0);
  }
  mm_stage_done();
#pragma unroll 1
  for (int c = 0; c < J; ++c) {
    if (e[c] >= a.E) break;
    float gs[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) gs[j] = s_g[c][wm + 16 * j + (lane & 15)];
    for (int k0 = 0; k0 < a.K; k0 += BK) {
      const bool same = k0 + BK < a.K, more = same || (c + 1 < J && e[c + 1 < J ? c + 1 : c] < a.E);
      if (more) load(same ? c : c + 1, same ? k0 + BK : 0, buf ^ 1);
      const uint4 *A = As + buf * BM * 8, *B = Bs + buf * BN * 8;
      mm_products<T, FN, FM, KS, SCALED>(
          acc,
          [&](int s, int i) {
            if constexpr (TRANS) return mm_read_kc<T>(B, wn + 16 * i, s, lane);
            else return mm_read_nc<T, UPR>(B, wn + 16 * i, s, lane);
          },
          [&](int s, int j) { return mm_read_kc<T>(A, wm + 16 * j, s, lane); }, gs);
      if (more) put(buf ^ 1);
      mm_stage_done();
      buf ^= 1;
    }
    if constexpr (SUM) {
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int m = wm + 16 * j + (lane & 15);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          if constexpr (DG) {
            float xv[4];
            mm_load4((const T*)a.x + s_x[m], n0 + wn + 16 * i + 4 * (lane >> 4), a.N, xv);
#pragma unroll
            for (int q = 0; q < 4; ++q) dot = fmaf(xv[q], acc[i][j][q], dot);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) sum[i][j][q] = fmaf(gs[j], acc[i][j][q], sum[i][j][q]);
          acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
        if constexpr (DG) {
          dot += __shfl_xor(dot, 16);
          dot += __shfl_xor(dot, 32);
          if (lane < 16) s_dg[wave / WM][m] = dot;
        }
      }
    }
    if constexpr (DG) {
      __syncthreads();
      if (tid < t.rows / a.M) {
        float d = 0.f;
        for (int m = tid * a.M; m < (tid + 1) * a.M; ++m) d += s_dg[0][m] + s_dg[1][m];
        a.dgates[list[t.row0 / a.M + tid]] = d;
      }
      __syncthreads();
    }
  }
  if constexpr (DG)
    if (e[0] >= a.E && tid < t.rows / a.M) a.dgates[list[t.row0 / a.M + tid]] = 0.f;
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int m = wm + 16 * j + (lane & 15);
    if (m >= t.rows || !a.out) continue;
    T* __restrict__ o = (T*)a.out + s_out[m];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const floatx4& v = SUM ? sum[SUM ? i : 0][SUM ? j : 0] : acc[i][j];
      mm_store4(o, n0 + wn + 16 * i + 4 * (lane >> 4), a.N, (const float*)&v);
    }
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// y[t, m] straight from the choices of row t, without a plan: a workgroup takes LC vectors of columns, its other
// threads share the sum over d, W is read once per row, coalesced along the columns, fp32 sums.  float operands that
// round to infinity in bfloat16 give NaN, as they do in the split operands of many rows.  Bound by latency: the sum
// over d is split as far as the workgroup goes, and the columns over many workgroups, with no branch between the loads
// (a check for cut vectors among them took 16 us instead of 8 for 1 row 1024 -> 1024 bfloat16, 4 of 64; 1 row 128 ->
// 128 float, k = 2: 3.5 us; 64 rows 64 -> 64: 3.4 us).
struct MMFew {
  const void *x, *W;
  const float* gates;
  const int* experts;
  long st, sm;
  int k, M, D, F, E;
};

// the least float that rounds to infinity in bfloat16
#define MM_SPLIT_LIMIT 0x1.ffp127f

template <typename T, int LC>
__global__ void __launch_bounds__(256) mm_expert_few_kernel(MMFew a, T* __restrict__ y) {
  constexpr int N = MMVec<T>::N, G = 256 / LC;
  __shared__ float red[4][LC * N];
  const long t = blockIdx.y;
  const int m = blockIdx.z, lc = threadIdx.x % LC, gd = threadIdx.x / LC, f0 = (blockIdx.x * LC + lc) * N;
  // a vector cut by the last column starts earlier instead: some columns are written twice, with the same bits
  const int f = a.F >= N ? min(f0, a.F - N) : f0;
  const T* __restrict__ x = (const T*)a.x + t * a.st + m * a.sm;
  float acc[N] = {};
  for (int j = 0; j < a.k; ++j) {
    const int e = a.experts[t * a.k + j];
    if ((unsigned)e >= (unsigned)a.E) continue;
    const float g = a.gates ? a.gates[t * a.k + j] : 1.f;
    const T* __restrict__ W = (const T*)a.W + (size_t)e * a.D * a.F;
    float sum[N] = {}, top[N] = {}, top_x = 0.f;   // largest magnitudes (float; a NaN is in the sum anyway)
    auto add = [&](int d, const float (&w)[N]) {
      const float xv = (float)x[d];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sum[i] = fmaf(xv, w[i], sum[i]);
        if constexpr (sizeof(T) == 4) top[i] = fmaxf(top[i], fabsf(w[i]));
      }
      if constexpr (sizeof(T) == 4) top_x = fmaxf(top_x, fabsf(xv));
    };
    if (a.F >= N) {
      if (f0 < a.F) {
#pragma unroll 8
        for (int d = gd; d < a.D; d += G) {
          const typename MMVec<T>::type v = *(const typename MMVec<T>::type*)(W + (size_t)d * a.F + f);
          float w[N];
#pragma unroll
          for (int i = 0; i < N; ++i) w[i] = (float)v[i];
          add(d, w);
        }
      }
    } else if (f == 0) {
#pragma unroll 1
      for (int d = gd; d < a.D; d += G) {
        float w[N];
        mm_load_vec(W + (size_t)d * a.F, 0, a.F, w);
        add(d, w);
      }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (fmaxf(top[i], top_x) >= MM_SPLIT_LIMIT) sum[i] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(g, sum[i], acc[i]);
  }
  // over the threads of a wave with the same columns, then over the waves
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int d = LC; d < 64; d <<= 1) acc[i] += __shfl_xor(acc[i], d);
    if ((threadIdx.x & 63) < LC) red[threadIdx.x >> 6][lc * N + i] = acc[i];
  }
  __syncthreads();
  if (threadIdx.x >= LC || f0 >= a.F) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    acc[i] = red[0][lc * N + i] + red[1][lc * N + i] + red[2][lc * N + i] + red[3][lc * N + i];
  mm_store_vec(y + (t * a.M + m) * a.F, f, a.F, acc);
}

// ------------------------------------------------------------------------------------------------ rows -> y
struct MMCombine {
  const float *rows, *gates;
  const int* experts;
  long T;
  int k, M, N, E;
};

// One vector of y a thread.  Bound by HBM: 65,536 rows of 1024 into bfloat16 59 us (5.1 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) mm_expert_combine_kernel(MMCombine a, T* __restrict__ y) {
  const int nv = (a.N + 3) / 4;
  const long i = (long)blockIdx.x * 256 + threadIdx.x, row = i / nv;
  if (row >= a.T * a.M) return;
  const int c = (int)(i - row * nv) * 4;
  const long t = row / a.M;
  const int m = (int)(row - t * a.M);
  float acc[4] = {};
  for (int j = 0; j < a.k; ++j) {
    const long s = t * a.k + j;
    if ((unsigned)a.experts[s] >= (unsigned)a.E) continue;
    const float g = a.gates ? a.gates[s] : 1.f;
    float v[4];
    mm_load4(a.rows + (s * a.M + m) * a.N, c, a.N, v);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = fmaf(g, v[q], acc[q]);
  }
  mm_store4(y + row * a.N, c, a.N, acc);
}

// One wave per row t: dx[t] = sum_j gate rows[t, j] and dgates[t, j] = sum_m <x[t, m], rows[t, j, m]>, KB choices at a
// time, so that rows are read once for up to KB choices.  Bound by HBM: 65,536 rows of 1024, bfloat16 x 69 us (4.8
// TB/s).
template <typename T, int KB>
__global__ void __launch_bounds__(256) mm_expert_combine_bwd_kernel(MMCombine a, const T* __restrict__ x, long st,
                                                                    long sm, T* __restrict__ dx,
                                                                    float* __restrict__ dgates) {
  const int lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  for (int j0 = 0; j0 < a.k; j0 += KB) {
    float g[KB], dg[KB];
    bool used[KB];
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const long s = t * a.k + j0 + j;
      used[j] = j0 + j < a.k && (unsigned)a.experts[s] < (unsigned)a.E;
      g[j] = used[j] && a.gates ? a.gates[s] : 1.f;
      dg[j] = 0.f;
    }
    for (int m = 0; m < a.M; ++m)
      for (int c = lane * 4; c < a.N; c += 256) {
        float acc[4] = {}, xv[4], v[KB][4];
        T* __restrict__ o = dx + (t * a.M + m) * a.N;
#pragma unroll
        for (int j = 0; j < KB; ++j)
          if (used[j]) mm_load4(a.rows + ((t * a.k + j0 + j) * a.M + m) * a.N, c, a.N, v[j]);
        if (dgates) mm_load4(x + t * st + m * sm, c, a.N, xv);
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          if (!used[j]) continue;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            acc[q] = fmaf(g[j], v[j][q], acc[q]);
            if (dgates) dg[j] = fmaf(xv[q], v[j][q], dg[j]);
          }
        }
        if (!dx) continue;
        // more choices than KB: the rows of the rest are added to the same sum, in order
        for (int j = KB; j < a.k; ++j) {
          const long s = t * a.k + j;
          if ((unsigned)a.experts[s] >= (unsigned)a.E) continue;
          const float gj = a.gates ? a.gates[s] : 1.f;
          float w[4];
          mm_load4(a.rows + (s * a.M + m) * a.N, c, a.N, w);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[q] = fmaf(gj, w[q], acc[q]);
        }
        mm_store4(o, c, a.N, acc);
      }
    if (dgates) {
#pragma unroll
      for (int j = 0; j < KB; ++j) {
        const float v = mm_lanes_sum<64>(dg[j]);
        if (lane == 0 && j0 + j < a.k) dgates[t * a.k + j0 + j] = used[j] ? v : 0.f;
      }
    }
    dx = nullptr;   // done in the first turn
    if (!dgates) return;
  }
}

// ------------------------------------------------------------------------------------------------ entry points
namespace {
// Narrow blocks take 64 columns a tile (33,456 float rows 368 -> 39: 56 us in tiles of 128, 37 so; 64,772 float16 rows
// 760 -> 32: 34, 26).  Tiles of 256 x 256 where the experts' lists and the columns fill them: twice the products per
// value loaded, but a cut tile at the end of every list.
bool big_tiles(long rows, int N, int E) { return rows >= 512L * E && N > 128; }

// two stages of both operands, then rows' offsets
template <int BM, int BN>
constexpr int rows_lds() { return 2 * (BM + BN) * 128 + BM * 8; }

template <typename T, bool TRANS, bool DMA, int BM, int BN, int WM, int WN>
int launch_rows_tile(const MMRows& a, int S, hipStream_t stream) {
  const int tiles_n = (a.N + BN - 1) / BN;
  // every expert's list may end in a cut tile
  const long wg = (((long)S * a.M + BM - 1) / BM + (a.E < S ? a.E : S)) * tiles_n;
  if (too_many(wg, 64 * WM * WN)) return range_error("mm_expert_rows", "output too large for one launch");
  constexpr auto kernel = mm_expert_rows_kernel<T, TRANS, DMA, BM, BN, WM, WN>;
  constexpr int lds = rows_lds<BM, BN>();
  if (!lds_granted<kernel>(lds)) return MM_ELAUNCH;
  hipLaunchKernelGGL(kernel, dim3((unsigned)wg), dim3(64 * WM * WN), lds, stream, a, tiles_n);
  return mm::launch_status("mm_expert_rows");
}

template <typename T, bool TRANS, bool DMA>
int launch_rows(const MMRows& a, int S, bool big, hipStream_t stream) {
  if constexpr (sizeof(T) == 2 && DMA)
    if (big) return launch_rows_tile<T, TRANS, DMA, 256, 256, 2, 4>(a, S, stream);
  if (a.N <= 64) return launch_rows_tile<T, TRANS, DMA, 128, 64, 2, 2>(a, S, stream);
  return launch_rows_tile<T, TRANS, DMA, 128, 128, 2, 2>(a, S, stream);
}

}  // namespace

extern "C" int mm_expert_rows(const void* in, long st, long sm, int dtype, int S, int k, int M, int K, int N,
                              const void* W, int transposed, int E, const int* offsets, const int* order, float* out,
                              hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(S >= 0 && k >= 1 && M >= 1 && K >= 1 && N >= 1 && E >= 1 && st >= 0 && sm >= 0, "bad sizes");
  if ((long)S * M > MM_EXPERT_MAX_ROWS) return range_error("mm_expert_rows", TOO_MANY_ROWS);
  if (too_wide(K, N)) return range_error("mm_expert_rows", TOO_WIDE);
  if (S == 0) return MM_OK;
  MM_CHECK_ARG(in && W && offsets && order && out, "a pointer is null");
  const MMRows a{in, W, offsets, order, out, st, sm, k, M, K, N, E};
  if (dtype == MM_F32 && K <= 128) return mm::launch_held("mm_expert_rows", a, S, nullptr, E, transposed, stream);
  const int unit = dtype == MM_F32 ? 4 : 8;
  const bool dma = aligned(in) && aligned(W) && st % unit == 0 && (M == 1 || sm % unit == 0) && K % unit == 0 &&
                   (transposed || N % unit == 0);
  int rc = MM_OK;
#define CALL(trans, dma)                                                          \
  if (dtype == MM_F32) rc = launch_rows<float, trans, dma>(a, S, false, stream);  \
  else if (dtype == MM_BF16) rc = launch_rows<__bf16, trans, dma>(a, S, big, stream); \
  else rc = launch_rows<_Float16, trans, dma>(a, S, big, stream);
  const bool big = big_tiles((long)S * M, N, E) && dma;
  if (transposed) { if (dma) { CALL(true, true) } else { CALL(true, false) } }
  else { if (dma) { CALL(false, true) } else { CALL(false, false) } }
#undef CALL
  return rc;
}

extern "C" int mm_expert_few(const void* x, long st, long sm, int dtype, int T, int k, int M, int D, int F,
                             const void* W, int E, const float* gates, const int* experts, void* y,
                             hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(T >= 0 && k >= 1 && M >= 1 && D >= 1 && F >= 1 && E >= 1 && st >= 0 && sm >= 0, "bad sizes");
  if (T > 65535 || M > 65535)
    return range_error("mm_expert_few", "more than 65535 rows or components are not supported");
  if (T == 0) return MM_OK;
  if (too_many(F / 16L + 1, 256)) return range_error("mm_expert_few", "output too large for one launch");
  if (too_wide(D, F)) return range_error("mm_expert_few", TOO_WIDE);
  MM_CHECK_ARG(x && W && experts && y, "a pointer is null");
  const MMFew a{x, W, gates, experts, st, sm, k, M, D, F, E};
#define CALL(T_)                                                                                             \
  hipLaunchKernelGGL((mm_expert_few_kernel<T_, 4>), dim3((F + 4 * MMVec<T_>::N - 1) / (4 * MMVec<T_>::N), T, M), \
                     dim3(256), 0, stream, a, (T_*)y)
  if (dtype == MM_F32) CALL(float);
  else if (dtype == MM_BF16) CALL(__bf16);
  else CALL(_Float16);
#undef CALL
  return mm::launch_status("mm_expert_few");
}

extern "C" int mm_expert_joined(const void* in, long st, long sm, int dtype, int T, int k, int M, int K, int N,
                                const void* W, int transposed, int E, const float* gates, const int* experts,
                                const int* offsets, const int* order, void* out, const void* x, long xt, long xm,
                                float* dgates, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(T >= 0 && M >= 1 && K >= 1 && N >= 1 && E >= 1 && st >= 0 && sm >= 0, "bad sizes");
  MM_CHECK_ARG(k == 1 || k == 2, "k must be 1 or 2");
  if (M > 64) return range_error("mm_expert_joined", "more than 64 components are not supported");
  if (too_wide(K, N)) return range_error("mm_expert_joined", TOO_WIDE);
  const int tiles_n = (N + 127) / 128, buckets = k == 1 ? E + 1 : E <= MM_PAIRS_MAX_E ? mm_pair_buckets(E) : 0;
  const int chunk = dtype == MM_F32 && K <= 128 && k == 2 && T ? mm::pairs_chunk((long)T * M, tiles_n, buckets, M) : 0;
  MM_CHECK_ARG(out || dgates, "nothing to compute");
  MM_CHECK_ARG(!dgates || (transposed && x && xt >= 0 && xm >= 0 && N <= 128 && (k == 1 || chunk || T == 0)),
               "dgates needs the transposed blocks, x, at most 128 columns, and one choice or short float rows");
  if (k == 2 && E > MM_PAIRS_MAX_E)
    return range_error("mm_expert_joined", "pairs of more than 21 experts are not supported");
  if ((long)T * M > MM_EXPERT_MAX_ROWS) return range_error("mm_expert_joined", TOO_MANY_ROWS);
  if (T == 0) return MM_OK;
  MM_CHECK_ARG(in && W && experts && offsets && order, "a pointer is null");
  if (dtype == MM_F32 && K <= 128 && k == 1 && !dgates && out) {
    const MMRows r{in, W, offsets, order, (float*)out, st, sm, 1, M, K, N, E};
    return mm::launch_held("mm_expert_joined", r, T, gates, E + 1, transposed, stream);
  }
  const int tile = (dtype == MM_F32 ? 128 : 64) / M;   // rows t a tile
  const long wg = (((long)T + tile - 1) / tile + (buckets < T ? buckets : T)) * tiles_n;
  if (too_many(wg, 256)) return range_error("mm_expert_joined", "output too large for one launch");
  if (chunk) {
    const MMPairs a{(const float*)in, (const float*)W, gates, (const float*)x, experts, offsets, order, (float*)out,
                    dgates, st, sm, xt, xm, T, M, K, N, E, buckets};
    return mm::launch_pairs("mm_expert_joined", a, transposed, chunk, stream);
  }
  const MMJoined a{in, W, x, gates, experts, offsets, order, out, dgates, st, sm, xt, xm, T, M, K, N, E, buckets};
  const int unit = dtype == MM_F32 ? 4 : 8;
  const bool dma = aligned(in) && aligned(W) && st % unit == 0 && (M == 1 || sm % unit == 0) && K % unit == 0 &&
                   (transposed || N % unit == 0);
#define CALL4(trans, dma, j, dg)                                                                                  \
  MM_DISPATCH(dtype,                                                                                              \
              hipLaunchKernelGGL((mm_expert_joined_kernel<T_, trans, dma, j, dg, sizeof(T_) == 4 ? 128 : 64>), \
                                 dim3((unsigned)wg), dim3(256), 0, stream, a, tiles_n))
#define CALL3(trans, j, dg) if (dma) { CALL4(trans, true, j, dg); } else { CALL4(trans, false, j, dg); }
#define CALL2(j) \
  if (transposed) { CALL3(true, j, false) } \
  else { CALL3(false, j, false) }
  if (dgates) { CALL3(true, 1, true) }
  else if (k == 1) { CALL2(1) }
  else { CALL2(2) }
#undef CALL2
#undef CALL3
#undef CALL4
  return mm::launch_status("mm_expert_joined");
}

extern "C" int mm_expert_combine(const float* rows, const float* gates, const int* experts, int dtype, long T, int k,
                                 int M, int N, int E, void* y, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(T >= 0 && k >= 1 && M >= 1 && N >= 1 && E >= 1, "bad sizes");
  if (too_wide(N, N)) return range_error("mm_expert_combine", TOO_WIDE);
  const long wg = (T * M * ((N + 3) / 4) + 255) / 256;
  if (too_many(wg, 256)) return range_error("mm_expert_combine", "output too large for one launch");
  if (wg == 0) return MM_OK;
  MM_CHECK_ARG(rows && experts && y, "a pointer is null");
  const MMCombine a{rows, gates, experts, T, k, M, N, E};
#define CALL hipLaunchKernelGGL((mm_expert_combine_kernel<T_>), dim3((unsigned)wg), dim3(256), 0, stream, a, (T_*)y)
  if (dtype == MM_F32) { using T_ = float; CALL; }
  else if (dtype == MM_BF16) { using T_ = __bf16; CALL; }
  else { using T_ = _Float16; CALL; }
#undef CALL
  return mm::launch_status("mm_expert_combine");
}

extern "C" int mm_expert_combine_bwd(const float* rows, const float* gates, const int* experts, const void* x, long st,
                                     long sm, int dtype, long T, int k, int M, int N, int E, void* dx, float* dgates,
                                     hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(T >= 0 && k >= 1 && M >= 1 && N >= 1 && E >= 1 && st >= 0 && sm >= 0, "bad sizes");
  if (too_wide(N, N)) return range_error("mm_expert_combine_bwd", TOO_WIDE);
  const long wg = (T + 3) / 4;
  if (too_many(wg, 256)) return range_error("mm_expert_combine_bwd", "too many rows for one launch");
  if (wg == 0) return MM_OK;
  MM_CHECK_ARG(rows && experts && (x || !dgates), "a pointer is null");
  const MMCombine a{rows, gates, experts, T, k, M, N, E};
#define CALL2(KB)                                                                                            \
  hipLaunchKernelGGL((mm_expert_combine_bwd_kernel<T_, KB>), dim3((unsigned)wg), dim3(256), 0, stream, a, \
                     (const T_*)x, st, sm, (T_*)dx, dgates);
#define CALL if (k == 1) { CALL2(1) } else if (k == 2) { CALL2(2) } else { CALL2(4) }
  if (dtype == MM_F32) { using T_ = float; CALL }
  else if (dtype == MM_BF16) { using T_ = __bf16; CALL }
  else { using T_ = _Float16; CALL }
#undef CALL
#undef CALL2
  return mm::launch_status("mm_expert_combine_bwd");
}

