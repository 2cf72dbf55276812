// Products of rows with the weight blocks of their experts:  y[t, m] = sum_j gate[t, j] x[t, m] @ W[expert[t, j]],
// with the gradients of x, W and the gates.  A slot is a (row, choice) pair s = t k + j; the plan lists the slots sorted
// by expert (stable), so that each expert's rows are consecutive and its block is read once per tile of rows.
//   mm_expert_plan     offsets [E + 1] and order [S]: the slots of expert e are order[offsets[e] .. offsets[e + 1])
//   mm_expert_rows     out[s, m] = in[s / k, m] @ W[e]  (or @ W[e]^T): fp32 rows in slot order
//   mm_expert_combine  y[t, m] = sum_j gate rows[t k + j, m];  mm_expert_combine_bwd  dx and dgates from the rows of dy
//   mm_expert_wgrad    dW[e] = sum of the expert's slots and components of gate x^T dy
// A slot whose expert lies outside [0, E) takes part nowhere.
#include "rowvec.h"

#define MM_EXPERT_MAX_E 1024
#define MM_PLAN_WAVE 1024   // slots per wave of the plan kernels

// ------------------------------------------------------------------------------------------------ plan
// counts[e][tile]: slots of expert e in the tile of 4 waves
__global__ void __launch_bounds__(256) mm_plan_count_kernel(const int* __restrict__ experts, int S, int E, int tiles,
                                                            int* __restrict__ counts) {
  extern __shared__ int h[];
  for (int e = threadIdx.x; e < E; e += 256) h[e] = 0;
  __syncthreads();
  for (int r = 0; r < 4 * MM_PLAN_WAVE; r += 256) {
    const long s = (long)blockIdx.x * (4 * MM_PLAN_WAVE) + r + threadIdx.x;
    if (s >= S) break;
    const int e = experts[s];
    if ((unsigned)e < (unsigned)E) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += 256) counts[(size_t)e * tiles + blockIdx.x] = h[e];
}

// one workgroup per expert: exclusive prefix sum over the tiles, and the total
__global__ void __launch_bounds__(256) mm_plan_scan_kernel(int* __restrict__ counts, int tiles,
                                                           int* __restrict__ totals) {
  __shared__ int s[4];
  int* __restrict__ row = counts + (size_t)blockIdx.x * tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + threadIdx.x;
    const int v = t < tiles ? row[t] : 0;
    int inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    if (lane == 63) s[wave] = inc;
    __syncthreads();
    int before = carry;
    for (int w = 0; w < wave; ++w) before += s[w];
    if (t < tiles) row[t] = before + inc - v;
    carry += s[0] + s[1] + s[2] + s[3];
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Scatter of a tile of NW waves: the waves count their slots, then each ranks 64 consecutive slots at a time among equal
// experts with one ballot per bit, on top of its counters.  SINGLE: the tile is the whole list, nothing was counted.
template <int NW, bool SINGLE>
__global__ void __launch_bounds__(64 * NW) mm_plan_kernel(const int* __restrict__ experts, int S, int E, int bits,
                                                          int tiles, const int* __restrict__ counts,
                                                          const int* __restrict__ totals, int* __restrict__ offsets,
                                                          int* __restrict__ order) {
  extern __shared__ int sm[];
  int* cnt = sm;            // [NW][E]
  int* base = sm + NW * E;  // [E]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long s0 = (long)blockIdx.x * (NW * MM_PLAN_WAVE) + wave * MM_PLAN_WAVE + lane;
  for (int i = tid; i < NW * E; i += 64 * NW) cnt[i] = 0;
  __syncthreads();
  for (int r = 0; r < MM_PLAN_WAVE; r += 64) {
    const int e = s0 + r < S ? experts[s0 + r] : -1;
    if ((unsigned)e < (unsigned)E) atomicAdd(&cnt[wave * E + e], 1);
  }
  __syncthreads();
  for (int e = tid; e < E; e += 64 * NW) {
    int t = 0;
    if constexpr (SINGLE) {
      for (int w = 0; w < NW; ++w) t += cnt[w * E + e];
    } else {
      t = totals[e];
    }
    base[e] = t;
  }
  __syncthreads();
  if (wave == 0) {   // exclusive prefix sum of the experts' totals
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int e = e0 + lane, v = e < E ? base[e] : 0;
      int inc = v;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(inc, d);
        if (lane >= d) inc += u;
      }
      if (e < E) {
        base[e] = carry + inc - v;
        if (blockIdx.x == 0) offsets[e] = carry + inc - v;
      }
      carry += __shfl(inc, 63);
    }
    if (blockIdx.x == 0 && lane == 0) offsets[E] = carry;
  }
  __syncthreads();
  for (int e = tid; e < E; e += 64 * NW) {
    int at = base[e];
    if constexpr (!SINGLE) at += counts[(size_t)e * tiles + blockIdx.x];
    for (int w = 0; w < NW; ++w) {
      const int c = cnt[w * E + e];
      cnt[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int r = 0; r < MM_PLAN_WAVE; r += 64) {
    const int e = s0 + r < S ? experts[s0 + r] : -1;
    const bool ok = (unsigned)e < (unsigned)E;
    unsigned long long same = __ballot(ok);
    if (same == 0) continue;
    for (int b = 0; b < bits; ++b) {
      const unsigned long long m = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? m : ~m;
    }
    const int before = __popcll(same & ((1ull << lane) - 1));
    const int at = ok ? cnt[wave * E + e] : 0;
    mm_wave_lds_sync();
    if (ok && before == 0) cnt[wave * E + e] = at + __popcll(same);
    mm_wave_lds_sync();
    if (ok) order[at + before] = (int)(s0 + r);
  }
}

// ------------------------------------------------------------------------------------------------ tiles of an expert
struct MMTile {
  int e, row0, rows;   // expert, first of its rows (slots x M), rows in the tile; e < 0: no such tile
};

// The tile-th tile of BM rows of the experts' row lists one after the other (every expert's list ends in a cut tile);
// every wave finds it by itself, 64 experts at a time.
__device__ __forceinline__ MMTile mm_expert_tile(const int* __restrict__ offsets, int E, int M, int BM, int tile) {
  const int lane = threadIdx.x & 63;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int e = e0 + lane;
    const int rows = e < E ? (offsets[e + 1] - offsets[e]) * M : 0, n = (rows + BM - 1) / BM;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    const unsigned long long past = __ballot(inc > tile);
    if (past) {
      const int src = __ffsll(past) - 1;
      const int first = (tile - __shfl(inc - n, src)) * BM, total = __shfl(rows, src);
      return MMTile{e0 + src, first, min(BM, total - first)};
    }
    tile -= __shfl(inc, 63);
  }
  return MMTile{-1, 0, 0};
}

// ------------------------------------------------------------------------------------------------ rows
struct MMRows {
  const void *in, *W;
  const int *offsets, *order;
  float* out;
  long st, sm;   // strides of in in elements: rows, components
  int k, M, K, N, E;
};

// 64 x 64 tiles, 4 x 4 values a thread, fp32 products and sums.  TRANS: W[e] is [N][K], else [K][N].
template <typename T, bool TRANS>
__global__ void __launch_bounds__(256) mm_expert_rows_kernel(MMRows a) {
  __shared__ float As[16][68], Bs[16][68];
  __shared__ long s_in[64], s_out[64];
  const MMTile t = mm_expert_tile(a.offsets, a.E, a.M, 64, blockIdx.x);
  if (t.e < 0) return;
  const int tid = threadIdx.x, n0 = blockIdx.y * 64;
  if (tid < 64) {
    const int r = t.row0 + min(tid, t.rows - 1), p = r / a.M, m = r - p * a.M;
    const int slot = a.order[a.offsets[t.e] + p];
    s_in[tid] = (slot / a.k) * a.st + m * a.sm;
    s_out[tid] = ((long)slot * a.M + m) * a.N;
  }
  __syncthreads();
  const T* __restrict__ in = (const T*)a.in;
  const T* __restrict__ W = (const T*)a.W + (size_t)t.e * a.K * a.N;
  float acc[4][4] = {};
  const int tr = tid >> 4, tc = tid & 15;
  for (int k0 = 0; k0 < a.K; k0 += 16) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int kk = tid & 15, r = (tid >> 4) + 16 * q;
      As[kk][r] = k0 + kk < a.K ? (float)in[s_in[r] + k0 + kk] : 0.f;
      if (TRANS) {
        const int n = n0 + r;
        Bs[kk][r] = k0 + kk < a.K && n < a.N ? (float)W[(size_t)n * a.K + k0 + kk] : 0.f;
      } else {
        const int kb = (tid >> 6) + 4 * q, n = n0 + (tid & 63);
        Bs[kb][tid & 63] = k0 + kb < a.K && n < a.N ? (float)W[(size_t)(k0 + kb) * a.N + n] : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[kk][tr * 4 + i], Bs[kk][tc * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (tr * 4 + i >= t.rows) continue;
    mm_store_vec(a.out + s_out[tr * 4 + i], n0 + tc * 4, a.N, acc[i]);
  }
}

// ------------------------------------------------------------------------------------------------ rows -> y
struct MMCombine {
  const float *rows, *gates;
  const int* experts;
  long T;
  int k, M, N, E;
};

// one vector of y a thread
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
    mm_load_vec(a.rows + (s * a.M + m) * a.N, c, a.N, v);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = fmaf(g, v[q], acc[q]);
  }
  T* __restrict__ o = y + row * a.N + c;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (c + q < a.N) o[q] = (T)acc[q];
}

// one wave per row t: dx[t] = sum_j gate rows[t, j] and dgates[t, j] = sum_m <x[t, m], rows[t, j, m]>
template <typename T>
__global__ void __launch_bounds__(256) mm_expert_combine_bwd_kernel(MMCombine a, const T* __restrict__ x, long st,
                                                                    long sm, T* __restrict__ dx,
                                                                    float* __restrict__ dgates) {
  const int lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  if (dx) {
    for (int m = 0; m < a.M; ++m)
      for (int c = lane * 4; c < a.N; c += 256) {
        float acc[4] = {};
        for (int j = 0; j < a.k; ++j) {
          const long s = t * a.k + j;
          if ((unsigned)a.experts[s] >= (unsigned)a.E) continue;
          const float g = a.gates ? a.gates[s] : 1.f;
          float v[4];
          mm_load_vec(a.rows + (s * a.M + m) * a.N, c, a.N, v);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[q] = fmaf(g, v[q], acc[q]);
        }
        T* __restrict__ o = dx + (t * a.M + m) * a.N + c;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (c + q < a.N) o[q] = (T)acc[q];
      }
  }
  if (dgates) {
    for (int j = 0; j < a.k; ++j) {
      const long s = t * a.k + j;
      const bool used = (unsigned)a.experts[s] < (unsigned)a.E;
      float acc = 0.f;
      if (used)
        for (int m = 0; m < a.M; ++m)
          for (int c = lane; c < a.N; c += 64)
            acc = fmaf((float)x[t * st + m * sm + c], a.rows[(s * a.M + m) * a.N + c], acc);
      acc = mm_lanes_sum<64>(acc);
      if (lane == 0) dgates[s] = used ? acc : 0.f;
    }
  }
}

// ------------------------------------------------------------------------------------------------ dW
struct MMWgrad {
  const void *x, *dy;
  const float* gates;
  const int *offsets, *order;
  void* dW;
  long xt, xm, yt, ym;
  int k, M, D, F, E;
};

// a workgroup: one 64 x 64 tile of dW[e] over all rows of expert e, 16 rows at a time in the order of the plan
template <typename T>
__global__ void __launch_bounds__(256) mm_expert_wgrad_kernel(MMWgrad a) {
  __shared__ float Xs[16][68], Ys[16][68];
  const int e = blockIdx.z, d0 = blockIdx.x * 64, f0 = blockIdx.y * 64, tid = threadIdx.x;
  const int first = a.offsets[e], rows = (a.offsets[e + 1] - first) * a.M;
  float acc[4][4] = {};
  const int tr = tid >> 4, tc = tid & 15;
  for (int r0 = 0; r0 < rows; r0 += 16) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int rr = (tid >> 6) + 4 * q, c = tid & 63, r = r0 + rr;
      float xv = 0.f, yv = 0.f;
      if (r < rows) {
        const int p = r / a.M, m = r - p * a.M, slot = a.order[first + p];
        const long t = slot / a.k;
        if (d0 + c < a.D) xv = (float)((const T*)a.x)[t * a.xt + m * a.xm + d0 + c];
        if (f0 + c < a.F) yv = (float)((const T*)a.dy)[t * a.yt + m * a.ym + f0 + c] * (a.gates ? a.gates[slot] : 1.f);
      }
      Xs[rr][c] = xv;
      Ys[rr][c] = yv;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(Xs[kk][tr * 4 + i], Ys[kk][tc * 4 + j], acc[i][j]);
    __syncthreads();
  }
  T* __restrict__ o = (T*)a.dW + (size_t)e * a.D * a.F;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = d0 + tr * 4 + i, f = f0 + tc * 4 + j;
      if (d < a.D && f < a.F) o[(size_t)d * a.F + f] = (T)acc[i][j];
    }
}

// ------------------------------------------------------------------------------------------------ entry points
namespace {
constexpr int kPlanTile = 4 * MM_PLAN_WAVE;

// waves of the one workgroup that plans S slots of E experts (its counters fit 64 KB of LDS); 0: several workgroups
int plan_waves(int S, int E) { return S <= 4 * MM_PLAN_WAVE ? 4 : S <= 16 * MM_PLAN_WAVE && E <= 512 ? 16 : 0; }

int range_error(const char* name, const char* what) {
  mm::set_error(std::string(name) + ": " + what);
  return MM_ERANGE;
}
}  // namespace

extern "C" int mm_expert_plan_scratch(int S, int E, long* ints) {
  MM_CHECK_ARG(S >= 0 && E >= 1 && ints, "bad sizes");
  *ints = plan_waves(S, E) ? 0 : (long)E * ((S + (long)kPlanTile - 1) / kPlanTile + 1);
  return MM_OK;
}

extern "C" int mm_expert_plan(const int* experts, int S, int E, int* offsets, int* order, int* scratch,
                              hipStream_t stream) {
  MM_CHECK_ARG(S >= 0 && E >= 1, "bad sizes");
  if (E > MM_EXPERT_MAX_E) return range_error("mm_expert_plan", "more than 1024 experts are not supported");
  int bits = 0;
  while (bits < 31 && (E - 1) >> bits) ++bits;
  const int waves = plan_waves(S, E);
  if (waves == 4)
    hipLaunchKernelGGL((mm_plan_kernel<4, true>), dim3(1), dim3(256), 5 * E * sizeof(int), stream, experts, S, E, bits,
                       1, nullptr, nullptr, offsets, order);
  else if (waves)
    hipLaunchKernelGGL((mm_plan_kernel<16, true>), dim3(1), dim3(1024), 17 * E * sizeof(int), stream, experts, S, E,
                       bits, 1, nullptr, nullptr, offsets, order);
  if (waves) return mm::launch_status("mm_expert_plan");
  MM_CHECK_ARG(scratch, "scratch is null");
  const int tiles = (int)((S + (long)kPlanTile - 1) / kPlanTile);
  int *counts = scratch, *totals = scratch + (size_t)E * tiles;
  hipLaunchKernelGGL(mm_plan_count_kernel, dim3(tiles), dim3(256), E * sizeof(int), stream, experts, S, E, tiles,
                     counts);
  hipLaunchKernelGGL(mm_plan_scan_kernel, dim3(E), dim3(256), 0, stream, counts, tiles, totals);
  hipLaunchKernelGGL((mm_plan_kernel<4, false>), dim3(tiles), dim3(256), 5 * E * sizeof(int), stream, experts, S, E,
                     bits, tiles, counts, totals, offsets, order);
  return mm::launch_status("mm_expert_plan");
}

extern "C" int mm_expert_rows(const void* in, long st, long sm, int dtype, int S, int k, int M, int K, int N,
                              const void* W, int transposed, int E, const int* offsets, const int* order, float* out,
                              hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(S >= 0 && k >= 1 && M >= 1 && K >= 1 && N >= 1 && E >= 1 && st >= 0 && sm >= 0, "bad sizes");
  if ((long)S * M > 2147483647L - 64) return range_error("mm_expert_rows", "2^31 rows or more are not supported");
  if (S == 0) return MM_OK;
  const MMRows a{in, W, offsets, order, out, st, sm, k, M, K, N, E};
  // every expert's list may end in a cut tile
  const dim3 grid((unsigned)(((long)S * M + 63) / 64 + (E < S ? E : S)), (unsigned)((N + 63) / 64));
  if (transposed)
    MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_rows_kernel<T, true>), grid, dim3(256), 0, stream, a));
  else
    MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_rows_kernel<T, false>), grid, dim3(256), 0, stream, a));
  return mm::launch_status("mm_expert_rows");
}

extern "C" int mm_expert_combine(const float* rows, const float* gates, const int* experts, int dtype, long T, int k,
                                 int M, int N, int E, void* y, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(T >= 0 && k >= 1 && M >= 1 && N >= 1 && E >= 1, "bad sizes");
  const long wg = (T * M * ((N + 3) / 4) + 255) / 256;
  if (wg > 2147483647L) return range_error("mm_expert_combine", "output too large for one launch");
  if (wg == 0) return MM_OK;
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
  const long wg = (T + 3) / 4;
  if (wg > 2147483647L) return range_error("mm_expert_combine_bwd", "too many rows for one launch");
  if (wg == 0) return MM_OK;
  const MMCombine a{rows, gates, experts, T, k, M, N, E};
#define CALL                                                                                                          \
  hipLaunchKernelGGL((mm_expert_combine_bwd_kernel<T_>), dim3((unsigned)wg), dim3(256), 0, stream, a, (const T_*)x, st, \
                     sm, (T_*)dx, dgates)
  if (dtype == MM_F32) { using T_ = float; CALL; }
  else if (dtype == MM_BF16) { using T_ = __bf16; CALL; }
  else { using T_ = _Float16; CALL; }
#undef CALL
  return mm::launch_status("mm_expert_combine_bwd");
}

extern "C" int mm_expert_wgrad(const void* x, long xt, long xm, const void* dy, long yt, long ym, int dtype, int S,
                               int k, int M, int D, int F, int E, const float* gates, const int* offsets,
                               const int* order, void* dW, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(S >= 0 && k >= 1 && M >= 1 && D >= 1 && F >= 1 && E >= 1, "bad sizes");
  MM_CHECK_ARG(xt >= 0 && xm >= 0 && yt >= 0 && ym >= 0, "bad strides");
  if (E > MM_EXPERT_MAX_E) return range_error("mm_expert_wgrad", "more than 1024 experts are not supported");
  if ((long)S * M > 2147483647L - 64) return range_error("mm_expert_wgrad", "2^31 rows or more are not supported");
  const MMWgrad a{x, dy, gates, offsets, order, dW, xt, xm, yt, ym, k, M, D, F, E};
  const dim3 grid((D + 63) / 64, (F + 63) / 64, E);
  MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_wgrad_kernel<T>), grid, dim3(256), 0, stream, a));
  return mm::launch_status("mm_expert_wgrad");
}
