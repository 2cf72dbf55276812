// Layer norm over the last axis of rows, forward and backward:
//     y = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//     g = dy w,  h = (x - mean) rstd:
//     dx = rstd (g - mean(g) - h mean(g h)),   dw = sum_rows dy h,   db = sum_rows dy
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx, with 8 and 14 operations an
// element. A row stays in the registers of LPR lanes (NV vectors of 16 bytes each), so it is read once and the
// variance is taken about the mean; all sums are fp32.  Several rows share a wave where they are short.  Backward: a
// workgroup walks over many rows with the sums of dy h and dy of its own columns in registers, writes them once as
// partial sums, and a second launch adds the workgroups' in a fixed order: no atomics, so the gradients are the same
// in every run.  Measured: 1,474,560 float rows of 64: forward 147 us (5.1 TB/s), backward 225 + 5 us (5.0 TB/s);
// 8,191 bfloat16 rows of 4096: 32 us (4.2 TB/s) and 44 + 11 us (the partial sums are a sixth of the traffic there).
#include "norm.h"

#define MM_NORM_MAX_D 16384
#define MM_NORM_WG 1024   // workgroups of the backward (partial sums of dw and db)

// sum over the LPR lanes of a row; LPR > 64: over the workgroup (s: one float per wave, two sets used in turn)
template <int LPR>
__device__ __forceinline__ float mm_norm_sum(float v, float* s) {
  if constexpr (LPR <= 64) {
    return mm_lanes_sum<LPR>(v);
  } else {
    v = mm_lanes_sum<64>(v);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < LPR / 64; ++w) t += s[w];
    return t;
  }
}

template <typename T, int LPR, int NV>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256)
mm_layernorm_fwd_kernel(const T* __restrict__ x, long ldx, long rows, int D, const void* __restrict__ w,
                        const void* __restrict__ b, int p_f32, float eps, T* __restrict__ y, long ldy,
                        float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int N = MMVec<T>::N, TPB = LPR > 256 ? LPR : 256, RPB = TPB / LPR;
  __shared__ float s[2][16];
  const int lane = threadIdx.x & (LPR - 1), sub = threadIdx.x / LPR;
  const float n = (float)D;
  float wv[NV][N], bv[NV][N];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * LPR + lane) * N;
    mm_norm_param<T>(w, p_f32, 1.f, c, D, wv[v]);
    mm_norm_param<T>(b, p_f32, 0.f, c, D, bv[v]);
  }
  for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += (long)gridDim.x * RPB) {
    const bool ok = r0 + sub < rows;
    const long r = ok ? r0 + sub : rows - 1;   // the same row twice instead of one past the end; not stored
    float v[NV][N], t = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) mm_load_vec(x + r * ldx, (j * LPR + lane) * N, D, v[j]);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) t += v[j][i];
    const float mu = mm_norm_sum<LPR>(t, s[0]) / n;   // divided: the mean of equal values is that value
    t = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[j][i] = (j * LPR + lane) * N + i < D ? v[j][i] - mu : 0.f;
        t = fmaf(v[j][i], v[j][i], t);
      }
    const float rs = 1.f / sqrtf(mm_norm_sum<LPR>(t, s[1]) / n + eps);
    if (ok) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[j][i] = fmaf(v[j][i] * rs, wv[j][i], bv[j][i]);
        mm_store_vec(y + r * ldy, (j * LPR + lane) * N, D, v[j]);
      }
      if (mean && lane == 0) {
        mean[r] = mu;
        rstd[r] = rs;
      }
    }
    if constexpr (LPR > 64) __syncthreads();   // the sums' LDS is free for the next row
  }
}

// part: [2][gridDim.x][D] partial sums of dw, then db
template <typename T, int LPR, int NV>
__global__ void __launch_bounds__(LPR > 256 ? LPR : 256)
mm_layernorm_bwd_kernel(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx, long rows, int D,
                        const void* __restrict__ w, int p_f32, const float* __restrict__ mean,
                        const float* __restrict__ rstd, T* __restrict__ dx, long lddx, float* __restrict__ part) {
  constexpr int N = MMVec<T>::N, TPB = LPR > 256 ? LPR : 256, RPB = TPB / LPR;
  __shared__ float s[2][16];
  const int lane = threadIdx.x & (LPR - 1), sub = threadIdx.x / LPR;
  const float n = (float)D;
  float wv[NV][N], dw[NV][N], db[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    mm_norm_param<T>(w, p_f32, 1.f, (j * LPR + lane) * N, D, wv[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) dw[j][i] = db[j][i] = 0.f;
  }
  for (long r0 = (long)blockIdx.x * RPB; r0 < rows; r0 += (long)gridDim.x * RPB) {
    const bool ok = r0 + sub < rows;
    const long r = ok ? r0 + sub : rows - 1;
    const float mu = mean[r], rs = rstd[r];
    float h[NV][N], g[NV][N], t0 = 0.f, t1 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      mm_load_vec(x + r * ldx, (j * LPR + lane) * N, D, h[j]);
      mm_load_vec(dy + r * lddy, (j * LPR + lane) * N, D, g[j]);   // 0 past the last column: such columns add nothing
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        h[j][i] = (h[j][i] - mu) * rs;
        if (ok) {
          dw[j][i] = fmaf(g[j][i], h[j][i], dw[j][i]);
          db[j][i] += g[j][i];
        }
        g[j][i] *= wv[j][i];
        t0 += g[j][i];
        t1 = fmaf(g[j][i], h[j][i], t1);
      }
    if (!dx) continue;
    if constexpr (LPR > 64) __syncthreads();   // the previous row's sums are read
    const float m0 = mm_norm_sum<LPR>(t0, s[0]) / n, m1 = mm_norm_sum<LPR>(t1, s[1]) / n;
    if (ok) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[j][i] = rs * (g[j][i] - m0 - h[j][i] * m1);
        mm_store_vec(dx + r * lddx, (j * LPR + lane) * N, D, g[j]);
      }
    }
  }
  if (!part) return;
  float* pw = part + (size_t)blockIdx.x * D;
  float* pb = part + ((size_t)gridDim.x + blockIdx.x) * D;
  if constexpr (LPR >= 256) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        mm_store_vec(pw, (j * LPR + lane) * N + i, D, dw[j] + i);
        mm_store_vec(pb, (j * LPR + lane) * N + i, D, db[j] + i);
      }
    }
  } else {
    // the rows of a wave by lane moves, the waves through LDS, one vector at a time
    __shared__ float red[2][4][64 * N];
    const int wave = threadIdx.x >> 6, l64 = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int d = LPR; d < 64; d <<= 1) {
          dw[j][i] += __shfl_xor(dw[j][i], d);
          db[j][i] += __shfl_xor(db[j][i], d);
        }
        if (l64 < LPR) {
          red[0][wave][l64 * N + i] = dw[j][i];
          red[1][wave][l64 * N + i] = db[j][i];
        }
      }
      __syncthreads();
      for (int q = threadIdx.x; q < 2 * LPR * N; q += 256) {
        const int which = q / (LPR * N), e = q - which * (LPR * N), c = j * LPR * N + e;
        const float t = red[which][0][e] + red[which][1][e] + red[which][2][e] + red[which][3][e];
        if (c < D) (which ? pb : pw)[c] = t;
      }
      __syncthreads();
    }
  }
}

// dw[c] (blockIdx.y 0) and db[c] (1): 16 columns by 64 groups of partial rows a workgroup
__global__ void __launch_bounds__(1024) mm_layernorm_sum_kernel(const float* __restrict__ part, int n_part, int D,
                                                                int out_dtype, void* __restrict__ dw,
                                                                void* __restrict__ db) {
  __shared__ float s[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
  const float* __restrict__ p = part + (size_t)blockIdx.y * n_part * D;
  float t = 0.f;
  if (c < D) {
    int r = q;
    for (; r + 448 < n_part; r += 512) {   // eight loads on their way
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[(size_t)(r + 64 * i) * D + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) t += v[i];
    }
    for (; r < n_part; r += 64) t += p[(size_t)r * D + c];
  }
  s[q][threadIdx.x & 15] = t;
  __syncthreads();
  if (q || c >= D) return;
  t = 0.f;
#pragma unroll
  for (int r = 0; r < 64; ++r) t += s[r][threadIdx.x];
  void* o = blockIdx.y ? db : dw;
  if (!o) return;
  if (out_dtype == MM_F32) ((float*)o)[c] = t;
  else if (out_dtype == MM_BF16) ((__bf16*)o)[c] = (__bf16)t;
  else ((_Float16*)o)[c] = (_Float16)t;
}

namespace {
long norm_rows_per_wg(int lpr) { return lpr > 256 ? 1 : 256 / lpr; }

// Lanes per row and vectors per lane: the least that hold D columns.  Rows of 1025 .. 2048 16-bit values take a
// workgroup: 32 values a lane of one wave leave too few waves for the loads (backward, bfloat16, us, a wave / a
// workgroup: 16,384 x 2048 72 / 54, 60,000 x 2000 224 / 164; forward 32 / 26, 107 / 97).
struct Shape { int lpr, nv; };
const Shape kShapes[] = {{4, 1}, {8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {64, 4}, {256, 1}, {256, 2}, {256, 4},
                         {1024, 2}, {1024, 4}};
constexpr int kUnused[] = {7, 6};   // shape that float, that 16-bit types do without

int shape_of(int D, int dtype) {
  const int n = dtype == MM_F32 ? 4 : 8, without = kUnused[dtype != MM_F32];
  int i = 0;
  while (kShapes[i].lpr * kShapes[i].nv * n < D || i == without) ++i;
  return i;
}

// Workgroups of the backward: as many as have rows, at most MM_NORM_WG.  Long rows, where the partial sums are a part
// of the traffic that counts: half of that below 32 rows each (us, 1024 / 512: float 8192 x 4096 92 / 82, 4096 x 8192
// 106 / 92, but 60,000 x 2000 278 / 307); not for 16-bit rows of up to 4096, whose loads need the waves (8192 x 4096:
// 58 / 73).
int bwd_workgroups(long rows, int D, int dtype) {
  const Shape sh = kShapes[shape_of(D, dtype)];
  const long rpb = norm_rows_per_wg(sh.lpr), n = (rows + rpb - 1) / rpb;
  const bool is_long = sh.lpr > 256 || (sh.lpr == 256 && (dtype == MM_F32 || sh.nv == 4));
  const long most = is_long && rows < 32L * MM_NORM_WG ? MM_NORM_WG / 2 : MM_NORM_WG;
  return (int)(n < most ? n : most);
}
}  // namespace

namespace mm {
void sum_partials(const float* part, int n_part, int D, int out_dtype, void* dw, void* db, hipStream_t stream) {
  hipLaunchKernelGGL(mm_layernorm_sum_kernel, dim3((D + 15) / 16, 2), dim3(1024), 0, stream, part, n_part, D, out_dtype,
                     dw, db);
}
}  // namespace mm

#define MM_NORM_SHAPES(X) X(0, 4, 1) X(1, 8, 1) X(2, 16, 1) X(3, 32, 1) X(4, 64, 1) X(5, 64, 2) X(6, 64, 4) \
  X(7, 256, 1) X(8, 256, 2) X(9, 256, 4) X(10, 1024, 2) X(11, 1024, 4)

extern "C" int mm_layernorm_fwd(const void* x, long ldx, int dtype, long rows, int D, const void* w, const void* b,
                                int p_dtype, float eps, void* y, long ldy, float* mean, float* rstd,
                                hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(p_dtype == dtype || p_dtype == MM_F32, "weight and bias must have the type of x or float");
  MM_CHECK_ARG(rows >= 0 && D > 0 && ldx >= 0 && ldy >= D, "bad sizes");
  MM_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "mean and rstd come together");
  if (D > MM_NORM_MAX_D) {
    mm::set_error("mm_layernorm_fwd: rows longer than 16384 are not supported");
    return MM_ERANGE;
  }
  if (rows == 0) return MM_OK;
  const int sh = shape_of(D, dtype), lpr = kShapes[sh].lpr;
  const long rpb = norm_rows_per_wg(lpr), n = (rows + rpb - 1) / rpb;
  const dim3 grid((unsigned)(n < 4096 ? n : 4096));
#define X(i, l, v)                                                                                              \
  if constexpr (l * v * MMVec<T_>::N <= MM_NORM_MAX_D && i != kUnused[sizeof(T_) == 2]) if (sh == i) \
    hipLaunchKernelGGL((mm_layernorm_fwd_kernel<T_, l, v>), grid, dim3(l > 256 ? l : 256), 0, stream, (const T_*)x, \
                       ldx, rows, D, w, b, p_dtype == MM_F32, eps, (T_*)y, ldy, mean, rstd);
  MM_DISPATCH(dtype, MM_NORM_SHAPES(X));
#undef X
  return mm::launch_status("mm_layernorm_fwd");
}

extern "C" int mm_layernorm_workspace(long rows, int D, int dtype, size_t* bytes) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16 && rows >= 0 && D > 0 && D <= MM_NORM_MAX_D && bytes, "bad sizes");
  *bytes = (size_t)2 * bwd_workgroups(rows, D, dtype) * D * sizeof(float);
  return MM_OK;
}

extern "C" int mm_layernorm_bwd(const void* dy, long lddy, const void* x, long ldx, int dtype, long rows, int D,
                                const void* w, int p_dtype, const float* mean, const float* rstd, void* dx, long lddx,
                                void* dw, void* db, float* workspace, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(p_dtype == dtype || p_dtype == MM_F32, "weight and bias must have the type of x or float");
  MM_CHECK_ARG(rows >= 0 && D > 0 && lddy >= 0 && ldx >= 0 && (!dx || lddx >= D), "bad sizes");
  MM_CHECK_ARG(!(dw || db) || rows == 0 || workspace, "dw and db need the workspace");
  if (D > MM_NORM_MAX_D) {
    mm::set_error("mm_layernorm_bwd: rows longer than 16384 are not supported");
    return MM_ERANGE;
  }
  const int sh = shape_of(D, dtype), n = bwd_workgroups(rows, D, dtype);
  float* part = dw || db ? workspace : nullptr;
#define X(i, l, v)                                                                                               \
  if constexpr (l * v * MMVec<T_>::N <= MM_NORM_MAX_D && i != kUnused[sizeof(T_) == 2]) if (sh == i) \
    hipLaunchKernelGGL((mm_layernorm_bwd_kernel<T_, l, v>), dim3(n), dim3(l > 256 ? l : 256), 0, stream,          \
                       (const T_*)dy, lddy, (const T_*)x, ldx, rows, D, w, p_dtype == MM_F32, mean, rstd, (T_*)dx,  \
                       lddx, part);
  if (n && (dx || part)) MM_DISPATCH(dtype, MM_NORM_SHAPES(X));
#undef X
  if (dw || db) mm::sum_partials(workspace, n, D, p_dtype, dw, db, stream);
  return mm::launch_status("mm_layernorm_bwd");
}
