// Group norm of rows of channels with an activation, forward and backward.  A structure is a run of rows, a group a run
// of cg = C / groups channels; over the n = rows x cg values of a (structure, group):
//     h = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  z = h w + b,  y = act(z)
//     dz = dy act'(z):  dw = sum_rows dz h,  db = sum_rows dz,  dx = rstd (dz w - mean(dz w) - h mean(dz w h))
// Bound by HBM.  A thread keeps one vector of 16 bytes of channels for several rows, and sums go by channel first (over
// a thread's rows, the lanes of a wave, the waves through LDS), then over the channels of a group: any group size works,
// whether or not it holds whole vectors.
//
// Two ways, by the number of rows of a structure, which the host need not know:
//   whole  a workgroup holds the structure (of its block of whole groups) in registers: every value is read once;
//   tiles  structures of more than `small` rows go in tiles of `small` rows: partial statistics of every tile, their
//          sum by structure, and a second reading.  Tiles lie at multiples of `small` rows, so a tile meets at most two
//          such structures: the one that holds its first row (part 0) and one that begins inside (part 1).
// Variances are about the mean (of a tile, joined as M2 + n (mean_i - mean)^2).  All sums are fp32 in a fixed order: no
// atomics, the same bits in every run.
#include "norm.h"

#define MM_GROUP_ACT_NONE 0
#define MM_GROUP_ACT_SILU 1
#define MM_GROUP_ACT_GELU 2
#define MM_GROUP_WG 1024   // workgroups of a backward kernel, at most (rows of partial sums of dw and db)

struct MMGroup {
  const int* offsets;   // [structs + 1]; null: structures of `each` rows
  long rows, each;
  int structs, C, G, cg;
  int gb, lpr, small;   // groups of a workgroup, lanes of a row (a power of two), rows that a workgroup holds
};

struct MMRange {
  long first;
  int n;
};

// rows of structure s (within the rows there are, whatever the offsets say)
__device__ __forceinline__ MMRange mm_group_range(const MMGroup& a, long s) {
  if (!a.offsets) return MMRange{s * a.each, (int)a.each};
  const long b = min(max((long)a.offsets[s], 0L), a.rows), e = min(max((long)a.offsets[s + 1], b), a.rows);
  return MMRange{b, (int)(e - b)};
}

// the last structure that begins at or before row r (0 if none does), found by a wave 64 offsets at a time
__device__ __forceinline__ int mm_group_find(const MMGroup& a, long r) {
  if (!a.offsets) return (int)(r / a.each);
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.structs;   // it lies in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const unsigned long long begun = __ballot(i < lo + n && a.offsets[min(i, a.structs)] <= r);
    const int k = begun ? 63 - __builtin_clzll(begun) : 0;
    n = min(step, lo + n - (lo + k * step));
    lo += k * step;
  }
  return lo;
}

// Distribution function of the normal distribution, given e = exp(-z^2 / 2): Hastings' approximation of erf (Abramowitz
// and Stegun 7.1.26), off by 0.75e-7 at most.  With it the activation shares its one exponential with the derivative; erff
// and expf bound the backward by their instructions.
__device__ __forceinline__ float mm_normal(float z, float e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
  const float p = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f),
                           0.254829592f);
  const float half = 0.5f * p * e;   // of the tail beyond |z|
  return z > 0.f ? 1.f - half : half;
}

template <int ACT>
__device__ __forceinline__ float mm_act(float z) {
  if constexpr (ACT == MM_GROUP_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if constexpr (ACT == MM_GROUP_ACT_GELU) return z * mm_normal(z, __expf(-0.5f * z * z));
  return z;
}

// derivative at z
template <int ACT>
__device__ __forceinline__ float mm_act_slope(float z) {
  if constexpr (ACT == MM_GROUP_ACT_SILU) {
    const float q = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return fmaf(z * q, 1.f - q, q);
  }
  if constexpr (ACT == MM_GROUP_ACT_GELU) {
    const float e = __expf(-0.5f * z * z);
    return fmaf(z * 0.39894228f, e, mm_normal(z, e));
  }
  return 1.f;
}

// This thread's place: channels c0 + c .. c0 + c + N of its block of groups, rows sub, sub + nsub, ...
template <typename T, int TPB>
struct MMGroupLane {
  static constexpr int N = MMVec<T>::N, VALS = TPB == 256 ? 64 : 32, NR = VALS / N;
  int g0, ng, c0, cw, c, sub, nsub, gi[N];
  float *red, *tot;   // LDS: [2][sets][lpr N] sums by channel, [2][gb] by group

  __device__ __forceinline__ MMGroupLane(const MMGroup& a, float* lds) {
    g0 = blockIdx.y * a.gb;
    ng = min(a.gb, a.G - g0);
    c0 = g0 * a.cg;
    cw = ng * a.cg;
    c = (threadIdx.x & (a.lpr - 1)) * N;
    sub = threadIdx.x / a.lpr;
    nsub = TPB / a.lpr;
#pragma unroll
    for (int i = 0; i < N; ++i) gi[i] = min((c + i) / a.cg, ng - 1);
    red = lds;
    tot = lds + 2 * (TPB / max(a.lpr, 64)) * a.lpr * N;
  }

  // out[k][i] = total of v[k] over the rows of all threads and the channels of the group of channel i; v: zero in
  // channels past the block.  Every thread of the workgroup comes here.
  template <int K>
  __device__ __forceinline__ void totals(const MMGroup& a, float (&v)[K][N], float (&out)[K][N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sets = TPB / max(a.lpr, 64), width = a.lpr * N;
    for (int d = a.lpr; d < 64; d <<= 1)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) v[k][i] += __shfl_xor(v[k][i], d);
    if (lane < a.lpr) {
      float* p = red + (threadIdx.x / max(a.lpr, 64)) * width + c;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) p[k * sets * width + i] = v[k][i];
    }
    __syncthreads();
    for (int g = wave; g < ng; g += TPB / 64)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float t = 0.f;
        for (int j = lane; j < a.cg; j += 64)
          for (int q = 0; q < sets; ++q) t += red[(k * sets + q) * width + g * a.cg + j];
        t = mm_lanes_sum<64>(t);
        if (lane == 0) tot[k * a.gb + g] = t;
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) out[k][i] = tot[k * a.gb + gi[i]];
  }
};

// v = the rows first + sub + j nsub < first + n of this thread's channels, zeros elsewhere (from the j on that no thread
// has, v is left alone: loops over j end there)
template <typename T, int TPB>
__device__ __forceinline__ void mm_group_load(const MMGroupLane<T, TPB>& l, const T* __restrict__ x, long ldx,
                                              long first, int n, float (&v)[MMGroupLane<T, TPB>::NR][MMVec<T>::N]) {
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    if (j * l.nsub >= n) break;
    const int r = l.sub + j * l.nsub;
    if (r < n && l.c < l.cw) {
      mm_load_vec(x + (first + r) * ldx + l.c0, l.c, l.cw, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[j][i] = 0.f;
    }
  }
}

// Mean and sum of squares about it of n <= small rows, by group; v becomes x - mean (0 outside).
template <typename T, int TPB>
__device__ __forceinline__ void mm_group_moments(const MMGroup& a, MMGroupLane<T, TPB>& l, int n,
                                                 float (&v)[MMGroupLane<T, TPB>::NR][MMVec<T>::N],
                                                 float (&mu)[1][MMVec<T>::N], float (&m2)[1][MMVec<T>::N]) {
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
  float t[1][N] = {};
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    if (j * l.nsub >= n) break;
#pragma unroll
    for (int i = 0; i < N; ++i) t[0][i] += v[j][i];
  }
  l.totals(a, t, mu);
  const float count = (float)n * (float)a.cg;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mu[0][i] /= count;   // divided: the mean of equal values is that value
    t[0][i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    if (j * l.nsub >= n) break;
    const bool on = l.sub + j * l.nsub < n;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[j][i] = on && l.c + i < l.cw ? v[j][i] - mu[0][i] : 0.f;
      t[0][i] = fmaf(v[j][i], v[j][i], t[0][i]);
    }
  }
  l.totals(a, t, m2);
}

// y or dx of the rows that belong to no structure: zeros
template <typename T, int TPB>
__device__ __forceinline__ void mm_group_outside(const MMGroup& a, const MMGroupLane<T, TPB>& l, T* __restrict__ y,
                                                 long ldy) {
  constexpr int N = MMVec<T>::N;
  if (!a.offsets || l.c >= l.cw) return;
  const long first = min(max((long)a.offsets[0], 0L), a.rows), last = min(max((long)a.offsets[a.structs], first), a.rows);
  const float zero[N] = {};
  for (long q = (long)blockIdx.x * l.nsub + l.sub; q < a.rows - (last - first); q += (long)gridDim.x * l.nsub)
    mm_store_vec(y + (q < first ? q : q + last - first) * ldy + l.c0, l.c, l.cw, zero);
}

template <typename T, int ACT, int TPB>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_whole_fwd_kernel(MMGroup a, const T* __restrict__ x, long ldx, const void* __restrict__ w,
                              const void* __restrict__ b, int p_f32, float eps, T* __restrict__ y, long ldy,
                              float* __restrict__ stats) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
  float wv[N], bv[N];
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long s = blockIdx.x; s < a.structs; s += gridDim.x) {
    const MMRange q = mm_group_range(a, s);
    if (q.n > a.small) continue;   // by tiles
    float v[NR][N], mu[1][N], m2[1][N];
    mm_group_load(l, x, ldx, q.first, q.n, v);
    if (q.n) {
      mm_group_moments(a, l, q.n, v, mu, m2);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) mu[0][i] = m2[0][i] = 0.f;
    }
    const float count = fmaxf((float)q.n * (float)a.cg, 1.f);
#pragma unroll
    for (int i = 0; i < N; ++i) m2[0][i] = 1.f / sqrtf(m2[0][i] / count + eps);
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      if (j * l.nsub >= q.n) break;
      const int r = l.sub + j * l.nsub;
      if (r < q.n && l.c < l.cw) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[j][i] = mm_act<ACT>(fmaf(v[j][i] * m2[0][i], wv[i], bv[i]));
        mm_store_vec(y + (q.first + r) * ldy + l.c0, l.c, l.cw, v[j]);
      }
    }
    if (stats && l.sub == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)   // the first channel of a group writes
        if (l.c + i < l.cw && (l.c + i) % a.cg == 0) {
          float* p = stats + (s * a.G + l.g0 + l.gi[i]) * 2;
          p[0] = mu[0][i];
          p[1] = m2[0][i];
        }
    }
  }
  mm_group_outside(a, l, y, ldy);
}

// The parts of tile `tile` that belong to structures of more than `small` rows: f(part, s, first row, rows).
template <typename F>
__device__ __forceinline__ void mm_group_tile(const MMGroup& a, long tile, F f) {
  const long r0 = tile * a.small, r1 = min(r0 + a.small, a.rows);
  int s = mm_group_find(a, r0);
  for (int part = 0; part < 2; ++part) {
    const MMRange q = mm_group_range(a, s);
    const long b = max(q.first, r0), e = min(q.first + q.n, r1);
    if (q.n > a.small && b < e) f(q.first > r0, s, b, (int)(e - b));
    if (e >= r1 || part) return;
    s = mm_group_find(a, r1 - 1);   // the structure of the tile's last row
    if (mm_group_range(a, s).first <= r0) return;
  }
}

// partial statistics: part [tiles][2][G][2]: mean and sum of squares about it
template <typename T, int TPB>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_stats_kernel(MMGroup a, const T* __restrict__ x, long ldx, long tiles, float* __restrict__ part) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int which, int s, long first, int n) {
      float v[NR][N], mu[1][N], m2[1][N];
      mm_group_load(l, x, ldx, first, n, v);
      mm_group_moments(a, l, n, v, mu, m2);
      if (l.sub == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (l.c + i < l.cw && (l.c + i) % a.cg == 0) {
            float* p = part + ((tile * 2 + which) * a.G + l.g0 + l.gi[i]) * 2;
            p[0] = mu[0][i];
            p[1] = m2[0][i];
          }
      }
    });
}

// One workgroup per structure of more than `small` rows, or per group of it where structures are few.  FWD: (mean, rstd) of the tiles' (mean, M2); else
// the sums of both numbers.
template <bool FWD>
__global__ void __launch_bounds__(256)
mm_groupnorm_join_kernel(MMGroup a, const float* __restrict__ part, float eps, float* __restrict__ out) {
  __shared__ float s0[4], s1[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto all = [&](float v, float* lds) {
    v = mm_lanes_sum<64>(v);
    if (lane == 0) lds[wave] = v;
    __syncthreads();
    v = lds[0] + lds[1] + lds[2] + lds[3];
    __syncthreads();
    return v;
  };
  for (long s = blockIdx.x; s < a.structs; s += gridDim.x) {
    const MMRange q = mm_group_range(a, s);
    if (q.n <= a.small) continue;
    const long t0 = q.first / a.small, t1 = (q.first + q.n - 1) / a.small;
    const long end = q.first + q.n;
    auto rows = [&](long t) {
      return (float)(int)(min((t + 1) * a.small, end) - max(t * (long)a.small, q.first));
    };
    for (int g = blockIdx.y; g < a.G; g += gridDim.y) {
      auto at = [&](long t) { return part + ((t * 2 + (t == t0 && q.first > t * a.small)) * a.G + g) * 2; };
      float u = 0.f, v = 0.f;
      for (long t = t0 + threadIdx.x; t <= t1; t += 256) {
        const float* p = at(t);
        u = FWD ? fmaf(p[0], rows(t), u) : u + p[0];
        v += p[1];
      }
      u = all(u, s0);
      v = all(v, s1);
      if constexpr (FWD) {
        const float mu = u / (float)q.n;
        u = mu;
        float d2 = 0.f;
        for (long t = t0 + threadIdx.x; t <= t1; t += 256) {
          const float d = at(t)[0] - mu;
          d2 = fmaf(d * d, rows(t), d2);
        }
        v = 1.f / sqrtf((v + all(d2, s0) * (float)a.cg) / ((float)q.n * (float)a.cg) + eps);
      }
      if (threadIdx.x == 0) {
        out[(s * a.G + g) * 2] = u;
        out[(s * a.G + g) * 2 + 1] = v;
      }
    }
  }
}

// y of the structures of more than `small` rows
template <typename T, int ACT, int TPB>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_fwd_kernel(MMGroup a, const T* __restrict__ x, long ldx, const void* __restrict__ w,
                             const void* __restrict__ b, int p_f32, T* __restrict__ y, long ldy, long tiles,
                             const float* __restrict__ stats) {
  MMGroupLane<T, TPB> l(a, nullptr);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N];
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int, int s, long first, int n) {
      if (l.c >= l.cw) return;   // here, as the whole wave looks for s
      float mu[N], rs[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float* p = stats + ((long)s * a.G + l.g0 + l.gi[i]) * 2;
        mu[i] = p[0];
        rs[i] = p[1];
      }
#pragma unroll 4
      for (int r = l.sub; r < n; r += l.nsub) {
        float v[N];
        mm_load_vec(x + (first + r) * ldx + l.c0, l.c, l.cw, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = mm_act<ACT>(fmaf((v[i] - mu[i]) * rs[i], wv[i], bv[i]));
        mm_store_vec(y + (first + r) * ldy + l.c0, l.c, l.cw, v);
      }
    });
}

// ------------------------------------------------------------------------------------------------ backward
// sums of dz h and dz of this thread's channels over the workgroup's rows, written as row `row` of part [2][rows][C]
template <typename T, int TPB>
__device__ __forceinline__ void mm_group_put(const MMGroup& a, const MMGroupLane<T, TPB>& l, float (&v)[2][MMVec<T>::N],
                                             float* __restrict__ part, long row, long rows) {
  constexpr int N = MMVec<T>::N;
  const int lane = threadIdx.x & 63, sets = TPB / max(a.lpr, 64), width = a.lpr * N;
  for (int d = a.lpr; d < 64; d <<= 1)
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) v[k][i] += __shfl_xor(v[k][i], d);
  __syncthreads();   // the last totals' sums are read
  if (lane < a.lpr) {
    float* p = l.red + (threadIdx.x / max(a.lpr, 64)) * width + l.c;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < N; ++i) p[k * sets * width + i] = v[k][i];
  }
  __syncthreads();
  for (int q = threadIdx.x; q < 2 * l.cw; q += TPB) {
    const int k = q >= l.cw, c = q - k * l.cw;
    float t = 0.f;
    for (int j = 0; j < sets; ++j) t += l.red[(k * sets + j) * width + c];
    part[(k * rows + row) * a.C + l.c0 + c] = t;
  }
}

// h (in place of x) and dz w (in place of dy), with the sums of dz h and dz by channel added to acc
template <typename T, int ACT, int TPB>
__device__ __forceinline__ void mm_group_slopes(const MMGroupLane<T, TPB>& l, int n, const float (&mu)[MMVec<T>::N],
                                                const float (&rs)[MMVec<T>::N], const float (&wv)[MMVec<T>::N],
                                                const float (&bv)[MMVec<T>::N],
                                                float (&x)[MMGroupLane<T, TPB>::NR][MMVec<T>::N],
                                                float (&dy)[MMGroupLane<T, TPB>::NR][MMVec<T>::N],
                                                float (&acc)[2][MMVec<T>::N], float (&sum)[2][MMVec<T>::N]) {
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
#pragma unroll
  for (int i = 0; i < N; ++i) sum[0][i] = sum[1][i] = 0.f;
#pragma unroll
  for (int j = 0; j < NR; ++j) {
    if (j * l.nsub >= n) break;
    if (l.sub + j * l.nsub >= n) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (l.c + i >= l.cw) continue;
      const float h = (x[j][i] - mu[i]) * rs[i], dz = dy[j][i] * mm_act_slope<ACT>(fmaf(h, wv[i], bv[i]));
      acc[0][i] = fmaf(dz, h, acc[0][i]);
      acc[1][i] += dz;
      x[j][i] = h;
      dy[j][i] = dz * wv[i];
      sum[0][i] += dy[j][i];
      sum[1][i] = fmaf(dy[j][i], h, sum[1][i]);
    }
  }
}

template <typename T, int ACT, int TPB>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_whole_bwd_kernel(MMGroup a, const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                              const void* __restrict__ w, const void* __restrict__ b, int p_f32,
                              const float* __restrict__ stats, T* __restrict__ dx, long lddx, float* __restrict__ part,
                              long part_rows) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
  float wv[N], bv[N], acc[2][N] = {};
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long s = blockIdx.x; s < a.structs; s += gridDim.x) {
    const MMRange q = mm_group_range(a, s);
    if (q.n > a.small || q.n == 0) continue;
    float h[NR][N], g[NR][N], mu[N], rs[N], sum[2][N], tot[2][N];
    mm_group_load(l, x, ldx, q.first, q.n, h);
    mm_group_load(l, dy, lddy, q.first, q.n, g);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float* p = stats + (s * a.G + l.g0 + l.gi[i]) * 2;
      mu[i] = p[0];
      rs[i] = p[1];
    }
    mm_group_slopes<T, ACT, TPB>(l, q.n, mu, rs, wv, bv, h, g, acc, sum);
    if (!dx) continue;
    l.totals(a, sum, tot);
    const float count = (float)q.n * (float)a.cg;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      tot[0][i] /= count;
      tot[1][i] /= count;
    }
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      if (j * l.nsub >= q.n) break;
      const int r = l.sub + j * l.nsub;
      if (r < q.n && l.c < l.cw) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[j][i] = rs[i] * (g[j][i] - tot[0][i] - h[j][i] * tot[1][i]);
        mm_store_vec(dx + (q.first + r) * lddx + l.c0, l.c, l.cw, g[j]);
      }
    }
  }
  if (dx) mm_group_outside(a, l, dx, lddx);
  if (part) mm_group_put(a, l, acc, part, blockIdx.x, part_rows);
}

// part [tiles][2][G][2]: sums of dz w and dz w h; wpart: as in the kernel above, rows from first_row on
template <typename T, int ACT, int TPB>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_sums_kernel(MMGroup a, const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                              const void* __restrict__ w, const void* __restrict__ b, int p_f32,
                              const float* __restrict__ stats, long tiles, float* __restrict__ part,
                              float* __restrict__ wpart, long first_row, long part_rows) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N, NR = MMGroupLane<T, TPB>::NR;
  float wv[N], bv[N], acc[2][N] = {};
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int which, int s, long first, int n) {
      float h[NR][N], g[NR][N], mu[N], rs[N], sum[2][N], tot[2][N];
      mm_group_load(l, x, ldx, first, n, h);
      mm_group_load(l, dy, lddy, first, n, g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float* p = stats + ((long)s * a.G + l.g0 + l.gi[i]) * 2;
        mu[i] = p[0];
        rs[i] = p[1];
      }
      mm_group_slopes<T, ACT, TPB>(l, n, mu, rs, wv, bv, h, g, acc, sum);
      if (!part) return;
      l.totals(a, sum, tot);
      if (l.sub == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (l.c + i < l.cw && (l.c + i) % a.cg == 0) {
            float* p = part + ((tile * 2 + which) * a.G + l.g0 + l.gi[i]) * 2;
            p[0] = tot[0][i];
            p[1] = tot[1][i];
          }
      }
    });
  if (wpart) mm_group_put(a, l, acc, wpart, first_row + blockIdx.x, part_rows);
}

// dx of the structures of more than `small` rows; sums [structs][G][2]
template <typename T, int ACT, int TPB>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_bwd_kernel(MMGroup a, const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                             const void* __restrict__ w, const void* __restrict__ b, int p_f32,
                             const float* __restrict__ stats, const float* __restrict__ sums, T* __restrict__ dx,
                             long lddx, long tiles) {
  MMGroupLane<T, TPB> l(a, nullptr);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N];
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int, int s, long first, int n) {
      if (l.c >= l.cw) return;   // here, as the whole wave looks for s
      float mu[N], rs[N], m0[N], m1[N];
      const float count = (float)mm_group_range(a, s).n * (float)a.cg;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const long at = ((long)s * a.G + l.g0 + l.gi[i]) * 2;
        mu[i] = stats[at];
        rs[i] = stats[at + 1];
        m0[i] = sums[at] / count;
        m1[i] = sums[at + 1] / count;
      }
#pragma unroll 4
      for (int r = l.sub; r < n; r += l.nsub) {
        float v[N], g[N];
        mm_load_vec(x + (first + r) * ldx + l.c0, l.c, l.cw, v);
        mm_load_vec(dy + (first + r) * lddy + l.c0, l.c, l.cw, g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float h = (v[i] - mu[i]) * rs[i], dz = g[i] * mm_act_slope<ACT>(fmaf(h, wv[i], bv[i]));
          g[i] = rs[i] * (fmaf(dz, wv[i], -m0[i]) - h * m1[i]);
        }
        mm_store_vec(dx + (first + r) * lddx + l.c0, l.c, l.cw, g);
      }
    });
}

// ------------------------------------------------------------------------------------------------ host
namespace {
struct Plan {
  MMGroup a;
  int tpb, blocks;     // threads of a workgroup, blocks of groups
  bool whole, tiles;   // which of the two ways may be needed
  long n_tiles;
  int wg_whole, wg_tiles;
  size_t lds;
};

// Channels of a workgroup: whole groups; as many as leave a workgroup's registers room for the rows of a structure (of
// structures with offsets eight times their mean), but no fewer than 64 bytes of a row.  Lanes of a row: the least
// power of two whose vectors hold them.
bool make_plan(const char* name, long rows, int structs, const int* offsets, int C, int G, int dtype, Plan* p) {
  const int N = dtype == MM_F32 ? 4 : 8, es = 16 / N, cg = C / G;
  if (cg > 1024 * N) {
    mm::set_error(std::string(name) + ": groups of more than 16384 bytes of channels are not supported");
    return false;
  }
  if (G > 65535) {
    mm::set_error(std::string(name) + ": more than 65535 groups are not supported");
    return false;
  }
  const long each = structs ? rows / structs : 0;
  const double want = offsets ? 8.0 * (double)rows / (structs ? structs : 1) : (double)each;
  int gb = 1;
  while (gb < G && gb < 256 && gb * 2 * cg <= 1024 * N) gb *= 2;
  if (gb > G) gb = G;
  auto lanes = [&](int g) {
    int l = 1;
    while (l * N < g * cg) l *= 2;
    return l;
  };
  auto threads = [](int l) { return l > 256 ? 1024 : 256; };
  auto held = [&](int l) { return (threads(l) == 256 ? 64 : 32) / N * (threads(l) / l); };
  int least = gb;
  while (least > 1 && held(lanes(least)) < want && (least + 1) / 2 * cg * es >= 64) least = (least + 1) / 2;
  if (offsets || held(lanes(least)) >= want) gb = least;   // else tiles: whole rows
  const int lpr = lanes(gb), tpb = threads(lpr);
  MMGroup& a = p->a;
  a = MMGroup{offsets, rows, each, structs, C, G, cg, gb, lpr, held(lpr)};
  p->tpb = tpb;
  p->blocks = (G + gb - 1) / gb;
  p->whole = offsets || each <= a.small;
  p->tiles = offsets ? rows > a.small : each > a.small;
  p->n_tiles = p->tiles ? (rows + a.small - 1) / a.small : 0;
  p->wg_whole = p->whole ? (int)(structs < MM_GROUP_WG ? (structs ? structs : 1) : MM_GROUP_WG) : 0;
  p->wg_tiles = (int)(p->n_tiles < MM_GROUP_WG ? p->n_tiles : MM_GROUP_WG);
  p->lds = ((size_t)2 * (tpb / (lpr > 64 ? lpr : 64)) * lpr * N + 2 * gb) * sizeof(float);
  return true;
}

dim3 join_grid(int structs, int groups) {
  return structs < 256 ? dim3(structs, groups) : dim3(structs < 4096 ? structs : 4096);
}

bool bad_sizes(long rows, int structs, const int* offsets, int C, int G) {
  return rows < 0 || structs < 0 || C <= 0 || G <= 0 || C % G || rows > 2147483647L - 65536 ||
         (!offsets && (structs ? rows % structs : rows)) || (offsets && structs == 0);
}
}  // namespace

#define MM_GROUP_DISPATCH(kernel, grid, lds, ...)                                                                     \
  MM_DISPATCH(dtype, {                                                                                                \
    auto go = [&](auto f) { hipLaunchKernelGGL(f, grid, dim3(p.tpb), lds, stream, __VA_ARGS__); };                    \
    if (p.tpb == 256) {                                                                                               \
      if (act == 0) go((kernel<T_, 0, 256>));                                                                         \
      else if (act == 1) go((kernel<T_, 1, 256>));                                                                    \
      else go((kernel<T_, 2, 256>));                                                                                  \
    } else {                                                                                                          \
      if (act == 0) go((kernel<T_, 0, 1024>));                                                                        \
      else if (act == 1) go((kernel<T_, 1, 1024>));                                                                   \
      else go((kernel<T_, 2, 1024>));                                                                                 \
    }                                                                                                                 \
  })

extern "C" int mm_groupnorm_workspace(long rows, int structs, int ragged, int C, int groups, int dtype, int backward,
                                      size_t* bytes) {
  static const int some = 0;
  const int* offsets = ragged ? &some : nullptr;   // not read
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16 && bytes, "bad dtype");
  MM_CHECK_ARG(!bad_sizes(rows, structs, offsets, C, groups), "bad sizes");
  Plan p;
  if (!make_plan("mm_groupnorm_workspace", rows, structs, offsets, C, groups, dtype, &p)) return MM_ERANGE;
  size_t n = (size_t)p.n_tiles * 4 * groups;
  if (backward) n += (p.n_tiles ? (size_t)structs * groups * 2 : 0) + (size_t)2 * (p.wg_whole + p.wg_tiles) * C;
  *bytes = n * sizeof(float);
  return MM_OK;
}

extern "C" int mm_groupnorm_fwd(const void* x, long ldx, int dtype, long rows, int structs, const int* offsets, int C,
                                int groups, const void* w, const void* b, int p_dtype, float eps, int act, void* y,
                                long ldy, float* stats, float* workspace, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(p_dtype == dtype || p_dtype == MM_F32, "weight and bias must have the type of x or float");
  MM_CHECK_ARG(!bad_sizes(rows, structs, offsets, C, groups) && ldx >= 0 && ldy >= C, "bad sizes");
  MM_CHECK_ARG(act >= 0 && act <= 2, "bad activation");
  Plan p;
  if (!make_plan("mm_groupnorm_fwd", rows, structs, offsets, C, groups, dtype, &p)) return MM_ERANGE;
  MM_CHECK_ARG(!p.tiles || (workspace && stats), "structures in tiles need the workspace and the statistics");
  if (structs == 0 || rows == 0) return MM_OK;
  if (p.whole) {
    MM_GROUP_DISPATCH(mm_groupnorm_whole_fwd_kernel, dim3(p.wg_whole, p.blocks), p.lds, p.a, (const T_*)x, ldx, w, b,
                      p_dtype == MM_F32, eps, (T_*)y, ldy, stats);
  }
  if (p.tiles) {
    const dim3 grid(p.wg_tiles, p.blocks);
    MM_DISPATCH(dtype, {
      auto go = [&](auto f) {
        hipLaunchKernelGGL(f, grid, dim3(p.tpb), p.lds, stream, p.a, (const T_*)x, ldx, p.n_tiles, workspace);
      };
      if (p.tpb == 256) go(mm_groupnorm_tile_stats_kernel<T_, 256>);
      else go(mm_groupnorm_tile_stats_kernel<T_, 1024>);
    });
    hipLaunchKernelGGL(mm_groupnorm_join_kernel<true>, join_grid(structs, groups), dim3(256), 0, stream,
                       p.a, workspace, eps, stats);
    MM_GROUP_DISPATCH(mm_groupnorm_tile_fwd_kernel, grid, 0, p.a, (const T_*)x, ldx, w, b, p_dtype == MM_F32, (T_*)y,
                      ldy, p.n_tiles, stats);
  }
  return mm::launch_status("mm_groupnorm_fwd");
}

extern "C" int mm_groupnorm_bwd(const void* dy, long lddy, const void* x, long ldx, int dtype, long rows, int structs,
                                const int* offsets, int C, int groups, const void* w, const void* b, int p_dtype,
                                int act, const float* stats, void* dx, long lddx, void* dw, void* db, float* workspace,
                                hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(p_dtype == dtype || p_dtype == MM_F32, "weight and bias must have the type of x or float");
  MM_CHECK_ARG(!bad_sizes(rows, structs, offsets, C, groups) && lddy >= 0 && ldx >= 0 && (!dx || lddx >= C), "bad sizes");
  MM_CHECK_ARG(act >= 0 && act <= 2, "bad activation");
  Plan p;
  if (!make_plan("mm_groupnorm_bwd", rows, structs, offsets, C, groups, dtype, &p)) return MM_ERANGE;
  const long part_rows = rows && structs ? p.wg_whole + p.wg_tiles : 0;
  MM_CHECK_ARG(workspace || part_rows == 0 || (!p.tiles && !dw && !db), "the workspace is needed");
  float* part = workspace;
  float* sums = part ? part + (size_t)p.n_tiles * 4 * groups : nullptr;
  float* wpart = part_rows && (dw || db) ? sums + (p.n_tiles ? (size_t)structs * groups * 2 : 0) : nullptr;
  if (part_rows && (dx || wpart)) {
    if (p.whole) {
      MM_GROUP_DISPATCH(mm_groupnorm_whole_bwd_kernel, dim3(p.wg_whole, p.blocks), p.lds, p.a, (const T_*)dy, lddy,
                        (const T_*)x, ldx, w, b, p_dtype == MM_F32, stats, (T_*)dx, lddx, wpart, part_rows);
    }
    if (p.tiles) {
      const dim3 grid(p.wg_tiles, p.blocks);
      MM_GROUP_DISPATCH(mm_groupnorm_tile_sums_kernel, grid, p.lds, p.a, (const T_*)dy, lddy, (const T_*)x, ldx, w, b,
                        p_dtype == MM_F32, stats, p.n_tiles, dx ? part : nullptr, wpart, (long)p.wg_whole, part_rows);
      if (dx) {
        hipLaunchKernelGGL(mm_groupnorm_join_kernel<false>, join_grid(structs, groups), dim3(256), 0,
                           stream, p.a, part, 0.f, sums);
        MM_GROUP_DISPATCH(mm_groupnorm_tile_bwd_kernel, grid, 0, p.a, (const T_*)dy, lddy, (const T_*)x, ldx, w, b,
                          p_dtype == MM_F32, stats, sums, (T_*)dx, lddx, p.n_tiles);
      }
    }
  }
  if (dw || db) mm::sum_partials(wpart, (int)part_rows, C, p_dtype, dw, db, stream);
  return mm::launch_status("mm_groupnorm_bwd");
}
