// Group norm with an activation, backward: see groupnorm.h.
#include "groupnorm.h"

// ------------------------------------------------------------------------------------------------ backward
// sums of dz h and dz of this thread's channels over the workgroup's rows, written as row `row` of part [2][rows][C]
template <int N, typename L>
__device__ __forceinline__ void mm_group_put(const MMGroup& a, const L& l, float (&v)[2][N], float* __restrict__ part,
                                             long row, long rows) {
  constexpr int TPB = L::THREADS;
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

template <typename T, int ACT, int TPB, int VALS, bool FULL>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_whole_bwd_kernel(MMGroup a, const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                              const void* __restrict__ w, const void* __restrict__ b, int p_f32,
                              const float* __restrict__ stats, T* __restrict__ dx, long lddx, float* __restrict__ part,
                              long part_rows) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB, VALS, FULL> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N], acc[2][N] = {};
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long s = blockIdx.x; s < a.structs; s += gridDim.x) {
    const MMRange q = mm_group_range(a, s);
    if (q.n > a.small || q.n == 0) continue;
    mm_group_rows<VALS / N, MMGroupLane<T, TPB, VALS, FULL>::LEAST>(q.n, l.nsub, [&](auto rows) {
      constexpr int R = decltype(rows)::value;
      float h[R][N], g[R][N], mu[N], rs[N], sum[2][N] = {}, tot[2][N];
      mm_group_load<R>(l, x, ldx, q.first, q.n, h);
      mm_group_load<R>(l, dy, lddy, q.first, q.n, g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float* p = stats + (s * a.G + l.g0 + l.gi[i]) * 2;
        mu[i] = p[0];
        rs[i] = p[1];
      }
#pragma unroll
      for (int j = 0; j < R; ++j) {
        // dy is 0 in rows and channels that are not there (h there is finite: x = 0)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          h[j][i] = (h[j][i] - mu[i]) * rs[i];
          const bool has = l.sub + j * l.nsub < q.n;
          const float dz = has ? g[j][i] * mm_act_slope<T, ACT>(fmaf(h[j][i], wv[i], bv[i])) : 0.f;
          sum[1][i] = has ? fmaf(dz, h[j][i], sum[1][i]) : sum[1][i];
          sum[0][i] += dz;
          g[j][i] = dz;
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[0][i] += sum[1][i];
        acc[1][i] += sum[0][i];
        sum[0][i] = l.c + i < l.cw ? sum[0][i] * wv[i] : 0.f;
        sum[1][i] = l.c + i < l.cw ? sum[1][i] * wv[i] : 0.f;
      }
      if (!dx) return;
      l.totals(a, sum, tot);
      const float by = 1.f / ((float)q.n * (float)a.cg);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        tot[0][i] *= by;
        tot[1][i] *= by;
      }
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int r = l.sub + j * l.nsub;
#pragma unroll
        for (int i = 0; i < N; ++i) g[j][i] = rs[i] * (fmaf(g[j][i], wv[i], -tot[0][i]) - h[j][i] * tot[1][i]);
        if (r < q.n && l.on) l.store(dx, lddx, q.first + r, g[j]);
      }
    });
  }
  if (dx) mm_group_outside(a, l, dx, lddx);
  if (part) mm_group_put<N>(a, l, acc, part, blockIdx.x, part_rows);
}

// part [tiles][2][G][2]: sums of dz w and dz w h; wpart: as in the kernel above, rows from first_row on
template <typename T, int ACT, int TPB, int VALS, bool FULL>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_sums_kernel(MMGroup a, const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                              const void* __restrict__ w, const void* __restrict__ b, int p_f32,
                              const float* __restrict__ stats, long tiles, float* __restrict__ part,
                              float* __restrict__ wpart, long first_row, long part_rows) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB, VALS, FULL> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N], acc[2][N] = {};
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int which, int s, long first, int n) {
      float mu[N], rs[N], sum[2][N] = {}, tot[2][N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float* p = stats + ((long)s * a.G + l.g0 + l.gi[i]) * 2;
        mu[i] = p[0];
        rs[i] = p[1];
      }
      if (l.on) {
#pragma unroll 4
        for (int r = l.sub; r < n; r += l.nsub) {
          float h[N], g[N];
          l.get(x, ldx, first + r, h);
          l.get(dy, lddy, first + r, g);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            h[i] = (h[i] - mu[i]) * rs[i];
            const float dz = g[i] * mm_act_slope<T, ACT>(fmaf(h[i], wv[i], bv[i]));
            sum[0][i] += dz;
            sum[1][i] = fmaf(dz, h[i], sum[1][i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[0][i] += sum[1][i];
        acc[1][i] += sum[0][i];
        sum[0][i] = l.c + i < l.cw ? sum[0][i] * wv[i] : 0.f;
        sum[1][i] = l.c + i < l.cw ? sum[1][i] * wv[i] : 0.f;
      }
      if (!part) return;
      l.totals(a, sum, tot);
      mm_group_write<N>(a, l, part + (tile * 2 + which) * a.G * 2, tot[0], tot[1]);
    });
  if (wpart) mm_group_put<N>(a, l, acc, wpart, first_row + blockIdx.x, part_rows);
}

// dx of the structures of more than `small` rows; sums [structs][G][2]
template <typename T, int ACT, int TPB, int VALS, bool FULL>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_bwd_kernel(MMGroup a, const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                             const void* __restrict__ w, const void* __restrict__ b, int p_f32,
                             const float* __restrict__ stats, const float* __restrict__ sums, T* __restrict__ dx,
                             long lddx, long tiles) {
  MMGroupLane<T, TPB, VALS, FULL> l(a, nullptr);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N];
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int, int s, long first, int n) {
      if (!l.on) return;   // here, as the whole wave looks for s
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
        l.get(x, ldx, first + r, v);
        l.get(dy, lddy, first + r, g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float h = (v[i] - mu[i]) * rs[i], dz = g[i] * mm_act_slope<T, ACT>(fmaf(h, wv[i], bv[i]));
          g[i] = rs[i] * (fmaf(dz, wv[i], -m0[i]) - h * m1[i]);
        }
        l.store(dx, lddx, first + r, g);
      }
    });
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
      MM_GROUP_DISPATCH(MM_GROUP_WAVES, p.tpb, mm_groupnorm_whole_bwd_kernel, dim3(p.wg_whole, p.blocks), p.lds, p.a,
                        (const T_*)dy, lddy, (const T_*)x, ldx, w, b, p_dtype == MM_F32, stats, (T_*)dx, lddx, wpart,
                         part_rows);
    }
    if (p.tiles) {
      const dim3 grid(p.wg_tiles, p.blocks);
      MM_GROUP_DISPATCH(MM_GROUP_SHAPES, p.tile_tpb, mm_groupnorm_tile_sums_kernel, grid, p.lds, p.a, (const T_*)dy, lddy,
                        (const T_*)x, ldx, w, b, p_dtype == MM_F32, stats, p.n_tiles, dx ? part : nullptr, wpart,
                        (long)p.wg_whole, part_rows);
      if (dx) {
        join_tiles<false>(p.a, part, 0.f, sums, stream);
        MM_GROUP_DISPATCH(MM_GROUP_SHAPES, p.tile_tpb, mm_groupnorm_tile_bwd_kernel, grid, 0, p.a, (const T_*)dy, lddy,
                          (const T_*)x, ldx, w, b, p_dtype == MM_F32, stats, sums, (T_*)dx, lddx, p.n_tiles);
      }
    }
  }
  if (dw || db) mm::sum_partials(wpart, (int)part_rows, C, p_dtype, dw, db, stream);
  return mm::launch_status("mm_groupnorm_bwd");
}
