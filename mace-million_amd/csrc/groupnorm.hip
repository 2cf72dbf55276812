// Group norm with an activation, forward: see groupnorm.h.
#include "groupnorm.h"

template <typename T, int ACT, int TPB, int VALS, bool FULL>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_whole_fwd_kernel(MMGroup a, const T* __restrict__ x, long ldx, const void* __restrict__ w,
                              const void* __restrict__ b, int p_f32, float eps, T* __restrict__ y, long ldy,
                              float* __restrict__ stats) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB, VALS, FULL> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N];
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long s = blockIdx.x; s < a.structs; s += gridDim.x) {
    const MMRange q = mm_group_range(a, s);
    if (q.n > a.small) continue;   // by tiles
    float mu[1][N] = {}, rs[1][N] = {};
    if (q.n) {
      mm_group_rows<VALS / N, MMGroupLane<T, TPB, VALS, FULL>::LEAST>(q.n, l.nsub, [&](auto rows) {
        constexpr int R = decltype(rows)::value;
        float v[R][N];
        mm_group_load<R>(l, x, ldx, q.first, q.n, v);
        mm_group_moments(a, l, q.n, v, mu, rs);
        const float count = (float)q.n * (float)a.cg;
#pragma unroll
        for (int i = 0; i < N; ++i) rs[0][i] = 1.f / sqrtf(rs[0][i] / count + eps);
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const int r = l.sub + j * l.nsub;
#pragma unroll
          for (int i = 0; i < N; ++i) v[j][i] = mm_act<T, ACT>(fmaf(v[j][i] * rs[0][i], wv[i], bv[i]));
          if (r < q.n && l.on) l.store(y, ldy, q.first + r, v[j]);
        }
      });
    }
    if (stats) mm_group_write<N>(a, l, stats + s * a.G * 2, mu[0], rs[0]);
  }
  mm_group_outside(a, l, y, ldy);
}

// partial statistics: part [tiles][2][G][2]: mean and sum of squares about it
template <typename T, int TPB, int VALS, bool FULL>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_stats_kernel(MMGroup a, const T* __restrict__ x, long ldx, long tiles, float* __restrict__ part) {
  extern __shared__ float mm_group_lds[];
  MMGroupLane<T, TPB, VALS, FULL> l(a, mm_group_lds);
  constexpr int N = MMVec<T>::N;
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int which, int, long first, int n) {
      float v[VALS / N][N], mu[1][N], m2[1][N];
      mm_group_load<VALS / N>(l, x, ldx, first, n, v);
      mm_group_moments(a, l, n, v, mu, m2);
      mm_group_write<N>(a, l, part + (tile * 2 + which) * a.G * 2, mu[0], m2[0]);
    });
}

// y of the structures of more than `small` rows
template <typename T, int ACT, int TPB, int VALS, bool FULL>
__global__ void __launch_bounds__(TPB)
mm_groupnorm_tile_fwd_kernel(MMGroup a, const T* __restrict__ x, long ldx, const void* __restrict__ w,
                             const void* __restrict__ b, int p_f32, T* __restrict__ y, long ldy, long tiles,
                             const float* __restrict__ stats) {
  MMGroupLane<T, TPB, VALS, FULL> l(a, nullptr);
  constexpr int N = MMVec<T>::N;
  float wv[N], bv[N];
  mm_norm_param<T>(w, p_f32, 1.f, l.c0 + l.c, l.c0 + l.cw, wv);
  mm_norm_param<T>(b, p_f32, 0.f, l.c0 + l.c, l.c0 + l.cw, bv);
  for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x)
    mm_group_tile(a, tile, [&](int, int s, long first, int n) {
      if (!l.on) return;   // here, as the whole wave looks for s
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
        l.get(x, ldx, first + r, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = mm_act<T, ACT>(fmaf((v[i] - mu[i]) * rs[i], wv[i], bv[i]));
        l.store(y, ldy, first + r, v);
      }
    });
}

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
    const dim3 grid(structs < 8192 ? structs : 8192, p.blocks);
    MM_GROUP_DISPATCH(MM_GROUP_WAVES, p.tpb, mm_groupnorm_whole_fwd_kernel, grid, p.lds, p.a, (const T_*)x, ldx, w, b,
                      p_dtype == MM_F32, eps, (T_*)y, ldy, stats);
  }
  if (p.tiles) {
    const dim3 grid(p.wg_tiles, p.blocks);
    MM_DISPATCH(dtype, {
      auto go = [&](auto f) {
        hipLaunchKernelGGL(f, grid, dim3(p.tile_tpb), p.lds, stream, p.a, (const T_*)x, ldx, p.n_tiles, workspace);
      };
      MM_GROUP_SHAPES(p.tile_tpb, mm_groupnorm_tile_stats_kernel, T_);
    });
    join_tiles<true>(p.a, workspace, eps, stats, stream);
    MM_GROUP_DISPATCH(MM_GROUP_SHAPES, p.tile_tpb, mm_groupnorm_tile_fwd_kernel, grid, 0, p.a, (const T_*)x, ldx, w, b,
                      p_dtype == MM_F32, (T_*)y,
                      ldy, p.n_tiles, stats);
  }
  return mm::launch_status("mm_groupnorm_fwd");
}

