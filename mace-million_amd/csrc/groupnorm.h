// Group norm of rows of channels with an activation: what forward (groupnorm.hip) and backward (groupnorm_bwd.hip)
// share.  A structure is a run of rows, a group a run of cg = C / groups channels; over the n = rows x cg values of a
// (structure, group):
//     h = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  z = h w + b,  y = act(z)
//     dz = dy act'(z):  dw = sum_rows dz h,  db = sum_rows dz,  dx = rstd (dz w - mean(dz w) - h mean(dz w h))
// Bound by HBM (500,000 x 128 bfloat16 values in one structure, gelu: forward 115 us, backward 210, 3.1 TB/s; 4096
// ragged structures of 90,001 x 128 floats, silu, whole: 37 and 43 us, 2.5 and 3.2 TB/s).  A thread keeps one vector of
// 16 bytes of channels for several rows, and sums go by channel first (over a thread's rows, the lanes of a wave, the
// waves through LDS), then over the channels of a group: any group size works, whether or not it holds whole vectors.
//
// Two ways, by the number of rows of a structure, which the host need not know:
//   whole  a workgroup holds the structure (of its block of whole groups) in registers: every value is read once;
//   tiles  structures of more than `small` rows go in tiles of `small` rows: partial statistics of every tile, their
//          sum by structure, and a second reading.  Tiles lie at multiples of `small` rows, so a tile meets at most two
//          such structures: the one that holds its first row (part 0) and one that begins inside (part 1).
// Variances are about the mean (of a tile, joined as M2 + n (mean_i - mean)^2).  All sums are fp32 in a fixed order: no
// atomics, the same bits in every run.
#pragma once
#include "norm.h"

#include <type_traits>

#define MM_GROUP_ACT_NONE 0
#define MM_GROUP_ACT_SILU 1
#define MM_GROUP_ACT_GELU 2
#define MM_GROUP_WG 1024   // workgroups of a backward kernel, at most (rows of partial sums of dw and db)

struct MMGroup {
  const int* offsets;   // [structs + 1]; null: structures of `each` rows
  long rows, each;
  int structs, C, G, cg;
  int gb, lpr, small;   // groups of a workgroup, lanes of a row (a power of two), rows that a workgroup holds
  int lanes;            // of a group, where it is 2^n lanes of a wave, else 0
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

// Distribution function of the normal distribution, given e = exp(-z^2 / 2).  The tail beyond |z| is e R(|z|), where R is
// a polynomial in t = 1 / (1 + p |z|), fitted here for the least largest relative error over |z| <= 14 (with fp32's
// roundings 5.2 x 2^-24; with two terms less 20 x 2^-24, for 16-bit rows, which then round to 2^-11 at best): the tail
// keeps its digits however small it is.  With it the activation shares its one exponential with the derivative; erff
// and expf bound the backward by their instructions (500,000 x 128 bfloat16 values: 309 us with nine terms, 303 with
// seven).
template <typename T>
__device__ __forceinline__ float mm_normal(float z, float e) {
  constexpr bool FLOAT = sizeof(T) == 4;
  constexpr int TERMS = FLOAT ? 9 : 7;
  constexpr float p = FLOAT ? 0.35f : 0.36f;
  constexpr float nine[] = {0.139621407f, 0.139861852f, 0.119833007f, 0.105507337f, -0.0231080018f,
                            0.15917109f,  -0.255711198f, 0.143970042f, -0.0291455518f};
  constexpr float seven[] = {0.143713027f, 0.141772658f,  0.139718115f, 0.0265525803f,
                             0.180949137f, -0.179760993f, 0.0470551737f};
  const float t = __builtin_amdgcn_rcpf(fmaf(p, fabsf(z), 1.f));
  float r = 0.f;
#pragma unroll
  for (int i = TERMS - 1; i >= 0; --i) r = fmaf(r, t, FLOAT ? nine[i] : seven[i < 7 ? i : 0]);
  const float tail = r * t * e;
  return z > 0.f ? 1.f - tail : tail;
}

template <typename T, int ACT>
__device__ __forceinline__ float mm_act(float z) {
  if constexpr (ACT == MM_GROUP_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if constexpr (ACT == MM_GROUP_ACT_GELU) return z * mm_normal<T>(z, __expf(-0.5f * z * z));
  return z;
}

// derivative at z
template <typename T, int ACT>
__device__ __forceinline__ float mm_act_slope(float z) {
  if constexpr (ACT == MM_GROUP_ACT_SILU) {
    const float q = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return fmaf(z * q, 1.f - q, q);
  }
  if constexpr (ACT == MM_GROUP_ACT_GELU) {
    const float e = __expf(-0.5f * z * z);
    return fmaf(z * 0.39894228f, e, mm_normal<T>(z, e));
  }
  return 1.f;
}

// This thread's place: channels c0 + c .. c0 + c + N of its block of groups, rows sub, sub + nsub, ...  VALS: values of a
// thread that a workgroup holds.  FULL: blocks are whole vectors, so that loads need no branches.
template <typename T, int TPB, int VALS, bool FULL>
struct MMGroupLane {
  static constexpr int N = MMVec<T>::N, NR = VALS / N, THREADS = TPB;
  static constexpr int LEAST = TPB == 1024 || !FULL ? NR : 1;   // row counts with code of their own
  int g0, ng, c0, cw, c, sub, nsub, gi[N], turn;
  bool on;            // has channels
  float *red, *tot;   // LDS: [2][sets][lpr N] sums by channel, [2][gb] by group; or [2 turns][2][waves][lpr] by lane

  __device__ __forceinline__ MMGroupLane(const MMGroup& a, float* lds) {
    g0 = blockIdx.y * a.gb;
    ng = min(a.gb, a.G - g0);
    c0 = g0 * a.cg;
    cw = ng * a.cg;
    c = (threadIdx.x & (a.lpr - 1)) * N;
    sub = threadIdx.x / a.lpr;
    nsub = TPB / a.lpr;
    on = c < cw;
#pragma unroll
    for (int i = 0; i < N; ++i) gi[i] = min((c + i) / a.cg, ng - 1);
    red = lds;
    tot = lds + 2 * (TPB / max(a.lpr, 64)) * a.lpr * N;
    turn = 0;
  }

  // v = channels of row r, zeros where there are none (mask: and where it is false)
  __device__ __forceinline__ void load(const T* __restrict__ x, long ldx, long r, bool mask, float (&v)[N]) const {
    if constexpr (FULL) {
      mm_load_vec(x + r * ldx + c0 + (on ? c : 0), 0, N, v);
      mask &= on;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = mask ? v[i] : 0.f;
    } else {
      if (mask) {
        mm_load_vec(x + r * ldx + c0, c, cw, v);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
      }
    }
  }
  // of a row and a thread that are there
  __device__ __forceinline__ void get(const T* __restrict__ x, long ldx, long r, float (&v)[N]) const {
    if constexpr (FULL) mm_load_vec(x + r * ldx + c0 + c, 0, N, v);
    else mm_load_vec(x + r * ldx + c0, c, cw, v);
  }
  __device__ __forceinline__ void store(T* __restrict__ y, long ldy, long r, const float* v) const {
    if constexpr (FULL) mm_store_vec(y + r * ldy + c0 + c, 0, N, v);
    else mm_store_vec(y + r * ldy + c0, c, cw, v);
  }

  // out[k][i] = total of v[k] over the rows of all threads and the channels of the group of channel i; v: zero in
  // channels past the block.  Every thread of the workgroup comes here.
  template <int K>
  __device__ __forceinline__ void totals(const MMGroup& a, float (&v)[K][N], float (&out)[K][N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (a.lanes) {   // a group is 2^n lanes of a wave: by lane moves, then over the waves, in LDS used in turn
      float t[K];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        t[k] = v[k][0];
#pragma unroll
        for (int i = 1; i < N; ++i) t[k] += v[k][i];
      }
      for (int d = 1; d < a.lanes; d <<= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) t[k] += __shfl_xor(t[k], d);
      for (int d = a.lpr; d < 64; d <<= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) t[k] += __shfl_xor(t[k], d);
      float* p = red + turn * (2 * (TPB / 64) * a.lpr) + (lane & (a.lpr - 1));
      turn ^= 1;
      if (lane < a.lpr) {
#pragma unroll
        for (int k = 0; k < K; ++k) p[(k * (TPB / 64) + wave) * a.lpr] = t[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        t[k] = 0.f;
#pragma unroll
        for (int w = 0; w < TPB / 64; ++w) t[k] += p[(k * (TPB / 64) + w) * a.lpr];
#pragma unroll
        for (int i = 0; i < N; ++i) out[k][i] = t[k];
      }
      return;
    }
    const int sets = TPB / max(a.lpr, 64), width = a.lpr * N;
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

// f(std::integral_constant<int, R>) with the least of R = NR, NR / 2, .. LEAST whose R nsub rows hold n
template <int NR, int LEAST, typename F>
__device__ __forceinline__ void mm_group_rows(int n, int nsub, F f) {
  if constexpr (NR > LEAST) {
    if (n <= NR / 2 * nsub) {
      mm_group_rows<NR / 2, LEAST>(n, nsub, f);
      return;
    }
  }
  f(std::integral_constant<int, NR>{});
}

// v = the rows first + sub + j nsub < first + n of this thread's channels, zeros elsewhere; n > 0
template <int R, typename T, typename L>
__device__ __forceinline__ void mm_group_load(const L& l, const T* __restrict__ x, long ldx, long first, int n,
                                              float (&v)[R][MMVec<T>::N]) {
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int r = l.sub + j * l.nsub;
    l.load(x, ldx, first + min(r, n - 1), r < n, v[j]);
  }
}

// Mean and sum of squares about it of n rows, by group; v becomes x - mean (0 outside).
template <int R, int N, typename L>
__device__ __forceinline__ void mm_group_moments(const MMGroup& a, L& l, int n, float (&v)[R][N], float (&mu)[1][N],
                                                 float (&m2)[1][N]) {
  float t[1][N] = {};
#pragma unroll
  for (int j = 0; j < R; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) t[0][i] += v[j][i];
  l.totals(a, t, mu);
  const float count = (float)n * (float)a.cg;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mu[0][i] /= count;   // divided: the mean of equal values is that value
    t[0][i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const bool has = l.sub + j * l.nsub < n;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[j][i] = has && l.c + i < l.cw ? v[j][i] - mu[0][i] : 0.f;
      t[0][i] = fmaf(v[j][i], v[j][i], t[0][i]);
    }
  }
  l.totals(a, t, m2);
}

// two numbers of every group, from the threads of its first channel
template <int N, typename L>
__device__ __forceinline__ void mm_group_write(const MMGroup& a, const L& l, float* __restrict__ p, const float* u,
                                               const float* v) {
  if (l.sub) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (l.c + i < l.cw && (l.c + i) % a.cg == 0) {
      p[(l.g0 + l.gi[i]) * 2] = u[i];
      p[(l.g0 + l.gi[i]) * 2 + 1] = v[i];
    }
}

// y or dx of the rows that belong to no structure: zeros
template <typename T, typename L>
__device__ __forceinline__ void mm_group_outside(const MMGroup& a, const L& l, T* __restrict__ y, long ldy) {
  if (!a.offsets || !l.on) return;
  const long first = min(max((long)a.offsets[0], 0L), a.rows);
  const long last = min(max((long)a.offsets[a.structs], first), a.rows);
  const float zero[MMVec<T>::N] = {};
  for (long q = (long)blockIdx.x * l.nsub + l.sub; q < a.rows - (last - first); q += (long)gridDim.x * l.nsub)
    l.store(y, ldy, q < first ? q : q + last - first, zero);
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

// WAVES waves per structure of more than `small` rows (and group, where blockIdx.y counts them).  FWD: (mean, rstd) of
// the tiles' (mean, M2); else the sums of both numbers.
template <bool FWD, int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
mm_groupnorm_join_kernel(MMGroup a, const float* __restrict__ part, float eps, float* __restrict__ out) {
  constexpr int PER = WAVES == 1 ? 4 : 1;   // structures of a workgroup
  __shared__ float s0[WAVES], s1[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto all = [&](float v, float* lds) {
    v = mm_lanes_sum<64>(v);
    if constexpr (WAVES > 1) {
      if (lane == 0) lds[wave] = v;
      __syncthreads();
      v = lds[0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v += lds[w];
      __syncthreads();
    }
    return v;
  };
  const int first = WAVES > 1 ? threadIdx.x : lane;
  const long step = (long)gridDim.x * PER;
  for (long s = (long)blockIdx.x * PER + (PER > 1 ? wave : 0); s < a.structs; s += step) {
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
#pragma unroll 8
      for (long t = t0 + first; t <= t1; t += 64 * WAVES) {
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
#pragma unroll 8
        for (long t = t0 + first; t <= t1; t += 64 * WAVES) {
          const float d = at(t)[0] - mu;
          d2 = fmaf(d * d, rows(t), d2);
        }
        v = 1.f / sqrtf((v + all(d2, s0) * (float)a.cg) / ((float)q.n * (float)a.cg) + eps);
      }
      if (first == 0) {
        out[(s * a.G + g) * 2] = u;
        out[(s * a.G + g) * 2 + 1] = v;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
namespace {
struct Plan {
  MMGroup a;
  int tpb, tile_tpb, blocks;   // threads of a workgroup (in tiles), blocks of groups
  bool full;               // blocks are whole vectors
  bool whole, tiles;       // which of the two ways may be needed
  long n_tiles;
  int wg_whole, wg_tiles;
  size_t lds;
};

// Threads of a workgroup and values a thread.  Small structures by one wave: sums without barriers, and four times as
// many of them at once (4096 structures of 5 to 39 rows of 128 float values, forward 64 -> 36 us).  1024 threads hold
// large ones.
struct Shape { int tpb, vals; };
constexpr Shape kShapes[] = {{64, 64}, {256, 32}, {1024, 32}};

// Channels of a workgroup: whole groups, no fewer than 64 bytes of a row unless a group has fewer; as many as leave the
// registers of a workgroup room for the rows of a structure (of structures with offsets, five times their mean).
// Structures that none of the shapes holds go in tiles, with all channels.  Lanes of a row: the least power of two
// whose vectors hold its channels.
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
  const double want = offsets ? 5.0 * (double)rows / (structs ? structs : 1) : (double)each;
  int most = 1;
  while (most < G && most < 256 && most * 2 * cg <= 1024 * N) most *= 2;
  if (most > G) most = G;
  auto lanes = [&](int g) {
    int l = 1;
    while (l * N < g * cg) l *= 2;
    return l;
  };
  auto held = [&](const Shape& s, int l) { return s.vals / N * (s.tpb / l); };
  auto whole_vectors = [&](int g) { return g * cg % N == 0 && C % N == 0; };
  int gb = most;
  Shape sh = kShapes[lanes(most) > 256 ? 2 : 1];
  bool found = false;
  for (int i = 0; i < 3 && !found; ++i)
    for (int g = most;; g = (g + 1) / 2) {
      const int l = lanes(g);
      const bool waves = i > 0 || (whole_vectors(g) && (long)structs * ((G + g - 1) / g) >= 2048);
      if (l <= kShapes[i].tpb && waves && held(kShapes[i], l) >= want) {
        gb = g;
        sh = kShapes[i];
        found = true;
        break;
      }
      if (g == 1 || (g + 1) / 2 * cg * es < 64) break;
    }
  const int lpr = lanes(gb);
  const bool full = whole_vectors(gb);
  const int lanes_of = cg / N;   // of a group
  const bool by_lanes = cg % N == 0 && (lanes_of & (lanes_of - 1)) == 0 && lpr <= 64;
  MMGroup& a = p->a;
  a = MMGroup{offsets, rows, each, structs, C, G, cg, gb, lpr, held(sh, lpr), by_lanes ? lanes_of : 0};
  p->tpb = sh.tpb;
  p->tile_tpb = sh.tpb == 64 ? 256 : sh.tpb;   // its 32 values a thread hold the rows of 64 threads with 64
  p->full = full;
  p->blocks = (G + gb - 1) / gb;
  p->whole = offsets || each <= a.small;
  p->tiles = offsets ? rows > a.small : each > a.small;
  p->n_tiles = p->tiles ? (rows + a.small - 1) / a.small : 0;
  p->wg_whole = p->whole ? (int)(structs < MM_GROUP_WG ? (structs ? structs : 1) : MM_GROUP_WG) : 0;
  p->wg_tiles = (int)(p->n_tiles < MM_GROUP_WG ? p->n_tiles : MM_GROUP_WG);
  p->lds = ((size_t)2 * (p->tile_tpb / (lpr > 64 ? lpr : 64)) * lpr * N + 2 * gb) * sizeof(float);
  return true;
}

// a workgroup for each group of few structures, else a wave for each structure
template <bool FWD>
void join_tiles(const MMGroup& a, const float* part, float eps, float* out, hipStream_t stream) {
  if (a.structs < 256) {
    hipLaunchKernelGGL((mm_groupnorm_join_kernel<FWD, 16>), dim3(a.structs, a.G), dim3(1024), 0, stream, a, part, eps,
                       out);
  } else {
    const int n = a.structs / 4 + 1;
    hipLaunchKernelGGL((mm_groupnorm_join_kernel<FWD, 1>), dim3(n < 4096 ? n : 4096), dim3(256), 0, stream, a, part, eps,
                       out);
  }
}

bool bad_sizes(long rows, int structs, const int* offsets, int C, int G) {
  return rows < 0 || structs < 0 || C <= 0 || G <= 0 || C % G || rows > 2147483647L - 65536 ||
         (!offsets && (structs ? rows % structs : rows)) || (offsets && structs == 0);
}
}  // namespace

// launches of kernel<T, activation, threads, values, full> by `go`, for the plan p
#define MM_GROUP_SHAPES(tpb, kernel, ...)                                                                \
  do {                                                                                                   \
    if ((tpb) == 1024) {                                                                                 \
      if (p.full) go(kernel<__VA_ARGS__, 1024, 32, true>);                                               \
      else go(kernel<__VA_ARGS__, 1024, 32, false>);                                                     \
    } else {                                                                                             \
      if (p.full) go(kernel<__VA_ARGS__, 256, 32, true>);                                                \
      else go(kernel<__VA_ARGS__, 256, 32, false>);                                                      \
    }                                                                                                    \
  } while (0)
#define MM_GROUP_WAVES(tpb, kernel, ...)                                                                 \
  do {                                                                                                   \
    if ((tpb) == 64) go(kernel<__VA_ARGS__, 64, 64, true>);                                              \
    else MM_GROUP_SHAPES(tpb, kernel, __VA_ARGS__);                                                      \
  } while (0)
#define MM_GROUP_DISPATCH(SHAPES, tpb, kernel, grid, lds, ...)                                           \
  MM_DISPATCH(dtype, {                                                                                   \
    auto go = [&](auto f) { hipLaunchKernelGGL(f, grid, dim3(tpb), lds, stream, __VA_ARGS__); };         \
    if (act == 0) SHAPES(tpb, kernel, T_, 0);                                                            \
    else if (act == 1) SHAPES(tpb, kernel, T_, 1);                                                       \
    else SHAPES(tpb, kernel, T_, 2);                                                                     \
  })
