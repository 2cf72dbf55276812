// Cross entropy of linear logits, without keeping them:
//     l[t, v] = x[t] . W[v],  top[t] = max_v l[t, v],  rest[t] = sum over v != y[t] of exp(l[t, v] - top[t])
//     s[t] = rest[t] + exp(l[t, y[t]] - top[t]),  loss[t] = top[t] - l[t, y[t]] + log s[t]
//     d[t, v] = exp(l[t, v] - top[t]) / s[t] - [v = y[t]]:  dx[t] = g[t] d[t] W,  dW = sum_t g[t] d[t]^T x[t]
// A row that is certain of its class has s = 1 + rest with a small rest: rounding s would leave 2^-24 of 1 in the loss
// and in d, whatever their size (1.5e-5 of a loss of 0.004).  So the sums leave the target out, and where it is the
// largest logit, loss = log1p(rest) and its d = -rest / (1 + rest), both as near as the exponentials.
// top and s (or rest) are kept, not log sum exp: its rounding (2^-24 of it) would be a relative error of a whole row of
// probabilities.  For the same reason backward takes the logits again in the forward's order of sums: few rows by the
// kernel for few rows, more by tiles.
// Rows whose target is ignored are taken out at the start: `list` has the asked rows in their order, and everything
// runs over their number, which stays on the GPU.  (8192 rows, 131,072 classes of 2048 bfloat16 values, both
// gradients: 16.5 ms, 800 TFLOP/s of the 13.2 T operations.  14,700 rows, 89 classes of 128 float values: 97 us,
// launches and the six products of small tiles.)
// Forward: tiles of logits in registers, of which every row's maximum, sum of exponentials and target's logit go out.
// Backward: pieces of the vocabulary; the logits of a piece are taken again and become d, stored in 16 bits by rows
// and transposed, and two products give the piece's part of dx (kept in fp32 over the pieces) and its rows of dW.
// Bound by the matrix cores: 2 T D V operations forward, 6 T D V backward.
//
// Operands (nt.h): 16-bit types as they are; float as three bfloat16 planes (six products, fp32 accuracy).  d is rounded
// to the type (relative error 2^-8 in bfloat16, 2^-11 in float16, of each of the many terms of dx and dW, as the
// operands themselves are); in float16 it is scaled by 2^14 first, so that probabilities down to 2^-28 keep all their
// bits and none above 2^-39 vanishes.  The incoming gradient g stays out of d in dx (applied in fp32 at the end) and
// enters the transposed d as g / max|g|.  All sums are fp32 and in a fixed order.
#include "nt.h"

#define MM_CE_SUM 1
#define MM_CE_MEAN 2

namespace {
// int buffer of a call: [0] number of asked rows, then list [T], y [T] (of the asked rows), pos [T] (-1: ignored)
struct Rows {
  int *count, *list, *y, *pos;
};
Rows rows_of(int* buf, long T) { return Rows{buf, buf + 4, buf + 4 + T, buf + 4 + 2 * T}; }
}  // namespace

// SCAN: rows of a thread, t0 + 1024 i.  16 where one workgroup lists them all, else 4 (98,304 rows, count and list: 16 ->
// 9 us) up to 4 million rows (each workgroup sums the numbers of those before it).

template <typename Y>
__device__ __forceinline__ int mm_ce_asked(const Y* __restrict__ y, long t, long T, long ignore) {
  return t < T && (long)y[t] != ignore;
}

// asked rows of every 1024 x SCAN
template <typename Y, int SCAN>
__global__ void __launch_bounds__(1024) mm_ce_count_kernel(const Y* __restrict__ y, long T, long ignore,
                                                           int* __restrict__ counts) {
  __shared__ int s[16];
  const long t0 = (long)blockIdx.x * 1024 * SCAN + threadIdx.x;
  int n = 0;
#pragma unroll
  for (int i = 0; i < SCAN; ++i) n += mm_ce_asked(y, t0 + 1024 * i, T, ignore);
#pragma unroll
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) n += s[w];
  counts[blockIdx.x] = n;
}

// list, y, pos and the count; loss (nullable): 0 for ignored rows.  A target outside [0, V) becomes -1.  Rows are taken
// 64 at a time by a wave, so that loads and stores are contiguous; the numbers of the SCAN x 16 runs of 64 are summed by
// one wave.  (16 rows in a row for each thread: 25 us instead of 5 for 8192 rows.)
template <typename Y, int SCAN>
__global__ void __launch_bounds__(1024) mm_ce_list_kernel(const Y* __restrict__ y, long T, int V, long ignore,
                                                          const int* __restrict__ counts, int* __restrict__ count,
                                                          int* __restrict__ list, int* __restrict__ yc,
                                                          int* __restrict__ pos, float* __restrict__ loss) {
  __shared__ int s[SCAN * 16], s_all;
  const long t0 = (long)blockIdx.x * 1024 * SCAN + threadIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long v[SCAN];
  int at[SCAN];
#pragma unroll
  for (int i = 0; i < SCAN; ++i) v[i] = t0 + 1024 * i < T ? (long)y[t0 + 1024 * i] : ignore;
#pragma unroll
  for (int i = 0; i < SCAN; ++i) {
    const unsigned long long asked = __ballot(v[i] != ignore);
    at[i] = __popcll(asked & ((1ull << lane) - 1));
    if (lane == 0) s[16 * i + wave] = __popcll(asked);
  }
  __syncthreads();
  if (wave == 0) {
    int before = 0;
    for (int b = lane; b < (int)blockIdx.x; b += 64) before += counts[b];
#pragma unroll
    for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d);
    constexpr int EACH = SCAN / 4;   // of a lane
    int c[EACH], sum = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) sum += c[i] = s[EACH * lane + i];
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    int first = before + inc - sum;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      s[EACH * lane + i] = first;
      first += c[i];
    }
    if (lane == 63) s_all = first;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SCAN; ++i) {
    const long t = t0 + 1024 * i;
    if (t >= T) break;
    if (v[i] != ignore) {
      const int k = s[16 * i + wave] + at[i];
      list[k] = (int)t;
      yc[k] = v[i] >= 0 && v[i] < V ? (int)v[i] : -1;
      pos[t] = k;
    } else {
      pos[t] = -1;
      if (loss) loss[t] = 0.f;
    }
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *count = s_all;
}

// ------------------------------------------------------------------------------------------------ operands
// Values of T as planes of H: three for float, one otherwise.
template <typename T>
struct MMCeType {
  typedef T H;
  static constexpr int P = 1, PLANES = 1;
};
template <>
struct MMCeType<float> {
  typedef __bf16 H;
  static constexpr int P = 6, PLANES = 3;
};

template <typename T>
__device__ __forceinline__ void mm_ce_put4(typename MMCeType<T>::H* __restrict__ p, long plane, const float* v) {
  typedef typename MMCeType<T>::H H;
  typedef H vec __attribute__((ext_vector_type(4)));
  float r[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int q = 0; q < MMCeType<T>::PLANES; ++q) {
    vec h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = (H)r[i];
      r[i] -= (float)h[i];
    }
    *(vec*)(p + q * plane) = h;
  }
}

struct MMPack {
  const void* src;          // [.., cols], rows ld apart
  const int *list, *count;  // rows list[0 .. *count) of src, or (null) rows row0 .. row0 + rows
  void *out, *outT;         // planes [rows, ldo] and [cols, ldt], each nullable; zeros past the last column (row)
  long ld, row0, ldo, ldt, plane, planeT;
  int rows, cols, blocks_r, blocks_c;   // blocks of 64 x 64
};

// rows of out [rows][N] that belong to no asked row: zeros
struct MMZero {
  const int* pos;
  void* out;
  long rows;
  int N, blocks;
};

// Two operands and the zeros in one launch, 64 x 64 values a workgroup.
template <typename T>
__global__ void __launch_bounds__(256) mm_ce_pack_kernel(MMPack first, MMPack second, MMZero z) {
  typedef typename MMCeType<T>::H H;
  __shared__ float s[64][65];
  const int one = first.blocks_r * first.blocks_c, two = second.blocks_r * second.blocks_c;
  int b = blockIdx.x;
  if (b >= one + two) {
    const int nv = (z.N + 3) / 4;
    const float none[4] = {};
    for (long i = (long)(b - one - two) * 256 + threadIdx.x; i < z.rows * nv; i += (long)z.blocks * 256) {
      const long row = i / nv;
      if (z.pos[row] < 0) mm_store4((T*)z.out + row * z.N, (int)(i - row * nv) * 4, z.N, none);
    }
    return;
  }
  const bool is_first = b < one;
  const MMPack& a = is_first ? first : second;
  if (!is_first) b -= one;
  const int rows = a.count ? *a.count : a.rows, r0 = b % a.blocks_r * 64, c0 = b / a.blocks_r * 64;
  if (r0 >= mm_up(rows, 64)) return;
  const int q = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = q + 16 * k;
    float v[4] = {};
    if (r0 + r < rows) {
      const long at = a.list ? a.list[r0 + r] : a.row0 + r0 + r;
      mm_load4((const T*)a.src + at * a.ld, c0 + c, a.cols, v);
      if (a.out) mm_ce_put4<T>((H*)a.out + (long)(r0 + r) * a.ldo + c0 + c, a.plane, v);
    }
    if (a.outT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[r][c + i] = v[i];
    }
  }
  if (!a.outT) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int col = q + 16 * k;
    if (c0 + col >= a.cols) continue;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = s[c + i][col];
    mm_ce_put4<T>((H*)a.outT + (long)(c0 + col) * a.ldt + r0 + c, a.planeT, v);
  }
}

// ------------------------------------------------------------------------------------------------ logits
struct MMCeRow {
  float top, sum;   // sum of exp(l - top) over the classes other than the target
};

__device__ __forceinline__ MMCeRow mm_ce_join(MMCeRow a, MMCeRow b) {
  const float top = fmaxf(a.top, b.top);   // drops a NaN, which has to reach the sum
  if (a.top == -INFINITY && b.top == -INFINITY) return MMCeRow{top, a.sum + b.sum};   // nothing yet, or -inf alone
  return MMCeRow{top, a.sum * __expf(a.top - top) + b.sum * __expf(b.top - top)};
}

// Loss of a row whose target's logit is `picked` (bad: target out of range), and what the backward keeps of its sums:
// s, or -rest where the target is the largest logit (-0 at least: the sign tells the two).
__device__ __forceinline__ float mm_ce_loss(const MMCeRow& r, float picked, bool bad, float* keep) {
  if (bad) {
    *keep = r.sum;
    return __builtin_nanf("");
  }
  const float gap = r.top - picked;
  if (gap == 0.f) {
    *keep = -r.sum;
    return log1pf(r.sum);
  }
  const float s = r.sum + __expf(-gap);   // NaN where logits are infinite
  *keep = s;
  return gap + logf(s);
}

// d of a row from what is kept: exp(l - top) inv, at the target times `by` plus `add`
struct MMCeD {
  float inv, by, add;
  __device__ __forceinline__ explicit MMCeD(float keep) {
    const bool sure = __builtin_signbitf(keep);
    inv = 1.f / (sure ? 1.f - keep : keep);
    by = sure ? 0.f : 1.f;
    add = sure ? keep * inv : -1.f;
  }
  __device__ __forceinline__ float operator()(float l, float top, bool target) const {
    const float p = __expf(l - top) * inv;
    return target ? fmaf(p, by, add) : p;
  }
};

// The incoming gradient: of every row's loss (g of the asked rows and the largest finite |g|), or (g null) of their sum
// or mean, dloss [1].
struct MMCeScale {
  const float *g, *gmax, *dloss;
  int mean;
  // what dW is multiplied by, a row's share of it, and a row's own
  __device__ __forceinline__ float whole(int count) const {
    return g ? *gmax : dloss[0] / (mean ? (float)max(count, 1) : 1.f);
  }
  __device__ __forceinline__ float share(int at) const { return !g ? 1.f : *gmax > 0.f ? g[at] / *gmax : g[at]; }
  __device__ __forceinline__ float row(int at, int count) const { return g ? g[at] : whole(count); }
};

template <typename H>
struct MMCeLogits {
  MMNtOperand<H> x, w;
  const int *count, *y;
  int V, K;              // K: stages
  // forward
  float *part, *picked;  // [tiles of columns][T][2], [T]
  long T;
  // backward: columns v0 .. v0 + n
  const float* stats;            // [2][T]: top, s or -rest
  MMCeScale by;
  H *d, *dT;                     // [T][ldd], [n][ldt] (planes)
  long ldd, ldt, plane, planeT;
  int v0, n;
  float scale;
};

// 8192 rows, 131,072 classes of 2048 bfloat16 values: 4.24 ms, 1040 TFLOP/s; the matrix cores are busy 0.56 of it.
template <typename T, typename Nt>
__global__ void __launch_bounds__(Nt::TH, Nt::PER_CU)
mm_ce_logits_kernel(MMCeLogits<typename MMCeType<T>::H> a, int tiles_n) {
  typedef typename MMCeType<T>::H H;
  constexpr int BM = Nt::BM, BN = Nt::BN;
  extern __shared__ uint4 mm_ce_lds[];
  const int count = *a.count;
  int e, tm, tn;
  if (!mm_nt_tile(blockIdx.x, 1, (count + BM - 1) / BM, tiles_n, &e, &tm, &tn)) return;
  const int m0 = tm * BM, n0 = tn * BN;
  MMNtOperand<H> x = a.x;
  x.rows = count;
  Nt t;
  t.run(x, m0, a.w, n0, 0, a.K, mm_ce_lds);
  MMCeRow* s = (MMCeRow*)mm_ce_lds;   // [WN][BM]
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j) {
    const int m = m0 + t.row(j), y = a.y[min(m, count - 1)];
    MMCeRow r{-INFINITY, 0.f};
    float hit = 0.f;
    bool has = false;
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + t.col(i) + q;
        if (n < a.V) r.top = fmaxf(r.top, t.acc[i][j][q]);
        if (n == y) {
          hit = t.acc[i][j][q];
          has = true;
          t.acc[i][j][q] = -INFINITY;   // stays out of the sum
        }
      }
    if (has && m < count) a.picked[m] = hit;
    const float top = r.top == -INFINITY ? 0.f : r.top;
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (n0 + t.col(i) + q < a.V) r.sum += __expf(t.acc[i][j][q] - top);
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) r = mm_ce_join(r, MMCeRow{__shfl_xor(r.top, d), __shfl_xor(r.sum, d)});
    if (t.lane < 16) s[(threadIdx.x >> 6) / Nt::WM * BM + t.row(j)] = r;
  }
  __syncthreads();
  if ((int)threadIdx.x < BM && m0 + (int)threadIdx.x < count) {
    MMCeRow r = s[threadIdx.x];
#pragma unroll
    for (int w = 1; w < Nt::WN; ++w) r = mm_ce_join(r, s[w * BM + threadIdx.x]);
    float* p = a.part + ((long)tn * a.T + m0 + threadIdx.x) * 2;
    p[0] = r.top;
    p[1] = r.sum;
  }
}

// 32 rows a workgroup, 32 threads for the tiles of each (one thread a row walks the tiles alone, far from filling the
// card); statistics and losses; sums [blocks] (nullable): of the losses
__global__ void __launch_bounds__(1024)
mm_ce_rows_kernel(const float* __restrict__ part, long T, int tiles_n, const int* __restrict__ count,
                  const int* __restrict__ list, const int* __restrict__ y, const float* __restrict__ picked,
                  float* __restrict__ stats, float* __restrict__ loss, float* __restrict__ sums) {
  __shared__ MMCeRow s[32][33];
  const int row = threadIdx.x & 31, q = threadIdx.x >> 5, n = *count;
  int i = blockIdx.x * 32 + row;
  if ((int)blockIdx.x * 32 >= n) return;
  MMCeRow r{-INFINITY, 0.f};
  if (i < n)
#pragma unroll 8
    for (int t = q; t < tiles_n; t += 32) {
      const float2 p = *(const float2*)(part + ((long)t * T + i) * 2);
      r = mm_ce_join(r, MMCeRow{p.x, p.y});
    }
  s[row][q] = r;
  __syncthreads();
  // a row by 32 lanes of one wave now
  const int k = threadIdx.x >> 5;
  r = s[k][threadIdx.x & 31];
#pragma unroll
  for (int d = 16; d; d >>= 1) r = mm_ce_join(r, MMCeRow{__shfl_xor(r.top, d), __shfl_xor(r.sum, d)});
  i = blockIdx.x * 32 + k;
  float l = 0.f;
  if (i < n && (threadIdx.x & 31) == 0) {
    stats[i] = r.top;
    l = mm_ce_loss(r, picked[i], y[i] < 0, stats + T + i);
    if (loss) loss[list[i]] = l;
  }
  if (!sums) return;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[0][k].top = l;
  __syncthreads();
  if (threadIdx.x) return;
  float t = 0.f;
  for (int w = 0; w < 32; ++w) t += s[0][w].top;
  sums[blockIdx.x] = t;
}

// The same for few rows of many tiles: a row a workgroup, sums [rows] (16 rows, 1563 tiles: 20 -> 6 us).
__global__ void __launch_bounds__(256)
mm_ce_row_kernel(const float* __restrict__ part, long T, int tiles_n, const int* __restrict__ count,
                 const int* __restrict__ list, const int* __restrict__ y, const float* __restrict__ picked,
                 float* __restrict__ stats, float* __restrict__ loss, float* __restrict__ sums) {
  __shared__ MMCeRow s[4];
  const int i = blockIdx.x;
  if (i >= *count) return;
  MMCeRow r{-INFINITY, 0.f};
#pragma unroll 4
  for (int t = threadIdx.x; t < tiles_n; t += 256) {
    const float2 p = *(const float2*)(part + ((long)t * T + i) * 2);
    r = mm_ce_join(r, MMCeRow{p.x, p.y});
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) r = mm_ce_join(r, MMCeRow{__shfl_xor(r.top, d), __shfl_xor(r.sum, d)});
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = r;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 4; ++w) r = mm_ce_join(r, s[w]);
  stats[i] = r.top;
  const float l = mm_ce_loss(r, picked[i], y[i] < 0, stats + T + i);
  if (loss) loss[list[i]] = l;
  if (sums) sums[i] = l;
}

// sum (mean) of the sums of `each` rows
__global__ void __launch_bounds__(1024)
mm_ce_total_kernel(const float* __restrict__ sums, const int* __restrict__ count, int each, int mean,
                   float* __restrict__ loss) {
  __shared__ double s[16];
  const int n = *count, blocks = (n + each - 1) / each;
  double t = 0.;
  for (int i = threadIdx.x; i < blocks; i += 1024) t += (double)sums[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) t += __shfl_xor(t, d);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) t += s[w];
  *loss = (float)(mean ? t / (double)max(n, 1) : t);
}

// ------------------------------------------------------------------------------------------------ few rows
// The forward of few rows, in one launch or two: rows of W go by in vectors, a few classes a wave, and meet all rows of x
// (fp32 in LDS); every workgroup lists the rows by itself.  Bound by reading W: one row, 100,003 classes of 4096
// bfloat16 values in 211 us, 3.9 TB/s.  One workgroup finishes the losses (small heads), more leave partial sums to the
// rows' kernel.  Backward (D) takes the same logits and leaves d for the products.
#define MM_CE_FEW 16     // rows, at most
#define MM_CE_FEW_LDS 16384   // floats of x in LDS
#define MM_CE_CLASSES 4  // of a wave at once

struct MMCeFew {
  const void *x, *w, *targets;
  long ldx, ignore;
  int T, D, V, targets64, reduction;
  int *count, *list, *y, *pos;
  float *part, *picked, *stats, *loss;
};

// D: d of the asked rows (nothing is listed) instead of the statistics, for classes v0 .. v0 + V of the head
template <typename T>
struct MMCeFewD {
  typename MMCeType<T>::H *d, *dT;   // [rows][ldd], [V][64] (planes)
  long ldd, plane, planeT;
  int v0;
  float scale;
  MMCeScale by;
};

template <typename T, int ROWS, int TH, bool D>
__global__ void __launch_bounds__(TH) mm_ce_few_kernel(MMCeFew a, MMCeFewD<T> b) {
  constexpr int N = MMVec<T>::N, W = TH / 64, C = MM_CE_CLASSES;
  constexpr bool SPLIT = MMCeType<T>::PLANES > 1;   // what the planes of more rows cannot hold gives NaN here too
  extern __shared__ float mm_ce_x[];   // [T][D rounded up to whole vectors of a wave]
  __shared__ MMCeRow s_row[W][ROWS];
  __shared__ float s_hit[W][ROWS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, Dp = (a.D + 64 * N - 1) / (64 * N) * (64 * N);
  // lane t of every wave: row t (rows that are left out are computed like the others and go nowhere); D: asked row t
  const int rows = D ? *a.count : a.T;
  const bool has = lane < rows;
  const long target = D || !has     ? a.ignore
                      : a.targets64 ? ((const long*)a.targets)[lane]
                                    : (long)((const int*)a.targets)[lane];
#pragma unroll
  for (int t = 0; t < ROWS; ++t) {
    if (t >= rows) continue;
    const long at = D ? a.list[t] : t;
    for (int c = threadIdx.x; c < Dp; c += TH) {
      const float v = c < a.D ? (float)((const T*)a.x)[at * a.ldx + c] : 0.f;
      mm_ce_x[t * Dp + c] = SPLIT && fabsf(v) >= MM_SPLIT_LIMIT ? __builtin_nanf("") : v;
    }
  }
  const unsigned long long asked = __ballot(target != a.ignore);
  const int at = __popcll(asked & ((1ull << lane) - 1)), n = __popcll(asked);
  const int y = D ? a.y[has ? lane : 0] : target >= 0 && target < a.V ? (int)target : -1;
  const float top = D ? a.stats[has ? lane : 0] : 0.f;
  const MMCeD d_of(D ? a.stats[a.T + (has ? lane : 0)] : 1.f);
  const float share = D ? b.by.share(has ? lane : 0) : 0.f;
  const int end = D ? (int)mm_up(a.V, MM_NT_K) : a.V;   // D: zeros past the last class
  if (!D && blockIdx.x == 0 && wave == 0) {
    if (target != a.ignore) {
      a.list[at] = lane;
      a.y[at] = y;
    }
    if (has) a.pos[lane] = target != a.ignore ? at : -1;
    if (has && target == a.ignore && a.reduction == 0) a.loss[lane] = 0.f;
    if (lane == 0) *a.count = n;
  }
  __syncthreads();
  MMCeRow r{-INFINITY, 0.f};
  float hit = 0.f;
  for (int v0 = (blockIdx.x * W + wave) * C; v0 < end; v0 += (int)gridDim.x * W * C) {
    float acc[ROWS][C] = {}, large[C] = {};   // the largest |w| (a NaN is in acc anyway)
    const T* __restrict__ p[C];
#pragma unroll
    for (int k = 0; k < C; ++k) p[k] = (const T*)a.w + (size_t)min(v0 + k, a.V - 1) * a.D;
    auto add = [&](int c, int end) {
      float w[C][N];
#pragma unroll
      for (int k = 0; k < C; ++k) mm_load_vec(p[k], c, end, w[k]);
      if constexpr (SPLIT) {
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int i = 0; i < N; ++i) large[k] = fmaxf(large[k], fabsf(w[k][i]));
      }
#pragma unroll
      for (int t = 0; t < ROWS; ++t) {
        if (ROWS > 1 && t >= rows) continue;   // not break, which would put acc into memory
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const floatx4 x = *(const floatx4*)(mm_ce_x + t * Dp + c + i);
#pragma unroll
          for (int k = 0; k < C; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[t][k] = fmaf(x[q], w[k][i + q], acc[t][k]);
        }
      }
    };
    int c = lane * N;
    const int whole = a.D / (64 * N) * (64 * N);
#pragma unroll 4
    for (; c < whole; c += 64 * N) add(c, c + N);
    if (whole < a.D && c < Dp) add(c, a.D);
    if constexpr (SPLIT) {
#pragma unroll
      for (int t = 0; t < ROWS; ++t)
#pragma unroll
        for (int k = 0; k < C; ++k) acc[t][k] = large[k] >= MM_SPLIT_LIMIT ? __builtin_nanf("") : acc[t][k];
    }
    float mine[C] = {};
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
      if (ROWS > 1 && t >= rows) continue;
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const float l = mm_lanes_sum<64>(acc[t][k]);
        if constexpr (D) {
          if (lane == t) mine[k] = l;
        } else if (lane == t && v0 + k < a.V) {
          r = mm_ce_join(r, MMCeRow{l, v0 + k == y ? 0.f : 1.f});
          if (v0 + k == y) hit = l;
        }
      }
    }
    if constexpr (D) {
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const float p = d_of(mine[k], top, v0 + k + b.v0 == y);
        // a target out of range (loss NaN) makes the row NaN
        mine[k] = has && v0 + k < a.V ? (y < 0 ? __builtin_nanf("") : p * b.scale) : 0.f;
      }
      if (has) mm_ce_put4<T>(b.d + lane * b.ldd + v0, b.plane, mine);
#pragma unroll
      for (int k = 0; k < C; ++k) {
        if (v0 + k >= a.V) break;
        float v = mine[k] * share;
#pragma unroll
        for (int q = 0; q < MMCeType<T>::PLANES; ++q) {
          const typename MMCeType<T>::H h = (typename MMCeType<T>::H)v;
          b.dT[q * b.planeT + (long)(v0 + k) * 64 + lane] = has ? h : (typename MMCeType<T>::H)0.f;
          v -= (float)h;
        }
      }
    }
  }
  if constexpr (D) return;
  if (gridDim.x > 1 && target != a.ignore && y >= 0 && y / C % (int)(gridDim.x * W) == (int)blockIdx.x * W + wave)
    a.picked[at] = hit;   // by the wave that has the target's class
  if (lane < ROWS) {
    s_row[wave][lane] = r;
    s_hit[wave][lane] = hit;
  }
  __syncthreads();
  if (wave) return;
  float l = 0.f;
  if (target != a.ignore) {
#pragma unroll
    for (int w = 1; w < W; ++w) {
      r = mm_ce_join(r, s_row[w][lane]);
      hit += s_hit[w][lane];   // 0 but for one wave
    }
    if (gridDim.x > 1) {
      float* p = a.part + ((long)blockIdx.x * a.T + at) * 2;
      p[0] = r.top;
      p[1] = r.sum;
      return;
    }
    a.stats[at] = r.top;
    l = mm_ce_loss(r, hit, y < 0, a.stats + a.T + at);
    if (a.reduction == 0) a.loss[lane] = l;
  }
  if (gridDim.x > 1 || a.reduction == 0) return;
  l = mm_lanes_sum<64>(l);
  if (lane == 0) *a.loss = a.reduction == MM_CE_MEAN ? l / (float)max(n, 1) : l;
}

// ------------------------------------------------------------------------------------------------ backward
// g of the asked rows and the largest finite |g|; one workgroup
__global__ void __launch_bounds__(1024) mm_ce_grad_kernel(const float* __restrict__ dloss,
                                                          const int* __restrict__ count, const int* __restrict__ list,
                                                          float* __restrict__ g, float* __restrict__ gmax) {
  __shared__ float s[16];
  const int n = *count;
  float top = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float v = dloss[list[i]];
    g[i] = v;
    if (fabsf(v) < INFINITY) top = fmaxf(top, fabsf(v));
  }
  top = mm_lanes_max<64>(top);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) top = fmaxf(top, s[w]);
  *gmax = top;
}

// The same product, with 32 bits of d and its transpose to store: 291 us for 8192 classes of it, 945 TFLOP/s.
template <typename T, typename Nt>
__global__ void __launch_bounds__(Nt::TH, Nt::PER_CU)
mm_ce_d_kernel(MMCeLogits<typename MMCeType<T>::H> a, int tiles_n) {
  typedef typename MMCeType<T>::H H;
  constexpr int BM = Nt::BM, BN = Nt::BN;
  extern __shared__ uint4 mm_ce_lds[];
  const int count = *a.count;
  int e, tm, tn;
  if (!mm_nt_tile(blockIdx.x, 1, (count + BM - 1) / BM, tiles_n, &e, &tm, &tn)) return;
  const int m0 = tm * BM, n0 = tn * BN;
  MMNtOperand<H> x = a.x;
  x.rows = count;
  Nt t;
  t.run(x, m0, a.w, n0, 0, a.K, mm_ce_lds);
  const int rows = (int)mm_up(count, MM_NT_K), cols = (int)mm_up(a.n, MM_NT_K);
  float share[Nt::FM];
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j) {
    const int m = m0 + t.row(j), at = min(m, count - 1), y = a.y[at];
    const float top = a.stats[at];
    const MMCeD d_of(a.stats[a.T + at]);
    share[j] = a.by.share(at);
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + t.col(i) + q;
        const float p = d_of(t.acc[i][j][q], top, n + a.v0 == y);
        // a target out of range (loss NaN) makes the row NaN
        t.acc[i][j][q] = n < a.n && m < count ? (y < 0 ? __builtin_nanf("") : p * a.scale) : 0.f;
      }
  }
  if constexpr (MMCeType<T>::PLANES > 1) {   // three planes: straight from the registers (27 us against 43 through LDS
                                             // for 14,700 rows, 89 classes)
#pragma unroll
    for (int j = 0; j < Nt::FM; ++j)
#pragma unroll
      for (int i = 0; i < Nt::FN; ++i) {
        const int m = m0 + t.row(j), n = n0 + t.col(i), mt = m & ~3, nt = n + (t.lane & 3);
        const floatx4 v = t.acc[i][j];
        if (m < count && n < cols) mm_ce_put4<T>(a.d + (long)m * a.ldd + n, a.plane, (const float*)&v);
        floatx4 r = v * share[j];
#pragma unroll
        for (int b = 0; b < MMCeType<T>::PLANES; ++b) {
          typedef H vec __attribute__((ext_vector_type(4)));
          H h[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            h[q] = (H)r[q];
            r[q] -= (float)h[q];
          }
          mm_quad_transpose(h);
          if (nt < a.n && mt < rows) *(vec*)(a.dT + b * a.planeT + (long)nt * a.ldt + mt) = vec{h[0], h[1], h[2], h[3]};
        }
      }
    return;
  }
  H* const tile = (H*)mm_ce_lds;
  mm_nt_store(t, tile, a.d + (long)m0 * a.ldd + n0, a.ldd, count - m0, cols - n0,
              [&](int i, int j) { return t.acc[i][j]; });
  mm_nt_store_transposed(t, tile, a.dT + (long)n0 * a.ldt + m0, a.ldt, rows - m0, a.n - n0,
                         [&](int i, int j) { return t.acc[i][j] * share[j]; });
}

// C = A B^T of a piece.  dx: rows of A are the asked rows (count), fp32 sums part [splits][T][N], added to what is there
// unless `first`, or (one piece, one split) the rows list[m] of dx themselves, times the row's g.  dW: the summed index
// is the asked rows; part [splits][M][N] (written), or with one split the rows of dW, times the whole gradient.
template <typename H>
struct MMCeProduct {
  MMNtOperand<H> a, b;
  const int *count, *list;
  int dx, M, N, K;      // K: stages (dx)
  int splits, first, tiles_n, blocks;
  float* part;
  long rows;            // of part
  void* out;
  MMCeScale by;
  float inv;
};

// both in one launch, as neither fills the card by itself where rows and classes are few (8192 rows and classes, 2048
// bfloat16 values: 490 us, 1120 TFLOP/s)
template <typename T, typename Nt>
__global__ void __launch_bounds__(Nt::TH, Nt::PER_CU)
mm_ce_product_kernel(MMCeProduct<typename MMCeType<T>::H> one, MMCeProduct<typename MMCeType<T>::H> two) {
  typedef typename MMCeType<T>::H H;
  constexpr int BM = Nt::BM, BN = Nt::BN;
  extern __shared__ uint4 mm_ce_lds[];
  const bool is_one = (int)blockIdx.x < one.blocks;
  const MMCeProduct<H>& a = is_one ? one : two;
  const int block = (int)blockIdx.x - (is_one ? 0 : one.blocks), count = *a.count, M = a.dx ? count : a.M;
  const int K = a.dx ? a.K : (count + MM_NT_K - 1) / MM_NT_K, tiles_m = (M + BM - 1) / BM;
  int split, tm, tn;
  if (!mm_nt_tile(block, a.splits, tiles_m, a.tiles_n, &split, &tm, &tn)) return;
  const int m0 = tm * BM, n0 = tn * BN;
  MMNtOperand<H> A = a.a;
  A.rows = M;
  Nt t;
  t.run(A, m0, a.b, n0, (int)((long)K * split / a.splits), (int)((long)K * (split + 1) / a.splits), mm_ce_lds);
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j) {
    const int m = m0 + t.row(j);
    if (m >= M) continue;
    float f = 1.f;
    T* out = nullptr;
    if (a.out) {
      f = (a.dx ? a.by.row(m, count) : a.by.whole(count)) * a.inv;
      out = (T*)a.out + (long)(a.dx ? a.list[m] : m) * a.N;
    }
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i) {
      const int n = n0 + t.col(i);
      floatx4 v = t.acc[i][j];
      if (out) {
        v *= f;
        mm_store4(out, n, a.N, (const float*)&v);
      } else {
        float* p = a.part + ((long)split * a.rows + m) * a.N;
        if (a.dx && !a.first) {
          floatx4 u;
          mm_load4(p, n, a.N, (float*)&u);
          v += u;
        }
        mm_store4(p, n, a.N, (const float*)&v);
      }
    }
  }
}

// out = the sum of the splits' sums: dx (pos: row of part, or none: 0; factor of the row) or dW (the whole factor).  A
// vector is summed by WAVES waves.
template <typename T, bool DX, int WAVES>
__global__ void __launch_bounds__(256)
mm_ce_join_kernel(const float* __restrict__ part, int splits, long part_rows, long rows, int N,
                  const int* __restrict__ pos, const int* __restrict__ count, MMCeScale by, float inv,
                  T* __restrict__ out) {
  constexpr int EACH = 256 / WAVES;
  __shared__ floatx4 s[WAVES][EACH];
  const int nv = (N + 3) / 4, lane = threadIdx.x % EACH, wave = threadIdx.x / EACH, asked = *count;
  for (long i0 = (long)blockIdx.x * EACH; i0 < rows * nv; i0 += (long)gridDim.x * EACH) {
    const long i = i0 + lane, row = i / nv, at = i >= rows * nv ? -1 : DX ? pos[row] : row;
    const int c = (int)(i - row * nv) * 4;
    floatx4 v = {};
    if (at >= 0) {
#pragma unroll 4
      for (int k = wave; k < splits; k += WAVES) {
        floatx4 u;
        mm_load4(part + (k * part_rows + at) * N, c, N, (float*)&u);
        v += u;
      }
    }
    if constexpr (WAVES > 1) {
      s[wave][lane] = v;
      __syncthreads();
    }
    if (wave == 0 && i < rows * nv) {
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v += s[w][lane];
      if (at >= 0) v *= (DX ? by.row((int)at, asked) : by.whole(asked)) * inv;   // 0 rows stay 0 whatever the factor
      mm_store4(out + row * N, c, N, (const float*)&v);
    }
    if constexpr (WAVES > 1) __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ host
namespace {
constexpr long MAX_SIDE = 2147483648L - 65536;
constexpr int BM = 64, BN = 64;   // the smallest tiles
constexpr float HALF_SCALE = 16384.f;   // of d in float16

struct Sizes {
  long T, D, V;
  int dtype;
  long Dp, Tp;
  int planes;
  bool w_in_place;   // the weights are operands as they are
  long piece, pieces, piece_p;
  int dx_splits, dw_splits;
  int dx_side, dw_side;
};

long div_up(long a, long b) { return (a + b - 1) / b; }
long clamp(long v, long lo, long hi) { return v < lo ? lo : v > hi ? hi : v; }

// Workspace regions, 256 bytes apart from each other.
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

int tiles(long m, long n, int side) { return (int)(div_up(m, side) * div_up(n, side)); }
int side_of(long m, long n, int P) { return mm_tile_side(P, tiles(m, n, 256), tiles(m, n, 128), tiles(m, n, 64)); }

// Tile and parts of the summed index K of an m x n product by the same rule, no part below 512 values; a part costs
// its sums' way through memory.  Whole passes with one side and number of parts for both products, us: 14,700 float
// rows, 89 classes of 128 values: 64 x 1 311, x 8 127, x 64 314 (each by its own: 87); 1000 x 3000 float of 512: 64 x
// 1 155, 128 x 4 144, x 64 376 (153); 8192 x 8192 bfloat16 of 2048: 256 x 1 1059, x 2 1143, x 8 1469 (1067).
int splits_of(long m, long n, long K, int P, int* side) {
  const long most = clamp(K / 512, 1, 64);
  const MMTileRates r = mm_tile_rates(P);
  double best = 1e30;
  int splits = 1;
  for (int i = 0; i < 3; ++i) {
    const long t = tiles(m, n, r.side[i]) < 1 ? 1 : tiles(m, n, r.side[i]), p = clamp(r.slots[i] / t, 1, most);
    const double cost = r.round[i] * (double)div_up(t * p, r.slots[i]) / (double)p + 0.002 * (double)p;
    if (cost < best) {
      best = cost;
      splits = (int)p;
      *side = r.side[i];
    }
  }
  return splits;
}

bool sizes_of(const char* name, long T, long D, long V, int dtype, const void* w, Sizes* s) {
  if (T > MAX_SIDE || D > MAX_SIDE || V > MAX_SIDE || div_up(T, BM) * div_up(V, BN) * 256 >= 4294967296L ||
      (div_up(T, 64) + div_up(V, 64) + 64) * (div_up(D, 64) + 16) * 256 >= 4294967296L) {
    mm::set_error(std::string(name) + ": sizes beyond the launches' limits");
    return false;
  }
  *s = Sizes{T, D, V, dtype};
  s->Dp = mm_up(D, MM_NT_K);
  s->Tp = mm_up(T ? T : 1, MM_NT_K);
  s->planes = dtype == MM_F32 ? 3 : 1;
  s->w_in_place = dtype != MM_F32 && D % MM_NT_K == 0 && (size_t)w % 16 == 0;
  // a piece: d by rows and transposed in 256 MB (a plane), but never fewer than 1024 columns
  const long most = clamp((268435456L / (s->Tp * 4)) / 256 * 256, 1024, 1 << 20);
  s->pieces = div_up(V, most);
  s->piece = s->pieces == 1 ? V : mm_up(div_up(V, s->pieces), 256);
  s->pieces = div_up(V, s->piece);
  s->piece_p = mm_up(s->piece, MM_NT_K);
  const int P = dtype == MM_F32 ? 6 : 1;
  s->dx_splits = splits_of(T, D, s->piece_p, P, &s->dx_side);
  s->dw_splits = splits_of(s->piece, D, s->Tp, P, &s->dw_side);
  return true;
}

// Few rows of a head: vectors of W without the matrix cores, where that takes less time.  Its adds and the sums over
// the lanes take 0.09 + 0.00015 D ns a row and class where they exceed the reading of W (bfloat16, 16 rows, 100,003
// classes of 512 and 1024 values: 238 and 330 us; float, 10 rows, 50,000 of 1024: 122); tiles take four launches more,
// read W once if it is an operand as it is (17 rows, 100,003 classes of 1024 values: 51 us in all), and three times its
// size if not (float: packed and read in 16 bytes a value).
bool few_rows(const Sizes& s) {
  const long Dp = mm_up(s.D, s.dtype == MM_F32 ? 256 : 512);
  if (s.T == 0 || s.T > MM_CE_FEW || s.T * Dp > MM_CE_FEW_LDS) return false;
  const double W = (double)s.V * s.D * (s.dtype == MM_F32 ? 4. : 2.);
  const double few = (double)s.T * s.V * (0.09 + 0.00015 * s.D), reading = W / 4000.;   // ns
  const double tiles = W * (s.dtype == MM_F32 ? 4. : s.D % MM_NT_K ? 3. : 1.) / 4200. + 25000.;
  return (few > reading ? few : reading) <= tiles;
}
// one workgroup where W has up to 128 KB
int few_workgroups(const Sizes& s) {
  if (s.V * s.D * (s.dtype == MM_F32 ? 4 : 2) <= 131072) return 1;
  return (int)clamp(div_up(s.V, 8 * MM_CE_CLASSES), 2, 512);
}

// few rows of many tiles: a workgroup each
#define MM_CE_ROW 256
bool row_each(const Sizes& s, int tiles_n) { return s.T < MM_CE_ROW && tiles_n >= 64; }

// tiles of the forward's logits
int logits_side(const Sizes& s) { return side_of(s.T, s.V, s.dtype == MM_F32 ? 6 : 1); }

struct Forward {
  void *x, *w;
  float *part, *picked, *sums;
  int* counts;
};
size_t forward_space(const Sizes& s, char* base, Forward* f) {
  Space p{base};
  if (few_rows(s)) {
    f->part = p.take<float>((size_t)few_workgroups(s) * s.T * 2);
    f->picked = p.take<float>(s.T);
    f->sums = p.take<float>(s.T);
    return p.used;
  }
  f->x = p.take<short>((size_t)s.planes * s.T * s.Dp);
  f->w = s.w_in_place ? nullptr : p.take<short>((size_t)s.planes * s.V * s.Dp);
  f->part = p.take<float>((size_t)div_up(s.V, logits_side(s)) * s.T * 2);
  f->picked = p.take<float>(s.T);
  f->sums = p.take<float>(s.T < MM_CE_ROW ? s.T : div_up(s.T, 32));
  f->counts = p.take<int>(div_up(s.T, 1024 * 4));
  return p.used;
}

struct Backward {
  void *x, *xT, *w, *wT, *d, *dT;
  float *g, *gmax, *dx, *dw;
};
size_t backward_space(const Sizes& s, bool dx, bool dw, char* base, Backward* b) {
  Space p{base};
  b->x = p.take<short>((size_t)s.planes * s.T * s.Dp);
  b->xT = dw ? p.take<short>((size_t)s.planes * s.D * s.Tp) : nullptr;
  b->w = s.w_in_place ? nullptr : p.take<short>((size_t)s.planes * s.piece * s.Dp);
  b->wT = dx ? p.take<short>((size_t)s.planes * s.D * s.piece_p) : nullptr;
  b->d = p.take<short>((size_t)s.planes * s.T * s.piece_p);
  b->dT = p.take<short>((size_t)s.planes * s.piece * s.Tp);
  b->g = p.take<float>(s.T);
  b->gmax = p.take<float>(1);
  b->dx = dx && (s.pieces > 1 || s.dx_splits > 1) ? p.take<float>((size_t)s.dx_splits * s.T * s.D) : nullptr;
  b->dw = dw && s.dw_splits > 1 ? p.take<float>((size_t)s.dw_splits * s.piece * s.D) : nullptr;
  return p.used;
}

template <typename T>
void pack(MMPack a, MMPack b, MMZero z, hipStream_t stream) {
  for (MMPack* p : {&a, &b}) {
    const bool any = p->out || p->outT;
    p->blocks_r = any ? (int)div_up(p->rows, 64) : 0;
    p->blocks_c = any ? (int)div_up(p->cols, 64) : 0;
  }
  z.blocks = z.out ? (int)clamp(div_up(z.rows * div_up(z.N, 4), 1024), 1, 4096) : 0;
  const long blocks = (long)a.blocks_r * a.blocks_c + (long)b.blocks_r * b.blocks_c + z.blocks;
  if (blocks) hipLaunchKernelGGL(mm_ce_pack_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, a, b, z);
}

template <auto KERNEL, typename Nt, typename... A>
bool launch(long blocks, hipStream_t stream, const A&... a) {
  if (!lds_granted<KERNEL>(Nt::LDS)) return false;
  hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(Nt::TH), Nt::LDS, stream, a...);
  return true;
}

template <typename T>
struct Tiles {
  typedef typename MMCeType<T>::H H;
  static constexpr int P = MMCeType<T>::P;
  typedef MMNtBig<H, P> Big;
  typedef MMNt<H, P, 128, 128, 2, P == 1 ? 2 : 4> Mid;   // planes leave room for one workgroup a CU
  typedef MMNt<H, P, 64, 64, 2, 2> Low;

  // the logits' statistics, or (D) d
  template <bool D>
  static bool logits(const MMCeLogits<H>& a, long rows, long n, int side, hipStream_t stream) {
    const int tn = (int)div_up(n, side), blocks = tiles(rows, n, side);
    if constexpr (D) {
      return side == 256   ? launch<mm_ce_d_kernel<T, Big>, Big>(blocks, stream, a, tn)
             : side == 128 ? launch<mm_ce_d_kernel<T, Mid>, Mid>(blocks, stream, a, tn)
                           : launch<mm_ce_d_kernel<T, Low>, Low>(blocks, stream, a, tn);
    } else {
      return side == 256   ? launch<mm_ce_logits_kernel<T, Big>, Big>(blocks, stream, a, tn)
             : side == 128 ? launch<mm_ce_logits_kernel<T, Mid>, Mid>(blocks, stream, a, tn)
                           : launch<mm_ce_logits_kernel<T, Low>, Low>(blocks, stream, a, tn);
    }
  }

  static bool products(MMCeProduct<H> a, MMCeProduct<H> b, int side, hipStream_t stream) {
    for (MMCeProduct<H>* p : {&a, &b}) {
      p->tiles_n = (int)div_up(p->N, side);
      p->blocks = p->blocks ? (int)mm_up((long)tiles(p->M, p->N, side) * p->splits, 8) : 0;   // the second one's XCDs
    }
    const long blocks = (long)a.blocks + b.blocks;
    return side == 256   ? launch<mm_ce_product_kernel<T, Big>, Big>(blocks, stream, a, b)
           : side == 128 ? launch<mm_ce_product_kernel<T, Mid>, Mid>(blocks, stream, a, b)
                         : launch<mm_ce_product_kernel<T, Low>, Low>(blocks, stream, a, b);
  }
};

// rows' statistics and losses from the tiles' (T > 0), then their sum or mean
void finish(const Sizes& s, const Forward& f, int tiles_n, const Rows& r, int reduction, float* stats, float* loss,
            hipStream_t stream) {
  const bool one = row_each(s, tiles_n);
  if (s.T) {
    const dim3 grid((unsigned)(one ? s.T : div_up(s.T, 32)));
    float *each = reduction == 0 ? loss : nullptr, *sums = reduction ? f.sums : nullptr;
    if (one)
      hipLaunchKernelGGL(mm_ce_row_kernel, grid, dim3(256), 0, stream, f.part, s.T, tiles_n, r.count, r.list, r.y, f.picked,
                         stats, each, sums);
    else
      hipLaunchKernelGGL(mm_ce_rows_kernel, grid, dim3(1024), 0, stream, f.part, s.T, tiles_n, r.count, r.list, r.y,
                         f.picked, stats, each, sums);
  }
  if (reduction)
    hipLaunchKernelGGL(mm_ce_total_kernel, dim3(1), dim3(1024), 0, stream, f.sums, r.count, one ? 1 : 32,
                       reduction == MM_CE_MEAN, loss);
}

template <typename T, int ROWS, int TH, bool D>
bool launch_few(const MMCeFew& a, const MMCeFewD<T>& b, int wg, hipStream_t stream) {
  const size_t lds = (size_t)a.T * mm_up(a.D, 64 * MMVec<T>::N) * sizeof(float);
  if (!lds_granted<mm_ce_few_kernel<T, ROWS, TH, D>>((int)lds)) return false;
  hipLaunchKernelGGL((mm_ce_few_kernel<T, ROWS, TH, D>), dim3(wg), dim3(TH), lds, stream, a, b);
  return true;
}

template <typename T, int TH, bool D>
bool few(const MMCeFew& a, const MMCeFewD<T>& b, int wg, hipStream_t stream) {
  return a.T == 1   ? launch_few<T, 1, TH, D>(a, b, wg, stream)
         : a.T <= 4 ? launch_few<T, 4, TH, D>(a, b, wg, stream)
                    : launch_few<T, MM_CE_FEW, TH, D>(a, b, wg, stream);
}

template <typename T>
int forward_few(const Sizes& s, const MMCeFew& a, const Rows& r, const Forward& f, hipStream_t stream) {
  const int wg = few_workgroups(s);
  const MMCeFewD<T> none{};
  const bool ok = wg == 1 ? few<T, 1024, false>(a, none, 1, stream) : few<T, 512, false>(a, none, wg, stream);
  if (!ok) return MM_ELAUNCH;
  if (wg > 1) finish(s, f, wg, r, a.reduction, a.stats, a.loss, stream);
  return mm::launch_status("mm_ce_fwd");
}

template <typename T>
int forward(const Sizes& s, const T* x, long ldx, const T* w, const Rows& r, int reduction, float* loss, float* stats,
            const Forward& f, hipStream_t stream) {
  typedef typename MMCeType<T>::H H;
  const int side = logits_side(s), tiles_n = (int)div_up(s.V, side);
  if (s.T) {
    const MMPack px{x, r.list, r.count, f.x, nullptr, ldx, 0, s.Dp, 0, s.T * s.Dp, 0, (int)s.T, (int)s.D};
    const MMPack pw{w, nullptr, nullptr, f.w, nullptr, s.D, 0, s.Dp, 0, s.V * s.Dp, 0, (int)s.V, (int)s.D};
    pack<T>(px, pw, MMZero{}, stream);
    MMCeLogits<H> a{};
    a.x = MMNtOperand<H>{(const H*)f.x, s.Dp, s.T * s.Dp, 0};
    a.w = s.w_in_place ? MMNtOperand<H>{(const H*)w, s.D, 0, (int)s.V}
                       : MMNtOperand<H>{(const H*)f.w, s.Dp, s.V * s.Dp, (int)s.V};
    a.count = r.count;
    a.y = r.y;
    a.V = (int)s.V;
    a.K = (int)(s.Dp / MM_NT_K);
    a.part = f.part;
    a.picked = f.picked;
    a.T = s.T;
    if (!Tiles<T>::template logits<false>(a, s.T, s.V, side, stream)) return MM_ELAUNCH;
  }
  finish(s, f, tiles_n, r, reduction, stats, loss, stream);
  return mm::launch_status("mm_ce_fwd");
}

template <typename T, bool DX>
void join(const float* part, int splits, long part_rows, long rows, int N, const int* pos, const int* count,
          const MMCeScale& by, float inv, T* out, hipStream_t stream) {
  const long vectors = rows * div_up(N, 4);
  if (splits < 4)
    hipLaunchKernelGGL((mm_ce_join_kernel<T, DX, 1>), dim3((unsigned)clamp(div_up(vectors, 256), 1, 4096)), dim3(256), 0,
                       stream, part, splits, part_rows, rows, N, pos, count, by, inv, out);
  else
    hipLaunchKernelGGL((mm_ce_join_kernel<T, DX, 4>), dim3((unsigned)clamp(div_up(vectors, 64), 1, 4096)), dim3(256), 0,
                       stream, part, splits, part_rows, rows, N, pos, count, by, inv, out);
}

template <typename T>
int backward(const Sizes& s, const T* x, long ldx, const T* w, const Rows& r, int reduction, const float* stats,
             const float* dloss, T* dx, T* dw, const Backward& b, hipStream_t stream) {
  typedef typename MMCeType<T>::H H;
  const float scale = s.dtype == MM_F16 ? HALF_SCALE : 1.f;
  const MMCeScale by{reduction ? nullptr : b.g, b.gmax, dloss, reduction == MM_CE_MEAN};
  if (!reduction)
    hipLaunchKernelGGL(mm_ce_grad_kernel, dim3(1), dim3(1024), 0, stream, dloss, r.count, r.list, b.g, b.gmax);
  const bool few_d = few_rows(s);
  const bool direct = s.pieces == 1 && s.dx_splits == 1;   // dx without sums in memory
  for (long p = 0; p < s.pieces; ++p) {
    const long v0 = p * s.piece, n = s.V - v0 < s.piece ? s.V - v0 : s.piece, np = mm_up(n, MM_NT_K);
    MMPack px{x, r.list, r.count, b.x, b.xT, ldx, 0, s.Dp, s.Tp, s.T * s.Dp, s.D * s.Tp, (int)s.T, (int)s.D};
    if (p) px.out = px.outT = nullptr;   // once
    MMPack pw{w, nullptr, nullptr, b.w, b.wT, s.D, v0, s.Dp, s.piece_p, s.piece * s.Dp, s.D * s.piece_p, (int)n,
                    (int)s.D};
    if (few_d) px.out = pw.out = nullptr;
    pack<T>(px, pw, MMZero{r.pos, direct ? dx : nullptr, s.T, (int)s.D}, stream);
    MMCeLogits<H> a{};
    a.x = MMNtOperand<H>{(const H*)b.x, s.Dp, s.T * s.Dp, 0};
    a.w = s.w_in_place ? MMNtOperand<H>{(const H*)w + v0 * s.D, s.D, 0, (int)n}
                       : MMNtOperand<H>{(const H*)b.w, s.Dp, s.piece * s.Dp, (int)n};
    a.count = r.count;
    a.y = r.y;
    a.K = (int)(s.Dp / MM_NT_K);
    a.T = s.T;
    a.stats = stats;
    a.by = by;
    a.d = (H*)b.d;
    a.dT = (H*)b.dT;
    a.ldd = s.piece_p;
    a.ldt = s.Tp;
    a.plane = s.T * s.piece_p;
    a.planeT = s.piece * s.Tp;
    a.v0 = (int)v0;
    a.n = (int)n;
    a.scale = scale;
    // d in three planes, twice: its stores need another workgroup's products beside them (8598 rows, 59,192 classes: 2.9
    // ms against 3.5 with tiles of 256)
    const int side = side_of(s.T, n, MMCeType<T>::P);
    bool ok;
    if (few_d) {
      const MMCeFew e{x, w + v0 * s.D, nullptr, ldx, 0, (int)s.T, (int)s.D, (int)n, 0, 0, r.count, r.list, r.y, r.pos,
                      nullptr, nullptr, (float*)stats, nullptr};
      const MMCeFewD<T> f{a.d, a.dT, a.ldd, a.plane, a.planeT, (int)v0, scale, by};
      ok = few<T, 512, true>(e, f, (int)clamp(div_up(np, 8 * MM_CE_CLASSES), 1, 512), stream);
    } else {
      ok = Tiles<T>::template logits<true>(a, s.T, n, MMCeType<T>::P > 1 && side > 128 ? 128 : side, stream);
    }
    MMCeProduct<H> q{}, u{};
    if (dx) {
      q.a = MMNtOperand<H>{(const H*)b.d, s.piece_p, s.T * s.piece_p, 0};
      q.b = MMNtOperand<H>{(const H*)b.wT, s.piece_p, s.D * s.piece_p, (int)s.D};
      q.count = r.count;
      q.list = r.list;
      q.dx = q.blocks = 1;
      q.M = (int)s.T;
      q.N = (int)s.D;
      q.K = (int)(np / MM_NT_K);
      q.splits = s.dx_splits;
      q.first = p == 0;
      q.part = b.dx;
      q.rows = s.T;
      q.out = direct ? dx : nullptr;
      q.by = by;
      q.inv = 1.f / scale;
    }
    if (dw) {
      u.a = MMNtOperand<H>{(const H*)b.dT, s.Tp, s.piece * s.Tp, 0};
      u.b = MMNtOperand<H>{(const H*)b.xT, s.Tp, s.D * s.Tp, (int)s.D};
      u.count = r.count;
      u.blocks = 1;
      u.M = (int)n;
      u.N = (int)s.D;
      u.splits = s.dw_splits;
      u.part = b.dw;
      u.rows = n;
      u.out = s.dw_splits == 1 ? dw + v0 * s.D : nullptr;
      u.by = by;
      u.inv = 1.f / scale;
    }
    if (dx && dw && s.dx_side == s.dw_side) {
      ok = ok && Tiles<T>::products(q, u, s.dx_side, stream);
    } else {
      if (dx) ok = ok && Tiles<T>::products(q, MMCeProduct<H>{}, s.dx_side, stream);
      if (dw) ok = ok && Tiles<T>::products(u, MMCeProduct<H>{}, s.dw_side, stream);
    }
    if (!ok) return MM_ELAUNCH;
    if (dw && s.dw_splits > 1)
      join<T, false>(b.dw, s.dw_splits, n, n, (int)s.D, nullptr, r.count, by, 1.f / scale, dw + v0 * s.D, stream);
  }
  if (dx && !direct)
    join<T, true>(b.dx, s.dx_splits, s.T, s.T, (int)s.D, r.pos, r.count, by, 1.f / scale, dx, stream);
  return mm::launch_status("mm_ce_bwd");
}
}  // namespace

#define MM_CE_CHECK(name)                                                                                    \
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");                                             \
  MM_CHECK_ARG(T >= 0 && D > 0 && V > 0, "bad sizes");                                                       \
  Sizes s;                                                                                                   \
  if (!sizes_of(name, T, D, V, dtype, w, &s)) return MM_ERANGE

extern "C" int mm_ce_workspace(long T, long D, long V, int dtype, const void* w, int dx, int dw, size_t* bytes) {
  MM_CHECK_ARG(bytes, "no result");
  MM_CE_CHECK("mm_ce_workspace");
  Forward f;
  Backward b;
  *bytes = dx || dw ? backward_space(s, dx, dw, nullptr, &b) : forward_space(s, nullptr, &f);
  return MM_OK;
}

extern "C" int mm_ce_fwd(const void* x, long ldx, int dtype, long T, long D, const void* w, long V, const void* targets,
                         int targets64, long ignore, int reduction, float* loss, float* stats, int* rows, void* workspace,
                         hipStream_t stream) {
  MM_CE_CHECK("mm_ce_fwd");
  MM_CHECK_ARG(ldx >= 0 && reduction >= 0 && reduction <= 2, "bad reduction");
  MM_CHECK_ARG(loss && rows && (T == 0 || (x && w && targets && stats && workspace)), "null pointer");
  Forward f;
  forward_space(s, (char*)workspace, &f);
  const Rows r = rows_of(rows, T);
  int rc = MM_OK;
  if (few_rows(s)) {
    const MMCeFew a{x, w, targets, ldx, ignore, (int)T, (int)D, (int)V, targets64, reduction, r.count, r.list, r.y, r.pos,
                    f.part, f.picked, stats, loss};
    MM_DISPATCH(dtype, rc = forward_few<T_>(s, a, r, f, stream));
    return rc;
  }
  auto list = [&](auto y, auto each) {
    typedef std::remove_const_t<std::remove_pointer_t<decltype(y)>> Y;
    constexpr int SCAN = decltype(each)::value;
    const unsigned blocks = T ? (unsigned)div_up(T, 1024 * SCAN) : 1;
    if (blocks > 1)
      hipLaunchKernelGGL((mm_ce_count_kernel<Y, SCAN>), dim3(blocks), dim3(1024), 0, stream, y, T, ignore, f.counts);
    hipLaunchKernelGGL((mm_ce_list_kernel<Y, SCAN>), dim3(blocks), dim3(1024), 0, stream, y, T, (int)V, ignore, f.counts,
                       r.count, r.list, r.y, r.pos, reduction == 0 ? loss : nullptr);
  };
  auto scan = [&](auto y) {
    if (T > 16384 && T <= 4194304) list(y, std::integral_constant<int, 4>{});
    else list(y, std::integral_constant<int, 16>{});
  };
  if (targets64) scan((const long*)targets);
  else scan((const int*)targets);
  MM_DISPATCH(dtype, rc = forward<T_>(s, (const T_*)x, ldx, (const T_*)w, r, reduction, loss, stats, f, stream));
  return rc;
}

extern "C" int mm_ce_bwd(const void* x, long ldx, int dtype, long T, long D, const void* w, long V, int reduction,
                         const float* stats, const int* rows, const float* dloss, void* dx, void* dw, void* workspace,
                         hipStream_t stream) {
  MM_CE_CHECK("mm_ce_bwd");
  MM_CHECK_ARG(ldx >= 0 && reduction >= 0 && reduction <= 2, "bad reduction");
  MM_CHECK_ARG(T > 0 && x && w && stats && rows && dloss && workspace, "null pointer");
  if (!dx && !dw) return MM_OK;
  Backward b;
  backward_space(s, dx, dw, (char*)workspace, &b);
  const Rows r = rows_of((int*)rows, T);
  int rc = MM_OK;
  MM_DISPATCH(dtype, rc = backward<T_>(s, (const T_*)x, ldx, (const T_*)w, r, reduction, stats, dloss, (T_*)dx, (T_*)dw, b,
                                       stream));
  return rc;
}
