// dW[e] = sum over the slots of expert e and their components of gate x^T dy.
#include "experts.h"

struct MMWgrad {
  const void *x, *dy;
  const float* gates;
  const int *offsets, *order;
  void* dW;
  long xt, xm, yt, ym;
  int k, M, D, F, E;
};

// A workgroup: a BD x BF tile of dW[e] over a chunk of the expert's rows (SPLIT: chunks of `chunk` rows, each into its
// own fp32 partial sums, which mm_expert_wgrad_sum_kernel adds in order; else all rows, straight into dW).  x and dy go
// into LDS as they are, float dy times its gate.  16-bit types with gates (GATED): gate x dy, taken in fp32, would lose
// bits and, in float16, its range if it were rounded to the type, so it enters the products as two bf16 parts
// (mm_products_gated).  Rows past the end are zeros on both sides.  Bound by the waits between stages and the vector
// instructions of the split: 65,536 rows, 64 blocks of 1024 x 1024, 2 of 64: bfloat16 380 us, float16 535 us (without
// gates 250 us, 550 TFLOP/s: one product instead of two or three); 98,304 float rows, 16 blocks of 128 x 128 41 + 7 us.
// Tiles of 64 where a side has no more (407,520 float rows 112 x 32: 140 -> 97 us).
#define MM_WG_ROWS 512   // rows whose offsets are kept in LDS at a time

template <typename T, bool SPLIT, bool DMA, bool GATED, int BD, int BF, int WD, int WF>
__global__ void __launch_bounds__(64 * WD * WF, 2) mm_expert_wgrad_kernel(MMWgrad a, int chunk, int tiles_f,
                                                                          int tiles_df, float* __restrict__ part) {
  constexpr int TH = 64 * WD * WF, BK = MM_TILE_K<T>, N = MMVec<T>::N, UD = BD / N, UF = BF / N, KS = BK / 32;
  constexpr int NX = BD * 8 / TH, NY = BF * 8 / TH, FD = BD / WD / 16, FF = BF / WF / 16;
  constexpr bool YDMA = BD == 256;   // the 256 x 256 tiles have no registers for dy on its way
  extern __shared__ uint4 mm_lds[];
  uint4 *Xs = mm_lds, *Ys = Xs + 2 * BD * 8;             // [2][BD * 8], [2][BF * 8]
  long *s_x = (long*)(Ys + 2 * BF * 8), *s_y = s_x + MM_WG_ROWS;
  float *s_g = (float*)(s_y + MM_WG_ROWS), *s_gate = s_g + MM_WG_ROWS;   // s_gate [2][BK]: of the stages (GATED)
  const int lane_id = threadIdx.x & 63;
  int df, tile;
  MMTile t;
  if constexpr (SPLIT) {
    t = mm_expert_tile(a.offsets, a.E, a.offsets[a.E], a.M, chunk, tiles_df, blockIdx.x, &df, &tile);
    if (t.e < 0) return;
  } else {
    // Each list is read by one XCD, whose L2 serves all tiles of dW[e].  The longest lists first, dealt out to the
    // XCDs forth and back, so that they end together (64 experts at most; beyond that every 8th as they come).  Lists
    // of uneven load (lognormal, 0.7), 64 experts, 1024 x 1024: 338 us in the order of the experts, 279 us so.
    const int x = blockIdx.x & 7, i = blockIdx.x >> 3, turn = i / tiles_df;
    tile = 8 * turn + x;
    df = i % tiles_df;
    if (tile >= a.E) return;
    if (a.E <= 64) {
      const int own = lane_id < a.E ? a.offsets[lane_id + 1] - a.offsets[lane_id] : -1;
      int rank = 0;
      for (int o = 0; o < a.E; ++o) {
        const int other = __builtin_amdgcn_readlane(own, o);
        rank += other > own || (other == own && o < lane_id);
      }
      const int snake = turn & 1 ? 8 * turn + 7 - x : tile;
      const int want = snake < a.E ? snake : tile;
      const unsigned long long is = __ballot(lane_id < a.E && rank == want);
      tile = __ffsll(is) - 1;
    }
    t = MMTile{tile, 0, (a.offsets[tile + 1] - a.offsets[tile]) * a.M};
  }
  const int d0 = df / tiles_f * BD, f0 = df % tiles_f * BF;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int* __restrict__ list = a.order + a.offsets[t.e];
  int qx[NX], left_d[NX], cx[NX], qy[NY], left_f[NY], cy[NY];
#pragma unroll
  for (int j = 0; j < NX; ++j) {
    const int pu = tid + TH * j;
    qx[j] = pu / UD;
    cx[j] = ((pu % UD) ^ mm_nc_swizzle<T, UD>(qx[j])) * N;
    left_d[j] = a.D - d0 - cx[j];
  }
#pragma unroll
  for (int j = 0; j < NY; ++j) {
    const int pu = tid + TH * j;
    qy[j] = pu / UF;
    cy[j] = ((pu % UF) ^ mm_nc_swizzle<T, UF>(qy[j])) * N;
    left_f[j] = a.F - f0 - cy[j];
  }
  MMStage<T, TH, NX, DMA> sx;
  MMStage<T, TH, NY, YDMA> sy;
  float gy[NY];
  auto load = [&](int r0, int buf) {   // rows r0 .. r0 + BK of the chunk, within one block of offsets
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const bool in = r0 + qx[j] < t.rows;
      const long at_x = in ? s_x[(r0 + qx[j]) & (MM_WG_ROWS - 1)] : 0;
      sx.load(Xs + buf * BD * 8, j, (const T*)a.x + at_x + d0 + cx[j], in ? left_d[j] : 0);
    }
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      const bool in = r0 + qy[j] < t.rows;
      const int r = (r0 + qy[j]) & (MM_WG_ROWS - 1);
      sy.load(Ys + buf * BF * 8, j, (const T*)a.dy + (in ? s_y[r] : 0) + f0 + cy[j], in ? left_f[j] : 0);
      gy[j] = in ? s_g[r] : 0.f;
    }
    if (GATED && tid < BK) s_gate[buf * BK + tid] = r0 + tid < t.rows ? s_g[(r0 + tid) & (MM_WG_ROWS - 1)] : 0.f;
  };
  auto put = [&](int buf) {
    sx.put(Xs + buf * BD * 8);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < NY; ++j) {
        floatx4 v = __builtin_bit_cast(floatx4, sy.v[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = gy[j] * v[i];
        sy.v[j] = __builtin_bit_cast(uint4, v);
      }
    }
    sy.put(Ys + buf * BF * 8);
  };
  auto rows_of = [&](int r0) {
    for (int i = tid; i < MM_WG_ROWS && r0 + i < t.rows; i += TH) {
      const int r = t.row0 + r0 + i, p = r / a.M, m = r - p * a.M, slot = list[p];
      const long tok = slot / a.k;
      s_x[i] = tok * a.xt + m * a.xm;
      s_y[i] = tok * a.yt + m * a.ym;
      s_g[i] = a.gates ? a.gates[slot] : 1.f;
    }
    __syncthreads();
  };
  floatx4 acc[FF][FD] = {};
  const int wd = (wave % WD) * (BD / WD), wf = (wave / WD) * (BF / WF);
  if (t.rows > 0) {
    rows_of(0);
    load(0, 0);
    put(0);
    mm_stage_done();
  }
  int buf = 0;
  for (int r0 = 0; r0 < t.rows; r0 += BK) {
    const int next = r0 + BK;
    const bool more = next < t.rows;
    if (more) {
      if (next % MM_WG_ROWS == 0) rows_of(next);   // the previous block's offsets are used up (the last barrier)
      load(next, buf ^ 1);
    }
    auto y_of = [&](int s, int i) { return mm_read_nc<T, UF>(Ys + buf * BF * 8, wf + 16 * i, s, lane); };
    auto x_of = [&](int s, int j) { return mm_read_nc<T, UD>(Xs + buf * BD * 8, wd + 16 * j, s, lane); };
    if constexpr (GATED) mm_products_gated<T, FF, FD, KS>(acc, y_of, x_of, s_gate + buf * BK, lane);
    else mm_products<T, FF, FD, KS>(acc, y_of, x_of);
    if (more) put(buf ^ 1);
    mm_stage_done();
    buf ^= 1;
  }
  const size_t base = SPLIT ? (size_t)tile * a.D * a.F : (size_t)t.e * a.D * a.F;
#pragma unroll
  for (int j = 0; j < FD; ++j) {
    const int d = d0 + wd + 16 * j + (lane & 15);
    if (d >= a.D) continue;
#pragma unroll
    for (int i = 0; i < FF; ++i) {
      const int f = f0 + wf + 16 * i + 4 * (lane >> 4);
      if constexpr (SPLIT) mm_store4(part + base + (size_t)d * a.F, f, a.F, (const float*)&acc[i][j]);
      else mm_store4((T*)a.dW + base + (size_t)d * a.F, f, a.F, (const float*)&acc[i][j]);
    }
  }
}

// dW[e] = the partial sums of the expert's chunks, in a fixed order.  V values a thread: 4 where that leaves threads
// for the card, from 2^19 values on (89 x 201 x 137: 11.6 -> 6.6 us; 16 x 128 x 128 would take 19 instead of 8).  G
// waves share the chunks: 4 where the values alone are too few, below 2^18 (2 x 216 x 72: 8 -> 5 us; 16 x 128 x 128: 8
// -> 9.7).
template <typename T, int V, int G>
__global__ void __launch_bounds__(256) mm_expert_wgrad_sum_kernel(MMWgrad a, int chunk,
                                                                  const float* __restrict__ part) {
  constexpr int COLUMNS = 256 / G * V;
  __shared__ float s_t[G][G > 1 ? 64 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.y;
  int first = 0;   // chunks of the experts before e
  for (int o = lane; o < e; o += 64) first += mm_pieces((a.offsets[o + 1] - a.offsets[o]) * a.M, chunk);
#pragma unroll
  for (int d = 32; d; d >>= 1) first += __shfl_xor(first, d);
  const int n = mm_pieces((a.offsets[e + 1] - a.offsets[e]) * a.M, chunk);
  const long size = (long)a.D * a.F, i = (long)blockIdx.x * COLUMNS + (G > 1 ? lane : V * (int)threadIdx.x);
  const int left = (int)(size - i < V ? size - i : V);
  const float* __restrict__ p = part + (size_t)first * size + i;
  float t[V] = {};
  if (left > 0) {
#pragma unroll 8
    for (int c = G > 1 ? wave : 0; c < n; c += G) {
      float v[V];
      if constexpr (V == 1) v[0] = p[c * size];
      else mm_load4(p + c * size, 0, left, v);
#pragma unroll
      for (int q = 0; q < V; ++q) t[q] += v[q];
    }
  }
  if constexpr (G > 1) {
    s_t[wave][lane] = t[0];
    __syncthreads();
    if (wave) return;
    t[0] = s_t[0][lane] + s_t[1][lane] + s_t[2][lane] + s_t[3][lane];
  }
  if (left <= 0) return;
  T* __restrict__ o = (T*)a.dW + (size_t)e * size + i;
  if constexpr (V == 1) *o = (T)t[0];
  else mm_store4(o, 0, left, t);
}

// ------------------------------------------------------------------------------------------------ entry points
namespace {
// two stages of both operands, then the offsets and gates of a block of rows, then the gates of two stages
template <int BD, int BF, int BK>
constexpr int wgrad_lds() { return 2 * (BD + BF) * 128 + MM_WG_ROWS * 20 + 2 * BK * 4; }

template <typename T, bool SPLIT, bool DMA, bool GATED, int BD, int BF, int WD, int WF>
int launch_wgrad_tile(const MMWgrad& a, int S, int chunk, float* part, hipStream_t stream) {
  const int tiles_f = (a.F + BF - 1) / BF, tiles_df = (a.D + BD - 1) / BD * tiles_f;
  const long wg = (SPLIT ? (long)S * a.M / chunk + (a.E < S ? a.E : S) : (a.E + 7L) / 8 * 8) * tiles_df;
  if (too_many(wg, 64 * WD * WF)) return range_error("mm_expert_wgrad", "output too large for one launch");
  constexpr auto kernel = mm_expert_wgrad_kernel<T, SPLIT, DMA, GATED, BD, BF, WD, WF>;
  constexpr int lds = wgrad_lds<BD, BF, MM_TILE_K<T>>();
  if (!lds_granted<kernel>(lds)) return MM_ELAUNCH;
  if (wg)
    hipLaunchKernelGGL(kernel, dim3((unsigned)wg), dim3(64 * WD * WF), lds, stream, a, chunk, tiles_f, tiles_df, part);
  return mm::launch_status("mm_expert_wgrad");
}

template <typename T, bool SPLIT, bool DMA, bool GATED>
int launch_wgrad_tiles(const MMWgrad& a, int S, int chunk, bool big, float* part, hipStream_t stream) {
  if constexpr (sizeof(T) == 2 && DMA && !SPLIT)
    if (big) return launch_wgrad_tile<T, SPLIT, DMA, GATED, 256, 256, 2, 4>(a, S, chunk, part, stream);
  if (a.D <= 64) {
    if (a.F <= 64) return launch_wgrad_tile<T, SPLIT, DMA, GATED, 64, 64, 2, 2>(a, S, chunk, part, stream);
    return launch_wgrad_tile<T, SPLIT, DMA, GATED, 64, 128, 2, 2>(a, S, chunk, part, stream);
  }
  if (a.F <= 64) return launch_wgrad_tile<T, SPLIT, DMA, GATED, 128, 64, 2, 2>(a, S, chunk, part, stream);
  return launch_wgrad_tile<T, SPLIT, DMA, GATED, 128, 128, 2, 2>(a, S, chunk, part, stream);
}

template <typename T, bool SPLIT, bool DMA>
int launch_wgrad(const MMWgrad& a, int S, int chunk, bool big, float* part, hipStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (a.gates) return launch_wgrad_tiles<T, SPLIT, DMA, true>(a, S, chunk, big, part, stream);
  return launch_wgrad_tiles<T, SPLIT, DMA, false>(a, S, chunk, big, part, stream);
}

// Rows per chunk of dW's sums; 0: no chunks.  A card of 256 CUs takes 512 workgroups at a time: with at least that
// many (expert, tile) pairs none are made; else chunks that fill those 512 once, of 128 rows or more, with room for the
// lists' cut chunks (half of one each on average, and 32 as these vary: a few workgroups past the 512 cost a second
// round, 24,544 bfloat16 rows 341 x 387 58 -> 72 us).  In us with the sums, against about 1024 workgroups and 256 rows
// or more: 72,166 bfloat16 rows 443 x 191, 12 experts 115 -> 86, 98,304 float rows 128 x 128, 16 experts 51 -> 50,
// 12,000 float rows 128 x 128, 16 experts 31 -> 23.
int wgrad_chunk(long rows, int D, int F, int E) {
  const long tiles = (long)((D + 127) / 128) * ((F + 127) / 128);
  if (E * tiles >= 512 || rows < 512) return 0;
  const long room = 480 - tiles * E / 2, wg = room < 128 ? 128 : room, c = (rows * tiles + wg - 1) / wg;
  return (int)(c < 128 ? 128 : ((c < rows ? c : rows) + 31) / 32 * 32);
}
}  // namespace

extern "C" int mm_expert_wgrad_workspace(int S, int M, int D, int F, int E, size_t* bytes) {
  MM_CHECK_ARG(S >= 0 && M >= 1 && D >= 1 && F >= 1 && E >= 1 && bytes, "bad sizes");
  if ((long)S * M > MM_EXPERT_MAX_ROWS) return range_error("mm_expert_wgrad_workspace", TOO_MANY_ROWS);
  if (too_wide(D, F)) return range_error("mm_expert_wgrad_workspace", TOO_WIDE);
  const long rows = (long)S * M, c = wgrad_chunk(rows, D, F, E);
  *bytes = c ? (size_t)(rows / c + (E < S ? E : S)) * D * F * sizeof(float) : 0;
  return MM_OK;
}

extern "C" int mm_expert_wgrad(const void* x, long xt, long xm, const void* dy, long yt, long ym, int dtype, int S,
                               int k, int M, int D, int F, int E, const float* gates, const int* offsets,
                               const int* order, void* dW, float* workspace, hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(S >= 0 && k >= 1 && M >= 1 && D >= 1 && F >= 1 && E >= 1, "bad sizes");
  MM_CHECK_ARG(xt >= 0 && xm >= 0 && yt >= 0 && ym >= 0, "bad strides");
  if (E > MM_EXPERT_MAX_E) return range_error("mm_expert_wgrad", "more than 1024 experts are not supported");
  if ((long)S * M > MM_EXPERT_MAX_ROWS) return range_error("mm_expert_wgrad", TOO_MANY_ROWS);
  if (too_wide(D, F)) return range_error("mm_expert_wgrad", TOO_WIDE);
  MM_CHECK_ARG(offsets && dW && (S == 0 || (x && dy && order)), "a pointer is null");
  const MMWgrad a{x, dy, gates, offsets, order, dW, xt, xm, yt, ym, k, M, D, F, E};
  const int chunk = wgrad_chunk((long)S * M, D, F, E);
  MM_CHECK_ARG(!chunk || workspace, "workspace is null");
  const int unit = dtype == MM_F32 ? 4 : 8;
  const bool dma = aligned(x) && xt % unit == 0 && (M == 1 || xm % unit == 0) && D % unit == 0;
  int rc = MM_OK;
#define CALL(split, dma)                                                                              \
  if (dtype == MM_F32) rc = launch_wgrad<float, split, dma>(a, S, chunk, false, workspace, stream);   \
  else if (dtype == MM_BF16) rc = launch_wgrad<__bf16, split, dma>(a, S, chunk, big, workspace, stream); \
  else rc = launch_wgrad<_Float16, split, dma>(a, S, chunk, big, workspace, stream);
  const bool dma_y = aligned(dy) && yt % unit == 0 && (M == 1 || ym % unit == 0) && F % unit == 0;
  const bool big = dma && dma_y && !chunk && D > 128 && F > 128 && E * ((D + 255) / 256) * ((F + 255) / 256) >= 512;
  if (chunk) { if (dma) { CALL(true, true) } else { CALL(true, false) } }
  else { if (dma) { CALL(false, true) } else { CALL(false, false) } }
#undef CALL
  if (rc != MM_OK) return rc;
  const long size = (long)D * F;
#define SUM(v, g)                                                                                               \
  MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_wgrad_sum_kernel<T_, v, g>),                                 \
                                        dim3((unsigned)((size + 256 / g * v - 1) / (256 / g * v)), E), dim3(256), 0, \
                                        stream, a, chunk, workspace))
  if (chunk) {
    if (E * size < 1 << 18) SUM(1, 4);
    else if (E * size < 1 << 19) SUM(1, 1);
    else SUM(4, 1);
  }
#undef SUM
  return mm::launch_status("mm_expert_wgrad");
}
