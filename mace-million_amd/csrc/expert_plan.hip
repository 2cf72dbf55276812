// The plan of the experts' products: slots, or rows of two choices, sorted by expert or pair of experts.
#include "experts.h"

// A stable counting sort by expert; slots without an expert are bucket E, at the end of the order.  Tiles of 4,096
// slots, each in the registers of one workgroup (16 a thread, loaded together).  Up to MM_PLAN_ONE tiles: one launch,
// whose workgroups count the other tiles' slots as well.  Beyond: the tiles' counts, then the scatter, whose
// workgroups add up the counts of all tiles themselves as long as that is at most MM_PLAN_SUM loads a thread; else a
// launch between them takes the prefix sums.  Bound by latency: 196,608 slots of 8 experts take 4.7 + 5.8 us, 98,304
// rows by pairs 4.9 + 7.4 us (0.8 MB in, 0.8 MB out: 0.3 us at HBM's rate).
#define MM_PLAN_TILE 4096
#define MM_PLAN_ONE 4
#define MM_PLAN_SUM 128

// Buckets of four consecutive slots of a tile, number 4 i of it on; -1 past the end.  PAIRS: of rows with two choices
// each, E being the number of buckets less one.
template <bool PAIRS>
__device__ __forceinline__ int4 mm_plan_load(const int* __restrict__ experts, int S, int E, int pairs_of, int tile,
                                             int i4) {
  const long s = (long)tile * MM_PLAN_TILE + 4 * i4;
  int v[4] = {-1, -1, -1, -1};
  if constexpr (PAIRS) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s + i < S) {
        const int a = experts[2 * (s + i)], b = experts[2 * (s + i) + 1];
        v[i] = mm_pair_bucket((unsigned)a < (unsigned)pairs_of ? a : pairs_of,
                              (unsigned)b < (unsigned)pairs_of ? b : pairs_of, pairs_of);
      }
  } else if (s + 4 <= S) {
    typedef int i4 __attribute__((ext_vector_type(4), aligned(4)));
    const i4 x = *(const i4*)(experts + s);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (unsigned)x[i] < (unsigned)E ? x[i] : E;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (s + i < S) v[i] = (unsigned)experts[s + i] < (unsigned)E ? experts[s + i] : E;
  }
  return make_int4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ void mm_plan_count(const int4& v, int* h) {
  if (v.x >= 0) atomicAdd(&h[v.x], 1);
  if (v.y >= 0) atomicAdd(&h[v.y], 1);
  if (v.z >= 0) atomicAdd(&h[v.z], 1);
  if (v.w >= 0) atomicAdd(&h[v.w], 1);
}

// counts[tile][bucket]
template <bool PAIRS>
__global__ void __launch_bounds__(1024) mm_plan_count_kernel(const int* __restrict__ experts, int S, int E,
                                                             int pairs_of, int* __restrict__ counts) {
  extern __shared__ int h[];
  const int4 v = mm_plan_load<PAIRS>(experts, S, E, pairs_of, blockIdx.x, threadIdx.x);
  for (int i = threadIdx.x; i <= E; i += 1024) h[i] = 0;
  __syncthreads();
  mm_plan_count(v, h);
  __syncthreads();
  for (int i = threadIdx.x; i <= E; i += 1024) counts[(size_t)blockIdx.x * (E + 1) + i] = h[i];
}

// one wave per bucket: its counts become exclusive prefix sums over the tiles, and the total
__global__ void __launch_bounds__(64) mm_plan_scan_kernel(int* __restrict__ counts, int tiles, int E,
                                                          int* __restrict__ totals) {
  const int e = blockIdx.x, lane = threadIdx.x;
  int carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += 64) {
    const int t = t0 + lane;
    const int v = t < tiles ? counts[(size_t)t * (E + 1) + e] : 0;
    int inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    if (t < tiles) counts[(size_t)t * (E + 1) + e] = carry + inc - v;
    carry += __shfl(inc, 63);
  }
  if (lane == 0) totals[e] = carry;
}

// threads of th side by side over the buckets (a power of two); the rest go over the tiles
__host__ __device__ inline int mm_plan_across(int buckets, int th) {
  int p = 1;
  while (p < buckets && p < th) p <<= 1;
  return p;
}

// One tile.  Each of the NW waves ranks its share of the slots, 64 consecutive ones at a time: one ballot per bit of
// the bucket finds the equals, the first of which takes places for all of them from the wave's counters.  Then the
// counters become places in the order.  Bound by the latency of these rounds, so as many waves as the counters leave
// room for share them (4 instead of 16: 12.6 us instead of 7.2 for 4,000 slots of 89 experts).  MODE 0:
// the other tiles are counted here; 1: the counts of all tiles are added up here; 2: counts are prefix sums, with the
// totals.  BITS: of the largest bucket, or more.
template <int MODE, int NW, int BITS, bool PAIRS>
__global__ void __launch_bounds__(64 * NW) mm_plan_kernel(const int* __restrict__ experts, int S, int E, int pairs_of,
                                                          int tiles,
                                                          const int* __restrict__ counts,
                                                          const int* __restrict__ totals, int* __restrict__ offsets,
                                                          int* __restrict__ order) {
  constexpr int TH = 64 * NW, SHARE = MM_PLAN_TILE / NW;
  extern __shared__ int sm[];
  __shared__ int s_e[MM_PLAN_TILE], s_at[MM_PLAN_TILE];
  const int B = E + 1;                                          // buckets
  int *cnt = sm, *total = sm + NW * B, *before = total + B;     // [NW][B], [B], [B]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < (NW + 2) * B; i += TH) sm[i] = 0;
  for (int i = tid; i < MM_PLAN_TILE / 4; i += TH)
    ((int4*)s_e)[i] = mm_plan_load<PAIRS>(experts, S, E, pairs_of, blockIdx.x, i);
  __syncthreads();
  if constexpr (MODE == 0) {
    for (int c = 0; c < tiles; ++c) {
      if (c == (int)blockIdx.x) continue;
      int* to = c < (int)blockIdx.x ? before : total;   // total: the tiles after this one, for now
      for (int i = tid; i < MM_PLAN_TILE / 4; i += TH)
        mm_plan_count(mm_plan_load<PAIRS>(experts, S, E, pairs_of, c, i), to);
    }
  }
  if constexpr (MODE == 1) {
    const int P = mm_plan_across(B, TH), G = TH / P, grp = tid / P;
    for (int i = tid % P; i < B; i += P) {
      int t = 0, f = 0;
#pragma unroll 8
      for (int c = grp; c < tiles; c += G) {
        const int v = counts[(size_t)c * B + i];
        t += v;
        f += c < (int)blockIdx.x ? v : 0;
      }
      atomicAdd(&total[i], t);
      atomicAdd(&before[i], f);
    }
  }
  if constexpr (MODE == 2)
    for (int i = tid; i < B; i += TH) {
      total[i] = totals[i];
      before[i] = counts[(size_t)blockIdx.x * B + i];
    }
  const int here = min(MM_PLAN_TILE, S - (int)blockIdx.x * MM_PLAN_TILE);   // slots of this tile
  const int end = min((wave + 1) * SHARE, here);
  // (the leaders' adds of one round are to different counters, those of successive rounds in order)
  for (int i = wave * SHARE + lane; i - lane < end; i += 64) {
    const int e = s_e[i];
    unsigned long long same = __ballot(e >= 0);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const unsigned long long m = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? m : ~m;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1)), first = __ffsll(same) - 1;
    int at = 0;
    if (e >= 0 && rank == 0) at = atomicAdd(&cnt[wave * B + e], (int)__popcll(same));
    at = __shfl(at, first & 63);
    s_at[i] = at + rank;
  }
  __syncthreads();
  if (wave == 0) {   // exclusive prefix sum of the buckets' totals
    int carry = 0;
    for (int e0 = 0; e0 < B; e0 += 64) {
      const int i = e0 + lane;
      int v = 0;
      if (i < B) {
        v = total[i];
        if constexpr (MODE == 0) {
          v += before[i];
#pragma unroll
          for (int w = 0; w < NW; ++w) v += cnt[w * B + i];
        }
      }
      int inc = v;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(inc, d);
        if (lane >= d) inc += u;
      }
      if (i < B) {
        total[i] = carry + inc - v;
        if (blockIdx.x == 0) offsets[i] = carry + inc - v;   // offsets[E] = slots with an expert
      }
      carry += __shfl(inc, 63);
    }
  }
  __syncthreads();
  for (int i = tid; i < B; i += TH) {
    int at = total[i] + before[i];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int c = cnt[w * B + i];
      cnt[w * B + i] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i = tid; i < here; i += TH) order[cnt[i / SHARE * B + s_e[i]] + s_at[i]] = blockIdx.x * MM_PLAN_TILE + i;
}

extern "C" int mm_expert_plan_scratch(int S, int E, long* ints) {
  MM_CHECK_ARG(S >= 0 && E >= 1 && ints, "bad sizes");
  const long tiles = ((long)S + MM_PLAN_TILE - 1) / MM_PLAN_TILE;
  *ints = tiles <= MM_PLAN_ONE ? 0 : (E + 1L) * (tiles + 1);   // counts, totals
  return MM_OK;
}

namespace {
// buckets 0 .. E; PAIRS: of S rows with two of pairs_of experts each, E + 1 = mm_pair_buckets(pairs_of)
template <bool PAIRS>
int launch_plan(const char* name, const int* experts, int S, int E, int pairs_of, int* offsets, int* order,
                int* scratch, hipStream_t stream) {
  const int tiles = (int)(((long)S + MM_PLAN_TILE - 1) / MM_PLAN_TILE), one = tiles <= MM_PLAN_ONE;
  MM_CHECK_ARG(one || scratch, "scratch is null");
  // 16 waves while their counters fit 64 KB of LDS beside the tile, else 4
  const int nw = E < 400 ? 16 : 4, th = 64 * nw, across = mm_plan_across(E + 1, th);
  const int lds = (nw + 2) * (E + 1) * (int)sizeof(int);
  int *counts = scratch, *totals = scratch + (size_t)tiles * (E + 1);
  if (!one)
    hipLaunchKernelGGL(mm_plan_count_kernel<PAIRS>, dim3(tiles), dim3(1024), (E + 1) * sizeof(int), stream, experts,
                       S, E, pairs_of, counts);
  const bool sums = ((long)tiles * across + th - 1) / th * ((E + across) / across) <= MM_PLAN_SUM;
  if (!one && !sums)
    hipLaunchKernelGGL(mm_plan_scan_kernel, dim3(E + 1), dim3(64), 0, stream, counts, tiles, E, totals);
#define CALL(mode, nw, bits)                                                                                 \
  hipLaunchKernelGGL((mm_plan_kernel<mode, nw, bits, PAIRS>), dim3(tiles ? tiles : 1), dim3(64 * nw), lds, stream, \
                     experts, S, E, pairs_of, tiles, counts, totals, offsets, order)
#define CALLS(mode)                      \
  if (nw == 4) CALL(mode, 4, 11);        \
  else if (E < 16) CALL(mode, 16, 4);    \
  else if (E < 128) CALL(mode, 16, 7);   \
  else CALL(mode, 16, 9);
  if (one) { CALLS(0) }
  else if (sums) { CALLS(1) }
  else { CALLS(2) }
#undef CALLS
#undef CALL
  return mm::launch_status(name);
}
}  // namespace

extern "C" int mm_expert_plan(const int* experts, int S, int E, int* offsets, int* order, int* scratch,
                              hipStream_t stream) {
  MM_CHECK_ARG(S >= 0 && E >= 1, "bad sizes");
  if (E > MM_EXPERT_MAX_E) return range_error("mm_expert_plan", "more than 1024 experts are not supported");
  MM_CHECK_ARG(S <= MM_PLAN_ONE * MM_PLAN_TILE || scratch, "scratch is null");
  return launch_plan<false>("mm_expert_plan", experts, S, E, 0, offsets, order, scratch, stream);
}

extern "C" int mm_expert_plan_pairs(const int* experts, int T, int E, int* offsets, int* order, int* scratch,
                                    hipStream_t stream) {
  MM_CHECK_ARG(T >= 0 && E >= 1, "bad sizes");
  if (E > MM_PAIRS_MAX_E) return range_error("mm_expert_plan_pairs", "pairs of more than 21 experts are not supported");
  MM_CHECK_ARG(T <= MM_PLAN_ONE * MM_PLAN_TILE || scratch, "scratch is null");
  return launch_plan<true>("mm_expert_plan_pairs", experts, T, mm_pair_buckets(E) - 1, E, offsets, order, scratch,
                           stream);
}

