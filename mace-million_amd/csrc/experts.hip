// Products of rows with the weight blocks of their experts:  y[t, m] = sum_j gate[t, j] x[t, m] @ W[expert[t, j]],
// with the gradients of x, W and the gates.  A slot is a (row, choice) pair s = t k + j; the plan lists the slots sorted
// by expert (stable), so that each expert's rows are consecutive and its block is read once per tile of rows.
//   mm_expert_plan     offsets [E + 1] and order [S]: the slots of expert e are order[offsets[e] .. offsets[e + 1])
//   mm_expert_rows     out[s, m] = in[s / k, m] @ W[e]  (or @ W[e]^T): fp32 rows in slot order
//   mm_expert_combine  y[t, m] = sum_j gate rows[t k + j, m];  mm_expert_combine_bwd  dx and dgates from the rows of dy
//   mm_expert_wgrad    dW[e] = sum of the expert's slots and components of gate x^T dy
// A slot whose expert lies outside [0, E) takes part nowhere.
#include "rowvec.h"

#include <atomic>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));

#define MM_EXPERT_MAX_E 1024
#define MM_PAIRS_MAX_E 21   // 253 pairs

// ------------------------------------------------------------------------------------------------ plan
// A stable counting sort by expert; slots without an expert are bucket E, at the end of the order.  Tiles of 4,096 slots,
// each in the registers of one workgroup (16 a thread, loaded together).  Up to MM_PLAN_ONE tiles: one launch, whose
// workgroups count the other tiles' slots as well.  Beyond: the tiles' counts, then the scatter, whose workgroups add up
// the counts of all tiles themselves as long as that is at most MM_PLAN_SUM loads a thread; else a launch between them
// takes the prefix sums.
#define MM_PLAN_TILE 4096
#define MM_PLAN_ONE 4
#define MM_PLAN_SUM 128

// Bucket of a pair of choices among E experts and none (number E), in any order: rows e1 <= e2 of a triangle, the pair of
// no expert at all last.
__host__ __device__ inline int mm_pair_bucket(int e1, int e2, int E) {
  const int lo = e1 < e2 ? e1 : e2, hi = e1 < e2 ? e2 : e1;
  return lo * (E + 1) - lo * (lo - 1) / 2 + hi - lo;
}
__host__ __device__ inline int mm_pair_buckets(int E) { return (E + 1) * (E + 2) / 2; }

// Buckets of four consecutive slots of a tile, number 4 i of it on; -1 past the end.  PAIRS: of rows with two choices each,
// E being the number of buckets less one.
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
__global__ void __launch_bounds__(1024) mm_plan_count_kernel(const int* __restrict__ experts, int S, int E, int pairs_of,
                                                             int* __restrict__ counts) {
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

// One tile.  Each of the NW waves ranks its share of the slots, 64 consecutive ones at a time: one ballot per bit of the
// bucket finds the equals, the first of which takes places for all of them from the wave's counters.  Then the counters
// become places in the order.  Bound by the latency of these rounds, so as many waves as the counters leave room for
// share them (4 instead of 16: 12.6 us instead of the figure below for 4,000 slots of 89 experts).  MODE 0: the other tiles are counted here; 1: the counts of all
// tiles are added up here; 2: counts are prefix sums, with the totals.  BITS: of the largest bucket, or more.
template <int MODE, int NW, int BITS, bool PAIRS>
__global__ void __launch_bounds__(64 * NW) mm_plan_kernel(const int* __restrict__ experts, int S, int E, int pairs_of, int tiles,
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
  for (int i = tid; i < MM_PLAN_TILE / 4; i += TH) ((int4*)s_e)[i] = mm_plan_load<PAIRS>(experts, S, E, pairs_of, blockIdx.x, i);
  __syncthreads();
  if constexpr (MODE == 0) {
    for (int c = 0; c < tiles; ++c) {
      if (c == (int)blockIdx.x) continue;
      int* to = c < (int)blockIdx.x ? before : total;   // total: the tiles after this one, for now
      for (int i = tid; i < MM_PLAN_TILE / 4; i += TH) mm_plan_count(mm_plan_load<PAIRS>(experts, S, E, pairs_of, c, i), to);
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

// ------------------------------------------------------------------------------------------------ tiles of an expert
struct MMTile {
  int e, row0, rows;   // expert, first of its rows (slots x M), rows in the tile; e < 0: no such tile
};

// Workgroup b of `per` for each of the tiles of BM rows that the row lists of the buckets have (every list ends in a cut
// tile); list i: entries offsets[i] .. offsets[i + 1], the last one to `end`, M rows each.  Every wave finds its tile by
// itself, 64 lists at a time.  Workgroups are dealt out to the 8 XCDs in turn; the work is numbered so that an XCD gets
// consecutive pieces, whose operands its L2 then holds.
__device__ __forceinline__ MMTile mm_expert_tile(const int* __restrict__ offsets, int lists, int end, int M, int BM,
                                                 int per, int b, int* part, int* number) {
  const int lane = threadIdx.x & 63;
  auto rows_of = [&](int i) {
    if (i >= lists) return 0;
    return ((i + 1 < lists ? offsets[i + 1] : end) - offsets[i]) * M;
  };
  const int head = rows_of(lane);
  int all = (head + BM - 1) / BM;
#pragma unroll 4
  for (int i = 64 + lane; i - lane < lists; i += 64) all += (rows_of(i) + BM - 1) / BM;
#pragma unroll
  for (int d = 32; d; d >>= 1) all += __shfl_xor(all, d);
  all *= per;
  if (b >= all) return MMTile{-1, 0, 0};
  const int share = all / 8, rest = all % 8, x = b % 8;
  const int at = x * share + min(x, rest) + b / 8;
  int tile = at / per;
  *part = at - tile * per;
  *number = tile;
  for (int i0 = 0; i0 < lists; i0 += 64) {
    const int rows = i0 ? rows_of(i0 + lane) : head, n = (rows + BM - 1) / BM;
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
      return MMTile{i0 + src, first, min(BM, total - first)};
    }
    tile -= __shfl(inc, 63);
  }
  return MMTile{-1, 0, 0};
}

// ------------------------------------------------------------------------------------------------ matrix products
// Operands of v_mfma_f32_16x16x32 (fp32 sums): lane (i, g) = (lane & 15, lane >> 4) holds the values k = 8 g .. 8 g + 7 of
// row (column) i.  16-bit types: one product.  float: three bf16 planes x = x0 + x1 + x2 (x0 = bf16(x), x1 = bf16(x - x0),
// x2 = bf16(x - x0 - x1), |x - x0 - x1 - x2| <= 2^-27 |x|) and the six products a_i b_j with i + j <= 2; those left out
// are below 3 * 2^-24 |a b|.  96 matrix cycles for 16 x 16 x 32 against 256 in fp32 products.
template <typename T>
struct MMFrag {
  typedef T vec __attribute__((ext_vector_type(8)));
  vec v;
};
template <>
struct MMFrag<float> {
  bf16x8 v[3];
};

__device__ __forceinline__ void mm_mma(floatx4& c, const MMFrag<__bf16>& a, const MMFrag<__bf16>& b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ void mm_mma(floatx4& c, const MMFrag<_Float16>& a, const MMFrag<_Float16>& b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ void mm_mma(floatx4& c, const MMFrag<float>& a, const MMFrag<float>& b) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[2], b.v[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[1], b.v[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[0], b.v[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[1], b.v[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[0], b.v[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[0], b.v[0], c, 0, 0, 0);
}

// an operand as it comes out of LDS
template <typename T>
struct MMRaw {
  MMFrag<T> f;
};
template <>
struct MMRaw<float> {
  float x[8];
};

// float operands may be scaled on the way
template <typename T, bool SCALED = false>
__device__ __forceinline__ MMFrag<T> mm_operand(const MMRaw<T>& r, float scale = 1.f) {
  if constexpr (sizeof(T) == 2) {
    return r.f;
  } else {
    MMFrag<float> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = SCALED ? scale * r.x[i] : r.x[i];
      const __bf16 h = (__bf16)x;
      const float d = x - (float)h;
      const __bf16 l = (__bf16)d;
      f.v[0][i] = h;
      f.v[1][i] = l;
      f.v[2][i] = (__bf16)(d - (float)l);
    }
    return f;
  }
}

// acc[i][j] += a(s, i) b(s, j) scale[j] over the KS steps of a stage (SCALED: float only): operands b are read two ahead of their products and turned
// into planes one ahead, the next step's operands a over the last products of this one.  The scheduling barriers keep the
// reads there: left alone, the compiler reads two operands, waits for them and multiplies.
template <typename T, int FN, int FM, int KS, bool SCALED = false, typename A, typename B>
__device__ __forceinline__ void mm_products(floatx4 (&acc)[FN][FM], A a, B b, const float* scale = nullptr) {
  auto second = [&](const MMRaw<T>& r, int j) { return mm_operand<T, SCALED>(r, SCALED ? scale[j] : 1.f); };
  constexpr int Q = KS * FM;
  MMFrag<T> fa[KS > 1 ? 2 : 1][FN], fb[2];
  MMRaw<T> rb[3];
  {
    MMRaw<T> ra[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) ra[i] = a(0, i);
    rb[0] = b(0, 0);
    rb[1] = b(1 / FM, 1 % FM);
#pragma unroll
    for (int i = 0; i < FN; ++i) fa[0][i] = mm_operand(ra[i]);
    fb[0] = second(rb[0], 0);
  }
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int s = q / FM, j = q % FM;
    if (q + 2 < Q) rb[(q + 2) % 3] = b((q + 2) / FM, (q + 2) % FM);
    if constexpr (KS > 1) {
      if (s + 1 < KS) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
          if ((FN < FM ? i + FM - FN : i * FM / FN) == j) fa[(s + 1) & 1][i] = mm_operand(a(s + 1, i));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (q + 1 < Q) fb[(q + 1) & 1] = second(rb[(q + 1) % 3], (q + 1) % FM);
#pragma unroll
    for (int i = 0; i < FN; ++i) mm_mma(acc[i][j], fa[KS > 1 ? s & 1 : 0][i], fb[q & 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Tiles in LDS, in units of 16 bytes.  MM_TILE_K<T> values of the summed index a stage.
//   KC (the summed index contiguous in memory): a row of 8 units (128 bytes), unit u of row r at 8 r + (u ^ (r & 7)): the
//   16 rows of an operand read spread over all banks.
//   NC (the other index contiguous): a row per value of the summed index, UPR units; unit u of row q at UPR q + (u ^ s(q)),
//   s(q) chosen so that the rows read together lie in different banks.  16-bit operands come out of it by transposing
//   reads (ds_read_b64_tr_b16: 16 lanes give the addresses of a 4 x 16 block, four lanes a row, and lane i receives its
//   column i), float operands value by value.
// Staged by loads straight into LDS (16 bytes a lane, the wave's units in order, so the swizzle is in the addresses of
// the sources) where the units are aligned, else through registers.
template <typename T>
constexpr int MM_TILE_K = 128 / sizeof(T);

typedef __attribute__((address_space(3))) void* mm_lds_ptr;
typedef const __attribute__((address_space(1))) void* mm_global_ptr;

__device__ uint4 mm_zero_unit;   // source of units outside the operands (zero-initialised, never written)

template <typename T, int UPR>
__device__ __forceinline__ int mm_nc_swizzle(int q) {
  if constexpr (sizeof(T) == 2) return ((q & 3) | (q >> 3 & 1) << 2) << 1 & (UPR - 1);
  else return (q >> 3 & 3) << 2 & (UPR - 1);
}

// operand rows n0 + i, values 32 s + 8 g .. of a KC tile
template <typename T>
__device__ __forceinline__ MMRaw<T> mm_read_kc(const uint4* tile, int n0, int s, int lane) {
  const int r = n0 + (lane & 15), g = lane >> 4;
  if constexpr (sizeof(T) == 2) {
    MMRaw<T> f;
    f.f.v = __builtin_bit_cast(typename MMFrag<T>::vec, tile[8 * r + ((4 * s + g) ^ (r & 7))]);
    return f;
  } else {
    MMRaw<T> f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const floatx4 v = __builtin_bit_cast(floatx4, tile[8 * r + ((2 * g + h) ^ (r & 7))]);
#pragma unroll
      for (int i = 0; i < 4; ++i) f.x[4 * h + i] = v[i];
    }
    return f;
  }
}

// operand columns n0 + i, values 32 s + 8 g .. of an NC tile
template <typename T, int UPR>
__device__ __forceinline__ MMRaw<T> mm_read_nc(const uint4* tile, int n0, int s, int lane) {
  const int i = lane & 15, g = lane >> 4;
  if constexpr (sizeof(T) == 2) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    s4 h[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int q = 32 * s + 8 * g + 4 * b + (i >> 2);
      const char* p = (const char*)&tile[UPR * q + ((n0 / 8 + (i >> 1 & 1)) ^ mm_nc_swizzle<T, UPR>(q))] + 8 * (i & 1);
      h[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
    }
    MMRaw<T> f;
    f.f.v = __builtin_bit_cast(typename MMFrag<T>::vec, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    return f;
  } else {
    MMRaw<T> f;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const int q = 8 * g + b, n = n0 + i;
      f.x[b] = ((const float*)&tile[UPR * q + ((n >> 2) ^ mm_nc_swizzle<T, UPR>(q))])[n & 3];
    }
    return f;
  }
}

// A thread's share of staging one tile by TH threads: NU units, unit number tid + TH j.  DMA: straight into LDS.
template <typename T, int TH, int NU, bool DMA>
struct MMStage {
  uint4 v[DMA ? 1 : NU];

  // unit j from p (left = values of T left at p; none: zeros)
  __device__ __forceinline__ void load(uint4* tile, int j, const T* p, int left) {
    constexpr int N = MMVec<T>::N;
    if constexpr (DMA) {
      const void* src = left > 0 ? (const void*)p : (const void*)&mm_zero_unit;
      __builtin_amdgcn_global_load_lds((mm_global_ptr)src, (mm_lds_ptr)(tile + TH * j + (threadIdx.x & ~63)), 16, 0, 0);
    } else {
      typename MMVec<T>::type x;
      if (left >= N) {
        x = *(const typename MMVec<T>::type*)p;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? p[i] : (T)0.f;
      }
      v[j] = __builtin_bit_cast(uint4, x);
    }
  }
  __device__ __forceinline__ void put(uint4* tile) {
    if constexpr (!DMA) {
#pragma unroll
      for (int j = 0; j < NU; ++j) tile[TH * j + threadIdx.x] = v[j];
    }
  }
};

// every load into LDS of this wave has arrived, and every wave's (and its LDS accesses are done)
__device__ __forceinline__ void mm_stage_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------ rows
struct MMRows {
  const void *in, *W;
  const int *offsets, *order;
  float* out;
  long st, sm;   // strides of in in elements: rows, components
  int k, M, K, N, E;
};

// A workgroup: a tile of BM rows of one expert by BN columns, its WM x WN waves with BM / WM x BN / WN each, two stages in
// LDS: the next stage is on its way while this one is multiplied.  The weights are the first operand, so that a lane ends
// with 4 consecutive columns of a row.  TRANS: W[e] is [N][K], else [K][N].
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

// ------------------------------------------------------------------------------------------------ held blocks
// Float rows of up to 128 values: the products of mm_expert_rows with the block in registers.  A workgroup is 4 waves; each
// holds 32 of 128 columns of its expert's block, split into planes (96 registers at K = 128), and streams up to `chunk` of
// the expert's rows past them, 32 (a stage) at a time.  A stage is loaded by the whole workgroup, split once and written
// to LDS in operand order, one stage ahead of the products and two ahead in registers, so an operand is split once where the tiles of
// mm_expert_rows split it in every wave, and the block is read once per chunk.  Bound by the products and the rows'
// traffic.  With gates (one choice a row) the rows are the result itself; list E, the slots without an expert, is then
// written as zeros.
#define MM_HELD_ROWS 1024   // rows of a workgroup at most
#define MM_HELD_AS 17       // LDS distance (16 B) of the groups of 8 values of a row tile: every bank once

struct MMHeld {
  MMRows r;
  const float* gates;
  int lists, S;   // E, or E + 1 with the slots without an expert
};

// four values of a row, number 4 k4 on, into the planes of a stage
template <int KG>
__device__ __forceinline__ void mm_held_put(uint4* stage, int row, int k4, const float (&x)[4]) {
  typedef __bf16 b4 __attribute__((ext_vector_type(4)));
  b4 v[3];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const __bf16 hi = (__bf16)x[q];
    const float d = x[q] - (float)hi;
    const __bf16 mid = (__bf16)d;
    v[0][q] = hi;
    v[1][q] = mid;
    v[2][q] = (__bf16)(d - (float)mid);
  }
#pragma unroll
  for (int p = 0; p < 3; ++p)
    ((uint2*)&stage[(((row >> 4) * 3 + p) * KG + (k4 >> 1)) * MM_HELD_AS + (row & 15)])[k4 & 1] =
        __builtin_bit_cast(uint2, v[p]);
}

// KS: steps of 32 values.  FULL: K = 32 KS and whole tiles of columns, so that no load or store stands behind a branch: the
// compiler then counts them and waits for the loads it needs only, not for the stores before them.  One row's 8 values g of step t, plane p at unit ((tile * 3 + p) * 4 KS + 4 t + g) * 17 + row.
template <bool TRANS, int KS, bool FULL>
__global__ void __launch_bounds__(256, 2) mm_expert_held_kernel(MMHeld h, int tiles_n, int chunk) {
  constexpr int KG = 4 * KS, UNITS = 2 * 3 * KG * MM_HELD_AS, PER = KS;   // float4 a thread and stage: 32 * 8 KS / 256
  __shared__ uint4 Al[2][UNITS];
  __shared__ long s_in[MM_HELD_ROWS];
  __shared__ int s_out[MM_HELD_ROWS];   // slot M + component
  __shared__ float s_g[MM_HELD_ROWS];
  const MMRows& a = h.r;
  int part, number;
  MMTile t = mm_expert_tile(a.offsets, h.lists, h.lists > a.E ? h.S : a.offsets[a.E], a.M, chunk, tiles_n, blockIdx.x,
                            &part, &number);
  if (t.e < 0) return;
  t = MMTile{__builtin_amdgcn_readfirstlane(t.e), __builtin_amdgcn_readfirstlane(t.row0),
             __builtin_amdgcn_readfirstlane(t.rows)};
  part = __builtin_amdgcn_readfirstlane(part);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, i = lane & 15, g = lane >> 4;
  const int n0 = part * 128 + 32 * wave;
  const int* __restrict__ list = a.order + a.offsets[t.e];
  if (t.e >= a.E) {   // slots without an expert
    for (int r = wave; r < t.rows; r += 4) {
      const int rr = t.row0 + r, p = rr / a.M;
      float* __restrict__ o = a.out + ((long)list[p] * a.M + rr - p * a.M) * a.N;
      for (int n = 128 * part + lane; n < min(128 * part + 128, a.N); n += 64) o[n] = 0.f;
    }
    return;
  }
  const int nst = (t.rows + 31) / 32;
  // the block's operands: column n0 + 16 c + i, values 32 s + 8 g ..
  MMRaw<float> rw[KS][2];
  {
    const float* __restrict__ W = (const float*)a.W + (size_t)t.e * a.K * a.N;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = n0 + 16 * c + i, k = 32 * s + 8 * g;
        if constexpr (TRANS) {
          mm_load4(W + (size_t)min(n, a.N - 1) * a.K, k, n < a.N ? a.K : 0, rw[s][c].x);
          mm_load4(W + (size_t)min(n, a.N - 1) * a.K, k + 4, n < a.N ? a.K : 0, rw[s][c].x + 4);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            rw[s][c].x[q] = n < a.N && k + q < a.K ? W[(size_t)(k + q) * a.N + n] : 0.f;
        }
      }
  }
  for (int r = tid; r < nst * 32; r += 256) {   // rows past the last one repeat it
    const int rr = t.row0 + min(r, t.rows - 1), p = rr / a.M, m = rr - p * a.M, slot = list[p];
    s_in[r] = (slot / a.k) * a.st + m * a.sm;
    s_out[r] = slot * a.M + m;
    s_g[r] = h.gates ? h.gates[slot] : 1.f;
  }
  __syncthreads();
  // this thread's part of a stage: values 4 k4 .. + 3 of rows rw0 + (256 / (8 KS)) j
  constexpr int ROWS = 32 / PER;
  const int k4 = tid % (8 * KS), row0 = tid / (8 * KS), left = a.K - 4 * k4;
  float x[2][PER][4];   // two stages on their way: one alone takes longer than the products of a stage
  auto load = [&](int st, float (&v)[PER][4]) {   // past the last stage that one again: no branch around the loads
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float* __restrict__ p = (const float*)a.in + s_in[32 * min(st, nst - 1) + row0 + ROWS * j];
      if constexpr (FULL) {
        const floatx4u f = *(const floatx4u*)(p + 4 * k4);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[j][q] = f[q];
      } else {
        mm_load4(p, 4 * k4, left > 0 ? a.K : 0, v[j]);
      }
    }
  };
  auto put = [&](int buf, int j, const float (&from)[PER][4]) {
    mm_held_put<KG>(Al[buf], row0 + ROWS * j, k4, from[j]);
  };
  load(0, x[0]);
  load(1, x[1]);
  MMFrag<float> w[KS][2];
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int c = 0; c < 2; ++c) w[s][c] = mm_operand(rw[s][c]);
#pragma unroll
  for (int j = 0; j < PER; ++j) put(0, j, x[0]);
  __syncthreads();
  for (int st0 = 0; st0 < nst; st0 += 2) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {   // stage st is in Al[b], stage st + 1 in x[b ^ 1]
      const int st = st0 + b;
      if (st >= nst) break;
      floatx4 acc[2][2] = {};   // [row tile][column tile]
      load(st + 2, x[b]);
      MMFrag<float> f[2][2];
      auto operands = [&](int s) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            f[s & 1][r].v[p] =
                __builtin_bit_cast(bf16x8, Al[b][((r * 3 + p) * KG + 4 * s + g) * MM_HELD_AS + i]);
      };
      operands(0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (s + 1 < KS) operands(s + 1);
        __builtin_amdgcn_sched_barrier(0);   // the reads of the next step stay ahead of the products of this one
        put(b ^ 1, s, x[b ^ 1]);             // a part of the next stage beside them (PER = KS)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) mm_mma(acc[r][c], w[s][c], f[s & 1][r]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = 32 * st + 16 * r + i;   // past the last row: that one again, with the same values
        float* __restrict__ o = a.out + (long)s_out[row] * a.N;
        const float gate = s_g[row];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const floatx4 v = acc[r][c];
          const float scaled[4] = {gate * v[0], gate * v[1], gate * v[2], gate * v[3]};
          if constexpr (FULL) *(floatx4u*)(o + n0 + 16 * c + 4 * g) = floatx4u{scaled[0], scaled[1], scaled[2], scaled[3]};
          else mm_store4(o, n0 + 16 * c + 4 * g, a.N, scaled);
        }
      }
      __syncthreads();
    }
  }
}

// The same for rows of two choices sorted by the pair of their experts: 8 waves hold 16 columns of both blocks (the same 96
// registers at K = 128), every operand of a row is read once for both, and the two products of a row are joined and
// written once.  64 rows a stage, one workgroup a CU.  DG: with the rows of dy and W[e]^T also dgates[t, j] = sum over m of
// <x[t, m], (dy W[e_j]^T)[t, m]>; all columns are then in one workgroup, and a chunk holds whole rows t.
struct MMPairs {
  const float *in, *W, *gates, *x;
  const int *experts, *offsets, *order;
  float *out, *dgates;
  long st, sm, xt, xm;
  int T, M, K, N, E, buckets;
};

template <bool TRANS, int KS, bool FULL, bool DG>
__global__ void __launch_bounds__(512, 2) mm_expert_held_pairs_kernel(MMPairs a, int tiles_n, int chunk) {
  constexpr int KG = 4 * KS, UNITS = 4 * 3 * KG * MM_HELD_AS, PER = KS;   // float4 a thread and stage: 64 * 8 KS / 512
  __shared__ uint4 Al[2][UNITS];
  __shared__ long s_in[MM_HELD_ROWS], s_x[DG ? MM_HELD_ROWS : 1];
  __shared__ int s_out[MM_HELD_ROWS];
  __shared__ float s_g[2][MM_HELD_ROWS], s_part[DG ? 2 : 1][8][2][64], s_dg[2][DG ? MM_HELD_ROWS : 1];
  int part, number;
  const MMTile tile = mm_expert_tile(a.offsets, a.buckets, a.T, a.M, chunk, tiles_n, blockIdx.x, &part, &number);
  if (tile.e < 0) return;
  const int rows = __builtin_amdgcn_readfirstlane(tile.rows), first = __builtin_amdgcn_readfirstlane(tile.row0);
  const int bucket = __builtin_amdgcn_readfirstlane(tile.e);
  part = __builtin_amdgcn_readfirstlane(part);
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, i = lane & 15, g = lane >> 4;
  const int n0 = part * 128 + 16 * wave;
  const int* __restrict__ list = a.order + a.offsets[bucket];
  int e0 = 0, e1 = bucket;
  while (e1 >= a.E + 1 - e0) e1 -= a.E + 1 - e0++;
  e1 += e0;
  if (e0 >= a.E) {   // rows without an expert
    for (int r = wave; r < rows; r += 8) {
      const int rr = first + r, p = rr / a.M;
      const long tok = list[p];
      if (a.out)
        for (int n = 128 * part + lane; n < min(128 * part + 128, a.N); n += 64)
          a.out[(tok * a.M + rr - p * a.M) * a.N + n] = 0.f;
      if (DG && lane < 2 && rr == p * a.M) a.dgates[2 * tok + lane] = 0.f;
    }
    return;
  }
  const int nst = (rows + 63) / 64;
  MMFrag<float> w[2][KS];
  int tok[MM_HELD_ROWS / 512];
  {
    MMRaw<float> rw[2][KS];
    const int n = n0 + i;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const bool there = n < a.N && (c ? e1 : e0) < a.E;
      const float* __restrict__ W = a.W + (size_t)(there ? (c ? e1 : e0) : 0) * a.K * a.N;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int k = 32 * s + 8 * g;
        if constexpr (TRANS) {
          mm_load4(W + (size_t)(there ? n : 0) * a.K, k, there ? a.K : 0, rw[c][s].x);
          mm_load4(W + (size_t)(there ? n : 0) * a.K, k + 4, there ? a.K : 0, rw[c][s].x + 4);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) rw[c][s].x[q] = there && k + q < a.K ? W[(size_t)(k + q) * a.N + n] : 0.f;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < MM_HELD_ROWS / 512; ++h) {   // rows past the last one repeat it
      const int r = tid + 512 * h;
      if (r >= nst * 64) break;
      const int rr = first + min(r, rows - 1), p = rr / a.M, m = rr - p * a.M;
      tok[h] = list[p];
      s_in[r] = tok[h] * a.st + m * a.sm;
      s_out[r] = tok[h] * a.M + m;
      if constexpr (DG) s_x[r] = tok[h] * a.xt + m * a.xm;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int s = 0; s < KS; ++s) w[c][s] = mm_operand(rw[c][s]);
  }
  __syncthreads();
  // this thread's part of a stage: values 4 k4 .. + 3 of rows row0 + ROWS j
  constexpr int ROWS = 64 / PER;
  const int k4 = tid % (8 * KS), row0 = tid / (8 * KS), left = a.K - 4 * k4;
  float x[2][PER][4];
  auto load = [&](int st, float (&v)[PER][4]) {   // past the last stage that one again
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float* __restrict__ p = a.in + s_in[64 * min(st, nst - 1) + row0 + ROWS * j];
      if constexpr (FULL) {
        const floatx4u f = *(const floatx4u*)(p + 4 * k4);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[j][q] = f[q];
      } else {
        mm_load4(p, 4 * k4, left > 0 ? a.K : 0, v[j]);
      }
    }
  };
  auto put = [&](int buf, int j, const float (&from)[PER][4]) {
    mm_held_put<KG>(Al[buf], row0 + ROWS * j, k4, from[j]);
  };
  load(0, x[0]);
  load(1, x[1]);
#pragma unroll
  for (int h = 0; h < MM_HELD_ROWS / 512; ++h) {   // the gates behind the first rows
    const int r = tid + 512 * h;
    if (r >= nst * 64) break;
    const int own = a.experts[2 * (long)tok[h]], swap = ((unsigned)own < (unsigned)a.E ? own : a.E) != e0;
    s_g[0][r] = a.gates ? a.gates[2 * (long)tok[h] + swap] : 1.f;
    s_g[1][r] = e1 < a.E ? a.gates ? a.gates[2 * (long)tok[h] + 1 - swap] : 1.f : 0.f;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) put(0, j, x[0]);
  __syncthreads();
  for (int st0 = 0; st0 < nst; st0 += 2) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {   // stage st is in Al[b], stage st + 1 in x[b ^ 1]
      const int st = st0 + b;
      if (st >= nst) break;
      float xv[DG ? 4 : 1][4];
      if constexpr (DG) {
#pragma unroll
        for (int r = 0; r < 4; ++r) mm_load4(a.x + s_x[64 * st + 16 * r + i], n0 + 4 * g, a.N, xv[r]);
      }
      load(st + 2, x[b]);
      floatx4 acc[2][4] = {};   // [choice][row tile]
      MMFrag<float> f[2][2];
      // row tiles 2 h, 2 h + 1 of step s: number 2 s + h
      auto operands = [&](int q) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            f[q & 1][r].v[p] = __builtin_bit_cast(
                bf16x8, Al[b][(((2 * (q & 1) + r) * 3 + p) * KG + 4 * (q >> 1) + g) * MM_HELD_AS + i]);
      };
      operands(0);
#pragma unroll
      for (int q = 0; q < 2 * KS; ++q) {
        if (q + 1 < 2 * KS) operands(q + 1);
        __builtin_amdgcn_sched_barrier(0);               // the reads of the next step stay ahead of the products
        if (q & 1) put(b ^ 1, q >> 1, x[b ^ 1]);         // a part of the next stage beside them (PER = KS)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) mm_mma(acc[c][2 * (q & 1) + r], w[c][q >> 1], f[q & 1][r]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 64 * st + 16 * r + i;   // past the last row: that one again, with the same values
        const float g0 = s_g[0][row], g1 = s_g[1][row];
        float v[4], d0 = 0.f, d1 = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = fmaf(g1, acc[1][r][q], g0 * acc[0][r][q]);
          if constexpr (DG) {
            d0 = fmaf(xv[r][q], acc[0][r][q], d0);
            d1 = fmaf(xv[r][q], acc[1][r][q], d1);
          }
        }
        if (!DG || a.out) {
          float* __restrict__ o = a.out + (long)s_out[row] * a.N;
          if constexpr (FULL) *(floatx4u*)(o + n0 + 4 * g) = floatx4u{v[0], v[1], v[2], v[3]};
          else mm_store4(o, n0 + 4 * g, a.N, v);
        }
        if constexpr (DG) {
          d0 += __shfl_xor(d0, 16);
          d1 += __shfl_xor(d1, 16);
          d0 += __shfl_xor(d0, 32);
          d1 += __shfl_xor(d1, 32);
          if (lane < 16) {
            s_part[b][wave][0][16 * r + i] = d0;
            s_part[b][wave][1][16 * r + i] = d1;
          }
        }
      }
      __syncthreads();
      if constexpr (DG) {   // the columns of a row, wave by wave; the other s_part is written next
        if (tid < 128) {
          const int c = tid >> 6;
          float d = 0.f;
#pragma unroll
          for (int v = 0; v < 8; ++v) d += s_part[b][v][c][lane];
          s_dg[c][64 * st + lane] = d;
        }
      }
    }
  }
  if constexpr (DG) {
    __syncthreads();
    for (int p = tid; p < rows / a.M; p += 512) {
      const long tok = list[first / a.M + p];
      const int own = a.experts[2 * tok], swap = ((unsigned)own < (unsigned)a.E ? own : a.E) != e0;
      float d[2] = {0.f, 0.f};
      for (int m = p * a.M; m < (p + 1) * a.M; ++m) {
        d[0] += s_dg[0][m];
        d[1] += s_dg[1][m];
      }
      a.dgates[2 * tok + swap] = d[0];
      a.dgates[2 * tok + 1 - swap] = e1 < a.E ? d[1] : 0.f;
    }
  }
}

// ------------------------------------------------------------------------------------------------ joined rows
// All k <= 2 choices of a row in one workgroup: rows sorted by the set of their experts (the plan of the slots for k = 1, of
// the pairs for k = 2) share both blocks, so that the products of a row are joined in registers and written once, in its
// type, where the path through slots writes k fp32 rows and reads them again.  Rows without an expert are written as
// zeros.  DG (k = 1): with the rows of dy and W[e]^T, also dgates[t] = sum over m of <x[t, m], (dy W^T)[t, m]>; a tile
// holds whole rows t (all M components) and all columns.
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
  // The gates: on the rows' values as they become operands (float without DG: one more rounding of 2^-24), or on each
  // choice's products, in sums of their own (16 bits, where the operands' rounding would show; DG, which needs the
  // products without the gates).
  constexpr bool SCALED = sizeof(T) == 4 && !DG, SUM = !SCALED;
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
    for (int i = 0; i < FN; ++i) mm_store4(o, n0 + wn + 16 * i + 4 * (lane >> 4), a.N, (const float*)&(SUM ? sum[SUM ? i : 0][SUM ? j : 0] : acc[i][j]));
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// y[t, m] straight from the choices of row t, without a plan: a workgroup takes LC vectors of columns, its other threads
// share the sum over d, W is read once per row, coalesced along the columns, fp32 sums.  Bound by latency: the sum over d is
// split as far as the workgroup goes, and the columns over many workgroups.
struct MMFew {
  const void *x, *W;
  const float* gates;
  const int* experts;
  long st, sm;
  int k, M, D, F, E;
};

template <typename T, int LC>
__global__ void __launch_bounds__(256) mm_expert_few_kernel(MMFew a, T* __restrict__ y) {
  constexpr int N = MMVec<T>::N, G = 256 / LC;
  __shared__ float red[4][LC * N];
  const long t = blockIdx.y;
  const int m = blockIdx.z, lc = threadIdx.x % LC, gd = threadIdx.x / LC, f = (blockIdx.x * LC + lc) * N;
  const T* __restrict__ x = (const T*)a.x + t * a.st + m * a.sm;
  float acc[N] = {};
  for (int j = 0; j < a.k; ++j) {
    const int e = a.experts[t * a.k + j];
    if ((unsigned)e >= (unsigned)a.E) continue;
    const float g = a.gates ? a.gates[t * a.k + j] : 1.f;
    const T* __restrict__ W = (const T*)a.W + (size_t)e * a.D * a.F;
    float sum[N] = {};
    if (f < a.F) {
#pragma unroll 8
      for (int d = gd; d < a.D; d += G) {
        float w[N];
        mm_load_vec(W + (size_t)d * a.F, f, a.F, w);
        const float xv = (float)x[d];
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = fmaf(xv, w[i], sum[i]);
      }
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
  if (threadIdx.x >= LC || f >= a.F) return;
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
    mm_load4(a.rows + (s * a.M + m) * a.N, c, a.N, v);
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] = fmaf(g, v[q], acc[q]);
  }
  mm_store4(y + row * a.N, c, a.N, acc);
}

// One wave per row t: dx[t] = sum_j gate rows[t, j] and dgates[t, j] = sum_m <x[t, m], rows[t, j, m]>, KB choices at a
// time, so that rows are read once for up to KB choices.
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

// ------------------------------------------------------------------------------------------------ dW
struct MMWgrad {
  const void *x, *dy;
  const float* gates;
  const int *offsets, *order;
  void* dW;
  long xt, xm, yt, ym;
  int k, M, D, F, E;
};

// A workgroup: a BD x BF tile of dW[e] over a chunk of the expert's rows (SPLIT: chunks of `chunk` rows, each into its own
// fp32 partial sums, which mm_expert_wgrad_sum_kernel adds in order; else all rows, straight into dW).  x goes into LDS as
// it is, dy through registers times its gate: in 16-bit types that rounds gate x dy to the type, an error of the size that
// dy's own rounding has.  Rows past the end are zeros on both sides.
#define MM_WG_ROWS 512   // rows whose offsets are kept in LDS at a time

template <typename T, bool SPLIT, bool DMA, int BD, int BF, int WD, int WF>
__global__ void __launch_bounds__(64 * WD * WF, 2) mm_expert_wgrad_kernel(MMWgrad a, int chunk, int tiles_f, int tiles_df,
                                                                          float* __restrict__ part) {
  constexpr int TH = 64 * WD * WF, BK = MM_TILE_K<T>, N = MMVec<T>::N, UD = BD / N, UF = BF / N, KS = BK / 32;
  constexpr int NX = BD * 8 / TH, NY = BF * 8 / TH, FD = BD / WD / 16, FF = BF / WF / 16;
  extern __shared__ uint4 mm_lds[];
  uint4 *Xs = mm_lds, *Ys = Xs + 2 * BD * 8;             // [2][BD * 8], [2][BF * 8]
  long *s_x = (long*)(Ys + 2 * BF * 8), *s_y = s_x + MM_WG_ROWS;
  float* s_g = (float*)(s_y + MM_WG_ROWS);
  const int lane_id = threadIdx.x & 63;
  int df, tile;
  MMTile t;
  if constexpr (SPLIT) {
    t = mm_expert_tile(a.offsets, a.E, a.offsets[a.E], a.M, chunk, tiles_df, blockIdx.x, &df, &tile);
    if (t.e < 0) return;
  } else {
    // Each list is read by one XCD, whose L2 serves all tiles of dW[e].  The longest lists first, dealt out to the XCDs
    // forth and back, so that they end together (64 experts at most; beyond that every 8th as they come).  Lists of uneven
    // load (lognormal, 0.7), 64 experts, 1024 x 1024: 338 us in the order of the experts, 279 us so.
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
  MMStage<T, TH, NY, false> sy;
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
  };
  auto put = [&](int buf) {
    sx.put(Xs + buf * BD * 8);
    if (a.gates) {
#pragma unroll
      for (int j = 0; j < NY; ++j) {
        typename MMVec<T>::type v = __builtin_bit_cast(typename MMVec<T>::type, sy.v[j]);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (T)(gy[j] * (float)v[i]);
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
      if (next % MM_WG_ROWS == 0) rows_of(next);   // the previous block's offsets are used up (barrier of the last step)
      load(next, buf ^ 1);
    }
    mm_products<T, FF, FD, KS>(
        acc, [&](int s, int i) { return mm_read_nc<T, UF>(Ys + buf * BF * 8, wf + 16 * i, s, lane); },
        [&](int s, int j) { return mm_read_nc<T, UD>(Xs + buf * BD * 8, wd + 16 * j, s, lane); });
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

// dW[e] = the partial sums of the expert's chunks, in order
template <typename T>
__global__ void __launch_bounds__(256) mm_expert_wgrad_sum_kernel(MMWgrad a, int chunk, const float* __restrict__ part) {
  const int lane = threadIdx.x & 63, e = blockIdx.y;
  int first = 0;   // chunks of the experts before e
  for (int o = lane; o < e; o += 64) first += ((a.offsets[o + 1] - a.offsets[o]) * a.M + chunk - 1) / chunk;
#pragma unroll
  for (int d = 32; d; d >>= 1) first += __shfl_xor(first, d);
  const int n = ((a.offsets[e + 1] - a.offsets[e]) * a.M + chunk - 1) / chunk;
  const long size = (long)a.D * a.F, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= size) return;
  const float* __restrict__ p = part + (size_t)first * size + i;
  float t = 0.f;
#pragma unroll 8
  for (int c = 0; c < n; ++c) t += p[c * size];
  ((T*)a.dW)[(size_t)e * size + i] = (T)t;
}

// ------------------------------------------------------------------------------------------------ entry points
namespace {
int range_error(const char* name, const char* what) {
  mm::set_error(std::string(name) + ": " + what);
  return MM_ERANGE;
}

// Tiles of 256 x 256 where the experts' lists and the columns fill them: twice the products per value loaded, but a cut
// tile at the end of every list.
bool big_tiles(long rows, int N, int E) { return rows >= 512L * E && N > 128; }

// two stages of both operands, then rows' offsets
template <int BM, int BN>
constexpr int rows_lds() { return 2 * (BM + BN) * 128 + BM * 8; }
template <int BD, int BF>
constexpr int wgrad_lds() { return 2 * (BD + BF) * 128 + MM_WG_ROWS * 20; }

// more than 64 KB of LDS has to be asked for, once per kernel and device
template <auto KERNEL>
bool lds_granted(int bytes) {
  static std::atomic<unsigned long long> granted{0};   // a bit per device
  int dev = 0;
  if (bytes <= 65536) return true;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const unsigned long long bit = 1ull << (dev & 63);
  if (granted.load(std::memory_order_relaxed) & bit) return true;
  if (hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
    return false;
  granted.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

template <typename T, bool TRANS, bool DMA, int BM, int BN, int WM, int WN>
int launch_rows_tile(const MMRows& a, int S, hipStream_t stream) {
  const int tiles_n = (a.N + BN - 1) / BN;
  // every expert's list may end in a cut tile
  const long wg = (((long)S * a.M + BM - 1) / BM + (a.E < S ? a.E : S)) * tiles_n;
  if (wg > 2147483647L) return range_error("mm_expert_rows", "output too large for one launch");
  constexpr auto kernel = mm_expert_rows_kernel<T, TRANS, DMA, BM, BN, WM, WN>;
  constexpr int lds = rows_lds<BM, BN>();
  if (!lds_granted<kernel>(lds)) return mm::launch_status("mm_expert_rows");
  hipLaunchKernelGGL(kernel, dim3((unsigned)wg), dim3(64 * WM * WN), lds, stream, a, tiles_n);
  return mm::launch_status("mm_expert_rows");
}

template <typename T, bool TRANS, bool DMA>
int launch_rows(const MMRows& a, int S, bool big, hipStream_t stream) {
  if constexpr (sizeof(T) == 2 && DMA)
    if (big) return launch_rows_tile<T, TRANS, DMA, 256, 256, 2, 4>(a, S, stream);
  return launch_rows_tile<T, TRANS, DMA, 128, 128, 2, 2>(a, S, stream);
}

// Rows per workgroup of the held blocks: for one round of the 512 that are resident (2 a CU), at most two and so on, with
// the experts' cut chunks taken off; 32 rows are a stage.
int held_chunk(long rows, long tiles_n, int lists) {
  for (long n = 1;; ++n) {
    const long wg = 512 * n - lists * tiles_n;
    if (wg < 256) continue;
    const long c = ((rows * tiles_n + wg - 1) / wg + 31) / 32 * 32;
    if (c <= MM_HELD_ROWS) return (int)(c < 32 ? 32 : c);
  }
}

int launch_held(const char* name, const MMRows& a, int S, const float* gates, int lists, int transposed,
                hipStream_t stream) {
  const int tiles_n = (a.N + 127) / 128, chunk = held_chunk((long)S * a.M, tiles_n, lists);
  const long wg = (((long)S * a.M + chunk - 1) / chunk + (lists < S ? lists : S)) * tiles_n;
  if (wg > 2147483647L) return range_error(name, "output too large for one launch");
  const MMHeld h{a, gates, lists, S};
#define CALL(trans, ks)                                                                                               \
  if (a.K == 32 * ks && a.N % 128 == 0)                                                                               \
    hipLaunchKernelGGL((mm_expert_held_kernel<trans, ks, true>), dim3((unsigned)wg), dim3(256), 0, stream, h, tiles_n, \
                       chunk);                                                                                        \
  else                                                                                                                \
    hipLaunchKernelGGL((mm_expert_held_kernel<trans, ks, false>), dim3((unsigned)wg), dim3(256), 0, stream, h, tiles_n, \
                       chunk)
#define CALLS(trans)                    \
  if (a.K <= 32) { CALL(trans, 1); }    \
  else if (a.K <= 64) { CALL(trans, 2); } \
  else { CALL(trans, 4); }
  if (transposed) { CALLS(true) } else { CALLS(false) }
#undef CALLS
#undef CALL
  return mm::launch_status(name);
}

// rows per workgroup of the pairs' blocks: one workgroup a CU, whole rows t and whole stages of 64; 0: no such chunk
int pairs_chunk(long rows, long tiles_n, int buckets, int M) {
  int step = 64;
  while (step % M) step += 64;
  if (step > MM_HELD_ROWS) return 0;
  for (long n = 1;; ++n) {
    const long wg = 256 * n - buckets / 2 * tiles_n;   // lists end in cut chunks, by half of one on average
    if (wg < 128) continue;
    const long c = ((rows * tiles_n + wg - 1) / wg + step - 1) / step * step;
    if (c <= MM_HELD_ROWS) return (int)(c < step ? step : c);
  }
}

int launch_pairs(const char* name, const MMPairs& a, int transposed, int chunk, hipStream_t stream) {
  const int tiles_n = (a.N + 127) / 128;
  const long wg = (((long)a.T * a.M + chunk - 1) / chunk + (a.buckets < a.T ? a.buckets : a.T)) * tiles_n;
  if (wg > 2147483647L) return range_error(name, "output too large for one launch");
#define CALL2(trans, ks, full, dg)                                                                                      \
  hipLaunchKernelGGL((mm_expert_held_pairs_kernel<trans, ks, full, dg>), dim3((unsigned)wg), dim3(512), 0, stream, a, \
                     tiles_n, chunk)
#define CALL(trans, ks, dg)                                          \
  if (a.K == 32 * ks && a.N % 128 == 0) CALL2(trans, ks, true, dg);  \
  else CALL2(trans, ks, false, dg);
#define CALLS(trans, dg)                              \
  if (a.K <= 32) { CALL(trans, 1, dg) }               \
  else if (a.K <= 64) { CALL(trans, 2, dg) }          \
  else { CALL(trans, 4, dg) }
  if (a.dgates) { CALLS(true, true) }
  else if (transposed) { CALLS(true, false) }
  else { CALLS(false, false) }
#undef CALLS
#undef CALL
#undef CALL2
  return mm::launch_status(name);
}

template <typename T, bool SPLIT, bool DMA, int BD, int BF, int WD, int WF>
int launch_wgrad_tile(const MMWgrad& a, int S, int chunk, float* part, hipStream_t stream) {
  const int tiles_f = (a.F + BF - 1) / BF, tiles_df = (a.D + BD - 1) / BD * tiles_f;
  const long wg = (SPLIT ? (long)S * a.M / chunk + (a.E < S ? a.E : S) : (a.E + 7L) / 8 * 8) * tiles_df;
  if (wg > 2147483647L) return range_error("mm_expert_wgrad", "output too large for one launch");
  constexpr auto kernel = mm_expert_wgrad_kernel<T, SPLIT, DMA, BD, BF, WD, WF>;
  constexpr int lds = wgrad_lds<BD, BF>();
  if (!lds_granted<kernel>(lds)) return mm::launch_status("mm_expert_wgrad");
  if (wg)
    hipLaunchKernelGGL(kernel, dim3((unsigned)wg), dim3(64 * WD * WF), lds, stream, a, chunk, tiles_f, tiles_df, part);
  return mm::launch_status("mm_expert_wgrad");
}

template <typename T, bool SPLIT, bool DMA>
int launch_wgrad(const MMWgrad& a, int S, int chunk, bool big, float* part, hipStream_t stream) {
  if constexpr (sizeof(T) == 2 && DMA && !SPLIT)
    if (big) return launch_wgrad_tile<T, SPLIT, DMA, 256, 256, 2, 4>(a, S, chunk, part, stream);
  return launch_wgrad_tile<T, SPLIT, DMA, 128, 128, 2, 2>(a, S, chunk, part, stream);
}

// base of a matrix whose 16-byte units can be loaded straight into LDS
bool aligned(const void* p) { return (size_t)p % 16 == 0; }

// Rows per chunk of dW's sums; 0: no chunks.  A card of 256 CUs takes 512 workgroups at a time: with at least that many
// (expert, tile) pairs none are made; else chunks for about 1024 workgroups, of 256 rows or more (a chunk's partial sums
// are 64 KB per tile to write and read, 256 rows of both operands 128 KB or more).
int wgrad_chunk(long rows, int D, int F, int E) {
  const long tiles = (long)((D + 127) / 128) * ((F + 127) / 128);
  if (E * tiles >= 512 || rows < 512) return 0;
  const long c = (rows * tiles + 1023) / 1024;
  return (int)(c < 256 ? 256 : (c + 63) / 64 * 64);
}

}  // namespace

extern "C" int mm_expert_plan_scratch(int S, int E, long* ints) {
  MM_CHECK_ARG(S >= 0 && E >= 1 && ints, "bad sizes");
  const long tiles = ((long)S + MM_PLAN_TILE - 1) / MM_PLAN_TILE;
  *ints = tiles <= MM_PLAN_ONE ? 0 : (E + 1L) * (tiles + 1);   // counts, totals
  return MM_OK;
}

namespace {
// buckets 0 .. E; PAIRS: of S rows with two of pairs_of experts each, E + 1 = mm_pair_buckets(pairs_of)
template <bool PAIRS>
int launch_plan(const char* name, const int* experts, int S, int E, int pairs_of, int* offsets, int* order, int* scratch,
                hipStream_t stream) {
  const int tiles = (int)(((long)S + MM_PLAN_TILE - 1) / MM_PLAN_TILE), one = tiles <= MM_PLAN_ONE;
  MM_CHECK_ARG(one || scratch, "scratch is null");
  // 16 waves while their counters fit 64 KB of LDS beside the tile, else 4
  const int nw = E < 400 ? 16 : 4, th = 64 * nw, across = mm_plan_across(E + 1, th);
  const int lds = (nw + 2) * (E + 1) * (int)sizeof(int);
  int *counts = scratch, *totals = scratch + (size_t)tiles * (E + 1);
  if (!one)
    hipLaunchKernelGGL(mm_plan_count_kernel<PAIRS>, dim3(tiles), dim3(1024), (E + 1) * sizeof(int), stream, experts, S, E,
                       pairs_of, counts);
  const bool sums = ((long)tiles * across + th - 1) / th * ((E + across) / across) <= MM_PLAN_SUM;
  if (!one && !sums)
    hipLaunchKernelGGL(mm_plan_scan_kernel, dim3(E + 1), dim3(64), 0, stream, counts, tiles, E, totals);
#define CALL(mode, nw, bits)                                                                                            \
  hipLaunchKernelGGL((mm_plan_kernel<mode, nw, bits, PAIRS>), dim3(tiles ? tiles : 1), dim3(64 * nw), lds, stream, experts, \
                     S, E, pairs_of, tiles, counts, totals, offsets, order)
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
  return launch_plan<true>("mm_expert_plan_pairs", experts, T, mm_pair_buckets(E) - 1, E, offsets, order, scratch, stream);
}

extern "C" int mm_expert_rows(const void* in, long st, long sm, int dtype, int S, int k, int M, int K, int N,
                              const void* W, int transposed, int E, const int* offsets, const int* order, float* out,
                              hipStream_t stream) {
  MM_CHECK_ARG(dtype >= MM_F32 && dtype <= MM_F16, "bad dtype");
  MM_CHECK_ARG(S >= 0 && k >= 1 && M >= 1 && K >= 1 && N >= 1 && E >= 1 && st >= 0 && sm >= 0, "bad sizes");
  if ((long)S * M > 2147483647L - 128) return range_error("mm_expert_rows", "2^31 rows or more are not supported");
  if (S == 0) return MM_OK;
  const MMRows a{in, W, offsets, order, out, st, sm, k, M, K, N, E};
  if (dtype == MM_F32 && K <= 128) return launch_held("mm_expert_rows", a, S, nullptr, E, transposed, stream);
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
  if (T > 65535 || M > 65535) return range_error("mm_expert_few", "more than 65535 rows or components are not supported");
  if (T == 0) return MM_OK;
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
  const int chunk = dtype == MM_F32 && K <= 128 && k == 2 && T
                        ? pairs_chunk((long)T * M, (N + 127) / 128, mm_pair_buckets(E <= MM_PAIRS_MAX_E ? E : 1), M) : 0;
  MM_CHECK_ARG(out || dgates, "nothing to compute");
  MM_CHECK_ARG(!dgates || (transposed && x && xt >= 0 && xm >= 0 && N <= 128 && (k == 1 || chunk || T == 0)),
               "dgates needs the transposed blocks, x, at most 128 columns, and one choice or float rows of up to 128 values");
  if (M > 64) return range_error("mm_expert_joined", "more than 64 components are not supported");
  if (k == 2 && E > MM_PAIRS_MAX_E)
    return range_error("mm_expert_joined", "pairs of more than 21 experts are not supported");
  if ((long)T * M > 2147483647L - 128) return range_error("mm_expert_joined", "2^31 rows or more are not supported");
  if (T == 0) return MM_OK;
  if (dtype == MM_F32 && K <= 128 && k == 1 && !dgates && out) {
    const MMRows r{in, W, offsets, order, (float*)out, st, sm, 1, M, K, N, E};
    return launch_held("mm_expert_joined", r, T, gates, E + 1, transposed, stream);
  }
  const int buckets = k == 1 ? E + 1 : mm_pair_buckets(E), tiles_n = (N + 127) / 128, tile = (dtype == MM_F32 ? 128 : 64) / M;   // rows t a tile
  const long wg = (((long)T + tile - 1) / tile + (buckets < T ? buckets : T)) * tiles_n;
  if (wg > 2147483647L) return range_error("mm_expert_joined", "output too large for one launch");
  if (chunk) {
    const MMPairs a{(const float*)in, (const float*)W, gates, (const float*)x, experts, offsets, order, (float*)out, dgates,
                    st, sm, xt, xm, T, M, K, N, E, buckets};
    return launch_pairs("mm_expert_joined", a, transposed, chunk, stream);
  }
  const MMJoined a{in, W, x, gates, experts, offsets, order, out, dgates, st, sm, xt, xm, T, M, K, N, E, buckets};
  const int unit = dtype == MM_F32 ? 4 : 8;
  const bool dma = aligned(in) && aligned(W) && st % unit == 0 && (M == 1 || sm % unit == 0) && K % unit == 0 &&
                   (transposed || N % unit == 0);
#define CALL4(trans, dma, j, dg) \
  MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_joined_kernel<T_, trans, dma, j, dg, sizeof(T_) == 4 ? 128 : 64>), dim3((unsigned)wg), dim3(256), 0, \
                                        stream, a, tiles_n))
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
#define CALL2(KB)                                                                                                     \
  hipLaunchKernelGGL((mm_expert_combine_bwd_kernel<T_, KB>), dim3((unsigned)wg), dim3(256), 0, stream, a, (const T_*)x, \
                     st, sm, (T_*)dx, dgates);
#define CALL if (k == 1) { CALL2(1) } else if (k == 2) { CALL2(2) } else { CALL2(4) }
  if (dtype == MM_F32) { using T_ = float; CALL }
  else if (dtype == MM_BF16) { using T_ = __bf16; CALL }
  else { using T_ = _Float16; CALL }
#undef CALL
#undef CALL2
  return mm::launch_status("mm_expert_combine_bwd");
}

extern "C" int mm_expert_wgrad_workspace(int S, int M, int D, int F, int E, size_t* bytes) {
  MM_CHECK_ARG(S >= 0 && M >= 1 && D >= 1 && F >= 1 && E >= 1 && bytes, "bad sizes");
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
  if ((long)S * M > 2147483647L - 128) return range_error("mm_expert_wgrad", "2^31 rows or more are not supported");
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
  const bool big = dma && !chunk && D > 128 && F > 128 && E * ((D + 255) / 256) * ((F + 255) / 256) >= 512;
  if (chunk) { if (dma) { CALL(true, true) } else { CALL(true, false) } }
  else { if (dma) { CALL(false, true) } else { CALL(false, false) } }
#undef CALL
  if (rc != MM_OK) return rc;
  if (chunk)
    MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_wgrad_sum_kernel<T_>),
                                          dim3((unsigned)(((long)D * F + 255) / 256), E), dim3(256), 0, stream, a, chunk,
                                          workspace));
  return mm::launch_status("mm_expert_wgrad");
}
