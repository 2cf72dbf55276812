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

template <typename T>
__device__ __forceinline__ MMFrag<T> mm_operand(const MMRaw<T>& r) {
  if constexpr (sizeof(T) == 2) {
    return r.f;
  } else {
    MMFrag<float> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __bf16 h = (__bf16)r.x[i];
      const float d = r.x[i] - (float)h;
      const __bf16 l = (__bf16)d;
      f.v[0][i] = h;
      f.v[1][i] = l;
      f.v[2][i] = (__bf16)(d - (float)l);
    }
    return f;
  }
}

// acc[i][j] += a(s, i) b(s, j) over the KS steps of a stage: operands b are read two ahead of their products and turned
// into planes one ahead, the next step's operands a over the last products of this one.  The scheduling barriers keep the
// reads there: left alone, the compiler reads two operands, waits for them and multiplies.
template <typename T, int FN, int FM, int KS, typename A, typename B>
__device__ __forceinline__ void mm_products(floatx4 (&acc)[FN][FM], A a, B b) {
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
    fb[0] = mm_operand(rb[0]);
  }
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int s = q / FM, j = q % FM;
    if (q + 2 < Q) rb[(q + 2) % 3] = b((q + 2) / FM, (q + 2) % FM);
    if constexpr (KS > 1) {
      if (s + 1 < KS && j >= FM - FN) fa[(s + 1) & 1][j - (FM - FN)] = mm_operand(a(s + 1, j - (FM - FN)));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (q + 1 < Q) fb[(q + 1) & 1] = mm_operand(rb[(q + 1) % 3]);
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

// Workgroups are dealt out to the 8 XCDs in turn: number them so that an XCD gets consecutive work, whose operands its L2
// then holds.
__device__ __forceinline__ int mm_xcd_order(int b, int n) {
  const int per = n / 8, rest = n % 8, x = b % 8, i = b / 8;
  return x < rest ? x * (per + 1) + i : x * per + rest + i;
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
  const int at = mm_xcd_order(blockIdx.x, gridDim.x), n0 = at % tiles_n * BN;
  const MMTile t = mm_expert_tile(a.offsets, a.E, a.M, BM, at / tiles_n);
  if (t.e < 0) return;
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

// ------------------------------------------------------------------------------------------------ rows -> y
struct MMCombine {
  const float *rows, *gates;
  const int* experts;
  long T;
  int k, M, N, E;
};

template <typename T>
__device__ __forceinline__ void mm_store4(T* __restrict__ p, int c, int N, const float* v) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (c + 4 <= N) {
    *(vec*)(p + c) = vec{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (c + q < N) p[c + q] = (T)v[q];
  }
}

template <typename T>
__device__ __forceinline__ void mm_load4(const T* __restrict__ p, int c, int N, float* v) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (c + 4 <= N) {
    const vec x = *(const vec*)(p + c);
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = (float)x[q];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = c + q < N ? (float)p[c + q] : 0.f;
  }
}

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
  const int at = mm_xcd_order(blockIdx.x, gridDim.x), tile = at / tiles_df, df = at % tiles_df;
  MMTile t;
  if constexpr (SPLIT) t = mm_expert_tile(a.offsets, a.E, a.M, chunk, tile);
  else t = MMTile{tile, 0, (a.offsets[tile + 1] - a.offsets[tile]) * a.M};
  if (t.e < 0) return;
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
  const long size = (long)a.D * a.F, i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= size) return;
  float t[4] = {};
  for (int c = 0; c < n; ++c) {
    const float* __restrict__ p = part + (size_t)(first + c) * size;
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (i + v < size) t[v] += p[i + v];
  }
  T* __restrict__ o = (T*)a.dW + (size_t)e * size;
#pragma unroll
  for (int v = 0; v < 4; ++v)
    if (i + v < size) o[i + v] = (T)t[v];
}

// ------------------------------------------------------------------------------------------------ entry points
namespace {
int range_error(const char* name, const char* what) {
  mm::set_error(std::string(name) + ": " + what);
  return MM_ERANGE;
}

constexpr int kPlanTile = 4 * MM_PLAN_WAVE;

// waves of the one workgroup that plans S slots of E experts (its counters fit 64 KB of LDS); 0: several workgroups
int plan_waves(int S, int E) { return S <= 4 * MM_PLAN_WAVE ? 4 : S <= 16 * MM_PLAN_WAVE && E <= 512 ? 16 : 0; }

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

template <typename T, bool SPLIT, bool DMA, int BD, int BF, int WD, int WF>
int launch_wgrad_tile(const MMWgrad& a, int S, int chunk, float* part, hipStream_t stream) {
  const int tiles_f = (a.F + BF - 1) / BF, tiles_df = (a.D + BD - 1) / BD * tiles_f;
  const long wg = (SPLIT ? (long)S * a.M / chunk + (a.E < S ? a.E : S) : a.E) * tiles_df;
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
  if ((long)S * M > 2147483647L - 128) return range_error("mm_expert_rows", "2^31 rows or more are not supported");
  if (S == 0) return MM_OK;
  const MMRows a{in, W, offsets, order, out, st, sm, k, M, K, N, E};
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
    MM_DISPATCH(dtype, hipLaunchKernelGGL((mm_expert_wgrad_sum_kernel<T>),
                                          dim3((unsigned)(((long)D * F + 1023) / 1024), E), dim3(256), 0, stream, a, chunk,
                                          workspace));
  return mm::launch_status("mm_expert_wgrad");
}
