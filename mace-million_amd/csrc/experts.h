// What the kernels of the experts' products share (expert_plan.hip, expert_rows.hip, expert_held.hip,
// expert_wgrad.hip):
//     y[t, m] = sum_j gate[t, j] x[t, m] @ W[expert[t, j]],   with the gradients of x, W and the gates.
// A slot is a (row, choice) pair s = t k + j; the plan lists the slots sorted by expert (stable), so that each
// expert's rows are consecutive and its block is read once per tile of rows.  A slot whose expert lies outside [0, E)
// takes part nowhere.
#pragma once
#include "rowvec.h"

#include <atomic>

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));   // 16 bytes known to be float-aligned only

#define MM_EXPERT_MAX_E 1024
#define MM_EXPERT_MAX_ROWS (2147483648L - 65536)   // rows (slots x M); an index a tile or stage past them fits an int
#define MM_PAIRS_MAX_E 21   // 253 pairs
#define MM_HELD_ROWS 1024   // rows of a workgroup with its blocks in registers, at most

// Bucket of a pair of choices among E experts and none (number E), in any order: rows e1 <= e2 of a triangle, the pair
// of no expert at all last.
__host__ __device__ inline int mm_pair_bucket(int e1, int e2, int E) {
  const int lo = e1 < e2 ? e1 : e2, hi = e1 < e2 ? e2 : e1;
  return lo * (E + 1) - lo * (lo - 1) / 2 + hi - lo;
}
__host__ __device__ inline int mm_pair_buckets(int E) { return (E + 1) * (E + 2) / 2; }

// ------------------------------------------------------------------------------------------------ tiles of an expert
struct MMTile {
  int e, row0, rows;   // expert, first of its rows (slots x M), rows in the tile; e < 0: no such tile
};

// pieces of `size` that n >= 0 values make (n + size may pass 2^31)
__host__ __device__ inline int mm_pieces(int n, int size) {
  return (int)(((unsigned)n + (unsigned)size - 1u) / (unsigned)size);
}

// Workgroup b of `per` for each of the tiles of BM rows that the row lists of the buckets have (every list ends in a
// cut tile); list i: entries offsets[i] .. offsets[i + 1], the last one to `end`, M rows each.  Every wave finds its
// tile by itself, 64 lists at a time.  Workgroups are dealt out to the 8 XCDs in turn; the work is numbered so that an
// XCD gets consecutive pieces, whose operands its L2 then holds.
__device__ __forceinline__ MMTile mm_expert_tile(const int* __restrict__ offsets, int lists, int end, int M, int BM,
                                                 int per, int b, int* part, int* number) {
  const int lane = threadIdx.x & 63;
  auto rows_of = [&](int i) {
    if (i >= lists) return 0;
    return ((i + 1 < lists ? offsets[i + 1] : end) - offsets[i]) * M;
  };
  const int head = rows_of(lane);
  int all = mm_pieces(head, BM);
#pragma unroll 4
  for (int i = 64 + lane; i - lane < lists; i += 64) all += mm_pieces(rows_of(i), BM);
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
    const int rows = i0 ? rows_of(i0 + lane) : head, n = mm_pieces(rows, BM);
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
// Operands of v_mfma_f32_16x16x32 (fp32 sums): lane (i, g) = (lane & 15, lane >> 4) holds the values k = 8 g .. 8 g +
// 7 of row (column) i.  16-bit types: one product.  float: three bf16 planes x = x0 + x1 + x2 (x0 = bf16(x), x1 =
// bf16(x - x0), x2 = bf16(x - x0 - x1), |x - x0 - x1 - x2| <= 2^-27 |x|) and the six products a_i b_j with i + j <= 2;
// those left out are below 3 * 2^-24 |a b|.  96 matrix cycles for 16 x 16 x 32 against 256 in fp32 products.
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

// acc[i][j] += a(s, i) b(s, j) scale[j] over the KS steps of a stage (SCALED: float only): operands b are read two
// ahead of their products and turned into planes one ahead, the next step's operands a over the last products of this
// one.  The scheduling barriers keep the reads there: left alone, the compiler reads two operands, waits for them and
// multiplies.
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

// Two bf16 parts of 8 values, scale x v in fp32: off by 2^-18 of each (float16 values without a scale: exact).
struct MMParts {
  bf16x8 v[2];
};

template <typename T, bool SCALED>
__device__ __forceinline__ MMParts mm_parts(const MMRaw<T>& r, const float* scale) {
  MMParts p;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = SCALED ? scale[i] * (float)r.f.v[i] : (float)r.f.v[i];
    const __bf16 h = (__bf16)x;
    p.v[0][i] = h;
    p.v[1][i] = (__bf16)(x - (float)h);
  }
  return p;
}

// acc[i][j] += sum over the values q of a stage of gate[q] a(s, i)[q] b(s, j)[q] for 16-bit types, as mm_products does
// without gates.  gate x a is taken in fp32 and enters as two bf16 parts: rounded to the type it would lose the bits
// below its own and, in float16, whatever is below 2^-25 or above 65504.  bfloat16 b: two products; float16 b: two
// parts as well and three products, the fourth being 2^-18 of the first.
template <typename T, int FN, int FM, int KS, typename A, typename B>
__device__ __forceinline__ void mm_products_gated(floatx4 (&acc)[FN][FM], A a, B b, const float* gates, int lane) {
  constexpr bool HALF = __is_same(T, _Float16);
  constexpr int Q = KS * FM;
  auto gates_of = [&](int s, float (&g)[8]) {   // of the values that this lane holds of step s
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const floatx4 v = *(const floatx4*)(gates + 32 * s + 8 * (lane >> 4) + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) g[4 * h + i] = v[i];
    }
  };
  MMParts fa[FN], fb[2];
  MMRaw<T> ra[FN], rb[3];
  float g[8];
  auto second = [&](const MMRaw<T>& r, MMParts& p) {
    if constexpr (HALF) p = mm_parts<T, false>(r, nullptr);
    else p.v[0] = r.f.v;
  };
  gates_of(0, g);
#pragma unroll
  for (int i = 0; i < FN; ++i) ra[i] = a(0, i);
  rb[0] = b(0, 0);
  rb[1] = b(1 / FM, 1 % FM);
#pragma unroll
  for (int i = 0; i < FN; ++i) fa[i] = mm_parts<T, true>(ra[i], g);
  second(rb[0], fb[0]);
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int s = q / FM, j = q % FM;
    if (q + 2 < Q) rb[(q + 2) % 3] = b((q + 2) / FM, (q + 2) % FM);
    if (s + 1 < KS) {   // the next step's operands, over the last products of this one
#pragma unroll
      for (int i = 0; i < FN; ++i)
        if ((FN < FM ? i + FM - FN : i * FM / FN) == j) ra[i] = a(s + 1, i);
      if (j == FM - 1) gates_of(s + 1, g);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (q + 1 < Q) second(rb[(q + 1) % 3], fb[(q + 1) & 1]);
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      floatx4& c = acc[i][j];
      const MMParts& x = fb[q & 1];
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i].v[1], x.v[0], c, 0, 0, 0);
      if constexpr (HALF) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i].v[0], x.v[1], c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i].v[0], x.v[0], c, 0, 0, 0);
      if (s + 1 < KS && j == FM - 1) fa[i] = mm_parts<T, true>(ra[i], g);   // beside the products of the others
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Tiles in LDS, in units of 16 bytes.  MM_TILE_K<T> values of the summed index a stage.
// KC (the summed index contiguous in memory): a row of 8 units (128 bytes), unit u of row r at 8 r + (u ^ (r & 7)), so
// that the 16 rows of an operand read spread over all banks.
// NC (the other index contiguous): a row per value of the summed index, UPR units; unit u of row q at
// UPR q + (u ^ s(q)), s(q) chosen so that the rows read together lie in different banks.  16-bit operands come out of
// it by transposing reads (ds_read_b64_tr_b16: 16 lanes give the addresses of a 4 x 16 block, four lanes a row, and
// lane i receives its column i), float operands value by value.
// Staged by loads straight into LDS (16 bytes a lane, the wave's units in order, so the swizzle is in the addresses of
// the sources) where the units are aligned, else through registers.
template <typename T>
constexpr int MM_TILE_K = 128 / sizeof(T);

typedef __attribute__((address_space(3))) void* mm_lds_ptr;
typedef const __attribute__((address_space(1))) void* mm_global_ptr;

static __device__ uint4 mm_zero_unit;   // source of units outside the operands (zero-initialised, never written)

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

// ------------------------------------------------------------------------------------------------ host
struct MMRows {
  const void *in, *W;
  const int *offsets, *order;
  float* out;
  long st, sm;   // strides of in in elements: rows, components
  int k, M, K, N, E;
};

struct MMPairs {
  const float *in, *W, *gates, *x;
  const int *experts, *offsets, *order;
  float *out, *dgates;
  long st, sm, xt, xm;
  int T, M, K, N, E, buckets;
};

namespace {
inline int range_error(const char* name, const char* what) {
  mm::set_error(std::string(name) + ": " + what);
  return MM_ERANGE;
}

constexpr char TOO_MANY_ROWS[] = "more than 2^31 - 2^16 rows are not supported";
constexpr char TOO_WIDE[] = "blocks of more than 2^31 - 2^16 rows or columns are not supported";
inline bool too_wide(long a, long b) { return a > MM_EXPERT_MAX_ROWS || b > MM_EXPERT_MAX_ROWS; }

// a launch takes fewer than 2^32 threads
inline bool too_many(long workgroups, long threads) { return workgroups * threads >= 4294967296L; }

// base of a matrix whose 16-byte units can be loaded straight into LDS
inline bool aligned(const void* p) { return (size_t)p % 16 == 0; }

// more than 64 KB of LDS has to be asked for, once per kernel and device
template <auto KERNEL>
bool lds_granted(int bytes) {
  static std::atomic<unsigned long long> granted{0};   // a bit per device
  int dev = 0;
  if (bytes <= 65536) return true;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const unsigned long long bit = 1ull << (dev & 63);
  if (granted.load(std::memory_order_relaxed) & bit) return true;
  if (hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
    mm::set_error("the kernel's LDS was not granted");
    return false;
  }
  granted.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

}  // namespace

namespace mm {
// expert_held.hip: float rows of up to 128 values.  launch_held: rows of slots, or with gates the rows of one choice
// (lists E + 1); launch_pairs: rows of two choices in chunks of pairs_chunk rows (0: not for this number of
// components).
int launch_held(const char* name, const MMRows& a, int S, const float* gates, int lists, int transposed,
                hipStream_t stream);
int pairs_chunk(long rows, long tiles_n, int buckets, int M);
int launch_pairs(const char* name, const MMPairs& a, int transposed, int chunk, hipStream_t stream);
}  // namespace mm
