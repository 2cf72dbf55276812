// What the kernels of the experts' products share (expert_plan.hip, expert_rows.hip, expert_held.hip,
// expert_wgrad.hip):
//     y[t, m] = sum_j gate[t, j] x[t, m] @ W[expert[t, j]],   with the gradients of x, W and the gates.
// A slot is a (row, choice) pair s = t k + j; the plan lists the slots sorted by expert (stable), so that each
// expert's rows are consecutive and its block is read once per tile of rows.  A slot whose expert lies outside [0, E)
// takes part nowhere.
#pragma once
#include "tile.h"


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
