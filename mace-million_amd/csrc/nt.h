// Tiles of C = A B^T with both operands rows of 16-bit values along the summed index:
//     C[m, n] = sum over the passes (i, j) and k of A_i[m, k] B_j[n, k]
// P = 1: one plane each.  P = 3: two planes (float16 high and low parts, 22 bits), the three products without low x
// low.  P = 6: three bfloat16 planes of float, the six products with i + j <= 2.  Rows are 16-byte aligned, their length
// a multiple of 64 values, zeros past the summed index.  Rows past the last one of an operand are read as the last one
// and give results that nobody stores.
#pragma once
#include "tile.h"

#include <type_traits>

#define MM_NT_K 64   // values of the summed index of a stage

template <typename H>
struct MMNtOperand {
  const H* p;
  long ld, plane;   // distances of rows and planes
  int rows;
};

// planes of pass q
template <int P>
__device__ __forceinline__ constexpr int mm_nt_first(int q) {
  return P == 1 ? 0 : P == 3 ? (q == 0 ? 1 : 0) : (q == 0 ? 2 : q == 1 || q == 3 ? 1 : 0);
}
template <int P>
__device__ __forceinline__ constexpr int mm_nt_second(int q) {
  return P == 1 ? 0 : P == 3 ? (q == 1 ? 1 : 0) : (q == 2 ? 2 : q == 1 || q == 4 ? 1 : 0);
}

// A workgroup's tile of BM rows of A by BN rows of B, WM x WN waves; lane's results acc[i][j][q]: row m = wm + 16 j +
// (lane & 15) of the tile, column n = wn + 16 i + 4 (lane >> 4) + q.
template <typename H, int P, int BM_, int BN_, int WM_, int WN_>
struct MMNtOne {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, PER_CU = 2;
  static constexpr int TH = 64 * WM * WN, UA = BM * 8 / TH, UB = BN * 8 / TH;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int LDS = 2 * (BM + BN) * 8 * 16;   // bytes
  floatx4 acc[FN][FM];
  int wm, wn, lane;

  __device__ __forceinline__ MMNtOne() {
    const int wave = threadIdx.x >> 6;
    lane = threadIdx.x & 63;
    wm = (wave % WM) * (BM / WM);
    wn = (wave / WM) * (BN / WN);
  }
  __device__ __forceinline__ int row(int j) const { return wm + 16 * j + (lane & 15); }
  __device__ __forceinline__ int col(int i) const { return wn + 16 * i + 4 * (lane >> 4); }

  // stages k0 .. k1 - 1 (of 64 values) of every pass; the LDS is free afterwards
  __device__ __forceinline__ void run(const MMNtOperand<H>& a, int m0, const MMNtOperand<H>& b, int n0, int k0, int k1,
                                      uint4* lds) {
    uint4 *As = lds, *Bs = lds + 2 * BM * 8;
    const int tid = threadIdx.x, ka = ((tid & 7) ^ (tid >> 3 & 7)) * 8;
    const H *pa[UA], *pb[UB];
#pragma unroll
    for (int j = 0; j < UA; ++j) pa[j] = a.p + (long)min(m0 + ((tid + TH * j) >> 3), a.rows - 1) * a.ld + ka;
#pragma unroll
    for (int j = 0; j < UB; ++j) pb[j] = b.p + (long)min(n0 + ((tid + TH * j) >> 3), b.rows - 1) * b.ld + ka;
    MMStage<H, TH, UA, true> sa;
    MMStage<H, TH, UB, true> sb;
    auto load = [&](int k, int q, int buf) {
      const long oa = mm_nt_first<P>(q) * a.plane + (long)k * MM_NT_K;
      const long ob = mm_nt_second<P>(q) * b.plane + (long)k * MM_NT_K;
#pragma unroll
      for (int j = 0; j < UA; ++j) sa.load(As + buf * BM * 8, j, pa[j] + oa, 8);
#pragma unroll
      for (int j = 0; j < UB; ++j) sb.load(Bs + buf * BN * 8, j, pb[j] + ob, 8);
    };
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    if (k0 >= k1) return;
    load(k0, 0, 0);
    mm_stage_done();
    int buf = 0, k = k0, q = 0;
    while (k < k1) {
      if (++q == P) {
        q = 0;
        ++k;
      }
      if (k < k1) load(k, q, buf ^ 1);
      const uint4 *A = As + buf * BM * 8, *B = Bs + buf * BN * 8;
      mm_products<H, FN, FM, 2>(
          acc, [&](int s, int i) { return mm_read_kc<H>(B, wn + 16 * i, s, lane); },
          [&](int s, int j) { return mm_read_kc<H>(A, wm + 16 * j, s, lane); });
      mm_stage_done();
      buf ^= 1;
    }
  }
};

// The same for operands of several planes (P > 1): a stage holds all planes of 32 values, so that a plane is loaded once
// for the products that it enters.  A ring of SLOTS stages, loads SLOTS - 1 stages ahead; units lie as in MMNtBig.
// Bound by the matrix cores and the reads of LDS before them: float, 2048 x 512 results of 8192 values, 103 G operations
// of bfloat16 in 112 us (920 TFLOP/s).
template <typename H, int P, int BM_, int BN_, int WM_, int WN_>
struct MMNtPlanes {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, TH = 64 * WM * WN, PL = P == 3 ? 2 : 3;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16, STAGE = PL * (BM + BN) * 4;   // units
  static constexpr int SLOTS = STAGE <= 1024 ? 4 : STAGE == 2048 ? 2 : 3, LDS = SLOTS * STAGE * 16;
  static constexpr int PER_CU = LDS <= 81920 ? 2 : 1, LOADS = STAGE / TH;
  floatx4 acc[FN][FM];
  int wm, wn, lane;

  __device__ __forceinline__ MMNtPlanes() {
    const int wave = threadIdx.x >> 6;
    lane = threadIdx.x & 63;
    wm = (wave % WM) * (BM / WM);
    wn = (wave / WM) * (BN / WN);
  }
  __device__ __forceinline__ int row(int j) const { return wm + 16 * j + (lane & 15); }
  __device__ __forceinline__ int col(int i) const { return wn + 16 * i + 4 * (lane >> 4); }
  static __device__ __forceinline__ int twist(int r) { return (r >> 1 & 3) ^ (r >> 3 & 1); }

  __device__ __forceinline__ void run(const MMNtOperand<H>& a, int m0, const MMNtOperand<H>& b, int n0, int k0, int k1,
                                      uint4* lds) {
    typedef typename MMFrag<H>::vec vec;
    constexpr int UA = BM * 4 / TH, UB = BN * 4 / TH;   // units of a thread and plane
    const int tid = threadIdx.x;
    const H *pa[UA], *pb[UB];
#pragma unroll
    for (int j = 0; j < UA; ++j) {
      const int r = (tid + TH * j) >> 2;
      pa[j] = a.p + (long)min(m0 + r, a.rows - 1) * a.ld + ((tid & 3) ^ twist(r)) * 8;
    }
#pragma unroll
    for (int j = 0; j < UB; ++j) {
      const int r = (tid + TH * j) >> 2;
      pb[j] = b.p + (long)min(n0 + r, b.rows - 1) * b.ld + ((tid & 3) ^ twist(r)) * 8;
    }
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int stages = (k1 - k0) * 2;
    if (stages <= 0) return;
    auto load = [&](int s) {
      const long at = (long)k0 * MM_NT_K + 32 * s;
      uint4* to = lds + s % SLOTS * STAGE + (tid & ~63);
#pragma unroll
      for (int p = 0; p < PL; ++p) {
#pragma unroll
        for (int j = 0; j < UA; ++j)
          __builtin_amdgcn_global_load_lds((mm_global_ptr)(pa[j] + p * a.plane + at),
                                           (mm_lds_ptr)(to + p * BM * 4 + TH * j), 16, 0, 0);
#pragma unroll
        for (int j = 0; j < UB; ++j)
          __builtin_amdgcn_global_load_lds((mm_global_ptr)(pb[j] + p * b.plane + at),
                                           (mm_lds_ptr)(to + (PL * BM + p * BN) * 4 + TH * j), 16, 0, 0);
      }
    };
    const int i16 = lane & 15, unit = 4 * i16 + ((lane >> 4) ^ twist(i16));
#pragma unroll
    for (int s = 0; s < SLOTS - 1; ++s)
      if (s < stages) load(s);
    for (int s = 0; s < stages; ++s) {
      // this wave's part of stage s has arrived; after the barrier every wave's has, and nobody reads stage s - 1
      if (s + SLOTS - 2 < stages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((SLOTS - 2) * LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + SLOTS - 1 < stages) load(s + SLOTS - 1);
      const uint4* A = lds + s % SLOTS * STAGE + 4 * wm + unit;
      const uint4* B = lds + s % SLOTS * STAGE + 4 * (PL * BM + wn) + unit;
      vec fb[PL][FN], fa[2][PL];
#pragma unroll
      for (int p = 0; p < PL; ++p) {
#pragma unroll
        for (int i = 0; i < FN; ++i) fb[p][i] = __builtin_bit_cast(vec, B[4 * BN * p + 64 * i]);
        fa[0][p] = __builtin_bit_cast(vec, A[4 * BM * p]);
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        if (j + 1 < FM) {
#pragma unroll
          for (int p = 0; p < PL; ++p) fa[(j + 1) & 1][p] = __builtin_bit_cast(vec, A[4 * BM * p + 64 * (j + 1)]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
          for (int i = 0; i < FN; ++i) {
            MMFrag<H> x{fb[mm_nt_second<P>(q)][i]}, y{fa[j & 1][mm_nt_first<P>(q)]};
            mm_mma(acc[i][j], x, y);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
  }
};

template <typename H, int P, int BM, int BN, int WM, int WN>
using MMNt = std::conditional_t<P == 1, MMNtOne<H, P, BM, BN, WM, WN>, MMNtPlanes<H, P, BM, BN, WM, WN>>;

// The same for tiles of 256 x 256 by 8 waves (2 x 4, 128 x 64 each) where there are enough of them for every CU.  128 KB
// of LDS hold a ring of four stages of 32 values: the loads of a stage have two stages' products (2048 cycles) to
// arrive, and a wave waits for its own part of the next stage only, once a stage.  Operands are read two products' rows
// ahead across the stages' borders, so that the matrix cores do not wait at the barrier either; the loads are issued
// between the products (all at the start of a stage they hold up its reads: 5 % slower).  Bound by LDS (96 KB read and 32
// written a stage, 1000 cycles at 128 bytes a cycle) and the matrix cores (1024 cycles) alike.  Four waves of 128 x 128
// would read a third less, but have nothing to run beside an epilogue (logits of 8192 x 131072, 2048 values: 6.1 ms
// against 4.1).  bfloat16, 8192 x 2048 results a piece, 8192 products each: 228 us, 1210 TFLOP/s.
// A row of a stage is 4 units of 16 bytes, unit u of row r at 4 r + (u ^ f(r)), so that any 8 or 16 consecutive rows of
// an operand read lie in different banks.
template <typename H, int P>
struct MMNtBig {
  static constexpr int BM = 256, BN = 256, WM = 2, WN = 4, TH = 512, FM = 8, FN = 4, PER_CU = 1, LOADS = 1024 / TH;
  static constexpr int LDS = 4 * (BM + BN) * 4 * 16;   // bytes
  floatx4 acc[FN][FM];
  int wm, wn, lane;

  __device__ __forceinline__ MMNtBig() {
    const int wave = threadIdx.x >> 6;
    lane = threadIdx.x & 63;
    wm = (wave % WM) * (BM / WM);
    wn = (wave / WM) * (BN / WN);
  }
  __device__ __forceinline__ int row(int j) const { return wm + 16 * j + (lane & 15); }
  __device__ __forceinline__ int col(int i) const { return wn + 16 * i + 4 * (lane >> 4); }
  static __device__ __forceinline__ int twist(int r) { return (r >> 1 & 3) ^ (r >> 3 & 1); }

  __device__ __forceinline__ void run(const MMNtOperand<H>& a, int m0, const MMNtOperand<H>& b, int n0, int k0, int k1,
                                      uint4* lds) {
    typedef typename MMFrag<H>::vec vec;
    constexpr int STAGE = (BM + BN) * 4;   // units
    const int tid = threadIdx.x;
    const H *pa[LOADS], *pb[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int r = (tid + TH * j) >> 2, u = ((tid & 3) ^ twist(r)) * 8;
      pa[j] = a.p + (long)min(m0 + r, a.rows - 1) * a.ld + u;
      pb[j] = b.p + (long)min(n0 + r, b.rows - 1) * b.ld + u;
    }
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int stages = (k1 - k0) * 2 * P;
    if (stages <= 0) return;
    long at = (long)k0 * MM_NT_K;   // of the next stage to load, and its pass
    int pass = 0;
    auto load = [&](int slot, int j) {   // part j of a stage, the last one moves on
      const long oa = mm_nt_first<P>(pass) * a.plane + at, ob = mm_nt_second<P>(pass) * b.plane + at;
      uint4* to = lds + slot * STAGE + (tid & ~63) + TH * j;
      __builtin_amdgcn_global_load_lds((mm_global_ptr)(pa[j] + oa), (mm_lds_ptr)to, 16, 0, 0);
      __builtin_amdgcn_global_load_lds((mm_global_ptr)(pb[j] + ob), (mm_lds_ptr)(to + BM * 4), 16, 0, 0);
      if (j + 1 < LOADS) return;
      if (P == 1) {
        at += 32;
      } else if (++pass == P) {
        pass = 0;
        at += 32;
      }
    };
    auto load_all = [&](int slot) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load(slot, j);
    };
    const int i16 = lane & 15, unit = 4 * i16 + ((lane >> 4) ^ twist(i16));
    const int ua = 4 * wm + unit, ub = 4 * (BM + wn) + unit;
    auto read_a = [&](int slot, int j) { return __builtin_bit_cast(vec, lds[slot * STAGE + ua + 64 * j]); };
    auto read_b = [&](int slot, int i) { return __builtin_bit_cast(vec, lds[slot * STAGE + ub + 64 * i]); };
    load_all(0);
    if (stages > 1) load_all(1);
    if (stages > 2) load_all(2);
    if (stages > 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * LOADS) : "memory");
    else if (stages > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    vec fa[4], fb[2][FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) fb[0][i] = read_b(0, i);
    fa[0] = read_a(0, 0);
    fa[1] = read_a(0, 1);
    auto step = [&](int s, auto odd) {
      constexpr int O = decltype(odd)::value;
      // this wave's part of stage s + 1 has arrived; after the barrier every wave's has, and nobody reads stage s - 1
      if (s + 2 < stages) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int now = s & 3, next = (s + 1) & 3;
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        if ((j == 1 || j == 4) && s + 3 < stages) load((s + 3) & 3, j / 4);   // apart: together they hold up the reads
        fa[(j + 2) & 3] = j + 2 < FM ? read_a(now, j + 2) : read_a(next, j + 2 - FM);
        if (j >= 2 && j < 2 + FN) fb[O ^ 1][j - 2] = read_b(next, j - 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          MMFrag<H> x{fb[O][i]}, y{fa[j & 3]};
          mm_mma(acc[i][j], x, y);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int s = 0; s < stages; s += 2) {   // stages come in pairs: 64 values
      step(s, std::integral_constant<int, 0>{});
      step(s + 1, std::integral_constant<int, 1>{});
    }
    __syncthreads();   // the last stage's reads (and those past it, of old values) are done
  }
};

// Four 16-bit values of every lane, lane l holding row l & 3 of a 4 x 4 block by its quad of lanes: transposed, so that
// lane l holds the block's column l & 3.  By lane moves inside the quad: pairs with the lane two further, then halves of
// pairs with the next one.
template <typename H>
__device__ __forceinline__ void mm_quad_transpose(H (&v)[4]) {
  typedef H pair __attribute__((ext_vector_type(2)));
  const int r = threadIdx.x & 3;
  const int w0 = __builtin_bit_cast(int, pair{v[0], v[1]}), w1 = __builtin_bit_cast(int, pair{v[2], v[3]});
  const int got = __builtin_amdgcn_mov_dpp(r < 2 ? w1 : w0, 0x4E, 0xF, 0xF, true);   // quad_perm [2, 3, 0, 1]
  const int lo = r < 2 ? w0 : got, hi = r < 2 ? got : w1;
  const int lo1 = __builtin_amdgcn_mov_dpp(lo, 0xB1, 0xF, 0xF, true);                // quad_perm [1, 0, 3, 2]
  const int hi1 = __builtin_amdgcn_mov_dpp(hi, 0xB1, 0xF, 0xF, true);
  // even lanes: the low halves of their own and the other's; odd lanes: the high halves of the other's and their own
  const unsigned pick = r & 1 ? 0x03020706 : 0x05040100;
  const pair a = __builtin_bit_cast(pair, __builtin_amdgcn_perm(lo1, lo, pick));
  const pair b = __builtin_bit_cast(pair, __builtin_amdgcn_perm(hi1, hi, pick));
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
}

// A workgroup's results as rows of 16-bit values, through LDS (`tile`, BM x BN values, free before and after) so that
// whole lines go out: out[m][n] for m < rows, n < cols, cols a multiple of 8 and rows of out 16-byte aligned.
// value(i, j): the four values of acc[i][j].  Units of 16 bytes are turned by their row's number, against bank conflicts.
template <typename H, typename Nt, typename F>
__device__ __forceinline__ void mm_nt_store(const Nt& t, H* tile, H* out, long ld, int rows, int cols, F value) {
  typedef H vec __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j)
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i) {
      const int m = t.row(j), n = t.col(i);
      const floatx4 v = value(i, j);
      *(vec*)(tile + m * Nt::BN + ((n >> 3 ^ (m & 7)) << 3) + (n & 4)) = vec{(H)v[0], (H)v[1], (H)v[2], (H)v[3]};
    }
  __syncthreads();
#pragma unroll 4
  for (int q = threadIdx.x; q < Nt::BM * Nt::BN / 8; q += Nt::TH) {
    const int m = q / (Nt::BN / 8), u = q % (Nt::BN / 8);
    if (m < rows && 8 * u < cols)
      *(uint4*)(out + (long)m * ld + 8 * u) = *(const uint4*)(tile + m * Nt::BN + ((u ^ (m & 7)) << 3));
  }
  __syncthreads();
}

// The same transposed: out[n][m] for n < cols, m < rows, rows a multiple of 8.
template <typename H, typename Nt, typename F>
__device__ __forceinline__ void mm_nt_store_transposed(const Nt& t, H* tile, H* out, long ld, int rows, int cols,
                                                       F value) {
  typedef H vec __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int j = 0; j < Nt::FM; ++j)
#pragma unroll
    for (int i = 0; i < Nt::FN; ++i) {
      const floatx4 v = value(i, j);
      H h[4] = {(H)v[0], (H)v[1], (H)v[2], (H)v[3]};
      mm_quad_transpose(h);   // this lane's column n + (lane & 3), rows of its quad of lanes
      const int m = t.row(j) & ~3, n = t.col(i) + (t.lane & 3);
      *(vec*)(tile + n * Nt::BM + ((m >> 3 ^ (n & 7)) << 3) + (m & 4)) = vec{h[0], h[1], h[2], h[3]};
    }
  __syncthreads();
#pragma unroll 4
  for (int q = threadIdx.x; q < Nt::BM * Nt::BN / 8; q += Nt::TH) {
    const int n = q / (Nt::BM / 8), u = q % (Nt::BM / 8);
    if (n < cols && 8 * u < rows)
      *(uint4*)(out + (long)n * ld + 8 * u) = *(const uint4*)(tile + n * Nt::BM + ((u ^ (n & 7)) << 3));
  }
  __syncthreads();
}

// Tile of workgroup b among `batch` times tiles_m x tiles_n: consecutive numbers on one XCD (workgroups are dealt out to
// the 8 XCDs in turn), in bands of 8 tiles of rows, so that neighbours share operands in that XCD's L2.  False: none.
__device__ __forceinline__ bool mm_nt_tile(int b, int batch, int tiles_m, int tiles_n, int* e, int* tm, int* tn) {
  const int one = tiles_m * tiles_n, all = batch * one;
  if (b >= all) return false;
  const int share = all / 8, rest = all % 8, x = b % 8;
  int at = x * share + min(x, rest) + b / 8;
  *e = at / one;
  at -= *e * one;
  const int band = at / (8 * tiles_n), high = min(8, tiles_m - 8 * band), r = at - band * 8 * tiles_n;
  *tm = 8 * band + r % high;
  *tn = r / high;
  return true;
}

// The same for the tiles on and below the diagonal of `batch` square products of `tiles` x `tiles`.
__device__ __forceinline__ bool mm_nt_lower(int b, int batch, int tiles, int* e, int* tm, int* tn) {
  const int one = tiles * (tiles + 1) / 2, all = batch * one;
  if (b >= all) return false;
  const int share = all / 8, rest = all % 8, x = b % 8;
  int at = x * share + min(x, rest) + b / 8, m = 0;
  *e = at / one;
  at -= *e * one;
  while (at > m) at -= ++m;   // row m has m + 1 tiles
  *tm = m;
  *tn = at;
  return true;
}

__host__ __device__ inline long mm_up(long n, long size) { return (n + size - 1) / size * size; }

// Tiles of 256, 128 and 64 for P products: how many run at once, and the time of such a round where one tile of 256 on
// every CU takes 1, by the rates that products of 1024 and more reach (planes leave room for fewer workgroups on a
// CU).  Logits of 1024 values and their sums, us by tiles of 256 | 128 | 64: bfloat16 1024 x 1024 47 | 32 | 27, 2048 x
// 8192 56 | 60 | 75, 4096 x 16,384 159 | 170 | 224; float (P = 6) 174 | 62 | 42, 212 | 214 | 259, 735 | 753 | 940.  P
// = 3, five steps of float matrices: 1024 x 1024 1545 | 582 | 278, 14 of them 3222 | 1829 | 1856 (in parts by their
// own tiles 1643).
struct MMTileRates {
  int side[3] = {256, 128, 64}, slots[3];
  double round[3];
};
inline MMTileRates mm_tile_rates(int P) {
  if (P == 1) return MMTileRates{{256, 128, 64}, {256, 512, 1024}, {1., 0.59, 0.5}};
  if (P == 3) return MMTileRates{{256, 128, 64}, {256, 512, 512}, {1., 0.59, 0.28}};
  return MMTileRates{{256, 128, 64}, {256, 256, 512}, {1., 0.31, 0.28}};
}

// Time of a launch that would have t256, t128 or t64 tiles of those sides, with the best of them.
inline double mm_tile_time(int P, long t256, long t128, long t64, int* side = nullptr) {
  const MMTileRates r = mm_tile_rates(P);
  const long t[] = {t256, t128, t64};
  double least = 1e30;
  for (int i = 0; i < 3; ++i) {
    const double time = r.round[i] * (double)((t[i] + r.slots[i] - 1) / r.slots[i]);
    if (time < least) {
      least = time;
      if (side) *side = r.side[i];
    }
  }
  return least;
}

inline int mm_tile_side(int P, long t256, long t128, long t64) {
  int side = 64;
  mm_tile_time(P, t256, t128, t64, &side);
  return side;
}
