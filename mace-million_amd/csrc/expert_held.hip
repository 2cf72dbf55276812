// Float rows of up to 128 values past weight blocks held in registers, for one expert or a pair of experts at a time.
#include "experts.h"

// Float rows of up to 128 values: the products of mm_expert_rows with the block in registers.  A workgroup is 4 waves;
// each holds 32 of 128 columns of its expert's block, split into planes (96 registers at K = 128), and streams up to
// `chunk` of the expert's rows past them, 32 (a stage) at a time.  A stage is loaded by the whole workgroup, split
// once and written to LDS in operand order, one stage ahead of the products and two ahead in registers, so an operand
// is split once where the tiles of mm_expert_rows split it in every wave, and the block is read once per chunk.  Bound
// by the products and the rows' traffic.  With gates (one choice a row) the rows are the result itself; list E, the
// slots without an expert, is then written as zeros.  65,536 rows 128 -> 128, one of 8 experts: 25 us (86 TFLOP/s).
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

// KS: steps of 32 values.  FULL: K = 32 KS and whole tiles of columns, so that no load or store stands behind a
// branch: the compiler then counts them and waits for the loads it needs only, not for the stores before them.  One
// row's 8 values g of step t, plane p at unit ((tile * 3 + p) * 4 KS + 4 t + g) * 17 + row.  RG = 2 (64 columns or
// fewer): the waves share a stage's row tiles as well as the columns, so that none is left without work.
template <bool TRANS, int KS, bool FULL, int RG>
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
  const int n0 = part * 128 + 32 * (RG == 1 ? wave : wave & 1), tile0 = RG == 1 ? 0 : wave >> 1;   // columns, row tile
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
      floatx4 acc[2 / RG][2] = {};   // [row tile][column tile]
      load(st + 2, x[b]);
      MMFrag<float> f[2][2 / RG];
      auto operands = [&](int s) {
#pragma unroll
        for (int r = 0; r < 2 / RG; ++r)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            f[s & 1][r].v[p] =
                __builtin_bit_cast(bf16x8, Al[b][(((tile0 + r) * 3 + p) * KG + 4 * s + g) * MM_HELD_AS + i]);
      };
      operands(0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if (s + 1 < KS) operands(s + 1);
        __builtin_amdgcn_sched_barrier(0);   // the reads of the next step stay ahead of the products of this one
        put(b ^ 1, s, x[b ^ 1]);             // a part of the next stage beside them (PER = KS)
#pragma unroll
        for (int r = 0; r < 2 / RG; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) mm_mma(acc[r][c], w[s][c], f[s & 1][r]);
      }
#pragma unroll
      for (int r = 0; r < 2 / RG; ++r) {
        const int row = 32 * st + 16 * (tile0 + r) + i;   // past the last row: that one again, with the same values
        float* __restrict__ o = a.out + (long)s_out[row] * a.N;
        const float gate = s_g[row];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const floatx4 v = acc[r][c];
          const float scaled[4] = {gate * v[0], gate * v[1], gate * v[2], gate * v[3]};
          if constexpr (FULL)
            *(floatx4u*)(o + n0 + 16 * c + 4 * g) = floatx4u{scaled[0], scaled[1], scaled[2], scaled[3]};
          else mm_store4(o, n0 + 16 * c + 4 * g, a.N, scaled);
        }
      }
      __syncthreads();
    }
  }
}

// The same for rows of two choices sorted by the pair of their experts: 8 waves hold 16 columns of both blocks (the
// same 96 registers at K = 128), every operand of a row is read once for both, and the two products of a row are
// joined and written once.  64 rows a stage, one workgroup a CU.  DG: with the rows of dy and W[e]^T also dgates[t, j]
// = sum over m of <x[t, m], (dy W[e_j]^T)[t, m]>; all columns are then in one workgroup, and a chunk holds whole rows
// t.  RG = 2 (64 columns or fewer): 4 waves a half of a stage's rows (203,760 rows 112 -> 32: 108 us without, 85 so).
// 98,304 rows 128 -> 128, 2 of 8 experts: 43 us (150 TFLOP/s of 207 that split operands allow); each further 98,304
// rows add 30 us, the rest is the first loads and the blocks' split.  DG, 49,152 rows: 43 us.
template <bool TRANS, int KS, bool FULL, bool DG, int RG>
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
  const int n0 = part * 128 + 16 * (RG == 1 ? wave : wave & 3);
  const int tile0 = RG == 1 ? 0 : wave >> 2 << 1;   // first row tile
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
      float xv[DG ? 4 / RG : 1][4];
      if constexpr (DG) {
#pragma unroll
        for (int r = 0; r < 4 / RG; ++r)
          mm_load4(a.x + s_x[64 * st + 16 * (tile0 + r) + i], n0 + 4 * g, a.N, xv[r]);
      }
      load(st + 2, x[b]);
      constexpr int H = 2 / RG;
      floatx4 acc[2][2 * H] = {};   // [choice][row tile]
      MMFrag<float> f[2][2];
      // row tiles 2 h, 2 h + 1 of this wave's, step s: number H s + h
      auto operands = [&](int q) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int p = 0; p < 3; ++p)
            f[q & 1][r].v[p] = __builtin_bit_cast(
                bf16x8, Al[b][(((tile0 + 2 * (q % H) + r) * 3 + p) * KG + 4 * (q / H) + g) * MM_HELD_AS + i]);
      };
      operands(0);
#pragma unroll
      for (int q = 0; q < H * KS; ++q) {
        if (q + 1 < H * KS) operands(q + 1);
        __builtin_amdgcn_sched_barrier(0);                     // the reads of the next step stay ahead of the products
        if (q % H == H - 1) put(b ^ 1, q / H, x[b ^ 1]);       // a part of the next stage beside them (PER = KS)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) mm_mma(acc[c][2 * (q % H) + r], w[c][q / H], f[q & 1][r]);
      }
#pragma unroll
      for (int r = 0; r < 2 * H; ++r) {
        const int row = 64 * st + 16 * (tile0 + r) + i;   // past the last row: that one again, with the same values
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
            s_part[b][wave][0][16 * (tile0 + r) + i] = d0;
            s_part[b][wave][1][16 * (tile0 + r) + i] = d1;
          }
        }
      }
      __syncthreads();
      if constexpr (DG) {   // the columns of a row, wave by wave; the other s_part is written next
        if (tid < 128) {
          const int c = tid >> 6, wave0 = RG == 2 ? lane / 32 * 4 : 0;   // the waves of this row
          float d = 0.f;
#pragma unroll
          for (int v = 0; v < 8 / RG; ++v) d += s_part[b][wave0 + v][c][lane];
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

// ------------------------------------------------------------------------------------------------ launches
namespace {
// Rows per workgroup of the held blocks: for one round of the 512 that are resident (2 a CU), at most two and so on,
// with the experts' cut chunks taken off; 32 rows are a stage.
int held_chunk(long rows, long tiles_n, int lists) {
  for (long n = 1;; ++n) {
    const long wg = 512 * n - lists * tiles_n;
    if (wg < 256) continue;
    const long c = ((rows * tiles_n + wg - 1) / wg + 31) / 32 * 32;
    if (c <= MM_HELD_ROWS) return (int)(c < 32 ? 32 : c);
  }
}

}  // namespace

namespace mm {
int launch_held(const char* name, const MMRows& a, int S, const float* gates, int lists, int transposed,
                hipStream_t stream) {
  const int tiles_n = (a.N + 127) / 128, chunk = held_chunk((long)S * a.M, tiles_n, lists);
  const long wg = (((long)S * a.M + chunk - 1) / chunk + (lists < S ? lists : S)) * tiles_n;
  if (too_many(wg, 256)) return range_error(name, "output too large for one launch");
  const MMHeld h{a, gates, lists, S};
  const bool whole = a.N % 128 == 0;
#define CALL2(trans, ks, full, rg)                                                                           \
  hipLaunchKernelGGL((mm_expert_held_kernel<trans, ks, full, rg>), dim3((unsigned)wg), dim3(256), 0, stream, \
                     h, tiles_n, chunk)
#define CALL(trans, ks)                                   \
  if (a.K == 32 * ks && whole) CALL2(trans, ks, true, 1); \
  else if (a.N <= 64) CALL2(trans, ks, false, 2);         \
  else CALL2(trans, ks, false, 1)
#define CALLS(trans)                    \
  if (a.K <= 32) { CALL(trans, 1); }    \
  else if (a.K <= 64) { CALL(trans, 2); } \
  else { CALL(trans, 4); }
  if (transposed) { CALLS(true) } else { CALLS(false) }
#undef CALLS
#undef CALL
#undef CALL2
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
  if (too_many(wg, 512)) return range_error(name, "output too large for one launch");
#define CALL2(trans, ks, full, dg, rg)                                                                             \
  hipLaunchKernelGGL((mm_expert_held_pairs_kernel<trans, ks, full, dg, rg>), dim3((unsigned)wg), dim3(512), 0, \
                     stream, a, tiles_n, chunk)
#define CALL(trans, ks, dg)                                             \
  if (a.K == 32 * ks && a.N % 128 == 0) CALL2(trans, ks, true, dg, 1);  \
  else if (a.N <= 64) CALL2(trans, ks, false, dg, 2);                   \
  else CALL2(trans, ks, false, dg, 1);
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

}  // namespace mm
