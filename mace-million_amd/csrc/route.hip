// Routing of rows (atoms, tokens) to experts: the choice of k of E experts by their logits, and the gates.
//     key_e = logit_e + bias_e (fp32, one rounding); a logit or key of -inf closes the expert
//     groups: the top_groups groups (of E / groups experts each) of largest key stay open
//     chosen: the k largest keys, ties to the lowest index; expert -1 and gate 0 where no open expert is left
//     score: softmax over the E logits, or sigmoid of each
//     gate_j = scale score_j / sum_chosen score, or scale score_j
// The bias moves the choice only, not the gates.  It is added to the logits: one rounded addition, so the choice does
// not depend on the order of a sum or the rounding of an exponential, and saturated sigmoids do not tie.  This is a
// rule of its own: with a bias that differs between experts, score + bias (or a group's key from the sum of its two
// best) orders them otherwise, so a router trained with that rule chooses other experts here; without a bias the orders
// are the same.  Renormalised gates are a softmax over the chosen of the scores' logarithms (of the logits, or of log
// sigmoid), so that scores that all underflow still give gates of sum scale.  A NaN logit is chosen first and makes the
// gates of its row NaN (of plain sigmoids: its own gate).
// A row lies in LPR lanes, C consecutive logits each; k rounds of a maximum over the lanes' best keys (as integers of
// the same order), the lowest lane with it giving its first such logit: no sort, no memory but the logits and the
// results.  Bound by vector instructions where there are many experts (1,000 a wave of 4 rows of 256 with k = 8 and
// groups, 470 of 89 with k = 3: the SIMDs issue them without a pause), by HBM for few.  Measured, forward and backward:
// 500,000 float rows of 16, k = 2: 17.6 and 10.2 us (40 and 44 MB); 65,536 bfloat16 rows of 256, k = 8 of 4 in 8
// groups: 29 and 13 us (38 MB each); 98,304 float16 rows of 89, k = 3, plain softmax: 18 us; one row: 2.7 us.
#include "rowvec.h"

#define MM_ROUTE_MAX_E 1024
#define MM_ROUTE_MAX_K 32
#define MM_ROUTE_MAX_G 64

// larger key, larger integer; NaN above all, 0 for -inf (closed)
__device__ __forceinline__ unsigned mm_route_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  if (x == -__builtin_inff()) return 0u;
  const unsigned u = __float_as_uint(x + 0.f);   // -0 + 0 = +0: equal keys are equal integers
  return u >> 31 ? ~u : u | 0x80000000u;
}

template <int CTRL>
__device__ __forceinline__ unsigned mm_dpp_u(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}

// maximum over the W lanes of a row, in every lane
template <int W>
__device__ __forceinline__ unsigned mm_route_max(unsigned v) {
  if constexpr (W >= 2) v = max(v, mm_dpp_u<0xB1>(v));
  if constexpr (W >= 4) v = max(v, mm_dpp_u<0x4E>(v));
  if constexpr (W >= 8) v = max(v, mm_dpp_u<0x141>(v));
  if constexpr (W >= 16) v = max(v, mm_dpp_u<0x140>(v));
  if constexpr (W >= 32) v = max(v, (unsigned)__shfl_xor((int)v, 16));
  if constexpr (W >= 64) v = max(v, (unsigned)__shfl_xor((int)v, 32));
  return v;
}

// exp(x) for x <= 0 (NaN stays NaN) to 2 units in the last place: 2^(x log2 e) with the rounding error of the product
// put back to first order.  A softmax over a whole row takes one per logit, and expf twice the instructions.
__device__ __forceinline__ float mm_exp_neg(float x) {
  x = x < -150.f ? -150.f : x;   // 0 either way
  const float t = x * 1.44269504088896340736f;
  const float lo = fmaf(x, 1.92596299112661746887e-8f, fmaf(x, 1.44269504088896340736f, -t));
  const float p = __builtin_amdgcn_exp2f(t);
  return fmaf(p, lo * 0.693147180559945309417f, p);
}

// C consecutive values of a row from column c on, `none` past the last one
template <typename T, int C>
__device__ __forceinline__ void mm_route_load(const T* __restrict__ p, int c, int E, float none, float* v) {
  constexpr int N = C < MMVec<T>::N ? C : MMVec<T>::N;
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
#pragma unroll
  for (int q = 0; q < C; q += N) {
    if (c + q + N <= E) {
      const vec x = *(const vec*)(p + c + q);
#pragma unroll
      for (int i = 0; i < N; ++i) v[q + i] = (float)x[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[q + i] = c + q + i < E ? (float)p[c + q + i] : none;
    }
  }
}

struct MMRoute {
  long T, ldl;
  int E, k, sigmoid, groups, top_groups, renorm;
  float scale;
};

// KM: results a lane keeps (choice q LPR + lane), enough for k
template <typename T, int LPR, int C, int KM>
__global__ void __launch_bounds__(256) mm_route_fwd_kernel(MMRoute a, const T* __restrict__ logits,
                                                           const float* __restrict__ bias, float* __restrict__ gates,
                                                           int* __restrict__ experts) {
  constexpr int RPB = 256 / LPR;   // rows per workgroup
  constexpr int G = LPR * C < MM_ROUTE_MAX_G ? LPR * C : MM_ROUTE_MAX_G;   // groups, at most
  __shared__ unsigned s_best[RPB][G], s_open[RPB][2];
  const int lane = threadIdx.x & (LPR - 1), sub = threadIdx.x / LPR, c0 = lane * C;
  const long row = (long)blockIdx.x * RPB + sub;
  const bool ok = row < a.T;
  const long r = ok ? row : a.T - 1;
  const float none = -__builtin_inff();
  float x[C], b[C] = {};
  unsigned key[C];
  mm_route_load<T, C>(logits + r * a.ldl, c0, a.E, none, x);
  if (bias) mm_route_load<float, C>(bias, c0, a.E, 0.f, b);
#pragma unroll
  for (int i = 0; i < C; ++i) key[i] = x[i] == none ? 0u : mm_route_key(x[i] + b[i]);
  if (a.groups > 1) {
    const int gs = a.E / a.groups, g0 = c0 / gs, rem = c0 - g0 * gs;
    for (int q = lane; q < a.groups; q += LPR) s_best[sub][q] = 0;
    if (lane < 2) s_open[sub][lane] = 0;
    mm_wave_lds_sync();
    const bool whole = gs % C == 0;   // a lane's logits belong to one group
    int g = g0, m = rem;
    if (whole) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < C; ++i) top = max(top, key[i]);
      if (c0 < a.E) atomicMax(&s_best[sub][g], top);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (c0 + i < a.E) atomicMax(&s_best[sub][g], key[i]);
        if (++m == gs) { m = 0; ++g; }
      }
    }
    mm_wave_lds_sync();
    for (int q = lane; q < a.groups; q += LPR) {
      const unsigned mine = s_best[sub][q];
      int before = 0;
      for (int o = 0; o < a.groups; ++o) {
        const unsigned other = s_best[sub][o];
        before += other > mine || (other == mine && o < q);
      }
      if (before < a.top_groups) atomicOr(&s_open[sub][q >> 5], 1u << (q & 31));
    }
    mm_wave_lds_sync();
    const unsigned open0 = s_open[sub][0], open1 = s_open[sub][1];
    g = g0;
    m = rem;
    if (whole) {
      const bool shut = !((g < 32 ? open0 : open1) >> (g & 31) & 1);
#pragma unroll
      for (int i = 0; i < C; ++i) key[i] = shut ? 0 : key[i];
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        if (!((g < 32 ? open0 : open1) >> (g & 31) & 1)) key[i] = 0;
        if (++m == gs) { m = 0; ++g; }
      }
    }
  }
  // softmax over all experts, where the gates keep its normalisation
  float top = 0.f, whole = 1.f;
  if (!a.renorm && !a.sigmoid) {
    top = none;
#pragma unroll
    for (int i = 0; i < C; ++i) top = fmaxf(top, x[i]);
    top = mm_lanes_max<LPR>(top);
    whole = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) whole += mm_exp_neg(x[i] - top);   // rows with nothing open have no gate that uses it
    whole = mm_lanes_sum<LPR>(whole);
  }
  // the rounds; a lane's keys lie in LDS by fours where it has more than four, and in registers only the fours' best:
  // taking the best one out is then one read, one write and a few maxima, where a pass over C registers was most of a
  // round (65,536 rows of 256, k = 8 of 4 in 8 groups: 55 us so, 29 us now)
  constexpr int Q = C / 4;
  __shared__ uint4 s_key[C > 4 ? RPB : 1][C > 4 ? Q * LPR : 1];
  __shared__ int s_pick[RPB][KM * LPR];
  unsigned four[Q], best = 0;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    four[q] = max(max(key[4 * q], key[4 * q + 1]), max(key[4 * q + 2], key[4 * q + 3]));
    best = max(best, four[q]);
    if constexpr (C > 4)
      s_key[sub][q * LPR + lane] = make_uint4(key[4 * q], key[4 * q + 1], key[4 * q + 2], key[4 * q + 3]);
  }
#pragma unroll
  for (int q = 0; q < KM; ++q) s_pick[sub][q * LPR + lane] = -1;
  const int first_lane = (threadIdx.x & 63) & ~(LPR - 1);
  for (int j = 0; j < a.k; ++j) {
    const unsigned m = mm_route_max<LPR>(best);
    if (__ballot(m != 0) == 0) break;   // no row of the wave has an open expert left
    const unsigned long long have = __ballot(best == m) >> first_lane;
    const int src = __ffsll((unsigned long long)have) - 1;   // the lane of this row with the lowest such index
    if (m != 0 && lane == src) {
      int qi = 0, i = 3;   // its first four with that key, and the first in it
#pragma unroll
      for (int q = Q - 1; q >= 0; --q) qi = four[q] == m ? q : qi;
      uint4 v = make_uint4(key[0], key[1], key[2], key[3]);
      if constexpr (C > 4) v = s_key[sub][qi * LPR + lane];
      i = v.z == m ? 2 : i;
      i = v.y == m ? 1 : i;
      i = v.x == m ? 0 : i;
      s_pick[sub][j] = c0 + 4 * qi + i;
      v = make_uint4(i == 0 ? 0 : v.x, i == 1 ? 0 : v.y, i == 2 ? 0 : v.z, i == 3 ? 0 : v.w);
      if constexpr (C > 4) {
        ((unsigned*)&s_key[sub][qi * LPR + lane])[i] = 0;
      } else {
        key[0] = v.x, key[1] = v.y, key[2] = v.z, key[3] = v.w;
      }
      const unsigned rest = max(max(v.x, v.y), max(v.z, v.w));
      best = 0;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        four[q] = q == qi ? rest : four[q];
        best = max(best, four[q]);
      }
    }
  }
  mm_wave_lds_sync();
  int ej[KM];
#pragma unroll
  for (int q = 0; q < KM; ++q) ej[q] = s_pick[sub][q * LPR + lane];
  float xj[KM];
#pragma unroll
  for (int q = 0; q < KM; ++q) xj[q] = ej[q] >= 0 ? (float)logits[r * a.ldl + ej[q]] : none;
  float gj[KM];
  if (a.renorm) {
    float m = none, sum = 0.f;
#pragma unroll
    for (int q = 0; q < KM; ++q) {
      gj[q] = a.sigmoid ? fminf(xj[q], 0.f) - log1pf(expf(-fabsf(xj[q]))) : xj[q];
      if (xj[q] != xj[q]) gj[q] = xj[q];   // fminf drops a NaN
      if (ej[q] >= 0) m = fmaxf(m, gj[q]);
    }
    m = mm_lanes_max<LPR>(m);
#pragma unroll
    for (int q = 0; q < KM; ++q) {
      gj[q] = ej[q] >= 0 ? expf(gj[q] - m) : 0.f;
      sum += gj[q];
    }
    sum = mm_lanes_sum<LPR>(sum);
#pragma unroll
    for (int q = 0; q < KM; ++q) gj[q] = gj[q] / sum;
  } else {
#pragma unroll
    for (int q = 0; q < KM; ++q) gj[q] = a.sigmoid ? 1.f / (1.f + expf(-xj[q])) : expf(xj[q] - top) / whole;
  }
  if (!ok) return;
#pragma unroll
  for (int q = 0; q < KM; ++q) {
    const int j = q * LPR + lane;
    if (j >= a.k) continue;
    gates[row * a.k + j] = ej[q] >= 0 ? a.scale * gj[q] : 0.f;
    experts[row * a.k + j] = ej[q];
  }
}

// dlogits from dgates, the gates and the chosen experts.  With w_j = gate_j / scale, over the chosen of a row:
//   renormalised       d log score_j = gate_j (dgate_j - sum_i w_i dgate_i)
//   sigmoid, plain     d log score_j = gate_j dgate_j
//   softmax, plain     dl_e = [e chosen] gate_e dgate_e - p_e sum_j gate_j dgate_j,  p over all E logits
// and d log score / dl = 1 (softmax, renormalised) or 1 - sigmoid(l).  The E values of a row are put together in LDS
// and written once; the logits are read where a formula has them.  Bound by HBM.
template <typename T, int LPR, int C, int KM>
__global__ void __launch_bounds__(256) mm_route_bwd_kernel(MMRoute a, const T* __restrict__ logits,
                                                           const float* __restrict__ gates,
                                                           const int* __restrict__ experts,
                                                           const float* __restrict__ dgates, T* __restrict__ dlogits) {
  constexpr int RPB = 256 / LPR;
  __shared__ floatx4 s_d[RPB][C / 4 * LPR];   // four q of lane l at q LPR + l: every bank once
  const int lane = threadIdx.x & (LPR - 1), sub = threadIdx.x / LPR, c0 = lane * C;
  const long row = (long)blockIdx.x * RPB + sub;
  const bool ok = row < a.T;
  const long r = ok ? row : a.T - 1;
  const bool plain_softmax = !a.renorm && !a.sigmoid;
  float x[C];
  if (plain_softmax) mm_route_load<T, C>(logits + r * a.ldl, c0, a.E, -__builtin_inff(), x);
  float d[KM], g[KM], sum = 0.f;
  int e[KM];
#pragma unroll
  for (int q = 0; q < KM; ++q) {
    const int j = q * LPR + lane;
    e[q] = j < a.k ? experts[r * a.k + j] : -1;
    const bool used = (unsigned)e[q] < (unsigned)a.E;
    g[q] = used ? gates[r * a.k + j] : 0.f;
    d[q] = used ? dgates[r * a.k + j] : 0.f;
    if (!used) e[q] = -1;
    sum = fmaf(g[q], d[q], sum);
  }
  sum = mm_lanes_sum<LPR>(sum);
#pragma unroll
  for (int q = 0; q < KM; ++q) {
    d[q] = g[q] * (a.renorm ? d[q] - sum / a.scale : d[q]);
    if (a.sigmoid && e[q] >= 0) d[q] /= 1.f + expf((float)logits[r * a.ldl + e[q]]);
  }
  float v[C];
  if (plain_softmax) {
    float top = -__builtin_inff(), whole = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) top = fmaxf(top, x[i]);
    top = mm_lanes_max<LPR>(top);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v[i] = mm_exp_neg(x[i] - top);
      whole += v[i];
    }
    whole = mm_lanes_sum<LPR>(whole);
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = x[i] == -__builtin_inff() ? 0.f : -(v[i] / whole) * sum;
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = 0.f;
  }
#pragma unroll
  for (int q = 0; q < C / 4; ++q)
    s_d[sub][q * LPR + lane] = floatx4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
  mm_wave_lds_sync();
#pragma unroll
  for (int q = 0; q < KM; ++q) {
    if (e[q] < 0) continue;   // the chosen of a row are different experts
    float* p = (float*)&s_d[sub][e[q] % C / 4 * LPR + e[q] / C] + e[q] % 4;
    *p += d[q];
  }
  mm_wave_lds_sync();
  if (!ok) return;
#pragma unroll
  for (int q = 0; q < C / 4; ++q) {
    const floatx4 t = s_d[sub][q * LPR + lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * q + i] = t[i];
  }
  T* __restrict__ o = dlogits + row * a.E;
  constexpr int N = C < MMVec<T>::N ? C : MMVec<T>::N;
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
#pragma unroll
  for (int q = 0; q < C; q += N) {
    if (c0 + q + N <= a.E) {
      vec y;
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = (T)v[q + i];
      *(vec*)(o + c0 + q) = y;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (c0 + q + i < a.E) o[c0 + q + i] = (T)v[q + i];
    }
  }
}

namespace {
unsigned route_wg(long rows, int lanes) { return (unsigned)((rows + 256 / lanes - 1) / (256 / lanes)); }

int route_args(const char* name, int dtype, long T, int E, int k, int scoring, int groups, int top_groups, long ldl,
               float scale, MMRoute* a, int renorm) {
  auto bad = [&](const char* what, int code) {
    mm::set_error(std::string(name) + ": " + what);
    return code;
  };
  if (dtype < MM_F32 || dtype > MM_F16) return bad("bad dtype", MM_EINVAL);
  if (T < 0 || E < 1 || k < 1 || k > E || ldl < E) return bad("bad sizes", MM_EINVAL);
  if (scoring != 0 && scoring != 1) return bad("scoring must be 0 (softmax) or 1 (sigmoid)", MM_EINVAL);
  if (groups < 1 || E % groups || top_groups < 1 || top_groups > groups) return bad("bad groups", MM_EINVAL);
  if (!(scale != 0.f)) return bad("scale must not be 0", MM_EINVAL);
  if (E > MM_ROUTE_MAX_E) return bad("more than 1024 experts are not supported", MM_ERANGE);
  if (k > MM_ROUTE_MAX_K) return bad("more than 32 experts a row are not supported", MM_ERANGE);
  if (groups > MM_ROUTE_MAX_G) return bad("more than 64 groups are not supported", MM_ERANGE);
  const int lanes = E <= 16 ? 4 : E <= 32 ? 8 : E <= 256 ? 16 : E <= 512 ? 32 : 64;   // of a row (MM_ROUTE_SHAPES)
  if ((T + 255) * lanes >= 4294967296L) return bad("too many rows for one launch", MM_ERANGE);   // of 2^32 threads
  *a = MMRoute{T, ldl, E, k, scoring, groups, top_groups, renorm != 0, scale};
  return MM_OK;
}
}  // namespace

// lanes a row and logits a lane by E: few lanes keep the rounds' lane maxima short and let a wave work on many rows,
// until a lane's own logits cost more; one result a lane where k allows it
#define MM_ROUTE_K(X, l, c) if (k <= l) { X(l, c, 1) } else { X(l, c, ((MM_ROUTE_MAX_K + l - 1) / l)) }
#define MM_ROUTE_SHAPES(X)  \
  if (E <= 16) { MM_ROUTE_K(X, 4, 4) }  \
  else if (E <= 32) { MM_ROUTE_K(X, 8, 4) } \
  else if (E <= 64) { MM_ROUTE_K(X, 16, 4) } \
  else if (E <= 128) { MM_ROUTE_K(X, 16, 8) } \
  else if (E <= 256) { MM_ROUTE_K(X, 16, 16) } \
  else if (E <= 512) { X(32, 16, 1) } \
  else { X(64, 16, 1) }

extern "C" int mm_route_fwd(const void* logits, long ldl, int dtype, long T, int E, int k, int scoring,
                            const float* bias, int groups, int top_groups, int renorm, float scale, float* gates,
                            int* experts, hipStream_t stream) {
  MMRoute a;
  const int rc = route_args("mm_route_fwd", dtype, T, E, k, scoring, groups, top_groups, ldl, scale, &a, renorm);
  if (rc != MM_OK || T == 0) return rc;
#define X(l, c, km)                                                                                             \
  hipLaunchKernelGGL((mm_route_fwd_kernel<T_, l, c, km>), dim3(route_wg(a.T, l)), dim3(256), 0, stream, a, \
                     (const T_*)logits, bias, gates, experts);
  if (dtype == MM_F32) { using T_ = float; MM_ROUTE_SHAPES(X) }
  else if (dtype == MM_BF16) { using T_ = __bf16; MM_ROUTE_SHAPES(X) }
  else { using T_ = _Float16; MM_ROUTE_SHAPES(X) }
#undef X
  return mm::launch_status("mm_route_fwd");
}

extern "C" int mm_route_bwd(const void* logits, long ldl, int dtype, long T, int E, int k, int scoring, int renorm,
                            float scale, const float* gates, const int* experts, const float* dgates, void* dlogits,
                            hipStream_t stream) {
  MMRoute a;
  const int rc = route_args("mm_route_bwd", dtype, T, E, k, scoring, 1, 1, ldl, scale, &a, renorm);
  if (rc != MM_OK || T == 0) return rc;
#define X(l, c, km)                                                                                             \
  hipLaunchKernelGGL((mm_route_bwd_kernel<T_, l, c, km>), dim3(route_wg(a.T, l)), dim3(256), 0, stream, a, \
                     (const T_*)logits, gates, experts, dgates, (T_*)dlogits);
  if (dtype == MM_F32) { using T_ = float; MM_ROUTE_SHAPES(X) }
  else if (dtype == MM_BF16) { using T_ = __bf16; MM_ROUTE_SHAPES(X) }
  else { using T_ = _Float16; MM_ROUTE_SHAPES(X) }
#undef X
  return mm::launch_status("mm_route_bwd");
}
