// Router of balanced MoE models, no counterpart in cvmm.py.  Per token, with
// logits l over E experts:
//   s_e = sigmoid(l_e), or softmax(l)_e
//   c_e = s_e + b_e                        (b: the balance bias, in the choice only)
//   experts stand in G groups of E / G; a group's score is the sum of its two
//   best c (of its one); the Gk groups of the highest scores stay
//   chosen: the k best c among the experts of those groups
//   w_j = scale * s_j / max(sum_i s_i, 1e-20)   (or scale * s_j)
// Ties go to the lower id, NaN ranks lowest.  The selection leaves sorted by
// expert, as the softmax router's does: each workgroup owns the tokens of one
// sort chunk and leaves its histogram to the scatter launch, or sorts all
// routes itself where it holds them.
//
// The choice is that of 64-bit scores: it is part of the answer, and between
// neighbours that 32 bits cannot tell apart it would depend on how exp was
// rounded (131072 choices of 128 experts see about one such pair per call).  It
// is made in 32 bits, with the candidates that are within the error of the ones
// before them ranked by their 64-bit scores, and in 64 bits throughout for the
// few tokens where that is not enough; without a bias and groups the logits
// themselves are compared, where different ones have different scores.  (64-bit
// exps for all: 32 tokens of 256 experts, on one CU, 33 us.)
#include <cmath>

#include "cvmm_common.h"
#include "cvmm_internal.h"
#include "cvmm_router.h"

namespace cvmm {

// Threads of a workgroup: one pass over a chunk's 64 tokens (top-8) with up to
// 128 experts.
template <int LPT> constexpr int scored_threads(bool one) { return one || LPT >= 16 ? 1024 : 512; }
constexpr int kScoredBwdThreads = 256;

template <int LPT>
__device__ __forceinline__ double seg_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < LPT; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}
template <int LPT>
__device__ __forceinline__ double seg_max_f64(double v) {
#pragma unroll
  for (int d = 1; d < LPT; d <<= 1) v = fmax(v, __shfl_xor(v, d, 64));
  return v;
}

// LDS written by lanes of this wave, about to be read by others of it.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

struct ScoredParams {
  int64_t ld, n_tokens;
  int32_t E, k;
  const float* bias;  // or NULL
  int32_t sigmoid, groups, topk_groups, renorm;
  double scale;
};

// A chosen expert's score, and for the sigmoid 1 minus it, from its logit: one
// inlined exp and division for both kinds.
__device__ __forceinline__ double score64(double x, bool sigmoid, double m, double total) {
  const double e = exp(sigmoid ? -x : x - m);
  return (sigmoid ? 1.0 : e) / (sigmoid ? 1.0 + e : total);
}

// The groups that stay, by one wave's lanes for its segments: the sum of the two
// best of the scores ct of each group, ranked.  Returns the experts of this lane
// that go, as bits of v; gap (32 bits): the distance between the last group that
// stays and the first that goes.
template <typename T, int LPT, int MAXV>
__device__ __forceinline__ uint32_t groups_out(const T* ct, T* gt, const ScoredParams& p, int li, T* gap) {
  const int32_t G = p.groups, per = p.E / G;
  wave_lds_fence();
#pragma unroll 1
  for (int g = li; g < G; g += LPT) {
    T b1 = ct[g * per], b2 = -INFINITY;
#pragma unroll 8
    for (int i = 1; i < per; ++i) {
      const T x = ct[g * per + i];
      b2 = fmax(b2, fmin(b1, x));
      b1 = fmax(b1, x);
    }
    const T s = per > 1 ? b1 + b2 : b1;
    gt[g] = isnan(s) ? -INFINITY : s;  // (+inf and -inf)
  }
  wave_lds_fence();
  T last = INFINITY, first = -INFINITY;
  uint32_t lo = 0, hi = 0;  // the groups that stay, as bits
#pragma unroll 1
  for (int g = li; g < G; g += LPT) {
    const T mine = gt[g];
    int rank = 0;  // groups ahead of this one
#pragma unroll 8
    for (int h = 0; h < G; ++h) {
      const T x = gt[h];
      rank += x > mine || (x == mine && h < g) ? 1 : 0;
    }
    if (rank < p.topk_groups) {
      last = fmin(last, mine);
      if (g < 32) lo |= 1u << g;
      else hi |= 1u << (g - 32);
    } else {
      first = fmax(first, mine);
    }
  }
  lo = seg_or<LPT>(lo);
  hi = seg_or<LPT>(hi);
  uint32_t out = 0;
  const float inv = 1.f / (float)per;  // e / per: exact for e + 0.5 (e < 1024)
#pragma unroll
  for (int v = 0; v < MAXV; ++v) {
    const int e = li + LPT * v, g = (int)(((float)e + 0.5f) * inv);
    const uint32_t stays = ((g < 32 ? lo : hi) >> (g & 31)) & 1u;
    if (e < p.E) out |= (stays ^ 1u) << v;
  }
  if constexpr (sizeof(T) == 4) *gap = -seg_max<LPT>(-last) - seg_max<LPT>(first);
  else *gap = 0;
  return out;
}

template <typename LT, int LPT, int MAXV, bool ONE, bool GROUPED, int THREADS>
__global__ __launch_bounds__(THREADS) void route_scored_kernel(
    const LT* __restrict__ logits, const ScoredParams p, int64_t tpc, float* __restrict__ weights,
    int64_t* __restrict__ sel, int32_t* __restrict__ counts, const RouteSortOut so) {
  constexpr int SEGS = THREADS / LPT;  // tokens per workgroup pass
  constexpr int SLOTS = 64 / LPT;      // results j held by lane j % LPT, slot j / LPT
  constexpr int PER = LPT * MAXV;      // expert slots per token
  constexpr int GMAX = PER < kRouteMaxGroups ? PER : kRouteMaxGroups;
  // per segment the biased scores, then (grouped) the groups'
  __shared__ double cs[GROUPED ? SEGS * (PER + GMAX) : 1];
  __shared__ int32_t hist[PER + 1];
  __shared__ __attribute__((aligned(16))) int32_t ids[ONE ? kRouteOneMax : 1];
  const int32_t E = p.E, k = p.k;
  const int64_t b = blockIdx.x;
  for (int e = threadIdx.x; e <= E; e += THREADS) hist[e] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int li = threadIdx.x % LPT, seg = threadIdx.x / LPT;
  const uint64_t seg_mask = (LPT == 64 ? ~0ull : ((1ull << (LPT & 63)) - 1)) << (lane - li);
  double* const ct = cs + (GROUPED ? seg * (PER + GMAX) : 0);
  const bool by_logit = !GROUPED && p.bias == nullptr;
  const int64_t t_lo = b * tpc, t_hi = t_lo + tpc < p.n_tokens ? t_lo + tpc : p.n_tokens;
  // every lane runs every pass (segment reductions need the whole wave); waves
  // of no token have none to run
  for (int64_t t0 = t_lo; t0 < t_hi && t0 + (threadIdx.x & ~63) / LPT < t_hi; t0 += SEGS) {
    const int64_t t = t0 + seg;
    const bool active = t < t_hi;
    const LT* row = logits + (active ? t : t_lo) * p.ld;
    // ---- 32 bits, and how far two of these scores can be off against each other,
    // in units of 2^-24.  exp(x): 2 + 1.22 |x| of itself (two roundings of its
    // argument and an ulp; 1 + 0.95 |x| measured).  Sigmoid: s (1 - s) of that,
    // below 0.8, and at most 1 each for the sum and the reciprocal: 2^-21 for both
    // sides.  Softmax: exp (l - m rounds too) and the product with 1 / sum, 3 of the
    // largest score on either side (8 for both, with the remainders).  The sum
    // scales all scores alike: its error counts once, of the distance of the two
    // scores, which is that of their biases where they nearly tie: 1 per addition,
    // of a lane's experts and over the lanes, 1 for the reciprocal, and the exps'
    // 2 + 2.22 times their weighted mean |x|, at most 4.5 for 1024 experts.
    // (Taken of the largest score instead, 17 of 16384 tokens of 128 experts would
    // be ranked in 64 bits, not 4.)  The sum with the bias rounds by half an ulp of
    // itself.
    // (Loads at clamped places: a guard around each made them
    // wait for one another.)
    float l[MAXV], c[MAXV];
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
      const int e = li + LPT * v;
      l[v] = (float)row[e < E ? e : E - 1];
      c[v] = 0.f;
    }
    if (p.bias != nullptr) {
#pragma unroll
      for (int v = 0; v < MAXV; ++v) c[v] = p.bias[li + LPT * v < E ? li + LPT * v : E - 1];
    }
    float m = -INFINITY, sum = 1.f, err = 0x1p-21f;
    bool unsure = false;  // NaN, or groups within the error
    if (p.sigmoid) {
#pragma unroll
      for (int v = 0; v < MAXV; ++v) c[v] += __frcp_rn(1.f + __expf(-l[v]));
    } else {
#pragma unroll
      for (int v = 0; v < MAXV; ++v) m = fmaxf(m, l[v]);  // (a repeated last one changes nothing)
      m = seg_max<LPT>(m);
      float s = 0.f, x[MAXV];
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        x[v] = __expf(l[v] - m);
        s += li + LPT * v < E ? x[v] : 0.f;
      }
      sum = seg_sum<LPT>(s);
      unsure = isnan(sum);
      const float inv = 1.f / sum;
      float b = 0.f;
      if (p.bias != nullptr) {
#pragma unroll
        for (int v = 0; v < MAXV; ++v) b = fmaxf(b, fabsf(c[v]));
        b = __int_as_float(seg_max_i<LPT>(__float_as_int(b)));  // (not negative: in the integers' order)
      }
      // (the largest score: 1 / sum)
      err = 0x1p-24f * (8.f * inv + (MAXV + __builtin_ctz(LPT) + 12) * fminf(2.f * b, inv));
#pragma unroll
      for (int v = 0; v < MAXV; ++v) c[v] += x[v] * inv;
    }
    // the scores as integers of the same order, the smallest for experts out of
    // the choice: one maximum finds the lane's best
    constexpr int32_t kOut = INT32_MIN;
    int32_t key[MAXV];
    float top = 0.f;
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
      const bool in = li + LPT * v < E;
      if (by_logit) c[v] = l[v];
      unsure |= in && isnan(c[v]);
      const int32_t i = __float_as_int(c[v] + 0.f);  // (-0 and 0 tie)
      key[v] = in ? i ^ ((i >> 31) & 0x7fffffff) : kOut;
      top = fmaxf(top, in ? fabsf(c[v]) : 0.f);
    }
    if constexpr (GROUPED) {
      float gap, *cf = reinterpret_cast<float*>(ct);
#pragma unroll
      for (int v = 0; v < MAXV; ++v) cf[li + LPT * v] = c[v];
      const uint32_t out = groups_out<float, LPT, MAXV>(cf, reinterpret_cast<float*>(ct + PER), p, li, &gap);
#pragma unroll
      for (int v = 0; v < MAXV; ++v) key[v] = (out >> v) & 1u ? kOut : key[v];
      // sums of two scores of size up to top, each rounded with its bias
      top = seg_max<LPT>(top);
      unsure |= !(gap > 2.f * err + 0x1p-21f * top);
    }
    // candidates by falling score: the k best, and those after them that the
    // error does not part from the one before; past the 64 that the lanes hold
    // the token is unsure
    int32_t res_e[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) res_e[q] = 0;
    float before = INFINITY;
    int n = 0;
    bool near = false, apart = true;
#pragma unroll 1
    for (;; ++n) {
      if (n == k && by_logit) break;
      int32_t bv = key[0];
#pragma unroll
      for (int v = 1; v < MAXV; ++v) bv = max(bv, key[v]);
      const int32_t mv = seg_max_i<LPT>(bv);
      if (mv == kOut) break;  // none is left
      int32_t bi = E;  // the lane's first of that score (its experts rise with v)
#pragma unroll
      for (int v = MAXV - 1; v >= 0; --v) bi = key[v] == mv ? li + LPT * v : bi;
      const int32_t win = seg_min_i<LPT>(bi);
      const float now = __int_as_float(mv ^ ((mv >> 31) & 0x7fffffff));
      apart = by_logit || n == 0 || before - now > err + 0x1p-23f * (fabsf(before) + fabsf(now));
      if (n >= k && (apart || n == 64)) break;
      near |= !apart;
      before = now;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) key[v] = win == li + LPT * v ? kOut : key[v];
#pragma unroll
      for (int q = 0; q < SLOTS; ++q)
        if (n == q * LPT + li) res_e[q] = win;
    }
    unsure |= n > k + 8 || n < k || (n == 64 && !apart);
    if (by_logit) {
      // Does every logit below a chosen one have a smaller 64-bit score?  From 2^-15 on
      // fp32 numbers lie 2^-40 apart, which exp and the sums keep (2^-43 at most is
      // lost) unless the score leaves the normal numbers (below e^-708), or a sigmoid
      // nears 1: up to 16 its steps are 2^-43 still, from 24 on it repeats values.
      unsure |= !(before - (p.sigmoid ? 0.f : m) > -700.f);
      if (before < 0x1p-15f) {
#pragma unroll
        for (int v = 0; v < MAXV; ++v) unsure |= l[v] >= before && fabsf(l[v]) < 0x1p-15f;
      }
      if (p.sigmoid) {
        float high = l[0];
#pragma unroll
        for (int v = 1; v < MAXV; ++v) high = fmaxf(high, l[v]);
        unsure |= high >= 16.f;
      }
    }
    // ---- all scores in 64 bits, for a wave with an unsure token: NaN, groups within
    // the error, or a crowd of candidates
    const bool again = active && (__ballot(unsure) & seg_mask) != 0;
    if (__any(again)) {
      double d[MAXV], den = 1.0;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) d[v] = exp(p.sigmoid ? -(double)l[v] : (double)l[v] - (double)m);
      if (!p.sigmoid) {
        double s = 0.0;
#pragma unroll
        for (int v = 0; v < MAXV; ++v) s += li + LPT * v < E ? d[v] : 0.0;
        den = seg_sum_f64<LPT>(s);
      }
      uint32_t taken = 0;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        const int e = li + LPT * v;
        d[v] = (p.sigmoid ? 1.0 : d[v]) / (p.sigmoid ? 1.0 + d[v] : den);
        if (e < E && p.bias != nullptr) d[v] += (double)p.bias[e];
        if (e >= E) taken |= 1u << v;
        if (e >= E || isnan(d[v])) d[v] = -INFINITY;
      }
      if constexpr (GROUPED) {
#pragma unroll
        for (int v = 0; v < MAXV; ++v) ct[li + LPT * v] = d[v];
        double gap;
        taken |= groups_out<double, LPT, MAXV>(ct, ct + PER, p, li, &gap);
      }
#pragma unroll 1
      for (int j = 0; j < k; ++j) {
        double bv = -INFINITY;
        int32_t bi = E;
#pragma unroll
        for (int v = 0; v < MAXV; ++v)
          if (!((taken >> v) & 1u) && (d[v] > bv || bi == E)) {
            bv = d[v];
            bi = li + LPT * v;
          }
        const double mv = seg_max_f64<LPT>(bi < E ? bv : -INFINITY);
        const int32_t win = seg_min_i<LPT>(bi < E && bv == mv ? bi : E);
        if (win == bi) taken |= 1u << (win / LPT);
#pragma unroll
        for (int q = 0; q < SLOTS; ++q)
          if (again && j == q * LPT + li) res_e[q] = win;
      }
      if (again) {
        n = k;
        near = false;
      }
    }
    // the candidates' scores in 64 bits, by the lanes that hold them; a softmax's
    // sum is 64-bit where it does not cancel (but for chosen scores under the clamp:
    // such weights are off by up to 2 ulp)
    double total = (double)sum;
    const bool rank = __any(active && near);
    if (!p.sigmoid && (rank || !p.renorm)) {
      double s = 0.0;
#pragma unroll 1
      for (int e = li; e < E; e += LPT) s += exp((double)(float)row[e] - (double)m);
      total = seg_sum_f64<LPT>(s);
    }
    double w[SLOTS], part = 0.0;
    int at[SLOTS];  // place among the chosen
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      w[q] = 0.0;
      at[q] = q * LPT + li;
      if (q * LPT + li < n) w[q] = score64((double)(float)row[res_e[q]], p.sigmoid, (double)m, total);
    }
    if (rank) {
      // ranked among the candidates, which hold the k best in some order
      double d[SLOTS];
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) {
        d[q] = w[q] + (p.bias != nullptr && q * LPT + li < n ? (double)p.bias[res_e[q]] : 0.0);
        if (near) at[q] = q * LPT + li < n ? 0 : 64;
      }
      const int most = (int)seg_max<64>((float)(near ? n : 0));
#pragma unroll
      for (int q2 = 0; q2 < SLOTS; ++q2) {
#pragma unroll 1
        for (int i = 0; i < LPT && q2 * LPT + i < most; ++i) {
          const int from = lane - li + i;
          const double x = __shfl(d[q2], from, 64);
          const int32_t e = __shfl(res_e[q2], from, 64);
#pragma unroll
          for (int q = 0; q < SLOTS; ++q)
            at[q] += near && q2 * LPT + i < n && (x > d[q] || (x == d[q] && e < res_e[q])) ? 1 : 0;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) part += at[q] < k ? w[q] : 0.0;
    double f = p.scale;
    if (p.renorm) {
      const double den = seg_sum_f64<LPT>(part);
      f = p.scale / (den < 1e-20 ? 1e-20 : den);  // clamp_min (NaN passes through)
    }
    if (active) {
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) {
        const int j = at[q];
        if (j < k) {
          sel[t * k + j] = res_e[q];
          weights[t * k + j] = (float)(w[q] * f);
          atomicAdd(&hist[res_e[q]], 1);
          if constexpr (ONE) ids[t * k + j] = res_e[q];
        }
      }
    }
  }
  __syncthreads();
  if constexpr (ONE) {
    route_sort_one<THREADS>(hist, ids, (int)(p.n_tokens * k), E, k, so);
    return;
  }
  for (int e = threadIdx.x; e <= E; e += THREADS) counts[b * (int64_t)(E + 1) + e] = hist[e];
}

// d logits.  With gw the weights' gradient, S = sum of the chosen scores:
//   renormalised: g_j = (scale gw_j - sum_i gw_i w_i) / S;  else g_j = scale gw_j
//   (S under the clamp is a constant: g_j = scale gw_j / 1e-20)
//   sigmoid: d l_j = g_j s_j (1 - s_j) at the chosen experts, 0 elsewhere
//   softmax: d l_e = s_e ([e chosen] g_e - sum_i g_i s_i)
// The per-choice terms are 64-bit (the difference in g cancels), the dense
// softmax row 32-bit.
template <typename LT, int LPT, int MAXV>
__global__ __launch_bounds__(kScoredBwdThreads) void route_scored_bwd_kernel(
    const LT* __restrict__ logits, const ScoredParams p, const int64_t* __restrict__ sel,
    const float* __restrict__ gw, LT* __restrict__ glog, int64_t gld) {
  constexpr int SEGS = kScoredBwdThreads / LPT;
  constexpr int SLOTS = 64 / LPT;
  constexpr int PER = LPT * MAXV;
  __shared__ float g_lds[SEGS * PER];  // per segment: g of every expert
  const int32_t E = p.E, k = p.k;
  const int li = threadIdx.x % LPT, seg = threadIdx.x / LPT;
  const int64_t t = (int64_t)blockIdx.x * SEGS + seg;
  const bool active = t < p.n_tokens;
  const LT* row = logits + (active ? t : 0) * p.ld;
  float l[MAXV];
  float mf = -INFINITY, sum = 1.f;
  if (!p.sigmoid) {
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
      const int e = li + LPT * v;
      l[v] = e < E ? (float)row[e] : -INFINITY;
      mf = fmaxf(mf, l[v]);
    }
    mf = seg_max<LPT>(mf);
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
      l[v] = li + LPT * v < E ? expf(l[v] - mf) : 0.f;
      s += l[v];
    }
    sum = seg_sum<LPT>(s);
  }
  float* gseg = g_lds + seg * PER;
#pragma unroll
  for (int v = 0; v < MAXV; ++v) gseg[li + LPT * v] = 0.f;
  int32_t sj[SLOTS];
  double pj[SLOTS], sg[SLOTS], dw[SLOTS], S = 0.0, dot = 0.0;
#pragma unroll
  for (int q = 0; q < SLOTS; ++q) {
    const int j = q * LPT + li;
    sj[q] = -1;
    pj[q] = sg[q] = dw[q] = 0.0;
    if (active && j < k) {
      const int64_t id = sel[t * k + j];
      if (id >= 0 && id < E) {
        sj[q] = (int32_t)id;
        const double x = (double)(float)row[id];
        const double e = exp(p.sigmoid ? -x : x - (double)mf);
        const double r = 1.0 / (p.sigmoid ? 1.0 + e : (double)sum);
        pj[q] = p.sigmoid ? r : e * r;
        // 1 - s = e / (1 + e), 1 where e overflows
        sg[q] = !p.sigmoid ? 0.0 : r > 0.0 ? e * r : 1.0;
        dw[q] = (double)gw[t * k + j] * p.scale;
      }
    }
    S += pj[q];
    dot += dw[q] * pj[q];
  }
  if (p.renorm) {
    S = seg_sum_f64<LPT>(S);
    dot = seg_sum_f64<LPT>(dot);
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) dw[q] = S < 1e-20 ? dw[q] / 1e-20 : (dw[q] - dot / S) / S;
  }
  float cdot = 0.f;
  if (!p.sigmoid) {
    double s = 0.0;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) s += dw[q] * pj[q];
    cdot = (float)seg_sum_f64<LPT>(s);
  }
  wave_lds_fence();  // the zeroed row before the chosen entries (one wave per segment)
#pragma unroll
  for (int q = 0; q < SLOTS; ++q)
    if (sj[q] >= 0) gseg[sj[q]] = (float)(p.sigmoid ? dw[q] * pj[q] * sg[q] : dw[q]);
  wave_lds_fence();
  if (!active) return;
  LT* out = glog + t * gld;
#pragma unroll
  for (int v = 0; v < MAXV; ++v) {
    const int e = li + LPT * v;
    if (e < E) out[e] = (LT)(p.sigmoid ? gseg[e] : l[v] / sum * (gseg[e] - cdot));
  }
}

template <typename LT, int LPT, int MAXV, bool GROUPED>
static void launch_scored(const LT* logits, const ScoredParams& p, int64_t tpc, int64_t n_chunks, float* w,
                          int64_t* sel, int32_t* counts, const RouteSortOut& so, hipStream_t s) {
  if (n_chunks == 1 && p.n_tokens * p.k <= kRouteOneMax)
    hipLaunchKernelGGL((route_scored_kernel<LT, LPT, MAXV, true, GROUPED, scored_threads<LPT>(true)>), dim3(1),
                       dim3(scored_threads<LPT>(true)), 0, s, logits, p, tpc, w, sel, counts, so);
  else
    hipLaunchKernelGGL((route_scored_kernel<LT, LPT, MAXV, false, GROUPED, scored_threads<LPT>(false)>), dim3((unsigned)n_chunks),
                       dim3(scored_threads<LPT>(false)), 0, s, logits, p, tpc, w, sel, counts, so);
}

// Tokens per workgroup (= per sort chunk).  Up to 128 routes one workgroup chooses
// and sorts them; past that its CU's instruction rate is the bound and a second
// launch to sort costs less (32 tokens, top-8 of 256 experts in 8 groups 22.1 ->
// 17.5 us in chunks of 8, of 64 experts 14.4 -> 12.5; but 16 tokens of 128
// experts 9.4 -> 12.3).  Then a workgroup per CU, of at most 64 tokens and at
// least 8, 32 or 64 (the tokens that a workgroup's lanes hold, by the experts):
// 500 / 4096 tokens of 256 experts 23 / 33 us, 35 / 47 in chunks of 64; 16384
// tokens, top-1 of 128, 17 in chunks of 64, 38 in chunks of 512.  Shorter ones
// cost the sort more than they save (16384 tokens, top-8: 27 / 33 / 47 us at 64
// / 32 / 16).  The count matrix stays within 64K entries.
static int64_t scored_chunk_tokens(int64_t n_tokens, int32_t n_experts, int64_t top_k) {
  const int64_t routes = n_tokens * top_k;
  if (routes <= 128 && n_tokens <= 64) return n_tokens > 0 ? n_tokens : 1;
  if (routes <= kRouteOneMax) return 8;
  const int64_t least = n_experts <= 64 ? 64 : n_experts <= 128 ? 32 : 8;
  int64_t tpc = (n_tokens + 255) / 256;
  tpc = tpc < least ? least : tpc > 64 ? 64 : tpc;
  const int64_t counts = (n_tokens * (int64_t)(n_experts + 1) + 65535) / 65536;
  return tpc > counts ? tpc : counts;
}

size_t scored_workspace_bytes(int64_t n_tokens, int32_t n_experts, int64_t top_k) {
  const int64_t tpc = scored_chunk_tokens(n_tokens, n_experts, top_k);
  const int64_t n_chunks = n_tokens > 0 ? (n_tokens + tpc - 1) / tpc : 1;
  // counts, bucket totals for the column scan, 256 bytes ending in n_invalid
  return sort_counts_bytes(n_chunks, n_experts) + align_up((size_t)(n_experts + 1) * sizeof(int32_t), 256) + 256;
}

hipError_t launch_route_scored(const void* logits, int32_t logits_dtype, int64_t n_tokens, int64_t logits_ld,
                               int32_t n_experts, int64_t top_k, const float* bias, int32_t sigmoid, int32_t groups,
                               int32_t topk_groups, int32_t renormalize, double scale, float* weights, int64_t* sel,
                               int32_t* sorted_sel, int64_t* perm, int64_t* token_index, int64_t* offsets,
                               int32_t* route_pos, void* workspace, hipStream_t stream) {
  if (n_tokens <= 0) return hipSuccess;
  const int64_t tpc = scored_chunk_tokens(n_tokens, n_experts, top_k);
  const int64_t n_chunks = (n_tokens + tpc - 1) / tpc;
  if (n_chunks > 0x7fffffffll) return hipErrorInvalidValue;
  int32_t* counts = (int32_t*)workspace;
  int32_t* n_invalid = (int32_t*)((char*)workspace + scored_workspace_bytes(n_tokens, n_experts, top_k) - 256);
  const ScoredParams p{logits_ld, n_tokens, n_experts, (int32_t)top_k, bias, sigmoid, groups, topk_groups,
                       renormalize, scale};
  const RouteSortOut so{sorted_sel, perm, token_index, offsets, route_pos};
  by_dtype(logits_dtype, [&](auto lt) {
    using LT = decltype(lt);
    by_experts(n_experts, [&](auto lpt, auto maxv) {
      constexpr int LPT = decltype(lpt)::value, MAXV = decltype(maxv)::value;
      // all groups kept: no expert is left out
      if (topk_groups < groups)
        launch_scored<LT, LPT, MAXV, true>((const LT*)logits, p, tpc, n_chunks, weights, sel, counts, so, stream);
      else
        launch_scored<LT, LPT, MAXV, false>((const LT*)logits, p, tpc, n_chunks, weights, sel, counts, so, stream);
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || (n_chunks == 1 && n_tokens * top_k <= kRouteOneMax)) return e;
  return launch_sort_scatter(sel, n_tokens * top_k, n_experts, tpc * top_k, top_k, counts, sorted_sel, perm,
                             token_index, offsets, route_pos, n_invalid, stream);
}

hipError_t launch_route_scored_backward(const void* logits, int32_t logits_dtype, int64_t n_tokens,
                                        int64_t logits_ld, int32_t n_experts, int64_t top_k, int32_t sigmoid,
                                        int32_t renormalize, double scale, const int64_t* sel,
                                        const float* grad_weights, void* grad_logits, int64_t grad_ld,
                                        hipStream_t stream) {
  if (n_tokens <= 0) return hipSuccess;
  if (n_tokens / 4 > 0x7fffffffll) return hipErrorInvalidValue;
  const ScoredParams p{logits_ld, n_tokens, n_experts, (int32_t)top_k, nullptr, sigmoid, 1, 1, renormalize, scale};
  by_dtype(logits_dtype, [&](auto lt) {
    using LT = decltype(lt);
    by_experts(n_experts, [&](auto lpt, auto maxv) {
      constexpr int LPT = decltype(lpt)::value, MAXV = decltype(maxv)::value;
      constexpr int SEGS = kScoredBwdThreads / LPT;
      hipLaunchKernelGGL((route_scored_bwd_kernel<LT, LPT, MAXV>), dim3((unsigned)((n_tokens + SEGS - 1) / SEGS)),
                         dim3(kScoredBwdThreads), 0, stream, (const LT*)logits, p, sel, grad_weights,
                         (LT*)grad_logits, grad_ld);
    });
  });
  return hipGetLastError();
}

}  // namespace cvmm
