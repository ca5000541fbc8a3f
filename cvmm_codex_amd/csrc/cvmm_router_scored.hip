// Router of balanced MoE models, no counterpart in cvmm.py.  Per token, with
// logits l over E experts:
//   s_e = sigmoid(l_e), or softmax(l)_e
//   c_e = s_e + b_e                        (b: the balance bias, in the choice only)
//   experts stand in G groups of E / G; a group's score is the sum of its two
//   best c (of its one); the Gk groups of the highest scores stay
//   chosen: the k best c among the experts of those groups
//   w_j = scale * s_j / sum_i s_i          (or scale * s_j)
// Ties go to the lower id, NaN ranks lowest.  The selection leaves sorted by
// expert, as the softmax router's does: each workgroup owns the tokens of one
// sort chunk and leaves its histogram to the scatter launch, or sorts all
// routes itself where it holds them.
//
// The scores, the biased scores and the group sums are computed and compared
// in 64 bits: the choice is part of the answer, and between neighbours that
// 32 bits cannot tell apart it would depend on how exp was rounded (131072
// choices of 128 experts see about one such pair per call).
//
// A selection round compares in two steps: the segment's maximum of the
// 32-bit roundings (rounding keeps the order, so the winner is among the
// lanes that attain it), and only where several lanes do, the 64-bit values.
#include <cmath>

#include "cvmm_common.h"
#include "cvmm_internal.h"
#include "cvmm_router.h"

namespace cvmm {

constexpr int kScoredThreads = 512;
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

__device__ __forceinline__ double sigmoid64(double l) { return 1.0 / (1.0 + exp(-l)); }

struct ScoredParams {
  int64_t ld, n_tokens;
  int32_t E, k;
  const float* bias;  // or NULL
  int32_t sigmoid, groups, topk_groups, renorm;
  double scale;
};

template <typename LT, int LPT, int MAXV, bool ONE, bool GROUPED>
__global__ __launch_bounds__(kScoredThreads) void route_scored_kernel(
    const LT* __restrict__ logits, const ScoredParams p, int64_t tpc, float* __restrict__ weights,
    int64_t* __restrict__ sel, int32_t* __restrict__ counts, const RouteSortOut so) {
  constexpr int SEGS = kScoredThreads / LPT;  // tokens per workgroup pass
  constexpr int SLOTS = 64 / LPT;             // results j held by lane j % LPT, slot j / LPT
  constexpr int PER = LPT * MAXV;             // expert slots per token
  constexpr int GMAX = PER < kRouteMaxGroups ? PER : kRouteMaxGroups;
  // grouped: per segment the biased scores, then the group scores
  __shared__ double cs[GROUPED ? SEGS * (PER + GMAX) : 1];
  __shared__ int32_t hist[PER + 1];
  __shared__ __attribute__((aligned(16))) int32_t ids[ONE ? kRouteOneMax : 1];
  const int32_t E = p.E, k = p.k;
  const int64_t b = blockIdx.x;
  for (int e = threadIdx.x; e <= E; e += kScoredThreads) hist[e] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int li = threadIdx.x % LPT, seg = threadIdx.x / LPT;
  const uint64_t seg_mask = (LPT == 64 ? ~0ull : ((1ull << (LPT & 63)) - 1)) << (lane - li);
  const int64_t t_lo = b * tpc, t_hi = t_lo + tpc < p.n_tokens ? t_lo + tpc : p.n_tokens;
  // every lane runs every pass (segment reductions need the whole wave)
  for (int64_t t0 = t_lo; t0 < t_hi; t0 += SEGS) {
    const int64_t t = t0 + seg;
    const bool active = t < t_hi;
    const LT* row = logits + (active ? t : t_lo) * p.ld;
    double c[MAXV];
    double m = 0.0, sum = 1.0;
    if (p.sigmoid) {
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        const int e = li + LPT * v;
        c[v] = e < E ? sigmoid64((double)(float)row[e]) : 0.0;
      }
    } else {
      float l[MAXV], mf = -INFINITY;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        const int e = li + LPT * v;
        l[v] = e < E ? (float)row[e] : -INFINITY;
        mf = fmaxf(mf, l[v]);
      }
      m = (double)seg_max<LPT>(mf);
      double s = 0.0;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        c[v] = li + LPT * v < E ? exp((double)l[v] - m) : 0.0;
        s += c[v];
      }
      sum = seg_sum_f64<LPT>(s);
#pragma unroll
      for (int v = 0; v < MAXV; ++v) c[v] = c[v] / sum;
    }
    uint32_t taken = 0;  // experts out of the choice
#pragma unroll
    for (int v = 0; v < MAXV; ++v) {
      const int e = li + LPT * v;
      if (e < E && p.bias != nullptr) c[v] += (double)p.bias[e];
      if (e >= E) taken |= 1u << v;
      c[v] = e >= E || isnan(c[v]) ? -INFINITY : c[v];
    }
    if constexpr (GROUPED) {
      const int32_t G = p.groups, per = E / G;
      double* ct = cs + seg * (PER + GMAX);
      double* gt = ct + PER;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) ct[li + LPT * v] = c[v];
      wave_lds_fence();
      for (int g = li; g < G; g += LPT) {
        double b1 = ct[g * per], b2 = -INFINITY;
        for (int i = 1; i < per; ++i) {
          const double x = ct[g * per + i];
          b2 = fmax(b2, fmin(b1, x));
          b1 = fmax(b1, x);
        }
        const double s = per > 1 ? b1 + b2 : b1;
        gt[g] = isnan(s) ? -INFINITY : s;  // (+inf and -inf)
      }
      wave_lds_fence();
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        const int e = li + LPT * v;
        if (e >= E) continue;
        const int g = e / per;
        const double mine = gt[g];
        int rank = 0;  // groups ahead of this one
        for (int h = 0; h < G; ++h) {
          const double x = gt[h];
          rank += x > mine || (x == mine && h < g) ? 1 : 0;
        }
        if (rank >= p.topk_groups) taken |= 1u << v;
      }
    }
    int32_t res_e[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) res_e[q] = 0;
    for (int j = 0; j < k; ++j) {
      // the lane's best, then the segment's
      double bv = -INFINITY;
      int32_t bi = E;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        const bool in = !((taken >> v) & 1u);
        // (a lane's experts rise with v: the first of equals is the lower id)
        if (in && (c[v] > bv || bi == E)) {
          bv = c[v];
          bi = li + LPT * v;
        }
      }
      const float hi = bi < E ? (float)bv : -INFINITY;
      const float mv = seg_max<LPT>(hi);
      bool cand = bi < E && hi == mv;
      const uint64_t ball = __ballot(cand) & seg_mask;
      if (__any(active && __popcll(ball) > 1)) {
        const double top = seg_max_f64<LPT>(cand ? bv : -INFINITY);
        cand = cand && bv == top;
      }
      const int32_t win = seg_min_i<LPT>(cand ? bi : E);
      if (win == bi) taken |= 1u << (win / LPT);
#pragma unroll
      for (int q = 0; q < SLOTS; ++q)
        if (j == q * LPT + li) res_e[q] = win;
    }
    // the winners' scores, by the lanes that hold them
    double w[SLOTS], part = 0.0;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      w[q] = 0.0;
      if (q * LPT + li < k) {
        const double l = (double)(float)row[res_e[q]];
        w[q] = p.sigmoid ? sigmoid64(l) : exp(l - m) / sum;
        part += w[q];
      }
    }
    double f = p.scale;
    if (p.renorm) {
      const double den = seg_sum_f64<LPT>(part);
      f = p.scale / (den < 1e-20 ? 1e-20 : den);  // clamp_min (NaN passes through)
    }
    if (active) {
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) {
        const int j = q * LPT + li;
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
    route_sort_one<kScoredThreads>(hist, ids, (int)(p.n_tokens * k), E, k, so);
    return;
  }
  for (int e = threadIdx.x; e <= E; e += kScoredThreads) counts[b * (int64_t)(E + 1) + e] = hist[e];
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
        pj[q] = p.sigmoid ? sigmoid64(x) : exp(x - (double)mf) / (double)sum;
        sg[q] = p.sigmoid ? sigmoid64(-x) : 0.0;
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
    hipLaunchKernelGGL((route_scored_kernel<LT, LPT, MAXV, true, GROUPED>), dim3(1), dim3(kScoredThreads), 0, s,
                       logits, p, tpc, w, sel, counts, so);
  else
    hipLaunchKernelGGL((route_scored_kernel<LT, LPT, MAXV, false, GROUPED>), dim3((unsigned)n_chunks),
                       dim3(kScoredThreads), 0, s, logits, p, tpc, w, sel, counts, so);
}

// Segment width: 8 experts per lane up to 512 experts, then 16.
template <typename F>
static void by_experts(int32_t E, F&& f) {
  if (E <= 32) f(std::integral_constant<int, 4>(), std::integral_constant<int, 8>());
  else if (E <= 64) f(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  else if (E <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
  else if (E <= 256) f(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
  else if (E <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

template <typename F>
static void by_dtype(int32_t dt, F&& f) {
  if (dt == kF32) f(float());
  else if (dt == kBF16) f(bf16_t());
  else f(f16_t());
}

hipError_t launch_route_scored(const void* logits, int32_t logits_dtype, int64_t n_tokens, int64_t logits_ld,
                               int32_t n_experts, int64_t top_k, const float* bias, int32_t sigmoid, int32_t groups,
                               int32_t topk_groups, int32_t renormalize, double scale, float* weights, int64_t* sel,
                               int32_t* sorted_sel, int64_t* perm, int64_t* token_index, int64_t* offsets,
                               int32_t* route_pos, void* workspace, hipStream_t stream) {
  if (n_tokens <= 0) return hipSuccess;
  const int64_t tpc = route_chunk_tokens(n_tokens, n_experts, top_k);
  const int64_t n_chunks = (n_tokens + tpc - 1) / tpc;
  if (n_chunks > 0x7fffffffll) return hipErrorInvalidValue;
  int32_t* counts = (int32_t*)workspace;
  int32_t* n_invalid = (int32_t*)((char*)workspace + route_workspace_bytes(n_tokens, n_experts, top_k) - 256);
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
