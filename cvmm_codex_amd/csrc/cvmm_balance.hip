// Balance loss of a router with the experts' counts, no counterpart in cvmm.py
// (its callers add such a term to their loss).  Tokens stand in groups of equal
// size (a sequence each, or all in one); those with mask 0 count nowhere.
//   p_te = softmax(l_t)_e, or sigmoid(l_te) / max(sum_j sigmoid(l_tj), 1e-20)
//   n_g live tokens of group g, c_ge their routes to e, P_ge = sum_t p_te / n_g
//   load:    B = mean_g sum_e (E c_ge / (k n_g)) P_ge     (1 where loads are even)
//   entropy: B = mean_g sum_e P_ge log P_ge
//   z = mean_t logsumexp(l_t)^2,   loss = weight B + z_weight z
// (the mean over the groups that have a live token).  Both gradients are one
// pass over the logits with a coefficient per group and expert, which the
// forward leaves behind: a_ge = weight dB/dP_ge / n_g, b = 2 z_weight / n:
//   softmax: dl_e = p_e (a_e - sum_j a_j p_j) + b lse p_e
//   sigmoid: dl_e = s_e (1 - s_e) (a_e - sum_j a_j p_j) / S + b lse softmax(l)_e
//
// Bound by launches and by the latency of one pass: 16384 tokens of 128 experts
// in bf16 are 4 MB, under a microsecond of the card's bandwidth.  So two
// launches forward (chunks of tokens, then one workgroup that adds them in a
// fixed order) and one backward.  Terms of a token are 32-bit; a chunk's sums
// too (at most some hundred addends per lane); sums over chunks are 64-bit.
#include <cmath>

#include "cvmm_common.h"
#include "cvmm_internal.h"
#include "cvmm_router.h"

namespace cvmm {

constexpr int kBalanceThreads = 256;
constexpr int kBalanceSumThreads = 1024;

// The expert of a lane's slot v: runs of 8, so that a lane's slots are whole
// 16-byte pieces of the row.
template <int LPT>
__device__ __forceinline__ int balance_expert(int li, int v) { return (v / 8) * (8 * LPT) + li * 8 + v % 8; }

// A row's logits in 32 bits, -inf in the slots past the last expert.
template <typename LT, int LPT, int MAXV, bool VEC>
__device__ __forceinline__ void balance_row(const LT* __restrict__ row, int li, int32_t E, float (&l)[MAXV]) {
#pragma unroll
  for (int b = 0; b < MAXV; b += 8) {
    const int e0 = balance_expert<LPT>(li, b);
    if constexpr (VEC) {  // E % 8 == 0: a run is inside the row or past it
      const LT* at = row + (e0 < E ? e0 : 0);
      if constexpr (sizeof(LT) == 4) {
        const float4 x = reinterpret_cast<const float4*>(at)[0], y = reinterpret_cast<const float4*>(at)[1];
        l[b] = x.x, l[b + 1] = x.y, l[b + 2] = x.z, l[b + 3] = x.w;
        l[b + 4] = y.x, l[b + 5] = y.y, l[b + 6] = y.z, l[b + 7] = y.w;
      } else {
        const uint4 raw = *reinterpret_cast<const uint4*>(at);
        const LT* x = reinterpret_cast<const LT*>(&raw);
#pragma unroll
        for (int v = 0; v < 8; ++v) l[b + v] = to_f32(x[v]);
      }
    } else {
#pragma unroll
      for (int v = 0; v < 8; ++v) l[b + v] = to_f32(row[e0 + v < E ? e0 + v : E - 1]);
    }
#pragma unroll
    for (int v = 0; v < 8; ++v) l[b + v] = e0 + v < E ? l[b + v] : -INFINITY;
  }
}

// p of a row, and (for z, or where p is that) its softmax and logsumexp.
template <int LPT, int MAXV>
struct BalanceTerms {
  float soft[MAXV], p[MAXV];
  float lse;
  bool clamped;  // the sigmoids' sum is below 1e-20
  __device__ __forceinline__ void make(const float (&l)[MAXV], bool sigmoid, bool want_z) {
    lse = 0.f;
    clamped = false;
    if (!sigmoid || want_z) {
      float m = l[0], s = 0.f;
#pragma unroll
      for (int v = 1; v < MAXV; ++v) m = fmaxf(m, l[v]);
      m = seg_max<LPT>(m);
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        soft[v] = expf(l[v] - m);
        s += soft[v];
      }
      s = seg_sum<LPT>(s);
      const float inv = 1.f / s;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) soft[v] *= inv;
      lse = m + logf(s);
    }
    if (sigmoid) {
      float s = 0.f;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) {
        p[v] = 1.f / (1.f + expf(-l[v]));  // (-inf: 0)
        s += p[v];
      }
      s = seg_sum<LPT>(s);
      clamped = s < 1e-20f;
      const float inv = 1.f / (clamped ? 1e-20f : s);
#pragma unroll
      for (int v = 0; v < MAXV; ++v) p[v] *= inv;
    } else {
#pragma unroll
      for (int v = 0; v < MAXV; ++v) p[v] = soft[v];
    }
  }
};

struct BalanceParams {
  int64_t ld, n_tokens, group_tokens;
  int32_t E, k;
  int64_t tpc;        // tokens per chunk
  int64_t per_group;  // chunks per group
  const uint8_t* mask;
  int32_t sigmoid, entropy;
  double weight, z_weight;
};

// One chunk: sums of p per expert, counts per expert, sum of lse^2, live tokens.
template <typename LT, int LPT, int MAXV, bool VEC>
__global__ __launch_bounds__(kBalanceThreads) void balance_chunk_kernel(
    const LT* __restrict__ logits, const void* __restrict__ sel, int32_t sel_is_int64, const BalanceParams p,
    float* __restrict__ part_p, int32_t* __restrict__ part_c, float* __restrict__ part_z,
    int32_t* __restrict__ part_n) {
  constexpr int SEGS = kBalanceThreads / LPT, PER = LPT * MAXV;
  __shared__ float sums[SEGS * PER];
  __shared__ int32_t hist[PER];
  __shared__ float zs[SEGS];
  __shared__ int32_t ns[SEGS];
  const int32_t E = p.E, k = p.k;
  const int li = threadIdx.x % LPT, seg = threadIdx.x / LPT;
  const int64_t b = blockIdx.x;
  const int64_t g0 = (b / p.per_group) * p.group_tokens;
  const int64_t t_lo = g0 + (b % p.per_group) * p.tpc;
  const int64_t t_end = t_lo + p.tpc < g0 + p.group_tokens ? t_lo + p.tpc : g0 + p.group_tokens;
  for (int e = threadIdx.x; e < PER; e += kBalanceThreads) hist[e] = 0;
  __syncthreads();
  // the counts
  const int64_t routes = (t_end - t_lo) * k;
  const float inv_k = 1.f / (float)k;
  for (int64_t i = threadIdx.x; i < routes; i += kBalanceThreads) {
    const int64_t r = t_lo * k + i;
    const int64_t id = sel_is_int64 ? ((const int64_t*)sel)[r] : (int64_t)((const int32_t*)sel)[r];
    // i / k: exact for i + 0.5 while i * 2^-24 < 0.5 / k (a chunk's routes, below 2^16; else by division)
    const int64_t t = t_lo + (i < 65536 ? (int64_t)(((float)i + 0.5f) * inv_k) : i / k);
    if (id >= 0 && id < E && (p.mask == nullptr || p.mask[t])) atomicAdd(&hist[(int)id], 1);
  }
  // the sums (every lane runs every pass: segment reductions need whole waves)
  float col[MAXV], z = 0.f;
  int32_t n = 0;
#pragma unroll
  for (int v = 0; v < MAXV; ++v) col[v] = 0.f;
  for (int64_t t0 = t_lo; t0 < t_end; t0 += SEGS) {
    const int64_t t = t0 + seg, at = t < t_end ? t : t_end - 1;
    const bool live = t < t_end && (p.mask == nullptr || p.mask[at]);
    float l[MAXV];
    balance_row<LT, LPT, MAXV, VEC>(logits + at * p.ld, li, E, l);
    BalanceTerms<LPT, MAXV> x;
    x.make(l, p.sigmoid != 0, true);
#pragma unroll
    for (int v = 0; v < MAXV; ++v) col[v] += live ? x.p[v] : 0.f;
    z += live ? x.lse * x.lse : 0.f;
    n += live ? 1 : 0;
  }
#pragma unroll
  for (int v = 0; v < MAXV; ++v) sums[seg * PER + balance_expert<LPT>(li, v)] = col[v];
  if (li == 0) {
    zs[seg] = z;
    ns[seg] = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kBalanceThreads) {
    float s = 0.f;
#pragma unroll 8
    for (int q = 0; q < SEGS; ++q) s += sums[q * PER + e];
    part_p[b * E + e] = s;
    part_c[b * E + e] = hist[e];
  }
  if (threadIdx.x == 0) {
    float zt = 0.f;
    int32_t nt = 0;
    for (int q = 0; q < SEGS; ++q) {
      zt += zs[q];
      nt += ns[q];
    }
    part_z[b] = zt;
    part_n[b] = nt;
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}

// The chunks' sums added, in chunk order per thread and threads in a fixed tree:
// the two terms, the counts and the coefficients of the backward pass.
__global__ __launch_bounds__(kBalanceSumThreads) void balance_sum_kernel(
    const BalanceParams p, int32_t groups, const float* __restrict__ part_p, const int32_t* __restrict__ part_c,
    const float* __restrict__ part_z, const int32_t* __restrict__ part_n, float* __restrict__ loss,
    float* __restrict__ terms, int64_t* __restrict__ counts, float* __restrict__ coef) {
  __shared__ int32_t n_of[kBalanceMaxGroups];  // live tokens of each group
  __shared__ int32_t c_of[kRouteMaxExperts];   // routes of each expert
  __shared__ double red_p[kBalanceSumThreads];
  __shared__ int32_t red_c[kBalanceSumThreads];
  __shared__ double wave_b[kBalanceSumThreads / 64], wave_z[kBalanceSumThreads / 64];
  __shared__ int32_t n_total, n_groups;
  const int tid = threadIdx.x;
  const int32_t E = p.E;
  for (int i = tid; i < groups; i += kBalanceSumThreads) n_of[i] = 0;
  for (int i = tid; i < E; i += kBalanceSumThreads) c_of[i] = 0;
  if (tid == 0) n_total = n_groups = 0;
  __syncthreads();
  const int64_t chunks = (int64_t)groups * p.per_group;
  double z = 0.0;
  for (int64_t c = tid; c < chunks; c += kBalanceSumThreads) {
    z += (double)part_z[c];
    atomicAdd(&n_of[c / p.per_group], part_n[c]);
  }
  __syncthreads();
  for (int i = tid; i < groups; i += kBalanceSumThreads)
    if (n_of[i] > 0) {
      atomicAdd(&n_total, n_of[i]);
      atomicAdd(&n_groups, 1);
    }
  __syncthreads();
  // pairs (group, expert), each by `splits` threads
  const int64_t pairs = (int64_t)groups * E;
  int splits = 1;
  while (splits < kBalanceSumThreads && pairs * splits * 2 <= kBalanceSumThreads) splits *= 2;
  const int per_pass = kBalanceSumThreads / splits, s = tid / per_pass;
  double total = 0.0;
  for (int64_t base = 0; base < pairs; base += per_pass) {
    const int64_t pair = base + tid % per_pass;
    const bool in = pair < pairs;
    const int32_t g = in ? (int32_t)(pair / E) : 0, e = in ? (int32_t)(pair - (int64_t)g * E) : 0;
    double P = 0.0;
    int32_t c = 0;
    if (in) {
      const int64_t at = (int64_t)g * p.per_group;
#pragma unroll 8
      for (int64_t i = s; i < p.per_group; i += splits) {
        P += (double)part_p[(at + i) * E + e];
        c += part_c[(at + i) * E + e];
      }
    }
    if (splits > 1) {
      __syncthreads();
      red_p[tid] = P;
      red_c[tid] = c;
      __syncthreads();
      if (s == 0)
        for (int q = 1; q < splits; ++q) {
          P += red_p[q * per_pass + tid];
          c += red_c[q * per_pass + tid];
        }
    }
    if (s != 0 || !in) continue;
    atomicAdd(&c_of[e], c);
    double a = 0.0;
    if (n_of[g] > 0) {
      const double n = (double)n_of[g], each = 1.0 / (double)n_groups;
      P /= n;
      if (p.entropy) {
        // P = 0: every p is 0 there, and so is its part of the gradient
        const double lg = P == 0.0 ? 0.0 : log(P);
        total += P * lg * each;
        a = P == 0.0 ? 0.0 : (lg + 1.0) * each / n;
      } else {
        const double f = (double)E * (double)c / ((double)p.k * n);
        total += f * P * each;
        a = f * each / n;
      }
    }
    coef[pair] = (float)(p.weight * a);
  }
  total = wave_sum_f64(total);
  z = wave_sum_f64(z);
  if (tid % 64 == 0) {
    wave_b[tid / 64] = total;
    wave_z[tid / 64] = z;
  }
  __syncthreads();
  for (int e = tid; e < E; e += kBalanceSumThreads) counts[e] = c_of[e];
  if (tid == 0) {
    double bt = 0.0, zt = 0.0;
    for (int w = 0; w < kBalanceSumThreads / 64; ++w) {
      bt += wave_b[w];
      zt += wave_z[w];
    }
    const double inv = n_total > 0 ? 1.0 / (double)n_total : 0.0;
    zt *= inv;
    terms[0] = (float)bt;
    terms[1] = (float)zt;
    // (a term of weight 0 does not pass its NaN or infinity on)
    loss[0] = (float)((p.weight != 0.0 ? p.weight * bt : 0.0) + (p.z_weight != 0.0 ? p.z_weight * zt : 0.0));
    coef[pairs] = (float)(2.0 * p.z_weight * inv);
  }
}

template <typename LT, int LPT, int MAXV, bool VEC>
__global__ __launch_bounds__(kBalanceThreads) void balance_bwd_kernel(
    const LT* __restrict__ logits, const BalanceParams p, int32_t groups, const float* __restrict__ coef,
    const float* __restrict__ grad_loss, LT* __restrict__ glog, int64_t gld) {
  constexpr int SEGS = kBalanceThreads / LPT;
  const int32_t E = p.E;
  const int li = threadIdx.x % LPT, seg = threadIdx.x / LPT;
  const int64_t t = (int64_t)blockIdx.x * SEGS + seg, at = t < p.n_tokens ? t : p.n_tokens - 1;
  float l[MAXV], a[MAXV];
  balance_row<LT, LPT, MAXV, VEC>(logits + at * p.ld, li, E, l);
  const float* arow = coef + (at / p.group_tokens) * E;
#pragma unroll
  for (int v = 0; v < MAXV; ++v) {
    const int e = balance_expert<LPT>(li, v);
    a[v] = arow[e < E ? e : E - 1];
  }
  const float b = coef[(int64_t)groups * E], g = *grad_loss;
  const bool live = p.mask == nullptr || p.mask[at];
  BalanceTerms<LPT, MAXV> x;
  x.make(l, p.sigmoid != 0, b != 0.f);
  float dot = 0.f;
#pragma unroll
  for (int v = 0; v < MAXV; ++v) dot += balance_expert<LPT>(li, v) < E ? a[v] * x.p[v] : 0.f;
  dot = seg_sum<LPT>(dot);
  const float zl = b * x.lse;
  // (S under the clamp is a constant: p = s / 1e-20)
  if (x.clamped) dot = 0.f;
#pragma unroll
  for (int v = 0; v < MAXV; ++v) {
    float d = x.p[v] * (a[v] - dot);
    if (p.sigmoid) {
      const float ex = expf(l[v]);  // 1 - s = 1 / (1 + e^l)
      d *= 1.f / (1.f + ex);
    }
    if (b != 0.f) d += zl * x.soft[v];
    l[v] = live ? d * g : 0.f;
  }
  if (t >= p.n_tokens) return;
  LT* out = glog + t * gld;
#pragma unroll
  for (int q = 0; q < MAXV; q += 8) {
    const int e0 = balance_expert<LPT>(li, q);
    if constexpr (VEC) {
      if (e0 >= E) continue;
      if constexpr (sizeof(LT) == 4) {
        reinterpret_cast<float4*>(out + e0)[0] = make_float4(l[q], l[q + 1], l[q + 2], l[q + 3]);
        reinterpret_cast<float4*>(out + e0)[1] = make_float4(l[q + 4], l[q + 5], l[q + 6], l[q + 7]);
      } else {
        LT o[8];
#pragma unroll
        for (int v = 0; v < 8; ++v) o[v] = from_f32<LT>(l[q + v]);
        *reinterpret_cast<uint4*>(out + e0) = *reinterpret_cast<uint4*>(o);
      }
    } else {
#pragma unroll
      for (int v = 0; v < 8; ++v)
        if (e0 + v < E) out[e0 + v] = from_f32<LT>(l[q + v]);
    }
  }
}

// Tokens per chunk: a workgroup per CU, of whole passes.
static int64_t balance_chunk_tokens(int64_t n_tokens, int64_t group_tokens, int32_t n_experts) {
  int64_t segs = 0;
  by_experts(n_experts, [&](auto lpt, auto) { segs = kBalanceThreads / decltype(lpt)::value; });
  int64_t tpc = ((n_tokens > 0 ? n_tokens : 1) + 255) / 256;
  tpc = (tpc + segs - 1) / segs * segs;
  return tpc < group_tokens ? tpc : group_tokens;
}

static int64_t balance_chunks(int64_t n_tokens, int64_t group_tokens, int32_t n_experts, int64_t* tpc) {
  *tpc = balance_chunk_tokens(n_tokens, group_tokens, n_experts);
  return (group_tokens + *tpc - 1) / *tpc;
}

size_t balance_workspace_bytes(int64_t n_tokens, int64_t group_tokens, int32_t n_experts) {
  int64_t tpc;
  const int64_t chunks = balance_chunks(n_tokens, group_tokens, n_experts, &tpc) * (n_tokens / group_tokens);
  return (size_t)chunks * ((size_t)n_experts + 1) * 8;
}

static bool balance_vec(const void* logits, int64_t ld, int32_t E) {
  return E % 8 == 0 && ld % 8 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
}

hipError_t launch_balance_loss(const void* logits, int32_t dtype, int64_t n_tokens, int64_t ld, int32_t n_experts,
                               const void* sel, int32_t sel_is_int64, int64_t top_k, const uint8_t* mask,
                               int64_t group_tokens, int32_t entropy, int32_t sigmoid, double weight,
                               double z_weight, float* loss, float* terms, int64_t* counts, float* coef,
                               void* workspace, hipStream_t stream) {
  BalanceParams p{ld, n_tokens, group_tokens, n_experts, (int32_t)top_k, 0, 0, mask, sigmoid, entropy, weight, z_weight};
  p.per_group = balance_chunks(n_tokens, group_tokens, n_experts, &p.tpc);
  const int32_t groups = (int32_t)(n_tokens / group_tokens);
  const int64_t chunks = p.per_group * groups;
  if (chunks > 0x7fffffffll) return hipErrorInvalidValue;
  float* part_p = (float*)workspace;
  int32_t* part_c = (int32_t*)(part_p + chunks * n_experts);
  float* part_z = (float*)(part_c + chunks * n_experts);
  int32_t* part_n = (int32_t*)(part_z + chunks);
  const bool vec = balance_vec(logits, ld, n_experts);
  if (chunks > 0) by_dtype(dtype, [&](auto lt) {
    using LT = decltype(lt);
    by_experts(n_experts, [&](auto lpt, auto maxv) {
      constexpr int LPT = decltype(lpt)::value, MAXV = decltype(maxv)::value;
      auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)chunks), dim3(kBalanceThreads), 0, stream, (const LT*)logits, sel,
                           sel_is_int64, p, part_p, part_c, part_z, part_n);
      };
      if (vec) go(balance_chunk_kernel<LT, LPT, MAXV, true>);
      else go(balance_chunk_kernel<LT, LPT, MAXV, false>);
    });
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(balance_sum_kernel, dim3(1), dim3(kBalanceSumThreads), 0, stream, p, groups, part_p, part_c,
                     part_z, part_n, loss, terms, counts, coef);
  return hipGetLastError();
}

hipError_t launch_balance_loss_backward(const void* logits, int32_t dtype, int64_t n_tokens, int64_t ld,
                                        int32_t n_experts, const uint8_t* mask, int64_t group_tokens,
                                        int32_t sigmoid, const float* coef, const float* grad_loss,
                                        void* grad_logits, int64_t grad_ld, hipStream_t stream) {
  const BalanceParams p{ld, n_tokens, group_tokens, n_experts, 1, 1, 1, mask, sigmoid, 0, 0.0, 0.0};
  const bool vec = balance_vec(logits, ld, n_experts) && balance_vec(grad_logits, grad_ld, n_experts);
  by_dtype(dtype, [&](auto lt) {
    using LT = decltype(lt);
    by_experts(n_experts, [&](auto lpt, auto maxv) {
      constexpr int LPT = decltype(lpt)::value, MAXV = decltype(maxv)::value;
      constexpr int SEGS = kBalanceThreads / LPT;
      auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)((n_tokens + SEGS - 1) / SEGS)), dim3(kBalanceThreads), 0, stream,
                           (const LT*)logits, p, (int32_t)(n_tokens / group_tokens), coef, grad_loss,
                           (LT*)grad_logits, grad_ld);
      };
      if (vec) go(balance_bwd_kernel<LT, LPT, MAXV, true>);
      else go(balance_bwd_kernel<LT, LPT, MAXV, false>);
    });
  });
  return hipGetLastError();
}

}  // namespace cvmm
