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
// launches forward (chunks of tokens, then their sums in a fixed order) and one
// backward.  Terms of a token are 32-bit; a chunk's sums
// too (at most 256 addends per lane, then at most 64 lanes); sums over chunks are 64-bit.
// Measured (chunks, sums, backward), us: 512 tokens of 16 experts 4.4, 6.2, 3.4; 16384 of
// 128 in bf16 5.4, 9.6, 7.3; 32768 of 256 in 8 sequences 12.8, 7.9, 20.7.  The sums are
// the latency of few workgroups (two of 16384 x 128) that walk all chunks.  The last
// backward is 34 MB at 1.6 TB/s: a wave has two tokens and then ends, so that each waits
// for its own loads (the logits, then 8 single words of coefficients), and issues 361
// vector instructions for them where the forward's passes take 213; vector instructions
// issue for about half of the time.
#include <cmath>

#include "cvmm_common.h"
#include "cvmm_internal.h"
#include "cvmm_router.h"

namespace cvmm {

constexpr int kBalanceThreads = 256;

// e^x to 2 ulp: x log2 e in two parts, the second (its rounding error, and log2 e's)
// to first order.  Below -150 it is 0 in 32 bits either way, and the parts of an
// infinity are none; NaN stays.
__device__ __forceinline__ float balance_exp(float x) {
  x = x < -150.f ? -150.f : x;
  const float t = x * 1.44269504f;
  const float r = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, r * 0.693147181f, e);
}
constexpr int kBalanceSumThreads = 512;

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
  // FORWARD: lse as it is for infinite logits too (their gradient is NaN either way).
  template <bool FORWARD>
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
        soft[v] = balance_exp(l[v] - m);
        s += soft[v];
      }
      s = seg_sum<LPT>(s);
      const float inv = 1.f / s;
#pragma unroll
      for (int v = 0; v < MAXV; ++v) soft[v] *= inv;
      lse = m + logf(s);
      if (FORWARD && __any(s != s)) {  // a NaN in the row, or an infinite maximum: that is its logsumexp
        float nan = 0.f;
#pragma unroll
        for (int v = 0; v < MAXV; ++v) nan = l[v] != l[v] ? 1.f : nan;
        nan = seg_max<LPT>(nan);
        lse = s != s && nan == 0.f ? m : lse;
      }
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

// The chunks' sums, rows of ld values (experts rounded up to 4), and what the sums'
// workgroups leave each other.
struct BalanceParts {
  int64_t ld;
  int32_t eb;           // workgroups per group of tokens: 64 experts each
  float* p;             // [chunks][ld]
  int32_t* c;           // [chunks][ld]
  float* z;             // [chunks]
  int32_t* n;           // [chunks]
  double* block_term;   // [groups * eb]
  int32_t* group_c;     // [groups][E]
  int32_t* arrived;
};

// One chunk: sums of p per expert, counts per expert, sum of lse^2, live tokens.
template <typename LT, int LPT, int MAXV, bool VEC>
__global__ __launch_bounds__(kBalanceThreads) void balance_chunk_kernel(
    const LT* __restrict__ logits, const void* __restrict__ sel, int32_t sel_is_int64, const BalanceParams p,
    const BalanceParts w) {
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
    x.template make<true>(l, p.sigmoid != 0, true);
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
  for (int e = threadIdx.x; e < w.ld; e += kBalanceThreads) {  // (ld <= PER)
    float s = 0.f;
#pragma unroll 8
    for (int q = 0; q < SEGS; ++q) s += sums[q * PER + e];
    w.p[b * w.ld + e] = s;
    w.c[b * w.ld + e] = hist[e];
  }
  if (threadIdx.x == 0) {
    float zt = 0.f;
    int32_t nt = 0;
    for (int q = 0; q < SEGS; ++q) {
      zt += zs[q];
      nt += ns[q];
    }
    w.z[b] = zt;
    w.n[b] = nt;
    if (b == 0) *w.arrived = 0;
  }
}

// Sums of a workgroup, in a fixed tree; every thread gets them.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = v;
  __syncthreads();
  T s = red[0];
#pragma unroll
  for (int w = 1; w < kBalanceSumThreads / 64; ++w) s += red[w];
  return s;
}

// The chunks' sums added, in a fixed order: a workgroup per group and 64 experts
// makes the coefficients of the backward pass, its part of the balance term and its
// counts; the last of them to end adds those, in their order.
__global__ __launch_bounds__(kBalanceSumThreads) void balance_sum_kernel(
    const BalanceParams p, int32_t groups, const BalanceParts w, float* __restrict__ loss, float* __restrict__ terms,
    int64_t* __restrict__ counts, float* __restrict__ coef) {
  constexpr int SLOTS = kBalanceSumThreads / 16;  // chunks at a time, four experts a thread
  __shared__ int32_t n_of[kBalanceMaxGroups];     // live tokens of each group
  __shared__ double s_p[SLOTS][64];
  __shared__ int32_t s_c[SLOTS][64];
  __shared__ double red_d[kBalanceSumThreads / 64];
  __shared__ int32_t red_i[kBalanceSumThreads / 64];
  __shared__ bool last;
  const int tid = threadIdx.x;
  const int32_t E = p.E, blocks = (int32_t)gridDim.x;
  const int32_t g = (int32_t)(blockIdx.x / (uint32_t)w.eb), e0 = (int32_t)(blockIdx.x % (uint32_t)w.eb) * 64;
  // this group's chunks
  {
    const int q = tid % 16, slot = tid / 16;
    double P[4] = {0.0, 0.0, 0.0, 0.0};
    int32_t c[4] = {0, 0, 0, 0};
    if (e0 + 4 * q < w.ld) {
      const int64_t at = (int64_t)g * p.per_group;
#pragma unroll 4
      for (int64_t i = slot; i < p.per_group; i += SLOTS) {
        const float4 v = *reinterpret_cast<const float4*>(w.p + (at + i) * w.ld + e0 + 4 * q);
        const int4 u = *reinterpret_cast<const int4*>(w.c + (at + i) * w.ld + e0 + 4 * q);
        P[0] += (double)v.x, P[1] += (double)v.y, P[2] += (double)v.z, P[3] += (double)v.w;
        c[0] += u.x, c[1] += u.y, c[2] += u.z, c[3] += u.w;
      }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      s_p[slot][4 * q + v] = P[v];
      s_c[slot][4 * q + v] = c[v];
    }
  }
  // live tokens, of all groups
  for (int i = tid; i < groups; i += kBalanceSumThreads) n_of[i] = 0;
  __syncthreads();
  const int64_t chunks = (int64_t)groups * p.per_group;
  double z = 0.0;
  for (int64_t i = tid; i < chunks; i += kBalanceSumThreads) {
    atomicAdd(&n_of[i / p.per_group], w.n[i]);
    z += (double)w.z[i];
  }
  __syncthreads();
  int32_t n_all = 0, n_live = 0;
  for (int i = tid; i < groups; i += kBalanceSumThreads) {
    n_all += n_of[i];
    n_live += n_of[i] > 0 ? 1 : 0;
  }
  n_all = block_sum(n_all, red_i);
  n_live = block_sum(n_live, red_i);
  double term = 0.0;
  if (tid < 64 && e0 + tid < E) {
    double P = 0.0, a = 0.0;
    int32_t c = 0;
#pragma unroll 8
    for (int i = 0; i < SLOTS; ++i) {
      P += s_p[i][tid];
      c += s_c[i][tid];
    }
    if (n_of[g] > 0) {
      const double n = (double)n_of[g], each = 1.0 / (double)n_live;
      P /= n;
      if (p.entropy) {
        // P = 0: every p is 0 there, and so is its part of the gradient
        const double lg = P == 0.0 ? 0.0 : log(P);
        term = P * lg * each;
        a = P == 0.0 ? 0.0 : (lg + 1.0) * each / n;
      } else {
        const double f = (double)E * (double)c / ((double)p.k * n);
        term = f * P * each;
        a = f * each / n;
      }
    }
    // (a weight of 0 passes no NaN of P on)
    coef[(int64_t)g * E + e0 + tid] = p.weight != 0.0 ? (float)(p.weight * a) : 0.f;
    __hip_atomic_store(&w.group_c[(int64_t)g * E + e0 + tid], c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  term = block_sum(term, red_d);
  if (tid == 0) __hip_atomic_store(&w.block_term[blockIdx.x], term, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  splitk_published();
  __syncthreads();
  if (tid == 0) last = splitk_arrive(w.arrived, blocks);
  __syncthreads();
  if (!last) return;
  splitk_acquired();
  double total = 0.0;
  for (int i = tid; i < blocks; i += kBalanceSumThreads)
    total += __hip_atomic_load(&w.block_term[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  total = block_sum(total, red_d);
  z = block_sum(z, red_d);
  for (int e = tid; e < E; e += kBalanceSumThreads) {
    int64_t c = 0;
#pragma unroll 4
    for (int i = 0; i < groups; ++i)
      c += __hip_atomic_load(&w.group_c[(int64_t)i * E + e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    counts[e] = c;
  }
  if (tid == 0) {
    const double inv = n_all > 0 ? 1.0 / (double)n_all : 0.0;
    z *= inv;
    terms[0] = (float)total;
    terms[1] = (float)z;
    // (a term of weight 0 does not pass its NaN or infinity on)
    loss[0] = (float)((p.weight != 0.0 ? p.weight * total : 0.0) + (p.z_weight != 0.0 ? p.z_weight * z : 0.0));
    coef[(int64_t)groups * E] = (float)(2.0 * p.z_weight * inv);
  }
}

// No tokens: zeros.
__global__ __launch_bounds__(256) void balance_none_kernel(int32_t E, float* __restrict__ loss,
                                                           float* __restrict__ terms, int64_t* __restrict__ counts,
                                                           float* __restrict__ coef) {
  for (int e = threadIdx.x; e < E; e += 256) counts[e] = 0;
  if (threadIdx.x == 0) loss[0] = terms[0] = terms[1] = coef[0] = 0.f;
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
  x.template make<false>(l, p.sigmoid != 0, b != 0.f);
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

// Tokens per chunk: two workgroups per CU, of whole passes (32768 tokens of 256 experts:
// 20.8 us forward; one per CU 24.3, four 25; 16384 of 128: 15, one 14.5, four 20), but
// at most 256 passes, whose 32-bit sums lose 256 half steps at most.
constexpr int64_t kBalancePasses = 256;
static int64_t balance_chunk_tokens(int64_t n_tokens, int64_t group_tokens, int32_t n_experts) {
  int64_t segs = 0;
  by_experts(n_experts, [&](auto lpt, auto) { segs = kBalanceThreads / decltype(lpt)::value; });
  int64_t tpc = ((n_tokens > 0 ? n_tokens : 1) + 511) / 512;
  tpc = (tpc + segs - 1) / segs * segs;
  if (tpc > kBalancePasses * segs) tpc = kBalancePasses * segs;
  return tpc < group_tokens ? tpc : group_tokens;
}

static int64_t balance_chunks(int64_t n_tokens, int64_t group_tokens, int32_t n_experts, int64_t* tpc) {
  *tpc = balance_chunk_tokens(n_tokens, group_tokens, n_experts);
  return (group_tokens + *tpc - 1) / *tpc;
}

static BalanceParts balance_parts(void* ws, int64_t chunks, int64_t groups, int32_t n_experts, size_t* bytes) {
  BalanceParts w{};
  w.ld = (n_experts + 3) / 4 * 4;
  w.eb = (n_experts + 63) / 64;
  size_t used = 0;
  auto take = [&](size_t n) {
    void* q = ws != nullptr ? (char*)ws + used : nullptr;
    used = align_up(used + n, 16);
    return q;
  };
  w.block_term = (double*)take((size_t)groups * (size_t)w.eb * 8);
  w.p = (float*)take((size_t)chunks * (size_t)w.ld * 4);
  w.c = (int32_t*)take((size_t)chunks * (size_t)w.ld * 4);
  w.z = (float*)take((size_t)chunks * 4);
  w.n = (int32_t*)take((size_t)chunks * 4);
  w.group_c = (int32_t*)take((size_t)groups * (size_t)n_experts * 4);
  w.arrived = (int32_t*)take(4);
  *bytes = used;
  return w;
}

size_t balance_workspace_bytes(int64_t n_tokens, int64_t group_tokens, int32_t n_experts) {
  if (n_tokens == 0) return 0;
  int64_t tpc;
  const int64_t groups = n_tokens / group_tokens;
  size_t bytes;
  balance_parts(nullptr, balance_chunks(n_tokens, group_tokens, n_experts, &tpc) * groups, groups, n_experts, &bytes);
  return bytes;
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
  if (chunks == 0) {
    hipLaunchKernelGGL(balance_none_kernel, dim3(1), dim3(256), 0, stream, n_experts, loss, terms, counts, coef);
    return hipGetLastError();
  }
  size_t bytes;
  const BalanceParts w = balance_parts(workspace, chunks, groups, n_experts, &bytes);
  const bool vec = balance_vec(logits, ld, n_experts);
  by_dtype(dtype, [&](auto lt) {
    using LT = decltype(lt);
    by_experts(n_experts, [&](auto lpt, auto maxv) {
      constexpr int LPT = decltype(lpt)::value, MAXV = decltype(maxv)::value;
      auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)chunks), dim3(kBalanceThreads), 0, stream, (const LT*)logits, sel,
                           sel_is_int64, p, w);
      };
      if (vec) go(balance_chunk_kernel<LT, LPT, MAXV, true>);
      else go(balance_chunk_kernel<LT, LPT, MAXV, false>);
    });
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(balance_sum_kernel, dim3((unsigned)(groups * w.eb)), dim3(kBalanceSumThreads), 0, stream, p,
                     groups, w, loss, terms, counts, coef);
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
