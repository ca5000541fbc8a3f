// Pieces the routers share: segment reductions, and the stable sort of the
// routes within one workgroup.
#pragma once

#include <type_traits>

#include "cvmm_common.h"

namespace cvmm {

// Segments of LPT lanes (4..64) each route one token: lane i of a segment
// holds experts i + LPT * v, v < MAXV.  Reductions over a segment use DPP
// (quad permutes, half-row and row mirrors) and, past 16 lanes, lane swaps; every
// lane of the segment ends with the same result.
template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ int32_t dpp_i(int32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

// The values of the lane and of the one 16 (32) lanes across, in the same order
// for both.
__device__ __forceinline__ void across16(uint32_t v, uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ void across32(uint32_t v, uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  a = r[0];
  b = r[1];
}

template <int LPT>
__device__ __forceinline__ float seg_max(float v) {
  v = fmaxf(v, dpp_f<kDppXor1>(v));
  v = fmaxf(v, dpp_f<kDppXor2>(v));
  if constexpr (LPT >= 8) v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
  if constexpr (LPT >= 16) v = fmaxf(v, dpp_f<kDppMirror>(v));
  uint32_t a, b;
  if constexpr (LPT >= 32) {
    across16(__float_as_uint(v), a, b);
    v = fmaxf(__uint_as_float(a), __uint_as_float(b));
  }
  if constexpr (LPT >= 64) {
    across32(__float_as_uint(v), a, b);
    v = fmaxf(__uint_as_float(a), __uint_as_float(b));
  }
  return v;
}
template <int LPT>
__device__ __forceinline__ float seg_sum(float v) {  // same two partials per step: same total in every lane
  v = v + dpp_f<kDppXor1>(v);
  v = v + dpp_f<kDppXor2>(v);
  if constexpr (LPT >= 8) v = v + dpp_f<kDppHalfMirror>(v);
  if constexpr (LPT >= 16) v = v + dpp_f<kDppMirror>(v);
  uint32_t a, b;
  if constexpr (LPT >= 32) {
    across16(__float_as_uint(v), a, b);
    v = __uint_as_float(a) + __uint_as_float(b);
  }
  if constexpr (LPT >= 64) {
    across32(__float_as_uint(v), a, b);
    v = __uint_as_float(a) + __uint_as_float(b);
  }
  return v;
}
template <int LPT>
__device__ __forceinline__ int32_t seg_min_i(int32_t v) {
  v = min(v, dpp_i<kDppXor1>(v));
  v = min(v, dpp_i<kDppXor2>(v));
  if constexpr (LPT >= 8) v = min(v, dpp_i<kDppHalfMirror>(v));
  if constexpr (LPT >= 16) v = min(v, dpp_i<kDppMirror>(v));
  uint32_t a, b;
  if constexpr (LPT >= 32) {
    across16((uint32_t)v, a, b);
    v = min((int32_t)a, (int32_t)b);
  }
  if constexpr (LPT >= 64) {
    across32((uint32_t)v, a, b);
    v = min((int32_t)a, (int32_t)b);
  }
  return v;
}
template <int LPT>
__device__ __forceinline__ int32_t seg_max_i(int32_t v) {
  v = max(v, dpp_i<kDppXor1>(v));
  v = max(v, dpp_i<kDppXor2>(v));
  if constexpr (LPT >= 8) v = max(v, dpp_i<kDppHalfMirror>(v));
  if constexpr (LPT >= 16) v = max(v, dpp_i<kDppMirror>(v));
  uint32_t a, b;
  if constexpr (LPT >= 32) {
    across16((uint32_t)v, a, b);
    v = max((int32_t)a, (int32_t)b);
  }
  if constexpr (LPT >= 64) {
    across32((uint32_t)v, a, b);
    v = max((int32_t)a, (int32_t)b);
  }
  return v;
}

template <int LPT>
__device__ __forceinline__ uint32_t seg_or(uint32_t v) {
  v |= (uint32_t)dpp_i<kDppXor1>((int32_t)v);
  v |= (uint32_t)dpp_i<kDppXor2>((int32_t)v);
  if constexpr (LPT >= 8) v |= (uint32_t)dpp_i<kDppHalfMirror>((int32_t)v);
  if constexpr (LPT >= 16) v |= (uint32_t)dpp_i<kDppMirror>((int32_t)v);
  uint32_t a, b;
  if constexpr (LPT >= 32) {
    across16(v, a, b);
    v = a | b;
  }
  if constexpr (LPT >= 64) {
    across32(v, a, b);
    v = a | b;
  }
  return v;
}

// Segment width: 8 experts per lane up to 512 experts, then 16.
template <typename F>
inline void by_experts(int32_t E, F&& f) {
  if (E <= 32) f(std::integral_constant<int, 4>(), std::integral_constant<int, 8>());
  else if (E <= 64) f(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  else if (E <= 128) f(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
  else if (E <= 256) f(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
  else if (E <= 512) f(std::integral_constant<int, 64>(), std::integral_constant<int, 8>());
  else f(std::integral_constant<int, 64>(), std::integral_constant<int, 16>());
}

template <typename F>
inline void by_dtype(int32_t dt, F&& f) {
  if (dt == kF32) f(float());
  else if (dt == kBF16) f(bf16_t());
  else f(f16_t());
}

// The sort's outputs, written by the router's own launch where one workgroup
// holds every route (ONE).
struct RouteSortOut {
  int32_t* sorted_sel;
  int64_t* perm;
  int64_t* token_index;  // or NULL
  int64_t* offsets;
  int32_t* route_pos;    // or NULL
};

// Routes that a single router workgroup sorts itself, at most.  Beyond them
// its ranking outlasts a second launch: 64 tokens, top-8, 128 / 256 / 512
// experts 26 / 42 / 76 us per call in one launch, 23 / 38 / 73 in two; 32
// tokens 14 / 22 / 39 and 20 / 23 / 41.
constexpr int kRouteOneMax = 256;
static_assert(kRouteOneMax % 64 == 0, "whole waves of ids");

// The sort of n = tokens * k routes by the workgroup that chose them: `hist`
// (E counts in LDS) turned into the experts' first positions by a scan, then
// each route's rank among the earlier routes of its expert, counted over `ids`
// (LDS, kRouteOneMax entries).  Enter past a barrier on hist and ids.
template <int THREADS>
__device__ __forceinline__ void route_sort_one(int32_t* hist, const int32_t* ids, int n, int32_t E, int32_t k,
                                               const RouteSortOut& so) {
  // hist -> first output position of each expert (exclusive scan, wave 0)
  if (threadIdx.x < 64) {
    int32_t carry = 0;
    for (int base = 0; base < E; base += 64) {
      const int e = base + (int)threadIdx.x;
      const int32_t c = e < E ? hist[e] : 0;
      const int32_t incl = wave_incl_scan(c) + carry;
      if (e < E) {
        hist[e] = incl - c;
        so.offsets[e] = incl;
      }
      carry = __builtin_amdgcn_readlane(incl, 63);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int32_t e = ids[i];
    // routes before i on the same expert, 16 ids per step (a wave's lanes
    // share their reads and the bound)
    int rank = 0;
    const int end = (i | 63) + 1;
    for (int j = 0; j < end; j += 16) {
      int4 o[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = *reinterpret_cast<const int4*>(ids + j + 4 * q);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = j + 4 * q;
        rank += (o[q].x == e && at < i) ? 1 : 0;
        rank += (o[q].y == e && at + 1 < i) ? 1 : 0;
        rank += (o[q].z == e && at + 2 < i) ? 1 : 0;
        rank += (o[q].w == e && at + 3 < i) ? 1 : 0;
      }
    }
    const int p = hist[e] + rank;
    so.sorted_sel[p] = e;
    so.perm[p] = i;
    if (so.token_index != nullptr) so.token_index[p] = i / k;
    if (so.route_pos != nullptr) so.route_pos[i] = p;
  }
}

}  // namespace cvmm
