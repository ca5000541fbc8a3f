// Low-rank adapters beside a shared projection (csrc/cvmm_lora*.hip):
//   out[t] = base[t] + x[t] W + h[t] B_i,   h[t] = rnd_op(s_i x[t] A_i),   i = ids[t]
// (calls of few rows do not round h); rows with an id outside [0, n) take the base and the projection alone.
#pragma once

#include "cvmm_common.h"

namespace cvmm {

constexpr int64_t kLoraMaxRank = 256;

struct LoraParams {
  // rows x [rows][K] in the op type
  const void* x;
  int64_t rows, x_ld;
  // W [K][N] (or NULL), A [n][K][rank], B [n][rank][N], op type, element strides
  const void* w;
  int64_t w_sk, w_sn;
  const void* a;
  int64_t a_se, a_sk, a_sr;
  const void* b;
  int64_t b_se, b_sr, b_sn;
  int32_t n;
  int64_t K, N, rank;
  const void* ids;
  int32_t ids_is_int64;
  const int64_t* order;  // a permutation of the rows with equal ids side by side, or NULL
  const float* scales;   // one per adapter, or NULL
  float scale;
  const void* base;      // or NULL; op type or fp32
  int32_t base_dtype;
  int64_t base_ld;
  void* out;             // op type
  int64_t out_ld;
  // h: [rows][h_ld], op type, zero from rank up to h_ld (a multiple of 32)
  void* h;
  int64_t h_ld;
  // or NULL: h transposed, [rank][ht_ld], column p the row order[p]
  void* ht;
  int64_t ht_ld;
  // 16-byte kernels: the output's own width and the rank that ht has (N and rank
  // count zero padding up to multiples of 8), and whether the rows of out and of
  // base are made of aligned pieces
  int64_t n_out, rank_out;
  int32_t out_vec, base_vec;
};

// K split over workgroups: fp32 partial products [splits][rows][part_ld], each
// of `slices` slices of 64 k; inner rows alike, [h_splits][rows][rank].
struct LoraSplit {
  float* part;
  int64_t part_ld;
  int32_t splits, slices;
  uint32_t gemm_blocks;  // the workgroups after them form inner rows
  float* h_part;
  int32_t h_splits;
  int32_t h_k;           // k per share of the inner rows
};

struct LoraWgradParams {
  // rows in the op type, and the inner rows transposed in sorted order
  const void* x;
  int64_t x_ld;
  const void* g;
  int64_t g_ld;
  const void* ht;  // [rank][t_ld]: s x A_i
  const void* ut;  // [rank][t_ld]: s g B_i^T
  int64_t t_ld, rows;
  int32_t n;
  int64_t d_in, d_out, rank;
  const int64_t* order;    // sorting permutation of the rows
  const int64_t* offsets;  // inclusive, one per adapter
  void* ga;                // [n][d_in][rank], contiguous, or NULL
  void* gb;                // [n][rank][d_out], contiguous, or NULL
  int32_t g_dtype;
  float* part;             // shares x (ga's values, then gb's), fp32
  int32_t shares;
};

__device__ __forceinline__ int32_t lora_id(const LoraParams& p, int64_t row) {
  const int64_t id = p.ids_is_int64 ? ((const int64_t*)p.ids)[row] : (int64_t)((const int32_t*)p.ids)[row];
  return id >= 0 && id < p.n ? (int32_t)id : -1;
}

__device__ __forceinline__ float lora_scale(const LoraParams& p, int32_t id) {
  return p.scales != nullptr ? p.scale * p.scales[id] : p.scale;
}

// The least of a wave's values, as a scalar.
__device__ __forceinline__ int32_t wave_min_i32(int32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t o = __shfl_xor(v, d, 64);
    v = o < v ? o : v;
  }
  return __builtin_amdgcn_readfirstlane(v);
}

}  // namespace cvmm
