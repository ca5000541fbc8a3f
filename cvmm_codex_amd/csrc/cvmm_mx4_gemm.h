// Routed products with 4-bit expert weights (cvmm_mx4.h), frozen: for every
// expert-sorted route p of expert e
//   forward     acc[p][n] = sum_k A[arow(p)][k] * W_e[k][n]
//   input grad  acc[p][k] = sum_n G[arow(p)][n] * W_e[k][n]
// The weights are read as they are stored, 17 bytes for 32 of them, and become
// matrix operands in registers; all sums are fp32.
//
// Three forms:
//  * 16-bit rows (mx4_gemm_kernel): v_mfma 16x16x32 with the weights converted
//    to the rows' type, which is exact (fp16: within its range).  A panel's
//    lane holds 32 consecutive k of one column; MFMA j of 4 takes its k 8 j ..
//    8 j + 8 and, as the other operand, the same k of the rows, so four MFMAs
//    cover a 128-k panel with no shuffles.  The weights go from L2 straight to
//    registers (a quarter of the bytes of a 16-bit copy), the gathered rows
//    through LDS by DMA.
//  * 4-bit rows (mx4_gemm4_kernel): v_mfma_scale 16x16x128 on the codes of
//    both sides, the block scales applied by the instruction: four times the
//    16-bit rate, an eighth of the LDS and L2 bytes per multiply-add.
//  * input gradient (mx4_gemm_t_kernel): the contraction runs over n, which a
//    panel's lane holds one of; each 64-n slice is converted once per
//    workgroup into LDS rows [n][k], read back through the transposing LDS
//    loads.
// Operands are swapped (C^T = W A^T), so a lane ends with 4 consecutive columns
// of one row.
#pragma once

#include <type_traits>

#include "cvmm_gemm_panel.h"
#include "cvmm_mx4.h"

namespace cvmm {

struct Mx4Params {
  GemmParams g;  // a: rows in the op type, or (4-bit rows) their codes; b unused
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t np, kp;           // panels of an expert
  const uint8_t* a_scales;  // 4-bit rows: 16 bytes per 512 values
  int64_t a_bytes;          // 4-bit rows: code bytes of a row
  int64_t a_groups;
  int32_t pieces;           // output rows not made of whole aligned 16-byte pieces
  int32_t dg_vec;           // x rows of the routing-weight gradient in 8-byte pieces
};

// acc[i][j] of lane (fr, fq): row j * 16 + fr, columns 16 i + 4 fq .. + 4 of
// the wave's 64.  Two lane swaps make 8 consecutive columns, one 16-byte store.
template <typename OutT, int MB, typename Row>
__device__ __forceinline__ void mx4_store(const Mx4Params& p, const f32x4_t (&acc)[4][MB], int64_t nwave, int fr,
                                          int fq, Row&& row) {
  const GemmParams& g = p.g;
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    float w;
    const int64_t orow = row(j, w);
    char* rowp = orow >= 0 ? reinterpret_cast<char*>(g.out) + orow * g.out_ld * (int64_t)sizeof(OutT) : nullptr;
    if constexpr (sizeof(OutT) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t n = nwave + i * 16 + 4 * fq;
        if (rowp == nullptr) continue;
        float* d = reinterpret_cast<float*>(rowp) + n;
        if (!p.pieces && n + 4 <= g.N) {
          *reinterpret_cast<float4*>(d) = make_float4(acc[i][j][0] * w, acc[i][j][1] * w, acc[i][j][2] * w, acc[i][j][3] * w);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n + q < g.N) d[q] = acc[i][j][q] * w;
        }
      }
    } else {
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        uint32_t a[2], b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          union { uint32_t u; OutT e[2]; } pa, pb;
          pa.e[0] = (OutT)(acc[2 * pr][j][2 * h] * w);
          pa.e[1] = (OutT)(acc[2 * pr][j][2 * h + 1] * w);
          pb.e[0] = (OutT)(acc[2 * pr + 1][j][2 * h] * w);
          pb.e[1] = (OutT)(acc[2 * pr + 1][j][2 * h + 1] * w);
          a[h] = pa.u;
          b[h] = pb.u;
        }
        const auto s0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
        const auto t0 = __builtin_amdgcn_permlane16_swap(s0[0], s0[1], false, false);
        const auto t1 = __builtin_amdgcn_permlane16_swap(s1[0], s1[1], false, false);
        const int64_t n = nwave + pr * 32 + 8 * fq;
        if (rowp == nullptr || n >= g.N) continue;
        if (!p.pieces) {  // N % 8 == 0
          *reinterpret_cast<uint4*>(rowp + n * 2) = make_uint4(t0[0], t1[0], t0[1], t1[1]);
        } else {
          const uint32_t d[4] = {t0[0], t1[0], t0[1], t1[1]};
          store_piece16(rowp + n * 2, d, g.N - n);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// 16-bit rows
// ---------------------------------------------------------------------------
template <int BM, int BN, int NW>
struct Mx4Cfg {
  static constexpr int NT = NW * 64;
  static constexpr int A_BYTES = BM * 256;             // one slice: 256 bytes of every row
  static constexpr int D = A_BYTES / (NW * 1024);      // DMA instructions per wave and slice
  static constexpr int WN = BN / 64, WM = NW / WN;
  static constexpr int WR = BM / WM, MB = WR / 16;
  static_assert(WM * WN == NW && WM * WR == BM && WR % 16 == 0 && A_BYTES % (NW * 1024) == 0, "tile");
};

// A row slice's 16-byte chunk c sits at c ^ (row & 15) of its 256-byte LDS row:
// the 16 rows of a fragment read then take 16 distinct bank groups.
template <typename OpT, int BM, int BN, int NW, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void mx4_gemm_kernel(const Mx4Params p) {
  using Cfg = Mx4Cfg<BM, BN, NW>;
  constexpr int MB = Cfg::MB;
  const GemmParams& g = p.g;
  // two LDS objects, named statically in each half of the loop: the compiler
  // then keeps the DMA into one in flight over the reads of the other
  __shared__ __attribute__((aligned(1024))) char stage0[Cfg::A_BYTES];
  __shared__ __attribute__((aligned(1024))) char stage1[Cfg::A_BYTES];
  __shared__ RouteMeta<BM> meta;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n_ntiles = (g.N + BN - 1) / BN;
  const bool tiled = gemm_schedule<BM, Cfg::NT>(g, n_ntiles, meta);
  const int64_t n0 = (int64_t)uniform_i32(meta.group) * BN;
  if (!tiled) {
    zero_unrouted_cols<BM, Cfg::NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + BN, -1);
    return;
  }
  const int32_t expert = uniform_i32(meta.expert);
  const char* zero = reinterpret_cast<const char*>(g_cvmm_zero_page);
  const char* src[Cfg::D];
  int kc[Cfg::D];
#pragma unroll
  for (int j = 0; j < Cfg::D; ++j) {
    const int q = (wave * Cfg::D + j) * 64 + lane, row = q / 16;
    kc[j] = ((q % 16) ^ (row & 15)) * 8;
    const int64_t ar = meta.arow[row];
    src[j] = ar >= 0 ? reinterpret_cast<const char*>(g.a) + (ar * g.a_ld + kc[j]) * 2 : nullptr;
  }
  auto issue = [&](int64_t s, char* buf) {
    const int64_t k0 = s * 128;
#pragma unroll
    for (int j = 0; j < Cfg::D; ++j)
      dma16(src[j] != nullptr && k0 + kc[j] < g.K ? src[j] + k0 * 2 : zero, buf + (wave * Cfg::D + j) * 1024);
  };
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t nwave = n0 + wn * 64;
  // (a wave past the last panel multiplies the last one and stores nothing)
  const int64_t pn = nwave / 64 < p.np ? nwave / 64 : p.np - 1;
  const int64_t panel0 = ((int64_t)expert * p.np + pn) * p.kp;
  const uint8_t* cp = p.codes + panel0 * kMx4PanelCodes + lane * 16;
  const uint8_t* sp = p.scales + panel0 * kMx4PanelScales + lane * 4;
  f32x4_t acc[4][MB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  uint4 w0[4], w1[4];
  uint32_t s0, s1;
  auto load_w = [&](int64_t s, uint4 (&w)[4], uint32_t& sc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(cp + s * kMx4PanelCodes + i * 1024);
    sc = *reinterpret_cast<const uint32_t*>(sp + s * kMx4PanelScales);
  };
  auto multiply = [&](const char* buf, const uint4 (&w)[4], uint32_t sc) {
    float scale[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[i] = mx4_scale((sc >> (8 * i)) & 255u);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      uint4 a[MB];
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const int ra = wm * Cfg::WR + j * 16 + fr;
        a[j] = *reinterpret_cast<const uint4*>(buf + ra * 256 + (((4 * fq + m) ^ (ra & 15)) << 4));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c = m == 0 ? w[i].x : m == 1 ? w[i].y : m == 2 ? w[i].z : w[i].w;
        const uint4 b = mx4_unpack8<OpT>(c, scale[i]);
#pragma unroll
        for (int j = 0; j < MB; ++j) MfmaOp<OpT>::step(acc[i][j], b, a[j]);
      }
    }
  };
  // slice s: everything it needs was requested a whole slice ago
  issue(0, stage0);
  load_w(0, w0, s0);
  for (int64_t s = 0; s < p.kp; s += 2) {
    vm_wait<0>();
    wg_barrier();
    if (s + 1 < p.kp) {
      issue(s + 1, stage1);
      load_w(s + 1, w1, s1);
    }
    multiply(stage0, w0, s0);
    if (s + 1 >= p.kp) break;
    vm_wait<0>();
    wg_barrier();
    if (s + 2 < p.kp) {
      issue(s + 2, stage0);
      load_w(s + 2, w0, s0);
    }
    multiply(stage1, w1, s1);
  }
  mx4_store<OpT, MB>(p, acc, nwave, fr, fq, [&](int j, float& w) {
    w = 1.f;
    return meta.orow[wm * Cfg::WR + j * 16 + fr];
  });
}

// Few routes per expert: 16-row tiles of one panel column, K split over the
// waves, every operand straight to registers; the partial tiles are added in
// wave order through LDS (deterministic).
template <typename OpT, int NW>
__global__ __launch_bounds__(NW * 64) void mx4_decode_kernel(const Mx4Params p) {
  constexpr int NT = NW * 64;
  const GemmParams& g = p.g;
  __shared__ __attribute__((aligned(16))) float part[NW][16][68];
  __shared__ RouteMeta<16> meta;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t n_ntiles = p.np;
  const bool tiled = gemm_schedule_tile<16>(g, n_ntiles, meta);
  const int64_t pn = uniform_i32(meta.group), n0 = pn * 64;
  if (!tiled) {
    zero_unrouted_cols<16, NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + 64, -1);
    return;
  }
  const int32_t expert = uniform_i32(meta.expert);
  const int64_t panel0 = ((int64_t)expert * p.np + pn) * p.kp;
  const uint8_t* cp = p.codes + panel0 * kMx4PanelCodes + lane * 16;
  const uint8_t* sp = p.scales + panel0 * kMx4PanelScales + lane * 4;
  // this wave's panels
  const int kp = (int)p.kp, per = (kp + NW - 1) / NW;
  const int b0 = wave * per, b1 = b0 + per < kp ? b0 + per : kp;
  auto load_w = [&](int s, uint4 (&w)[4], uint32_t& sc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(cp + s * kMx4PanelCodes + i * 1024);
    sc = *reinterpret_cast<const uint32_t*>(sp + s * kMx4PanelScales);
  };
  uint4 w0[4], w1[4], a0[4], a1[4];
  uint32_t s0 = 0, s1 = 0;
  // the first weights are requested before the route rows are known
  if (b0 < b1) load_w(b0, w0, s0);
  gemm_route_meta<16, NT>(g, meta);
  const int64_t ar = meta.arow[fr];
  const char* arow = ar >= 0 ? static_cast<const char*>(g.a) + ar * g.a_ld * 2 : nullptr;
  auto load_a = [&](int s, uint4 (&a)[4]) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int64_t k = (int64_t)s * 128 + fq * 32 + m * 8;
      a[m] = arow != nullptr && k < g.K ? *reinterpret_cast<const uint4*>(arow + k * 2) : make_uint4(0, 0, 0, 0);
    }
  };
  f32x4_t acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const uint4 (&w)[4], uint32_t sc, const uint4 (&a)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float scale = mx4_scale((sc >> (8 * i)) & 255u);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const uint32_t c = m == 0 ? w[i].x : m == 1 ? w[i].y : m == 2 ? w[i].z : w[i].w;
        MfmaOp<OpT>::step(acc[i], mx4_unpack8<OpT>(c, scale), a[m]);
      }
    }
  };
  if (b0 < b1) {
    load_a(b0, a0);
    for (int s = b0; s < b1; s += 2) {
      if (s + 1 < b1) {
        load_w(s + 1, w1, s1);
        load_a(s + 1, a1);
      }
      multiply(w0, s0, a0);
      if (s + 1 >= b1) break;
      if (s + 2 < b1) {
        load_w(s + 2, w0, s0);
        load_a(s + 2, a0);
      }
      multiply(w1, s1, a1);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float4*>(&part[wave][fr][i * 16 + 4 * fq]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  __syncthreads();
  for (int pc = tid; pc < 128; pc += NT) {
    const int r = pc / 8, c = (pc % 8) * 8;
    const int64_t orow = meta.orow[r], n = n0 + c;
    if (orow < 0 || n >= g.N) continue;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += part[w][r][c + q];
    }
    union { uint32_t d[4]; OpT e[8]; } h;
#pragma unroll
    for (int q = 0; q < 8; ++q) h.e[q] = from_f32<OpT>(v[q]);
    char* dst = static_cast<char*>(g.out) + (orow * g.out_ld + n) * 2;
    if (!p.pieces) *reinterpret_cast<uint4*>(dst) = make_uint4(h.d[0], h.d[1], h.d[2], h.d[3]);
    else store_piece16(dst, h.d, g.N - n);
  }
}

// ---------------------------------------------------------------------------
// 4-bit rows
// ---------------------------------------------------------------------------
typedef int mx4_i32x8 __attribute__((ext_vector_type(8)));

template <int OpselW, int OpselA>
__device__ __forceinline__ void mx4_mfma(f32x4_t& c, const uint4& w, uint32_t sw, const uint4& a, uint32_t sa) {
  const mx4_i32x8 vw = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const mx4_i32x8 va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vw, va, c, 4, 4, OpselW, (int)sw, OpselA, (int)sa);
}

// A slice is 512 k: 256 bytes of codes per row, chunk 4 s + q block q of its
// s-th 128 k, with the swizzle of the 16-bit rows' slices.
template <typename OutT, int BM, int BN, int NW, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void mx4_gemm4_kernel(const Mx4Params p) {
  using Cfg = Mx4Cfg<BM, BN, NW>;
  constexpr int MB = Cfg::MB;
  const GemmParams& g = p.g;
  __shared__ __attribute__((aligned(1024))) char stage0[Cfg::A_BYTES];
  __shared__ __attribute__((aligned(1024))) char stage1[Cfg::A_BYTES];
  __shared__ RouteMeta<BM> meta;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n_ntiles = (g.N + BN - 1) / BN;
  const bool tiled = gemm_schedule<BM, Cfg::NT>(g, n_ntiles, meta);
  const int64_t n0 = (int64_t)uniform_i32(meta.group) * BN;
  if (!tiled) {
    zero_unrouted_cols<BM, Cfg::NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + BN, -1);
    return;
  }
  const int32_t expert = uniform_i32(meta.expert);
  const char* zero = reinterpret_cast<const char*>(g_cvmm_zero_page);
  const char* src[Cfg::D];
  int bc[Cfg::D];
#pragma unroll
  for (int j = 0; j < Cfg::D; ++j) {
    const int q = (wave * Cfg::D + j) * 64 + lane, row = q / 16;
    bc[j] = ((q % 16) ^ (row & 15)) * 16;
    const int64_t ar = meta.arow[row];
    src[j] = ar >= 0 ? reinterpret_cast<const char*>(g.a) + ar * p.a_bytes + bc[j] : nullptr;
  }
  auto issue = [&](int64_t s, char* buf) {
    const int64_t b = s * 256;
#pragma unroll
    for (int j = 0; j < Cfg::D; ++j)
      dma16(src[j] != nullptr && b + bc[j] < p.a_bytes ? src[j] + b : zero, buf + (wave * Cfg::D + j) * 1024);
  };
  const int wm = wave / Cfg::WN, wn = wave % Cfg::WN;
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t nwave = n0 + wn * 64;
  const int64_t pn = nwave / 64 < p.np ? nwave / 64 : p.np - 1;
  const int64_t panel0 = ((int64_t)expert * p.np + pn) * p.kp;
  const uint8_t* cp = p.codes + panel0 * kMx4PanelCodes + lane * 16;
  const uint8_t* sp = p.scales + panel0 * kMx4PanelScales + lane * 4;
  const uint8_t* asp[MB];
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    const int64_t ar = meta.arow[wm * Cfg::WR + j * 16 + fr];
    asp[j] = p.a_scales + (ar >= 0 ? ar : 0) * p.a_groups * 16 + fq * 4;  // (no row: zero codes)
  }
  f32x4_t acc[4][MB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int64_t slices = (p.kp + 3) / 4;
  uint32_t sa0[MB], sa1[MB];
  auto load_sa = [&](int64_t s, uint32_t (&sa)[MB]) {
#pragma unroll
    for (int j = 0; j < MB; ++j) sa[j] = *reinterpret_cast<const uint32_t*>(asp[j] + s * 16);
  };
  uint4 w0[4], w1[4];
  uint32_t c0 = 0, c1 = 0;
  auto load_w = [&](int64_t s, uint4 (&w)[4], uint32_t& sc) {
    if (s >= p.kp) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(cp + s * kMx4PanelCodes + i * 1024);
    sc = *reinterpret_cast<const uint32_t*>(sp + s * kMx4PanelScales);
  };
  // step m of a slice
  auto step = [&](auto mc, const char* buf, const uint4 (&w)[4], uint32_t sc, const uint32_t (&sa)[MB]) {
    constexpr int m = decltype(mc)::value;
    uint4 a[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int ra = wm * Cfg::WR + j * 16 + fr;
      a[j] = *reinterpret_cast<const uint4*>(buf + ra * 256 + (((4 * m + fq) ^ (ra & 15)) << 4));
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      mx4_mfma<0, m>(acc[0][j], w[0], sc, a[j], sa[j]);
      mx4_mfma<1, m>(acc[1][j], w[1], sc, a[j], sa[j]);
      mx4_mfma<2, m>(acc[2][j], w[2], sc, a[j], sa[j]);
      mx4_mfma<3, m>(acc[3][j], w[3], sc, a[j], sa[j]);
    }
  };
  auto slice = [&](int64_t s, const char* buf, const uint32_t (&sa)[MB]) {
    const int64_t k = s * 4;
    load_w(k + 1, w1, c1);
    step(std::integral_constant<int, 0>(), buf, w0, c0, sa);
    if (k + 1 >= p.kp) return;
    load_w(k + 2, w0, c0);
    step(std::integral_constant<int, 1>(), buf, w1, c1, sa);
    if (k + 2 >= p.kp) return;
    load_w(k + 3, w1, c1);
    step(std::integral_constant<int, 2>(), buf, w0, c0, sa);
    if (k + 3 >= p.kp) return;
    load_w(k + 4, w0, c0);
    step(std::integral_constant<int, 3>(), buf, w1, c1, sa);
  };
  issue(0, stage0);
  load_w(0, w0, c0);
  load_sa(0, sa0);
  for (int64_t s = 0; s < slices; s += 2) {
    vm_wait<0>();
    wg_barrier();
    if (s + 1 < slices) {
      issue(s + 1, stage1);
      load_sa(s + 1, sa1);
    }
    slice(s, stage0, sa0);
    if (s + 1 >= slices) break;
    vm_wait<0>();
    wg_barrier();
    if (s + 2 < slices) {
      issue(s + 2, stage0);
      load_sa(s + 2, sa0);
    }
    slice(s + 1, stage1, sa1);
  }
  mx4_store<OutT, MB>(p, acc, nwave, fr, fq, [&](int j, float& w) {
    w = 1.f;
    return meta.orow[wm * Cfg::WR + j * 16 + fr];
  });
}

// ---------------------------------------------------------------------------
// input gradient: BN = 128 columns (one k panel), 64-n slices
// ---------------------------------------------------------------------------
typedef short mx4_s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint2 mx4_read_tr(const char* p) {
  const mx4_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mx4_s16x4*)p);
  return __builtin_bit_cast(uint2, v);
}

template <typename OpT, typename OutT, int BM, int OCC>
__global__ __launch_bounds__(256, OCC) void mx4_gemm_t_kernel(const Mx4Params p) {
  constexpr int NW = 4, NT = 256, BN = 128, MB = BM / 2 / 16;
  constexpr int A_BYTES = BM * 128, B_BYTES = 64 * 256, D = A_BYTES / (NW * 1024);
  static_assert(BM % 32 == 0 && A_BYTES % (NW * 1024) == 0, "tile");
  const GemmParams& g = p.g;  // K = d_out, N = d_in
  __shared__ __attribute__((aligned(1024))) char stage0[A_BYTES + B_BYTES];
  __shared__ __attribute__((aligned(1024))) char stage1[A_BYTES + B_BYTES];
  __shared__ RouteMeta<BM> meta;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n_ntiles = (g.N + BN - 1) / BN;
  const bool tiled = gemm_schedule<BM, NT>(g, n_ntiles, meta);
  const int64_t ntile = uniform_i32(meta.group), n0 = ntile * BN;
  if (!tiled) {
    // (the routing-weight gradient's partials: one per 64 columns)
    zero_unrouted_cols<BM, NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + BN, 2 * ntile,
                               2 * ntile + 1 < g.dg_ntiles ? 2 : 1);
    return;
  }
  const int32_t expert = uniform_i32(meta.expert);
  const char* zero = reinterpret_cast<const char*>(g_cvmm_zero_page);
  const char* src[D];
  int kc[D];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int q = (wave * D + j) * 64 + lane, row = q / 8;
    kc[j] = ((q % 8) ^ (row & 7)) * 8;
    const int64_t ar = meta.arow[row];
    src[j] = ar >= 0 ? reinterpret_cast<const char*>(g.a) + (ar * g.a_ld + kc[j]) * 2 : nullptr;
  }
  auto issue = [&](int64_t s, char* buf) {
    const int64_t k0 = s * 64;
#pragma unroll
    for (int j = 0; j < D; ++j)
      dma16(src[j] != nullptr && k0 + kc[j] < g.K ? src[j] + k0 * 2 : zero, buf + (wave * D + j) * 1024);
  };
  // this thread's part of a panel: column (of W) 16 wave + lane % 16, the 32 k of block lane / 16
  const uint8_t* cp = p.codes + ((int64_t)expert * p.np * p.kp + ntile) * kMx4PanelCodes + wave * 1024 + lane * 16;
  const uint8_t* sp = p.scales + ((int64_t)expert * p.np * p.kp + ntile) * kMx4PanelScales + lane * 4 + wave;
  uint4 w;
  uint32_t sb;
  auto load_w = [&](int64_t s) {
    w = *reinterpret_cast<const uint4*>(cp + s * p.kp * kMx4PanelCodes);
    sb = sp[s * p.kp * kMx4PanelScales];
  };
  auto put_w = [&](char* buf) {  // LDS row (of 128 k) of this n, chunks 4 (lane / 16) .. + 4
    const int r = wave * 16 + (lane & 15);
    const float scale = mx4_scale(sb);
    const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int m = 0; m < 4; ++m)
      *reinterpret_cast<uint4*>(buf + A_BYTES + r * 256 + (((4 * (lane >> 4) + m) ^ tr_row_swz<16>(r)) << 4)) =
          mx4_unpack8<OpT>(c[m], scale);
  };
  const int wm = wave >> 1, wn = wave & 1;
  const int fr = lane & 15, fq = lane >> 4;
  f32x4_t acc[4][MB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const char* buf) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 a[MB];
#pragma unroll
      for (int j = 0; j < MB; ++j) {
        const int ra = wm * (BM / 2) + j * 16 + fr;
        a[j] = *reinterpret_cast<const uint4*>(buf + ra * 128 + (((kk * 4 + fq) ^ (ra & 7)) << 4));
      }
      // rows kk * 32 + 8 fq + fr / 4 (+ 4) of the slice, 4 of the 16 columns
      const int r = kk * 32 + fq * 8 + (fr >> 2);
      const int lane_lo = ((fr & 1) << 3) + (((fr >> 1) & 1) << 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* at = buf + A_BYTES + r * 256 + lane_lo + (((wn * 8 + 2 * i) ^ tr_row_swz<16>(r)) << 4);
        const uint2 lo = mx4_read_tr(at), hi = mx4_read_tr(at + 4 * 256);
        const uint4 b = make_uint4(lo.x, lo.y, hi.x, hi.y);
#pragma unroll
        for (int j = 0; j < MB; ++j) MfmaOp<OpT>::step(acc[i][j], b, a[j]);
      }
    }
  };
  const int64_t slices = p.np;
  // slice s is converted into its buffer while slice s - 1 is multiplied
  issue(0, stage0);
  load_w(0);
  put_w(stage0);
  if (slices > 1) load_w(1);
  for (int64_t s = 0; s < slices; s += 2) {
    vm_wait<0>();
    lds_barrier();
    if (s + 1 < slices) {
      issue(s + 1, stage1);
      put_w(stage1);
      if (s + 2 < slices) load_w(s + 2);
    }
    multiply(stage0);
    if (s + 1 >= slices) break;
    vm_wait<0>();
    lds_barrier();
    if (s + 2 < slices) {
      issue(s + 2, stage0);
      put_w(stage0);
      if (s + 3 < slices) load_w(s + 3);
    }
    multiply(stage1);
  }
  const int64_t nwave = n0 + wn * 64;
  if (g.out != nullptr)
    mx4_store<OutT, MB>(p, acc, nwave, fr, fq, [&](int j, float& wt) {
      const int m = wm * (BM / 2) + j * 16 + fr;
      wt = meta.w[m];
      return meta.orow[m];
    });
  if (g.dg != nullptr && nwave < g.dg_n) {
    // routing-weight gradient: sum over the wave's 64 columns of acc * x, in
    // the order of the lane's 16 columns, then the row's 4 lanes
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int m = wm * (BM / 2) + j * 16 + fr;
      const int64_t xr = meta.dgrow[m];
      float sum = 0.f;
      if (xr >= 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t n = nwave + i * 16 + 4 * fq;
          if (p.dg_vec && n + 4 <= g.dg_n) {
            union { uint2 u; OpT e[4]; } c;
            c.u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g.dg_x) + xr * g.dg_x_ld + n);
#pragma unroll
            for (int q = 0; q < 4; ++q) sum += acc[i][j][q] * to_f32(c.e[q]);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (n + q < g.dg_n) sum += acc[i][j][q] * load_as_f32(g.dg_x, g.dg_x_dtype, xr * g.dg_x_ld + n + q);
          }
        }
      }
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (fq == 0 && meta.widx[m] >= 0) g.dg[meta.widx[m] * g.dg_ntiles + nwave / 64] = sum;
    }
  }
}

template <int BM>
inline int64_t mx4_grid(const GemmParams& g, int64_t n_ntiles) {
  const int64_t m_tiles = (g.n_routes + BM - 1) / BM + (g.n_experts < g.n_routes ? g.n_experts : g.n_routes);
  return m_tiles * n_ntiles;
}

}  // namespace cvmm
