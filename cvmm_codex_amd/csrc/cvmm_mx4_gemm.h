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

typedef unsigned int mx4_u32x4 __attribute__((ext_vector_type(4)));

struct Mx4Params {
  GemmParams g;  // a: rows in the op type, or (4-bit rows) their codes; b unused
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t np, kp;           // panels of an expert
  const uint8_t* a_scales;  // 4-bit rows: 16 bytes per 512 values
  int64_t a_bytes;          // 4-bit rows: code bytes of a row
  int64_t a_groups;
  int32_t passes;           // 4-bit rows: column tiles per workgroup
  FastDiv a_div;            // input gradient: routes per row of A
  int32_t stream;           // 16-bit output stored past the caches
  int32_t pieces;           // output rows not made of whole aligned 16-byte pieces
  int32_t dg_vec;           // x rows of the routing-weight gradient in 8-byte pieces
};

// The tile's rows: A row and output row of each, -1 for none (indices below
// 2^31; the general metadata divides in 64 bits).
template <int BM, int NT>
__device__ __forceinline__ void mx4_route_meta(const Mx4Params& p, RouteMeta<BM>& m) {
  const GemmParams& g = p.g;
  for (int r = threadIdx.x; r < BM; r += NT) {
    int64_t a = -1, o = -1, wi = -1, d = -1;
    float w = 1.f;
    if (r < m.rows) {
      const int64_t q = m.row0 + r;
      a = g.a_idx[q];
      o = g.o_idx != nullptr ? g.o_idx[q] : q;
      wi = g.w_idx[q];
      if (g.dg != nullptr) d = g.dg_x_idx[q];
      a = a < 0 || a >= g.n_routes ? -1 : p.a_div.div(a);
      if (a >= g.a_rows) a = -1;
      if (o < 0 || o >= g.out_rows) o = -1;
      if (wi < 0 || wi >= g.n_routes) wi = -1;
      if (d < 0 || d >= g.dg_x_rows) d = -1;
      if (g.w != nullptr && wi >= 0) w = static_cast<const float*>(g.w)[wi];
    }
    m.arow[r] = a;
    m.orow[r] = o;
    m.widx[r] = wi;
    m.dgrow[r] = d;
    m.w[r] = w;
  }
  __syncthreads();
}
template <int BM>
struct Mx4Rows {
  int32_t a[BM], o[BM];
};
template <int BM, int NT>
__device__ __forceinline__ void mx4_rows(const GemmParams& g, const RouteMeta<BM>& m, Mx4Rows<BM>& rows) {
  for (int r = threadIdx.x; r < BM; r += NT) {
    int64_t a = -1, o = -1;
    if (r < m.rows) {
      const int64_t q = m.row0 + r;
      a = g.a_idx[q];
      o = g.o_idx != nullptr ? g.o_idx[q] : q;
      if (a < 0 || a >= g.a_rows) a = -1;
      if (o < 0 || o >= g.out_rows) o = -1;
    }
    rows.a[r] = (int32_t)a;
    rows.o[r] = (int32_t)o;
  }
  __syncthreads();
}

// acc[i][j] of lane (fr, fq): row j * 16 + fr, columns 16 i + 4 fq .. + 4 of
// the wave's 64.  Two lane swaps make 8 consecutive columns, one 16-byte store.
// row(j, w): the output row, or -1, and its scale.
template <typename OutT, int MB, bool SCALED, typename Row>
__device__ __forceinline__ void mx4_store(const Mx4Params& p, const f32x4_t (&acc)[4][MB], int64_t nwave, int fr,
                                          int fq, Row&& row) {
  const GemmParams& g = p.g;
  const uint32_t ldb = (uint32_t)(g.out_ld * (int64_t)sizeof(OutT));  // (columns below 2^30)
  const int64_t left = g.N - nwave;                                   // columns from the wave's first on
#pragma unroll
  for (int j = 0; j < MB; ++j) {
    float w = 1.f;
    const int32_t orow = row(j, w);
    char* rowp = reinterpret_cast<char*>(g.out) + nwave * (int64_t)sizeof(OutT) + (uint64_t)(uint32_t)orow * ldb;
    auto val = [&](int i, int q) { return SCALED ? acc[i][j][q] * w : acc[i][j][q]; };
    if constexpr (sizeof(OutT) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = i * 16 + 4 * fq;
        float* d = reinterpret_cast<float*>(rowp) + n;
        if (orow < 0) continue;
        if (!p.pieces && n + 4 <= left) {
          *reinterpret_cast<float4*>(d) = make_float4(val(i, 0), val(i, 1), val(i, 2), val(i, 3));
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (n + q < left) d[q] = val(i, q);
        }
      }
    } else {
#pragma unroll
      for (int pr = 0; pr < 2; ++pr) {
        uint32_t a[2], b[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          union { uint32_t u; OutT e[2]; } pa, pb;
          pa.e[0] = (OutT)val(2 * pr, 2 * h);
          pa.e[1] = (OutT)val(2 * pr, 2 * h + 1);
          pb.e[0] = (OutT)val(2 * pr + 1, 2 * h);
          pb.e[1] = (OutT)val(2 * pr + 1, 2 * h + 1);
          a[h] = pa.u;
          b[h] = pb.u;
        }
        const auto s0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
        const auto t0 = __builtin_amdgcn_permlane16_swap(s0[0], s0[1], false, false);
        const auto t1 = __builtin_amdgcn_permlane16_swap(s1[0], s1[1], false, false);
        const int n = pr * 32 + 8 * fq;
        if (orow < 0 || n >= left) continue;
        if (!p.pieces) {  // N % 8 == 0
          const mx4_u32x4 d = {t0[0], t1[0], t0[1], t1[1]};
          if (p.stream) __builtin_nontemporal_store(d, reinterpret_cast<mx4_u32x4*>(rowp + n * 2));
          else *reinterpret_cast<mx4_u32x4*>(rowp + n * 2) = d;
        } else {
          const uint32_t d[4] = {t0[0], t1[0], t0[1], t1[1]};
          store_piece16(rowp + n * 2, d, left - n);
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
  __shared__ Mx4Rows<BM> rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n_ntiles = (g.N + BN - 1) / BN;
  const bool tiled = gemm_schedule_tile<BM>(g, n_ntiles, meta);
  const int64_t n0 = (int64_t)uniform_i32(meta.group) * BN;
  if (!tiled) {
    zero_unrouted_cols<BM, Cfg::NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + BN, -1);
    return;
  }
  mx4_rows<BM, Cfg::NT>(g, meta, rows);
  const int32_t expert = uniform_i32(meta.expert);
  const char* zero = reinterpret_cast<const char*>(g_cvmm_zero_page);
  // DMA instruction j of this wave fills 4 rows of 16 pieces
  const int r0 = wave * Cfg::D * 4 + (lane >> 4), kl = (lane & 15) ^ (lane >> 4);
  auto issue = [&](int s, char* buf) {
    int l = kl, rr = r0;
    asm volatile("" : "+v"(l), "+v"(rr));  // (addresses made here, not kept over the loop)
    int32_t ar[Cfg::D];
#pragma unroll
    for (int j = 0; j < Cfg::D; ++j) ar[j] = rows.a[rr + 4 * j];
#pragma unroll
    for (int j = 0; j < Cfg::D; ++j) {
      // piece (lane & 15) ^ (row & 15), row = r0 + 4 j
      const int64_t k = (int64_t)s * 128 + (l ^ ((4 * (wave * Cfg::D + j)) & 15)) * 8;
      const char* row = reinterpret_cast<const char*>(g.a) + ((int64_t)ar[j] * g.a_ld + k) * 2;
      dma16(ar[j] >= 0 && k < g.K ? row : zero, buf + (wave * Cfg::D + j) * 1024);
    }
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
  auto load_w = [&](uint4 (&w)[4], uint32_t& sc) {  // the next panel
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(cp + i * 1024);
    sc = *reinterpret_cast<const uint32_t*>(sp);
    cp += kMx4PanelCodes;
    sp += kMx4PanelScales;
    issue_fence();
  };
  // row wm * WR + 16 j + fr, chunk 4 fq + m, at chunk ^ fr
  const int a_at = (wm * Cfg::WR + fr) * 256 + (((4 * fq) ^ fr) << 4);
  auto multiply = [&](const char* buf, const uint4 (&w)[4], uint32_t sc) {
    float scale[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) scale[i] = mx4_scale((sc >> (8 * i)) & 255u);
    int at = a_at;
    asm volatile("" : "+v"(at));
    uint4 a[2][MB];
    auto read = [&](int m) {
#pragma unroll
      for (int j = 0; j < MB; ++j) a[m & 1][j] = *reinterpret_cast<const uint4*>(buf + (at ^ (m << 4)) + j * 16 * 256);
    };
    read(0);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (m < 3) read(m + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t c = m == 0 ? w[i].x : m == 1 ? w[i].y : m == 2 ? w[i].z : w[i].w;
        const uint4 b = mx4_unpack8<OpT>(c, scale[i]);
#pragma unroll
        for (int j = 0; j < MB; ++j) MfmaOp<OpT>::step(acc[i][j], b, a[m & 1][j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // slice s: everything it needs was requested a whole slice ago.  Slices go in
  // pairs, an odd one first: a loop left in the middle held two sets of sums.
  const int kp = (int)p.kp;
  int s = kp & 1;
  if (s) {
    issue(0, stage1);
    load_w(w1, s1);
    vm_wait<0>();
    wg_barrier();
    if (kp > 1) {
      issue(1, stage0);
      load_w(w0, s0);
    }
    multiply(stage1, w1, s1);
  } else {
    issue(0, stage0);
    load_w(w0, s0);
  }
  for (; s < kp; s += 2) {
    vm_wait<0>();
    wg_barrier();
    issue(s + 1, stage1);
    load_w(w1, s1);
    multiply(stage0, w0, s0);
    vm_wait<0>();
    wg_barrier();
    if (s + 2 < kp) {
      issue(s + 2, stage0);
      load_w(w0, s0);
    }
    multiply(stage1, w1, s1);
  }
  mx4_store<OpT, MB, false>(p, acc, nwave, fr, fq,
                            [&](int j, float&) { return rows.o[wm * Cfg::WR + j * 16 + fr]; });
}

// Few tiles: 16 rows x 64 columns, every operand straight to registers.  Each of
// the NW waves takes a part of K; the partial tiles are added in wave order
// through LDS (deterministic).  A wave requests its first four panels before the
// route rows are known, and each further one as soon as its registers are free.
template <typename OpT, int NW>
__global__ __launch_bounds__(NW * 64) void mx4_decode_kernel(const Mx4Params p) {
  constexpr int NT = NW * 64, BN = 64;
  const GemmParams& g = p.g;
  __shared__ __attribute__((aligned(16))) float part[NW][16][68];
  __shared__ RouteMeta<16> meta;
  __shared__ Mx4Rows<16> rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t n_ntiles = p.np;
  const bool tiled = gemm_schedule_tile<16>(g, n_ntiles, meta);
  const int64_t pn = uniform_i32(meta.group), n0 = pn * BN;
  if (!tiled) {
    zero_unrouted_cols<16, NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + BN, -1);
    return;
  }
  const int32_t expert = uniform_i32(meta.expert);
  const int64_t panel0 = ((int64_t)expert * p.np + pn) * p.kp;
  const uint8_t* cp = p.codes + panel0 * kMx4PanelCodes + lane * 16;
  const uint8_t* sp = p.scales + panel0 * kMx4PanelScales + lane * 4;
  // this wave's panels
  const int kp = (int)p.kp, per = (kp + NW - 1) / NW;
  const int b0 = wave * per, b1 = b0 + per < kp ? b0 + per : kp;
  uint4 w[4][4], a[2][4];
  uint32_t sc[4];
  auto load_w = [&](int k, int set) {
    if (k >= b1) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[set][i] = *reinterpret_cast<const uint4*>(cp + (int64_t)k * kMx4PanelCodes + i * 1024);
    sc[set] = *reinterpret_cast<const uint32_t*>(sp + (int64_t)k * kMx4PanelScales);
  };
#pragma unroll
  for (int u = 0; u < 4; ++u) load_w(b0 + u, u);
  mx4_rows<16, NT>(g, meta, rows);
  const int32_t ar = rows.a[fr];
  const char* arow = static_cast<const char*>(g.a) + ((int64_t)(ar >= 0 ? ar : 0) * g.a_ld + fq * 32) * 2;
  auto load_a = [&](int k, int set) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int64_t k0 = (int64_t)k * 128 + m * 8;
      a[set][m] = ar >= 0 && k < b1 && k0 + fq * 32 < g.K ? *reinterpret_cast<const uint4*>(arow + k0 * 2)
                                                          : make_uint4(0, 0, 0, 0);
    }
  };
  f32x4_t acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  load_a(b0, 0);
  for (int k = b0; k < b1; k += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (k + u < b1) {
        load_a(k + u + 1, (u + 1) & 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float scale = mx4_scale((sc[u] >> (8 * i)) & 255u);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const uint32_t c = m == 0 ? w[u][i].x : m == 1 ? w[u][i].y : m == 2 ? w[u][i].z : w[u][i].w;
            MfmaOp<OpT>::step(acc[i], mx4_unpack8<OpT>(c, scale), a[u & 1][m]);
          }
        }
        load_w(k + u + 4, u);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<float4*>(&part[wave][fr][i * 16 + 4 * fq]) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  __syncthreads();
  for (int pc = tid; pc < 128; pc += NT) {
    const int r = pc / 8, c = (pc % 8) * 8;
    const int64_t orow = rows.o[r], n = n0 + c;
    if (orow < 0 || n >= g.N) continue;
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.f;
#pragma unroll
    for (int s = 0; s < NW; ++s) {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += part[s][r][c + q];
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

// Four waves, each all BM rows x 64 columns of the tile's 256.  The rows' codes
// of up to 1024 k (512 bytes of every row) sit in LDS, chunk 4 s + q block
// q of the s-th 128 k, at c ^ (row & 15) of each 16 chunks; with them the rows'
// scales.  The weights stream past them straight into registers, RING sets of
// one panel in turn, so the loop over panels and column tiles holds no barrier
// and no DMA: the waits for the weights are the compiler's own counts.  A tile
// of K <= 1024 is loaded once for all of the workgroup's `passes` column tiles.
constexpr int kMx4ChunkK = 1024;
template <typename OutT, int BM, int OCC>
__global__ __launch_bounds__(256, OCC) void mx4_gemm4_kernel(const Mx4Params p) {
  constexpr int BN = 256, NW = 4, NT = 256, MB = BM / 16, RING = 2, PD = RING - 1;
  constexpr int STEPS = kMx4ChunkK / 128;  // panels per chunk
  constexpr int ROWB = kMx4ChunkK / 2, D = BM * ROWB / (NW * 1024);
  static_assert(STEPS % RING == 0, "sets by the panel's place in its chunk");
  const GemmParams& g = p.g;
  __shared__ __attribute__((aligned(1024))) char codes[BM * ROWB];
  // [512 k][16 rows][q][row]: a fragment's 64 scales are 64 consecutive dwords
  __shared__ __attribute__((aligned(16))) uint32_t row_scales[kMx4ChunkK / 512][BM / 16][4][16];
  __shared__ RouteMeta<BM> meta;
  __shared__ Mx4Rows<BM> rows;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n_ntiles = (g.N + BN - 1) / BN, n_groups = (n_ntiles + p.passes - 1) / p.passes;
  const bool tiled = gemm_schedule_tile<BM>(g, n_groups, meta);
  const int64_t t0 = (int64_t)uniform_i32(meta.group) * p.passes;
  const int64_t t1 = t0 + p.passes < n_ntiles ? t0 + p.passes : n_ntiles;
  if (!tiled) {
    zero_unrouted_cols<BM, NT>(g, meta, gridDim.x / n_groups, t0 * BN, t1 * BN, -1);
    return;
  }
  mx4_rows<BM, NT>(g, meta, rows);
  const int32_t expert = uniform_i32(meta.expert);
  const char* zero = reinterpret_cast<const char*>(g_cvmm_zero_page);
  const int kp = (int)p.kp, chunks = (kp + STEPS - 1) / STEPS;
  const int fr = lane & 15, fq = lane >> 4;
  auto load_rows = [&](int c) {
    // instruction j of this wave: 2 rows of 32 16-byte pieces
    int l = lane;
    asm volatile("" : "+v"(l));  // (addresses made here, not kept over the tile)
    const int r0 = wave * D * 2 + (l >> 5);
    int32_t ar[D];
#pragma unroll
    for (int j = 0; j < D; ++j) ar[j] = rows.a[r0 + 2 * j];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int64_t b = (int64_t)c * ROWB + (((l & 31) ^ ((r0 + 2 * j) & 15)) << 4);
      const char* sp_ = reinterpret_cast<const char*>(g.a) + ((int64_t)ar[j] * p.a_bytes + b);
      dma16(ar[j] >= 0 && b < p.a_bytes ? sp_ : zero, codes + (wave * D + j) * 1024);
    }
    // one 16-byte scale group per thread: row tid / 2, group tid % 2
    if (tid >= 2 * BM) return;
    const int64_t sr = rows.a[tid >> 1], gr = (int64_t)c * (kMx4ChunkK / 512) + (tid & 1);
    uint4 s = make_uint4(0, 0, 0, 0);
    if (sr >= 0 && gr < p.a_groups) s = *reinterpret_cast<const uint4*>(p.a_scales + (sr * p.a_groups + gr) * 16);
    uint32_t* d = &row_scales[tid & 1][tid >> 5][0][(tid >> 1) & 15];
    d[0] = s.x; d[16] = s.y; d[32] = s.z; d[48] = s.w;
  };
  const int a_at = fr * ROWB + ((fq ^ fr) << 4);
  f32x4_t acc[4][MB];
  uint4 w[RING][4];
  uint32_t sc[RING];
  const uint8_t *cp, *sp;
  auto load_w = [&](int k, int set) {  // (past the last panel: the last again, unused)
    k = k < kp ? k : kp - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[set][i] = *reinterpret_cast<const uint4*>(cp + (int64_t)k * kMx4PanelCodes + i * 1024);
    sc[set] = *reinterpret_cast<const uint32_t*>(sp + (int64_t)k * kMx4PanelScales);
  };
  auto step = [&](auto mc, int k) {
    constexpr int m = decltype(mc)::value, set = m % RING;
    load_w(k + PD, (m + PD) % RING);
    issue_fence();
    // chunk (4 m + fq) ^ fr of row 16 j + fr
    int at = a_at;
    asm volatile("" : "+v"(at));  // (one address, not one per panel)
    const char* ap = codes + (at ^ (m << 6));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 a[MB / 2];
      uint32_t sa[MB / 2];
#pragma unroll
      for (int j = 0; j < MB / 2; ++j) {
        a[j] = *reinterpret_cast<const uint4*>(ap + (h * (MB / 2) + j) * 16 * ROWB);
        sa[j] = row_scales[m / 4][h * (MB / 2) + j][fq][fr];
      }
#pragma unroll
      for (int j = 0; j < MB / 2; ++j) {
        mx4_mfma<0, m % 4>(acc[0][h * (MB / 2) + j], w[set][0], sc[set], a[j], sa[j]);
        mx4_mfma<1, m % 4>(acc[1][h * (MB / 2) + j], w[set][1], sc[set], a[j], sa[j]);
        mx4_mfma<2, m % 4>(acc[2][h * (MB / 2) + j], w[set][2], sc[set], a[j], sa[j]);
        mx4_mfma<3, m % 4>(acc[3][h * (MB / 2) + j], w[set][3], sc[set], a[j], sa[j]);
      }
    }
  };
  auto start = [&](int64_t t) {
    const int64_t nwave = t * BN + wave * 64;
    const int64_t pn = nwave / 64 < p.np ? nwave / 64 : p.np - 1;
    const int64_t panel0 = ((int64_t)expert * p.np + pn) * p.kp;
    cp = p.codes + panel0 * kMx4PanelCodes + lane * 16;
    sp = p.scales + panel0 * kMx4PanelScales + lane * 4;
#pragma unroll
    for (int k = 0; k < PD; ++k) load_w(k, k);
  };
  for (int64_t t = t0; t < t1; ++t) {
    const int64_t nwave = t * BN + wave * 64;
    start(t);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < MB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < chunks; ++c) {
      const int k0 = c * STEPS;
      if (chunks > 1 || t == t0) {
        if (c > 0 || t > t0) wg_barrier();  // every wave is past the chunk before
        load_rows(c);
        vm_wait<0>();
        lds_barrier();
      }
      const int left = kp - k0;
      step(std::integral_constant<int, 0>(), k0);
      if (left > 1) step(std::integral_constant<int, 1>(), k0 + 1);
      if (left > 2) step(std::integral_constant<int, 2>(), k0 + 2);
      if (left > 3) step(std::integral_constant<int, 3>(), k0 + 3);
      if (left > 4) step(std::integral_constant<int, 4>(), k0 + 4);
      if (left > 5) step(std::integral_constant<int, 5>(), k0 + 5);
      if (left > 6) step(std::integral_constant<int, 6>(), k0 + 6);
      if (left > 7) step(std::integral_constant<int, 7>(), k0 + 7);
    }
    mx4_store<OutT, MB, false>(p, acc, nwave, fr, fq, [&](int j, float&) { return rows.o[j * 16 + fr]; });
  }
}

// ---------------------------------------------------------------------------
// input gradient: BN = 128 columns (one k panel), 64-n slices
// ---------------------------------------------------------------------------
typedef short mx4_s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint2 mx4_read_tr(const char* p) {
  const mx4_s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mx4_s16x4*)p);
  return __builtin_bit_cast(uint2, v);
}

template <typename OpT, typename OutT, int BM, int OCC, bool DG>
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
  const bool tiled = gemm_schedule_tile<BM>(g, n_ntiles, meta);
  const int64_t ntile = uniform_i32(meta.group), n0 = ntile * BN;
  if (!tiled) {
    // (the routing-weight gradient's partials: one per 64 columns)
    zero_unrouted_cols<BM, NT>(g, meta, gridDim.x / n_ntiles, n0, n0 + BN, 2 * ntile,
                               2 * ntile + 1 < g.dg_ntiles ? 2 : 1);
    return;
  }
  mx4_route_meta<BM, NT>(p, meta);
  const int32_t expert = uniform_i32(meta.expert);
  const char* zero = reinterpret_cast<const char*>(g_cvmm_zero_page);
  // DMA instruction j of this wave fills 8 rows of 8 pieces
  const int r0 = wave * D * 8 + (lane >> 3), kl = (lane & 7) ^ (lane >> 3);
  int32_t ar[D];
#pragma unroll
  for (int j = 0; j < D; ++j) ar[j] = (int32_t)meta.arow[r0 + 8 * j];
  auto issue = [&](int s, char* buf) {
    const int64_t k = (int64_t)s * 64 + kl * 8;
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const char* row = reinterpret_cast<const char*>(g.a) + ((int64_t)ar[j] * g.a_ld + k) * 2;
      dma16(ar[j] >= 0 && k < g.K ? row : zero, buf + (wave * D + j) * 1024);
    }
  };
  // this thread's part of a panel: column (of W) 16 wave + lane % 16, the 32 k of block lane / 16
  const uint8_t* cp = p.codes + ((int64_t)expert * p.np * p.kp + ntile) * kMx4PanelCodes + wave * 1024 + lane * 16;
  const uint8_t* sp = p.scales + ((int64_t)expert * p.np * p.kp + ntile) * kMx4PanelScales + lane * 4 + wave;
  uint4 w;
  uint32_t sb;
  auto load_w = [&](int s) {
    w = *reinterpret_cast<const uint4*>(cp + (int64_t)s * p.kp * kMx4PanelCodes);
    sb = sp[(int64_t)s * p.kp * kMx4PanelScales];
  };
  // LDS row (of 128 k) of this n, chunks 4 (lane / 16) .. + 4; the swizzle is even
  const int w_at = A_BYTES + (wave * 16 + (lane & 15)) * 256 +
                   (((4 * (lane >> 4)) ^ tr_row_swz<16>(wave * 16 + (lane & 15))) << 4);
  auto put_w = [&](char* buf) {
    const float scale = mx4_scale(sb);
    const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int m = 0; m < 4; ++m) *reinterpret_cast<uint4*>(buf + (w_at ^ (m << 4))) = mx4_unpack8<OpT>(c[m], scale);
  };
  const int wm = wave >> 1, wn = wave & 1;
  const int fr = lane & 15, fq = lane >> 4;
  f32x4_t acc[4][MB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < MB; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // A row wm * BM / 2 + 16 j + fr, chunk 4 kk + fq at chunk ^ (fr & 7); W rows
  // 32 kk + 8 fq + fr / 4 (+ 4) of the slice, 4 of 16 columns
  const int a_at = (wm * (BM / 2) + fr) * 128 + ((fq ^ (fr & 7)) << 4);
  const int wr = fq * 8 + (fr >> 2);  // (the swizzle of row + 32 is the row's)
  const int b_at = A_BYTES + wr * 256 + ((fr & 1) << 3) + (((fr >> 1) & 1) << 4) + (((wn * 8) ^ tr_row_swz<16>(wr)) << 4);
  auto multiply = [&](const char* buf) {
    int aa = a_at, ba = b_at;
    asm volatile("" : "+v"(aa), "+v"(ba));
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 a[MB];
#pragma unroll
      for (int j = 0; j < MB; ++j) a[j] = *reinterpret_cast<const uint4*>(buf + (aa ^ (kk << 6)) + j * 16 * 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* at = buf + (ba ^ (i << 5)) + kk * 32 * 256;
        const uint2 lo = mx4_read_tr(at), hi = mx4_read_tr(at + 4 * 256);
        const uint4 b = make_uint4(lo.x, lo.y, hi.x, hi.y);
#pragma unroll
        for (int j = 0; j < MB; ++j) MfmaOp<OpT>::step(acc[i][j], b, a[j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // slice s is converted into its buffer while slice s - 1 is multiplied, an odd
  // one first, then pairs
  const int np = (int)p.np;
  int s = np & 1;
  if (s) {
    issue(0, stage1);
    load_w(0);
    put_w(stage1);
    if (np > 1) load_w(1);
    vm_wait<0>();
    lds_barrier();
    if (np > 1) {
      issue(1, stage0);
      put_w(stage0);
      load_w(2);
    }
    multiply(stage1);
  } else {
    issue(0, stage0);
    load_w(0);
    put_w(stage0);
    load_w(1);
  }
  for (; s < np; s += 2) {
    vm_wait<0>();
    lds_barrier();
    issue(s + 1, stage1);
    put_w(stage1);
    if (s + 2 < np) load_w(s + 2);
    multiply(stage0);
    vm_wait<0>();
    lds_barrier();
    if (s + 2 < np) {
      issue(s + 2, stage0);
      put_w(stage0);
      load_w(s + 3);
    }
    multiply(stage1);
  }
  const int64_t nwave = n0 + wn * 64;
  // the x pieces of the routing-weight gradient, all in flight over the stores
  uint2 xv[DG ? MB : 1][4];
  const bool dg_whole = DG && p.dg_vec && nwave + 64 <= g.dg_n && g.dg_x_rows > 0;
  if (dg_whole) {
#pragma unroll
    for (int j = 0; j < MB; ++j) {
      const int64_t xr = meta.dgrow[wm * (BM / 2) + j * 16 + fr];
      const uint16_t* x = static_cast<const uint16_t*>(g.dg_x) + (xr >= 0 ? xr : 0) * g.dg_x_ld + nwave + 4 * fq;
#pragma unroll
      for (int i = 0; i < 4; ++i) xv[j][i] = *reinterpret_cast<const uint2*>(x + i * 16);
    }
    issue_fence();
  }
  if (g.out != nullptr)
    mx4_store<OutT, MB, true>(p, acc, nwave, fr, fq, [&](int j, float& wt) {
      const int m = wm * (BM / 2) + j * 16 + fr;
      wt = meta.w[m];
      return (int32_t)meta.orow[m];
    });
  if (DG && nwave < g.dg_n) {
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
          if (dg_whole) {
            union { uint2 u; OpT e[4]; } c;
            c.u = xv[j][i];
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
