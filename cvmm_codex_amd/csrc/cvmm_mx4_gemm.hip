// Launchers of the 4-bit weight products (cvmm_mx4_gemm.h).
#include "cvmm_mx4_gemm.h"

namespace cvmm {

template <typename K>
static hipError_t launch(K kernel, const Mx4Params& p, int64_t grid, int threads, hipStream_t s) {
  if (grid <= 0) return hipSuccess;
  if (grid > 0x7fffffffll) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), 0, s, p);
  return hipGetLastError();
}

template <typename OpT, int BM, int BN, int NW, int OCC>
static hipError_t tile16(const Mx4Params& p, hipStream_t s) {
  return launch(mx4_gemm_kernel<OpT, BM, BN, NW, OCC>, p, mx4_grid<BM>(p.g, (p.g.N + BN - 1) / BN), NW * 64, s);
}

// 16-bit rows.  Times of bf16 launches, 128 experts of 2048 x 512 (512 x 2048):
//   routes per expert     2           8     16          32          64          96          124         1024
//   16-row tiles      14.1 (14.6)  16.3  17.0 (18.7)  21.8 (24.3)  32.5 (36.8)  43.7 (51.1)  53.9 (64.1)  423
//   32-row            15.5 (15.5)  16.5  19.6 (19.7)  21.3 (22.9)  29.8 (31.9)  36.8 (41.4)  46.0 (51.1)  323
//   64-row            21.2 (20.3)  21.7  22.2 (23.9)  29.5 (25.9)  33.2 (32.2)  35.3 (40.6)  44.6 (48.7)  276
// 256-column tiles, 4 waves of 64 columns; 128-column ones where the columns
// end there (64 experts of 1024 x 128, 250 routes: 18.1 -> 14.1 us) or
// where they leave less than four fifths of the wide tiles filled.  A launch
// of fewer than 256 16-row tiles splits K over the waves of a workgroup
// instead: 8 tokens, top-8, 128 experts of 2048 x 512: 11.3 -> 8.1 us; 16
// tokens, 64 experts of 1024 x 128: 7.0 -> 4.6.
template <typename OpT>
static hipError_t fwd16(const Mx4Params& p, hipStream_t s) {
  const GemmParams& g = p.g;
  const int64_t E = g.n_experts < g.n_routes ? g.n_experts : g.n_routes, R = g.n_routes;
  if (((R + 15) / 16 + E) * ((g.N + 255) / 256) < 256 && p.kp >= 4) {
    // eight parts of K where four leave CUs idle (4 tokens, 1024 x 128: 5.0 -> 4.5 us; 8, 2048 x 512: 8.1 -> 9.9)
    if (E * p.np <= 256 && p.kp >= 8)
      return launch(mx4_decode_kernel<OpT, 8>, p, mx4_grid<16>(g, p.np), 512, s);
    return launch(mx4_decode_kernel<OpT, 4>, p, mx4_grid<16>(g, p.np), 256, s);
  }
  const int64_t w128 = (g.N + 127) / 128 * 128, w256 = (g.N + 255) / 256 * 256;
  const bool narrow = 5 * w128 < 4 * w256;
  if (R <= 24 * E) return narrow ? tile16<OpT, 16, 128, 2, 4>(p, s) : tile16<OpT, 16, 256, 4, 4>(p, s);
  if (R <= 88 * E) return narrow ? tile16<OpT, 32, 128, 2, 4>(p, s) : tile16<OpT, 32, 256, 4, 4>(p, s);
  return narrow ? tile16<OpT, 64, 128, 4, 4>(p, s) : tile16<OpT, 64, 256, 4, 3>(p, s);
}

// 4-bit rows.  A tile of K <= 1024 keeps its rows for two column tiles: 16384
// tokens, top-8 of 128 experts of 512 x 2048 take 239 / 212 / 219 us with 1 / 2
// / 4 tiles per workgroup; past that the rows are read again either way, and
// one tile each fills the GPU better (2048 x 512: 107 / 124 us with 1 / 2).
template <typename OutT, int BM, int OCC>
static hipError_t tile4(Mx4Params p, hipStream_t s) {
  const int64_t tiles = (p.g.N + 255) / 256;
  p.passes = p.g.K <= kMx4ChunkK && tiles > 1 ? 2 : 1;
  return launch(mx4_gemm4_kernel<OutT, BM, OCC>, p, mx4_grid<BM>(p.g, (tiles + p.passes - 1) / p.passes), 256, s);
}

// Times of bf16 outputs, 128 experts of 2048 x 512 (512 x 2048), us:
//   routes per expert     4           32          64          128         187
//   32-row tiles      13.7 (13.6)  16.2 (18.1)  19.1 (23.2)  26.3 (33.9)  33.7 (44.4)
//   64-row            14.5 (14.9)  17.5 (20.6)  18.2 (21.6)  23.1 (32.4)  29.0 (39.0)
//   128-row           16.2 (17.4)  17.7 (20.9)  21.9 (29.0)  24.2 (36.7)  25.5 (39.9)
template <typename OutT>
static hipError_t fwd4(const Mx4Params& p, hipStream_t s) {
  const GemmParams& g = p.g;
  const int64_t E = g.n_experts < g.n_routes ? g.n_experts : g.n_routes;
  if (g.n_routes <= 48 * E) return tile4<OutT, 32, 4>(p, s);
  if (g.n_routes <= 160 * E) return tile4<OutT, 64, 3>(p, s);
  return tile4<OutT, 128, 2>(p, s);
}

// Input gradient: 160-row tiles unless they cost over 5 % more than 128-row ones
// in rounds of 512 tiles x tile height (65536 routes of 64 experts, 1024 -> 128:
// 32.4 / 46.4 us, one round against two; 512 x 2048: 248 / 270); 64-row ones
// where the average expert fills no more.
static int bwd_rows(const GemmParams& g) {
  const int64_t E = g.n_experts < g.n_routes ? g.n_experts : g.n_routes, nt = (g.N + 127) / 128;
  if (g.n_routes <= 64 * E) return 64;
  auto rounds = [&](int64_t bm) { return (((g.n_routes + bm - 1) / bm + E / 2) * nt + 511) / 512; };
  return 20 * 160 * rounds(160) <= 21 * 128 * rounds(128) ? 160 : 128;
}

template <typename OpT, typename OutT, int BM, int OCC>
static hipError_t tile_t(const Mx4Params& p, hipStream_t s) {
  const int64_t grid = mx4_grid<BM>(p.g, (p.g.N + 127) / 128);
  if (p.g.dg != nullptr) return launch(mx4_gemm_t_kernel<OpT, OutT, BM, OCC, true>, p, grid, 256, s);
  return launch(mx4_gemm_t_kernel<OpT, OutT, BM, OCC, false>, p, grid, 256, s);
}

template <typename OpT, typename OutT>
static hipError_t bwd_out(const Mx4Params& p, hipStream_t s) {
  switch (bwd_rows(p.g)) {
    case 64: return tile_t<OpT, OutT, 64, 3>(p, s);
    case 160: return tile_t<OpT, OutT, 160, 2>(p, s);
    default: return tile_t<OpT, OutT, 128, 2>(p, s);
  }
}

template <typename OpT>
static hipError_t bwd(const Mx4Params& p, hipStream_t s) {
  return p.g.out_dtype == kF32 ? bwd_out<OpT, float>(p, s) : bwd_out<OpT, OpT>(p, s);
}

// Output rows in whole aligned 16-byte pieces?
static void finish(Mx4Params& p) {
  const GemmParams& g = p.g;
  const int64_t per = g.out_dtype == kF32 ? 4 : 8;
  p.pieces = g.out == nullptr || g.N % per != 0 || g.out_ld % per != 0 || (reinterpret_cast<uintptr_t>(g.out) & 15) != 0;
  // (134 MB, which the Infinity Cache holds for its reader, 65 us stored and
  // summed, 73 past it; 393 MB 276 and 226: launch_combine_rows)
  p.stream = g.out != nullptr && g.n_routes * g.out_ld * 2 >= kStreamBytes;
  p.dg_vec = g.dg != nullptr && g.dg_x_dtype != kF32 && g.dg_x_ld % 4 == 0 && (reinterpret_cast<uintptr_t>(g.dg_x) & 7) == 0;
}

hipError_t launch_mx4_fwd(const GemmParams& g, const void* codes, const void* scales, const void* a_scales,
                          int32_t op_dtype, hipStream_t stream) {
  Mx4Params p{};
  p.g = g;
  p.codes = (const uint8_t*)codes;
  p.scales = (const uint8_t*)scales;
  p.np = mx4_panels_n(g.N);
  p.kp = mx4_panels_k(g.K);
  finish(p);
  if (a_scales != nullptr) {
    p.a_scales = (const uint8_t*)a_scales;
    p.a_bytes = mx4_row_code_bytes(g.K);
    p.a_groups = mx4_row_scale_bytes(g.K) / 16;
    return op_dtype == kBF16 ? fwd4<bf16_t>(p, stream) : fwd4<f16_t>(p, stream);
  }
  return op_dtype == kBF16 ? fwd16<bf16_t>(p, stream) : fwd16<f16_t>(p, stream);
}

hipError_t launch_mx4_bwd_x(const GemmParams& g, const void* codes, const void* scales, int32_t op_dtype,
                            hipStream_t stream) {
  Mx4Params p{};
  p.g = g;
  p.codes = (const uint8_t*)codes;
  p.scales = (const uint8_t*)scales;
  p.np = mx4_panels_n(g.K);
  p.kp = mx4_panels_k(g.N);
  p.a_div = make_fast_div(g.a_div);
  finish(p);
  return op_dtype == kBF16 ? bwd<bf16_t>(p, stream) : bwd<f16_t>(p, stream);
}

}  // namespace cvmm
