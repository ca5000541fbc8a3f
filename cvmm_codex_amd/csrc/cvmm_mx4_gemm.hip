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

template <typename OpT>
static hipError_t fwd16(const Mx4Params& p, hipStream_t s) {
  const GemmParams& g = p.g;
  if (g.n_routes <= 16 * (int64_t)g.n_experts)
    return launch(mx4_decode_kernel<OpT, 4>, p, mx4_grid<16>(g, p.np), 256, s);
  return launch(mx4_gemm_kernel<OpT, 128, 128, 4, 2>, p, mx4_grid<128>(g, (g.N + 127) / 128), 256, s);
}

template <typename OutT>
static hipError_t fwd4(const Mx4Params& p, hipStream_t s) {
  return launch(mx4_gemm4_kernel<OutT, 128, 128, 4, 2>, p, mx4_grid<128>(p.g, (p.g.N + 127) / 128), 256, s);
}

template <typename OpT>
static hipError_t bwd(const Mx4Params& p, hipStream_t s) {
  const int64_t grid = mx4_grid<128>(p.g, (p.g.N + 127) / 128);
  if (p.g.out_dtype == kF32) return launch(mx4_gemm_t_kernel<OpT, float, 128, 2>, p, grid, 256, s);
  return launch(mx4_gemm_t_kernel<OpT, OpT, 128, 2>, p, grid, 256, s);
}

// Output rows in whole aligned 16-byte pieces?
static void finish(Mx4Params& p) {
  const GemmParams& g = p.g;
  const int64_t per = g.out_dtype == kF32 ? 4 : 8;
  p.pieces = g.out == nullptr || g.N % per != 0 || g.out_ld % per != 0 || (reinterpret_cast<uintptr_t>(g.out) & 15) != 0;
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
  finish(p);
  return op_dtype == kBF16 ? bwd<bf16_t>(p, stream) : bwd<f16_t>(p, stream);
}

}  // namespace cvmm
