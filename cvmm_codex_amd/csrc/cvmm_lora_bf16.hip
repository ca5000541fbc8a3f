// Low-rank adapters with bf16_t operands (cvmm_lora_gemm.h, cvmm_lora_rows.h).
#include "cvmm_lora_gemm.h"

namespace cvmm {
template hipError_t launch_lora_gemm_op<bf16_t>(const LoraParams& p, hipStream_t s);
template hipError_t launch_lora_inner_op<bf16_t>(const LoraParams& p, hipStream_t s);
template hipError_t launch_lora_few_op<bf16_t>(const LoraParams& p, const LoraSplit& sp, hipStream_t s);
template hipError_t launch_lora_wgrad_op<bf16_t>(const LoraWgradParams& p, hipStream_t s);
}  // namespace cvmm
