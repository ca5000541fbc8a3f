// Microscaled 4-bit values (MX4): blocks of 32 values along one dimension
// share a scale 2^s, s = floor(log2 max|v|) - 2, and each value is the nearest
// of +-{0, .5, 1, 1.5, 2, 3, 4, 6} * 2^s (ties to the even code; beyond 6 * 2^s
// the largest).  A scale is held as the byte s + 127 (s clamped to -127), 255
// marks a block with a NaN or an infinity: all its values are NaN.
//
// Layouts (codes: two per byte, the lower index in the low 4 bits):
//  rows [T][K] in blocks along K, for activations: a row holds K128 / 2 bytes
//    of codes (K128: K up to a multiple of 128) and 16 scale bytes per 512
//    values, [q][s] for the block 4 s + q of the 16 (a lane of the 4-bit
//    product takes the 4 scales of its blocks in one dword);
//  keys [E][K][N] in blocks along K, for expert weights: panels of 64 columns
//    x 128 k, [E][NP][KP] of them (NP = ceil(N / 64), KP = ceil(K / 128)), each
//    4096 bytes of codes, [tile of 16 columns][lane][16 bytes], lane
//    16 q + c holding the 32 k of block q of column c, and 256 bytes of
//    scales, [lane][tile].  A wave reads a panel as the operands of its matrix
//    instructions, 16 bytes per lane and tile.
// Values past K or N are zeros (codes 0).
#pragma once

#include "cvmm_common.h"

namespace cvmm {

inline int64_t mx4_k128(int64_t K) { return (K + 127) / 128 * 128; }
inline int64_t mx4_row_code_bytes(int64_t K) { return mx4_k128(K) / 2; }
inline int64_t mx4_row_scale_bytes(int64_t K) { return (K + 511) / 512 * 16; }
inline int64_t mx4_panels_n(int64_t N) { return (N + 63) / 64; }
inline int64_t mx4_panels_k(int64_t K) { return (K + 127) / 128; }
constexpr int64_t kMx4PanelCodes = 4096, kMx4PanelScales = 256;

// The scale byte of a block whose largest |v| has the float bits `top`.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t top) {
  const uint32_t e = top >> 23;  // biased exponent: 0 below 2^-126
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}
// 2^s as a float, by its byte: the conversions take the scale by its exponent
// bits, of which 0 stands for 2^-127 (a subnormal) and 255 for NaN.
__device__ __forceinline__ float mx4_scale(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
}

// 8 values to 8 codes.  The hardware conversion divides by the scale, rounds
// to the nearest code, ties to even, and keeps what lies beyond at 6.
__device__ __forceinline__ uint32_t mx4_pack8(const float (&v)[8], float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  return c;
}

typedef __bf16 mx4_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 mx4_f16x2 __attribute__((ext_vector_type(2)));
typedef float mx4_f32x2 __attribute__((ext_vector_type(2)));

// 8 codes to 8 values of a 16-bit type, exact where they are normal or
// subnormal numbers of it (bf16: always up to 3.4e38; fp16: values below 2^-25
// become 0 and from 65520 on infinities, as in a cast of the weights).
template <typename T> __device__ __forceinline__ uint4 mx4_unpack8(uint32_t c, float scale);
template <> __device__ __forceinline__ uint4 mx4_unpack8<bf16_t>(uint32_t c, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3)));
}
template <> __device__ __forceinline__ uint4 mx4_unpack8<f16_t>(uint32_t c, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3)));
}
__device__ __forceinline__ void mx4_unpack8_f32(uint32_t c, float scale, float (&v)[8]) {
  const mx4_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0);
  const mx4_f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
  const mx4_f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2);
  const mx4_f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
  v[4] = d[0]; v[5] = d[1]; v[6] = e[0]; v[7] = e[1];
}

}  // namespace cvmm
