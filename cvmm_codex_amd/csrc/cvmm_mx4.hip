// Quantisation to microscaled 4-bit values and back (cvmm_mx4.h: the format
// and its two layouts).  One pass over the data each way: bound by the bytes
// read and written.
#include <cmath>

#include "cvmm_common.h"
#include "cvmm_internal.h"
#include "cvmm_mx4.h"

namespace cvmm {

constexpr int kMx4Threads = 256;

// 8 consecutive values of a row from k on, zeros past K.
template <typename T>
__device__ __forceinline__ void mx4_load8(const T* __restrict__ row, int64_t k, int64_t K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(row + k);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(row[k + i]) : 0.f;
  }
}

__device__ __forceinline__ uint32_t mx4_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Rows: a wave takes 512 values of one row (lane l the 8 from 8 l on, 4 lanes
// a block), so its codes are 256 contiguous bytes.  134 MB of bf16 rows 33 us,
// 5.2 TB/s with the codes (a copy: 5.1).
template <typename T>
__global__ __launch_bounds__(kMx4Threads) void mx4_quantize_rows_kernel(const T* __restrict__ src, int64_t ld,
                                                                        int64_t rows, int64_t K, int64_t k128,
                                                                        int64_t groups, FastDiv by_groups, bool vec,
                                                                        uint8_t* __restrict__ codes,
                                                                        uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * (kMx4Threads / 64) + (threadIdx.x >> 6);
  if (item >= rows * groups) return;
  const int64_t r = by_groups.div(item), g = item - r * groups;
  const int64_t k = g * 512 + lane * 8;
  float v[8];
  mx4_load8<T>(src + r * ld, k, K, vec, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, mx4_abs_bits(v[i]));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));
  const uint32_t sb = mx4_scale_byte(top);
  const uint32_t c = mx4_pack8(v, mx4_scale(sb));
  if (k < k128) *reinterpret_cast<uint32_t*>(codes + r * (k128 / 2) + k / 2) = c;
  // block 4 s + q of the 16 at byte 4 q + s
  const int b = lane >> 2;
  if ((lane & 3) == 0) scales[(r * groups + g) * 16 + (b & 3) * 4 + (b >> 2)] = (uint8_t)sb;
}

template <bool NT, typename T>
__device__ __forceinline__ float mx4_load1(const T* p) {
  if constexpr (!NT) {
    return to_f32(*p);
  } else if constexpr (sizeof(T) == 4) {
    return __builtin_nontemporal_load(reinterpret_cast<const float*>(p));
  } else {
    const uint16_t u = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(p));
    return to_f32(__builtin_bit_cast(T, u));
  }
}

// Keys: a workgroup takes one panel, thread (q, n) the 32 k of block q of
// column n.
// NT: a tensor larger than the Infinity Cache (kStreamBytes) read around the
// caches: 537 MB of fp32 keys 133 -> 102 us, 6.0 TB/s with the codes (a bare
// read reaches 6.5).
template <typename T, bool NT>
__global__ __launch_bounds__(kMx4Threads) void mx4_quantize_keys_kernel(const T* __restrict__ src, int64_t se,
                                                                        int64_t sk, int64_t sn, int64_t K, int64_t N,
                                                                        int64_t np, int64_t kp,
                                                                        uint8_t* __restrict__ codes,
                                                                        uint8_t* __restrict__ scales) {
  const int64_t panel = blockIdx.x;  // (e, n panel, k panel)
  const int64_t pk = panel % kp, en = panel / kp, pn = en % np, e = en / np;
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int64_t n = pn * 64 + c, k0 = pk * 128 + q * 32;
  const T* col = src + e * se + n * sn;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = 0.f;
  if (n < N) {
    if (k0 + 32 <= K) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = mx4_load1<NT>(col + (k0 + i) * sk);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (k0 + i < K) v[i] = to_f32(col[(k0 + i) * sk]);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, mx4_abs_bits(v[i]));
  const uint32_t sb = mx4_scale_byte(top);
  const float scale = mx4_scale(sb);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = v[8 * j + i];
    w[j] = mx4_pack8(u, scale);
  }
  const int tile = c >> 4, lane = q * 16 + (c & 15);
  *reinterpret_cast<uint4*>(codes + panel * kMx4PanelCodes + tile * 1024 + lane * 16) =
      make_uint4(w[0], w[1], w[2], w[3]);
  scales[panel * kMx4PanelScales + lane * 4 + tile] = (uint8_t)sb;
}

template <typename T>
__device__ __forceinline__ void mx4_unpack_to(uint32_t c, float scale, T (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    mx4_unpack8_f32(c, scale, v);
  } else {
    const uint4 u = mx4_unpack8<T>(c, scale);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e[i];
  }
}

// Rows back, into contiguous rows of K values: a wave takes 512 values of a row,
// as above.
template <typename T>
__global__ __launch_bounds__(kMx4Threads) void mx4_dequantize_rows_kernel(const uint8_t* __restrict__ codes,
                                                                          const uint8_t* __restrict__ scales,
                                                                          int64_t rows, int64_t K, int64_t k128,
                                                                          int64_t groups, FastDiv by_groups,
                                                                          T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * (kMx4Threads / 64) + (threadIdx.x >> 6);
  if (item >= rows * groups) return;
  const int64_t r = by_groups.div(item), g = item - r * groups;
  const int64_t k = g * 512 + lane * 8;
  if (k >= K) return;
  const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + r * (k128 / 2) + k / 2);
  const int b = lane >> 2;
  T v[8];
  mx4_unpack_to<T>(c, mx4_scale(scales[(r * groups + g) * 16 + (b & 3) * 4 + (b >> 2)]), v);
  T* dst = out + r * K + k;
  if (K % 8 == 0) {  // (rows and out 16-byte aligned)
    __builtin_memcpy(__builtin_assume_aligned(dst, 16), v, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) dst[i] = v[i];
  }
}

// Keys back, into contiguous [E][K][N]: thread (q, n) writes the 32 k of
// block q of column n.
template <typename T>
__global__ __launch_bounds__(kMx4Threads) void mx4_dequantize_keys_kernel(const uint8_t* __restrict__ codes,
                                                                          const uint8_t* __restrict__ scales,
                                                                          int64_t K, int64_t N, int64_t np, int64_t kp,
                                                                          T* __restrict__ out) {
  const int64_t panel = blockIdx.x;
  const int64_t pk = panel % kp, en = panel / kp, pn = en % np, e = en / np;
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6;
  const int64_t n = pn * 64 + c, k0 = pk * 128 + q * 32;
  if (n >= N) return;
  const int tile = c >> 4, lane = q * 16 + (c & 15);
  const uint4 u = *reinterpret_cast<const uint4*>(codes + panel * kMx4PanelCodes + tile * 1024 + lane * 16);
  const float scale = mx4_scale(scales[panel * kMx4PanelScales + lane * 4 + tile]);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  T* col = out + (e * K + k0) * N + n;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    T v[8];
    mx4_unpack_to<T>(w[j], scale, v);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + 8 * j + i < K) col[(8 * j + i) * N] = v[i];
  }
}

template <typename F>
static void by_dtype(int32_t dt, F&& f) {
  if (dt == kF32) f(float());
  else if (dt == kBF16) f(bf16_t());
  else f(f16_t());
}

hipError_t launch_mx4_quantize_rows(const void* src, int32_t dtype, int64_t ld, int64_t rows, int64_t K, void* codes,
                                    void* scales, hipStream_t stream) {
  if (rows <= 0 || K <= 0) return hipSuccess;
  const int64_t groups = (K + 511) / 512;
  const int64_t blocks = (rows * groups + kMx4Threads / 64 - 1) / (kMx4Threads / 64);
  if (rows * groups > 0x7fffffffll) return hipErrorInvalidValue;
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && (ld * (int64_t)dtype_size(dtype)) % 16 == 0;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((mx4_quantize_rows_kernel<T>), dim3((unsigned)blocks), dim3(kMx4Threads), 0, stream,
                       (const T*)src, ld, rows, K, mx4_k128(K), groups, make_fast_div(groups), vec, (uint8_t*)codes,
                       (uint8_t*)scales);
  });
  return hipGetLastError();
}

hipError_t launch_mx4_quantize_keys(const void* src, int32_t dtype, int64_t se, int64_t sk, int64_t sn, int64_t E,
                                    int64_t K, int64_t N, void* codes, void* scales, hipStream_t stream) {
  const int64_t np = mx4_panels_n(N), kp = mx4_panels_k(K), blocks = E * np * kp;
  if (blocks <= 0) return hipSuccess;
  if (blocks > 0x7fffffffll) return hipErrorInvalidValue;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto kernel = sn == 1 && E * K * N * (int64_t)sizeof(T) >= kStreamBytes ? mx4_quantize_keys_kernel<T, true>
                                                                            : mx4_quantize_keys_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kMx4Threads), 0, stream, (const T*)src, se, sk, sn, K, N,
                       np, kp, (uint8_t*)codes, (uint8_t*)scales);
  });
  return hipGetLastError();
}

hipError_t launch_mx4_dequantize_rows(const void* codes, const void* scales, int64_t rows, int64_t K, void* out,
                                      int32_t dtype, hipStream_t stream) {
  if (rows <= 0 || K <= 0) return hipSuccess;
  const int64_t groups = (K + 511) / 512;
  const int64_t blocks = (rows * groups + kMx4Threads / 64 - 1) / (kMx4Threads / 64);
  if (rows * groups > 0x7fffffffll) return hipErrorInvalidValue;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((mx4_dequantize_rows_kernel<T>), dim3((unsigned)blocks), dim3(kMx4Threads), 0, stream,
                       (const uint8_t*)codes, (const uint8_t*)scales, rows, K, mx4_k128(K), groups, make_fast_div(groups),
                       (T*)out);
  });
  return hipGetLastError();
}

hipError_t launch_mx4_dequantize_keys(const void* codes, const void* scales, int64_t E, int64_t K, int64_t N,
                                      void* out, int32_t dtype, hipStream_t stream) {
  const int64_t np = mx4_panels_n(N), kp = mx4_panels_k(K), blocks = E * np * kp;
  if (blocks <= 0) return hipSuccess;
  if (blocks > 0x7fffffffll) return hipErrorInvalidValue;
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((mx4_dequantize_keys_kernel<T>), dim3((unsigned)blocks), dim3(kMx4Threads), 0, stream,
                       (const uint8_t*)codes, (const uint8_t*)scales, K, N, np, kp, (T*)out);
  });
  return hipGetLastError();
}

}  // namespace cvmm
