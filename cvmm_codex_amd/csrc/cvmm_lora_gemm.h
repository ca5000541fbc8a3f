// The projection with its rows' adapters in 16-bit operands of whole 16-byte
// pieces (cvmm_lora.h): a plain GEMM whose accumulators start from base and take,
// after the shared weights' k slices, a slice of 32 inner values of each adapter
// that occurs in the tile.
//
// A workgroup of four waves owns BM rows x BN columns; a wave MI x NJ blocks of
// 16 x 16.  Slices of 32 k (64-byte row pieces of x, 64-byte pieces or whole rows
// of W, by which of its strides is 1) go by buffer loads straight into a ring of
// four LDS buffers, three in flight while one is multiplied; the fragments of
// slice s + 1 are read while the products of slice s run.  Every slice is the
// same number of loads, those past the last k included (offsets past the
// descriptor's range read zeros), so every wait is an exact vmcnt.  Operands are
// swapped (C^T = W^T x^T): a lane ends with 4 consecutive columns of one row, 8
// after two lane swaps, stored as one 16-byte write.
//
// Adapters: the tile walks the adapters of its rows by rising id.  A block of 16
// rows that all have the adapter takes its product in its accumulators; one that
// has it in some rows forms it apart and adds it where it belongs (no product
// with zero: infinities of one request's adapter stay with its rows); others skip
// it.  Rows of a request stand together, so nearly all blocks are of the first or
// the last kind, and the adapters' slices cost what they add: rank / 32 slices
// beside K / 32.
#pragma once

#include <type_traits>
#include <utility>

#include "cvmm_lora_rows.h"

namespace cvmm {

// A buffer offset that reads zeros, and the descriptors' range (cvmm_topk_gemm.hip
// says why): 2^31.  The bases sit kLoraBack before the data: instruction j's
// immediate 1024 (j % 4) moves the LDS address and the memory's, and is taken off
// the lane's offset.
constexpr uint32_t kLoraOob = 0x80000000u;
constexpr uint32_t kLoraBack = 4096;

template <typename F, int... I>
__device__ __forceinline__ void static_for_seq(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_seq(f, std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t lora_rsrc(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)(reinterpret_cast<const char*>(p) - kLoraBack), (short)0,
                                           (int)kLoraOob, kBufferRsrcWord3);
}

template <int N>
__device__ __forceinline__ void lora_wait(lds_u32x4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}
template <int N>
__device__ __forceinline__ void lora_wait(lds_u32x2 (&x)[N][2]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i][0]), "+v"(x[i][1]));
}
__device__ __forceinline__ uint4 lora_frag(const lds_u32x4& v) { return make_uint4(v.x, v.y, v.z, v.w); }
__device__ __forceinline__ uint4 lora_frag(const lds_u32x2 (&v)[2]) {
  return make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
}

template <int MI, int NJ, int WMW, int WNW>
struct LoraTile {
  static_assert(WMW * WNW == 4, "four waves");
  static constexpr int BM = 16 * MI * WMW, BN = 16 * NJ * WNW;
  static constexpr int A_INSTS = BM / 16, B_INSTS = BN / 16;  // 1 KB each
  static_assert((A_INSTS + B_INSTS) % 4 == 0, "whole instructions per wave");
  static constexpr int D = (A_INSTS + B_INSTS) / 4;
  static constexpr int A_BYTES = BM * 64, SLICE = (BM + BN) * 64, STAGES = 4;
  static constexpr int OCC = MI * NJ > 16 ? 1 : 2;
};

// Lane offsets of a slice's B half.  KC: [n][k] pieces, as the A half; else [k][n]
// rows of BN columns, read back transposed.
template <bool KC, int BN>
__device__ __forceinline__ void lora_b_lane(int inst, int lane, int64_t sk, int64_t sn, int64_t cols, uint32_t& off,
                                            int& k) {
  if constexpr (KC) {
    const int n = inst * 16 + (lane >> 2), c = (lane & 3) ^ ((n >> 1) & 3);
    k = c * 8;
    off = n < cols ? (uint32_t)(n * sn * 2) + (uint32_t)c * 16 + kLoraBack : kLoraOob;
  } else {
    constexpr int CPR = BN / 8;
    const int q = inst * 64 + lane, row = q / CPR, c = (q % CPR) ^ tr_row_swz<CPR>(row);
    k = row;
    off = c * 8 < cols ? (uint32_t)(row * sk * 2) + (uint32_t)c * 16 + kLoraBack : kLoraOob;
  }
}

template <typename OpT, int MI, int NJ, int WMW, int WNW, bool WKC, bool BKC, bool SPLIT>
__global__ __launch_bounds__(256, (LoraTile<MI, NJ, WMW, WNW>::OCC)) void lora_gemm_kernel(const LoraParams p,
                                                                                           const LoraSplit sp) {
  using T = LoraTile<MI, NJ, WMW, WNW>;
  constexpr int BM = T::BM, BN = T::BN, D = T::D, SLICE = T::SLICE;
  __shared__ __attribute__((aligned(1024))) char ring[T::STAGES * SLICE];
  __shared__ int32_t s_row[BM], s_id[BM];

  if constexpr (SPLIT) {
    if (blockIdx.x >= sp.gemm_blocks) {
      lora_inner_row<OpT>(p, sp, blockIdx.x - sp.gemm_blocks, reinterpret_cast<float*>(ring));
      return;
    }
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WNW, wn = wave % WNW;
  const int fr = lane & 15, fq = lane >> 4;
  const uint32_t tiles_n = (uint32_t)((p.N + BN - 1) / BN);
  uint32_t id = xcd_remap((uint32_t)blockIdx.x, SPLIT ? sp.gemm_blocks : (uint32_t)gridDim.x);
  int64_t k_lo = 0, k_hi = p.w != nullptr ? p.K : 0;
  uint32_t split = 0;
  if constexpr (SPLIT) {
    split = id % (uint32_t)sp.splits;
    id /= (uint32_t)sp.splits;
    k_lo = (int64_t)split * sp.slices * 32;
    k_hi = k_lo + (int64_t)sp.slices * 32 < p.K ? k_lo + (int64_t)sp.slices * 32 : p.K;
  }
  const int64_t m0 = (int64_t)(id / tiles_n) * BM, n0 = (int64_t)(id % tiles_n) * BN;

  for (int i = tid; i < BM; i += 256) {
    const int64_t m = m0 + i;
    int64_t row = m < p.rows ? (p.order != nullptr ? p.order[m] : m) : -1;
    if (row < 0 || row >= p.rows) row = -1;
    s_row[i] = (int32_t)row;
    if constexpr (!SPLIT) s_id[i] = row >= 0 ? lora_id(p, row) : -1;
  }
  __syncthreads();

  // ---- sources of this wave's loads: instruction g = wave * D + j fills 1 KB of
  // the slice, A rows first
  // (without an order x is addressed from the tile's first row)
  const int64_t first = p.order != nullptr ? 0 : m0;
  const __amdgpu_buffer_rsrc_t ra = lora_rsrc(reinterpret_cast<const OpT*>(p.x) + first * p.x_ld + k_lo);
  const __amdgpu_buffer_rsrc_t rw = lora_rsrc(reinterpret_cast<const OpT*>(p.w) + n0 * p.w_sn + k_lo * p.w_sk);
  uint32_t off[D];
  int kc[D];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int g = wave * D + j;
    if (g < T::A_INSTS) {
      const int r = g * 16 + (lane >> 2), c = (lane & 3) ^ ((r >> 1) & 3);
      const int32_t row = s_row[r];
      kc[j] = c * 8;
      off[j] = row >= 0 ? (uint32_t)(((int64_t)row - first) * p.x_ld * 2) + (uint32_t)c * 16 + kLoraBack : kLoraOob;
    } else {
      lora_b_lane<WKC, BN>(g - T::A_INSTS, lane, p.w_sk, p.w_sn, p.N - n0, off[j], kc[j]);
    }
    if (off[j] != kLoraOob) off[j] -= 1024u * (uint32_t)(j & 3);
  }
  const int32_t kw = (int32_t)(k_hi - k_lo);
  const uint32_t b_step = (uint32_t)((WKC ? 1 : p.w_sk) * 64);  // bytes a slice moves W by
  auto issue_one = [&](auto jc, __amdgpu_buffer_rsrc_t rsa, __amdgpu_buffer_rsrc_t rsb, uint32_t o, uint32_t sa,
                       uint32_t sb, char* dst) {
    constexpr int J = decltype(jc)::value;
    const bool is_a = wave * D + J < T::A_INSTS;
    buf_dma<16, (J & 3) * 1024>(is_a ? rsa : rsb, o, is_a ? sa : sb, dst + (wave * D + (J & ~3)) * 1024);
  };
  int32_t i_k = 0;       // k of the slice to be issued, and its offsets
  uint32_t i_a = 0, i_b = 0;
  auto issue_part = [&](auto jc, char* dst) {
    constexpr int J = decltype(jc)::value;
    issue_one(jc, ra, rw, i_k + kc[J] < kw ? off[J] : kLoraOob, i_a, i_b, dst);
  };
  auto issue_next = [&]() {
    i_k += 32;
    i_a += 64;
    i_b += b_step;
    if (i_k >= kw) i_a = i_b = 0;  // (only offsets past the range from here on)
  };

  // ---- fragments
  const uint32_t st0 = lds_addr(ring);
  const uint32_t a_f = st0 + (uint32_t)((wm * MI * 16 + fr) * 64 + ((fq ^ ((fr >> 1) & 3)) << 4));
  uint32_t kc_f, tr_f[NJ];
  kc_f = st0 + T::A_BYTES + (uint32_t)((wn * NJ * 16 + fr) * 64 + ((fq ^ ((fr >> 1) & 3)) << 4));
  {
    constexpr int CPR = BN / 8;
    const int r = fq * 8 + (fr >> 2);
    const int lo = ((fr & 1) << 3) + (((fr >> 1) & 1) << 4);
#pragma unroll
    for (int i = 0; i < NJ; ++i)
      tr_f[i] = st0 + T::A_BYTES + (uint32_t)(r * BN * 2 + lo + (((wn * NJ * 2 + 2 * i) ^ tr_row_swz<CPR>(r)) << 4));
  }
  auto read_a = [&](uint32_t at, lds_u32x4 (&f)[MI]) {
    static_for<MI>([&](auto i) { f[i] = lds_read128_at<decltype(i)::value * 1024>(a_f + at); });
  };
  auto read_b = [&](uint32_t at, auto& f) {
    if constexpr (std::is_same_v<std::remove_reference_t<decltype(f)>, lds_u32x4[NJ]>) {
      static_for<NJ>([&](auto i) { f[i] = lds_read128_at<decltype(i)::value * 1024>(kc_f + at); });
    } else {
#pragma unroll
      for (int i = 0; i < NJ; ++i) {
        f[i][0] = lds_read_tr<0>(tr_f[i] + at);
        f[i][1] = lds_read_tr<4 * BN * 2>(tr_f[i] + at);
      }
    }
  };

  // ---- accumulators, from base: acc[j][i] holds columns 16 j + 4 fq + {0..3} of row 16 i + fr
  f32x4_t acc[NJ][MI];
  const int64_t nw = n0 + wn * NJ * 16;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if constexpr (!SPLIT) {
    if (p.base != nullptr) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int64_t row = s_row[(wm * MI + i) * 16 + fr];
        if (row < 0) continue;
        const int64_t at = row * p.base_ld;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int64_t n = nw + j * 16 + 4 * fq;
          if (n + 4 <= p.n_out && p.base_vec) {
            if (p.base_dtype == kF32) {
              const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.base) + at + n);
              acc[j][i] = f32x4_t{v.x, v.y, v.z, v.w};
            } else {
              const uint2 raw = *reinterpret_cast<const uint2*>(reinterpret_cast<const OpT*>(p.base) + at + n);
              const OpT* v = reinterpret_cast<const OpT*>(&raw);
              acc[j][i] = f32x4_t{to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3])};
            }
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (n + v < p.n_out) acc[j][i][v] = load_as_f32(p.base, p.base_dtype, at + n + v);
          }
        }
      }
    }
  }

  // ---- the shared weights
  using WFrag = std::conditional_t<WKC, lds_u32x4[NJ], lds_u32x2[NJ][2]>;
  const int32_t S = (kw + 31) / 32;
  if (S > 0) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      static_for<D>([&](auto j) { issue_part(j, ring + s * SLICE); });
      issue_next();
      issue_fence();
    }
    lds_u32x4 a0[MI], a1[MI];
    WFrag b0, b1;
    vm_wait<3 * D>();
    lds_barrier();
    read_a(0, a0);
    read_b(0, b0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    lora_wait(a0);
    lora_wait(b0);
    int buf = 0;
    // slice s is in (ca, cb): slice s + 1 is read into (na, nb), slice s + 4
    // issued into the buffer of s, which every wave has read
    auto step = [&](lds_u32x4 (&ca)[MI], WFrag& cb, lds_u32x4 (&na)[MI], WFrag& nb) {
      const int nbuf = (buf + 1) & 3;
      vm_wait<2 * D>();
      lds_barrier();
      char* dst = ring + buf * SLICE;
      read_a((uint32_t)nbuf * SLICE, na);
      read_b((uint32_t)nbuf * SLICE, nb);
      static_for<NJ>([&](auto jb) {
        constexpr int JB = decltype(jb)::value;
        const uint4 w = lora_frag(cb[JB]);
#pragma unroll
        for (int i = 0; i < MI; ++i) MfmaOp<OpT>::step(acc[JB][i], w, lora_frag(ca[i]));
        static_for<D>([&](auto j) {
          if constexpr (decltype(j)::value * NJ / D == JB) issue_part(j, dst);
        });
        __builtin_amdgcn_sched_barrier(0);
      });
      issue_next();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      lora_wait(na);
      lora_wait(nb);
      buf = nbuf;
    };
    // in pairs; an odd count gets a slice of zeros
    for (int32_t s = 0; s < S; s += 2) {
      step(a0, b0, a1, b1);
      step(a1, b1, a0, b0);
    }
    vm_wait<0>();
  }

  if constexpr (SPLIT) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int32_t row = s_row[(wm * MI + i) * 16 + fr];
      if (row < 0) continue;
      float* dst = sp.part + ((int64_t)split * p.rows + row) * sp.part_ld;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int64_t n = nw + j * 16 + 4 * fq;
        if (n < p.N)
          *reinterpret_cast<float4*>(dst + n) = make_float4(acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]);
      }
    }
    return;
  }

  // ---- the adapters of the tile's rows
  using BFrag = std::conditional_t<BKC, lds_u32x4[NJ], lds_u32x2[NJ][2]>;
  int32_t ids[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) ids[i] = s_id[(wm * MI + i) * 16 + fr];
  const __amdgpu_buffer_rsrc_t rh = lora_rsrc(reinterpret_cast<const OpT*>(p.h) + first * p.h_ld);
  uint32_t hoff[D];
  int hk[D];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int g = wave * D + j;
    if (g < T::A_INSTS) {
      const int r = g * 16 + (lane >> 2), c = (lane & 3) ^ ((r >> 1) & 3);
      const int32_t row = s_row[r];
      hk[j] = 0;  // (zeros up to h_ld)
      hoff[j] = row >= 0 ? (uint32_t)(((int64_t)row - first) * p.h_ld * 2) + (uint32_t)c * 16 + kLoraBack : kLoraOob;
    } else {
      lora_b_lane<BKC, BN>(g - T::A_INSTS, lane, p.b_sr, p.b_sn, p.N - n0, hoff[j], hk[j]);
    }
    if (hoff[j] != kLoraOob) hoff[j] -= 1024u * (uint32_t)(j & 3);
  }
  const int32_t rank = (int32_t)p.rank;
  const uint32_t hb_step = (uint32_t)((BKC ? 1 : p.b_sr) * 64);
  for (int32_t cur = -1;;) {
    int32_t a = INT32_MAX;
#pragma unroll
    for (int i = 0; i < BM / 64; ++i) {
      const int32_t v = s_id[i * 64 + lane];
      a = v > cur && v < a ? v : a;
    }
    a = wave_min_i32(a);  // the same in every wave
    if (a == INT32_MAX) break;
    cur = a;
    const __amdgpu_buffer_rsrc_t rb = lora_rsrc(reinterpret_cast<const OpT*>(p.b) + a * p.b_se + n0 * p.b_sn);
    for (int32_t r0 = 0; r0 < rank; r0 += 128) {  // four slices at a time
      lds_barrier();                              // the buffers' last reads
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int32_t k = r0 + s * 32;
        if (k < rank)
          static_for<D>([&](auto j) {
            constexpr int J = decltype(j)::value;
            issue_one(j, rh, rb, k + hk[J] < rank ? hoff[J] : kLoraOob, (uint32_t)k * 2,
                      (uint32_t)(k / 32) * hb_step, ring + s * SLICE);
          });
      }
      vm_wait<0>();
      lds_barrier();
      for (int s = 0; s < 4 && r0 + s * 32 < rank; ++s) {
        lds_u32x4 af[MI];
        BFrag bf;
        read_a((uint32_t)s * SLICE, af);
        read_b((uint32_t)s * SLICE, bf);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        lora_wait(af);
        lora_wait(bf);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const bool mine = ids[i] == a;
          const uint64_t in = __ballot(mine);
          if (in == 0) continue;
          if (in == ~0ull) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) MfmaOp<OpT>::step(acc[j][i], lora_frag(bf[j]), lora_frag(af[i]));
          } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              f32x4_t t{0.f, 0.f, 0.f, 0.f};
              MfmaOp<OpT>::step(t, lora_frag(bf[j]), lora_frag(af[i]));
#pragma unroll
              for (int v = 0; v < 4; ++v) acc[j][i][v] = mine ? acc[j][i][v] + t[v] : acc[j][i][v];
            }
          }
        }
      }
    }
  }

  // ---- stores
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t row = s_row[(wm * MI + i) * 16 + fr];
    OpT* dst = reinterpret_cast<OpT*>(p.out) + row * p.out_ld;
#pragma unroll
    for (int pr = 0; pr < NJ / 2; ++pr) {
      uint32_t a[2], b[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        union { uint32_t u; OpT e[2]; } pa, pb;
        pa.e[0] = from_f32<OpT>(acc[2 * pr][i][2 * h]);
        pa.e[1] = from_f32<OpT>(acc[2 * pr][i][2 * h + 1]);
        pb.e[0] = from_f32<OpT>(acc[2 * pr + 1][i][2 * h]);
        pb.e[1] = from_f32<OpT>(acc[2 * pr + 1][i][2 * h + 1]);
        a[h] = pa.u;
        b[h] = pb.u;
      }
      const auto s0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
      const auto s1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
      const auto u0 = __builtin_amdgcn_permlane16_swap(s0[0], s0[1], false, false);
      const auto u1 = __builtin_amdgcn_permlane16_swap(s1[0], s1[1], false, false);
      const int64_t n = nw + pr * 32 + 8 * fq;
      if (row < 0 || n >= p.n_out) continue;
      const uint4 v = make_uint4(u0[0], u1[0], u0[1], u1[1]);
      if (p.out_vec) {
        *reinterpret_cast<uint4*>(dst + n) = v;
      } else {
        const OpT* e = reinterpret_cast<const OpT*>(&v);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (n + q < p.n_out) dst[n + q] = e[q];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// launchers of one op type (cvmm_lora_bf16.hip, cvmm_lora_f16.hip)
// ---------------------------------------------------------------------------
template <typename OpT, bool WKC, bool BKC>
hipError_t launch_lora_gemm_kc(const LoraParams& p, hipStream_t s) {
  auto tiles = [&](int64_t bm, int64_t bn) { return ((p.rows + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  auto go = [&](auto mi, auto nj, auto wm, auto wn) {
    constexpr int MI = decltype(mi)::value, NJ = decltype(nj)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    using T = LoraTile<MI, NJ, WM, WN>;
    const int64_t n = tiles(T::BM, T::BN);
    if (n > 0x7fffffffll) return hipErrorInvalidValue;
    hipLaunchKernelGGL((lora_gemm_kernel<OpT, MI, NJ, WM, WN, WKC, BKC, false>), dim3((unsigned)n), dim3(256), 0, s, p,
                       LoraSplit{});
    return hipGetLastError();
  };
  using std::integral_constant;
  using i2 = integral_constant<int, 2>;
  using i4 = integral_constant<int, 4>;
  using i8 = integral_constant<int, 8>;
  if (tiles(256, 256) >= 192) return go(i8(), i8(), i2(), i2());
  if (tiles(128, 128) >= 192) return go(i4(), i4(), i2(), i2());
  return go(i2(), i4(), i2(), i2());
}

template <typename OpT>
hipError_t launch_lora_gemm_op(const LoraParams& p, hipStream_t s) {
  const bool wkc = p.w != nullptr && p.w_sn != 1, bkc = p.b_sn != 1;
  if (wkc) return bkc ? launch_lora_gemm_kc<OpT, true, true>(p, s) : launch_lora_gemm_kc<OpT, true, false>(p, s);
  return bkc ? launch_lora_gemm_kc<OpT, false, true>(p, s) : launch_lora_gemm_kc<OpT, false, false>(p, s);
}

template <typename OpT>
hipError_t launch_lora_inner_op(const LoraParams& p, hipStream_t s) {
  const bool akc = p.a_sr != 1;
  auto go = [&](auto rb, auto kw) {
    constexpr int RB = decltype(rb)::value, KW = decltype(kw)::value;
    const int64_t wg = (p.rows + (KW == 1 ? 63 : 15)) / (KW == 1 ? 64 : 16);
    if (akc)
      hipLaunchKernelGGL((lora_inner_tile_kernel<OpT, RB, KW, true>), dim3((unsigned)wg), dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((lora_inner_tile_kernel<OpT, RB, KW, false>), dim3((unsigned)wg), dim3(256), 0, s, p);
  };
  auto by_rank = [&](auto kw) {
    using std::integral_constant;
    if (p.rank <= 16) go(integral_constant<int, 1>(), kw);
    else if (p.rank <= 32) go(integral_constant<int, 2>(), kw);
    else if (p.rank <= 64) go(integral_constant<int, 4>(), kw);
    else if (p.rank <= 128) go(integral_constant<int, 8>(), kw);
    else go(integral_constant<int, 16>(), kw);
  };
  if (p.rows >= 8192) by_rank(std::integral_constant<int, 1>());
  else by_rank(std::integral_constant<int, 4>());
  return hipGetLastError();
}

template <typename OpT>
hipError_t launch_lora_few_op(const LoraParams& p, const LoraSplit& sp, hipStream_t s) {
  const uint32_t row_blocks = (uint32_t)(p.rows * sp.h_splits);
  if (p.w == nullptr) {
    hipLaunchKernelGGL((lora_inner_row_kernel<OpT>), dim3(row_blocks), dim3(256), 0, s, p, sp);
  } else {
    const dim3 grid(sp.gemm_blocks + row_blocks);
    if (p.w_sn == 1)
      hipLaunchKernelGGL((lora_gemm_kernel<OpT, 2, 4, 2, 2, false, false, true>), grid, dim3(256), 0, s, p, sp);
    else
      hipLaunchKernelGGL((lora_gemm_kernel<OpT, 2, 4, 2, 2, true, false, true>), grid, dim3(256), 0, s, p, sp);
  }
  hipLaunchKernelGGL((lora_join_kernel<OpT>),
                     dim3((unsigned)((p.n_out + kLoraJoinThreads * 4 - 1) / (kLoraJoinThreads * 4)), (unsigned)p.rows),
                     dim3(kLoraJoinThreads), 0, s, p, sp);
  return hipGetLastError();
}

template <typename OpT>
hipError_t launch_lora_wgrad_op(const LoraWgradParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.d_in + 127) / 128 + (p.d_out + 127) / 128), (unsigned)((p.rank + 63) / 64),
                  (unsigned)(p.n * p.shares));
  if (p.rank <= 16) hipLaunchKernelGGL((lora_wgrad_fast_kernel<OpT, 1>), grid, dim3(256), 0, s, p);
  else if (p.rank <= 32) hipLaunchKernelGGL((lora_wgrad_fast_kernel<OpT, 2>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((lora_wgrad_fast_kernel<OpT, 4>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace cvmm
