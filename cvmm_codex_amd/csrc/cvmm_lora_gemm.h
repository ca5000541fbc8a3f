// The projection with its rows' adapters in 16-bit operands of whole 16-byte
// pieces (cvmm_lora.h): a plain GEMM whose accumulators start from base and take,
// after the shared weights' k slices, a slice of 32 inner values of each adapter
// that occurs in the tile.
//
// A workgroup of four waves owns BM rows x BN columns; a wave MI x NJ blocks of
// 16 x 16.  Slices of 64 k (128-byte row pieces of x: whole lines; such pieces or
// whole rows of W, by which of its strides is 1) go by buffer loads straight into a
// ring of LDS buffers; the fragments of one half of a slice are read while the
// products of the other run.  Every slice is the same number of loads, those past
// the last k included (offsets past the descriptor's range read zeros), so every
// wait is an exact vmcnt.  Operands are
// swapped (C^T = W^T x^T): a lane ends with 4 consecutive columns of one row, 8
// after two lane swaps, stored as one 16-byte write.
//
// Adapters: the tile walks the adapters of its rows by rising id, each a product
// of the rows' inner values, zero in the rows of others, with B_i's columns.  Rows
// of a request stand together, so most tiles have one, and the adapters cost rank /
// 32 slices beside K / 32.  Zero times an infinity or a NaN would carry one
// request's to another's rows: where a tile has several adapters such values of
// B_i are left out, and added to their own rows after the stores.  (Chosen per
// element of the accumulators instead, 256 of them through branches, the compiler
// spilled: 800 us against 130 for 16384 rows of 2048 -> 2048.)
//
// Measured, bf16: 16384 rows, 2048 -> 2048, rank 64: 121-135 us (146 GFLOP: 1.08-1.21
// PFLOP/s; the library's product without adapters 113).  Bound by the matrix pipe,
// busy for 60 % of the cycles: a further 2048 k cost 1.4 PFLOP/s, but each round of
// tiles starts with an empty ring and ends with its CU's stores, 11 us together.
// 8192 rows, 1024 -> 1024, rank 16: 24.6 (library 23.2), each way.
// Without W, 16384 rows of 1024 with base, rank 16: 22.9, 67 MB at 2.9 TB/s: a tile
// is a chain of loads (order, id, inner row) before its stores.
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

// Infinities and NaN of a fragment's 16-bit values -> 0; dropped: there were some.
template <typename OpT>
__device__ __forceinline__ uint32_t lora_finite_pair(uint32_t v, bool& dropped) {
  constexpr uint32_t kExp = DTypeOf<OpT>::value == kBF16 ? 0x7f80u : 0x7c00u;
  const bool lo = (v & kExp) == kExp, hi = (v & (kExp << 16)) == (kExp << 16);
  dropped |= lo | hi;
  return (lo ? 0u : v & 0xffffu) | (hi ? 0u : v & 0xffff0000u);
}
template <typename OpT, int N>
__device__ __forceinline__ void lora_finite(lds_u32x4 (&f)[N], bool& dropped) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) f[i][q] = lora_finite_pair<OpT>(f[i][q], dropped);
}
template <typename OpT, int N>
__device__ __forceinline__ void lora_finite(lds_u32x2 (&f)[N][2], bool& dropped) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) f[i][q / 2][q % 2] = lora_finite_pair<OpT>(f[i][q / 2][q % 2], dropped);
}

// c += w x^T.  AGPR: in accumulation registers by name.  Of 256 accumulators the
// compiler moved 200 to other registers and back in every slice, as many
// instructions as the matrix unit leaves room for.  It does not see a matrix
// instruction here: lora_mfma_ready comes before the first of a slice, whose operands
// vector instructions may have written (two wait states), and lora_mfma_done before
// an accumulator is read.
template <typename OpT, bool AGPR>
__device__ __forceinline__ void lora_mfma_one(f32x4_t& c, const uint4& w, const lds_u32x4& x) {
  if constexpr (!AGPR) {
    MfmaOp<OpT>::step(c, w, make_uint4(x.x, x.y, x.z, x.w));
  } else {
    const lds_u32x4 a{w.x, w.y, w.z, w.w};
    if constexpr (DTypeOf<OpT>::value == kBF16)
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(x));
    else
      asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(x));
  }
}
// Operands that vector instructions made, in their registers from here on.
template <int N, int M>
__device__ __forceinline__ void lora_operands(uint4 (&w)[N], lds_u32x4 (&x)[M]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    lds_u32x4 v{w[i].x, w[i].y, w[i].z, w[i].w};
    asm volatile("" : "+v"(v));
    w[i] = make_uint4(v.x, v.y, v.z, v.w);
  }
#pragma unroll
  for (int i = 0; i < M; ++i) asm volatile("" : "+v"(x[i]));
}
__device__ __forceinline__ void lora_mfma_ready() { asm volatile("s_nop 1" ::: "memory"); }
// After the last of them: more wait states than the last result needs before a
// vector instruction reads it, and every accumulator handed on, so that no read of
// one comes earlier.
template <int NJ, int MI>
__device__ __forceinline__ void lora_mfma_done(f32x4_t (&c)[NJ][MI]) {
  asm volatile("s_nop 15\n\ts_nop 15" : "+a"(c[0][0]));
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) asm volatile("" : "+a"(c[j][i]));
}

template <int MI, int NJ, int WMW, int WNW, int STAGES_>
struct LoraTile {
  static_assert(WMW * WNW == 4, "four waves");
  static constexpr int BM = 16 * MI * WMW, BN = 16 * NJ * WNW, STAGES = STAGES_;
  static constexpr int A_INSTS = BM / 8, B_INSTS = BN / 8;  // 1 KB each
  static_assert((A_INSTS + B_INSTS) % 4 == 0, "whole instructions per wave");
  static constexpr int D = (A_INSTS + B_INSTS) / 4;
  static constexpr int A_BYTES = BM * 128, SLICE = (BM + BN) * 128;
  static constexpr int LDS = STAGES * SLICE + BM * 8;
  static constexpr int OCC = MI * NJ > 16 || LDS > 80 * 1024 ? 1 : 2;
  static constexpr bool AGPR = MI * NJ == 64;
  static constexpr bool MIXED = A_INSTS % D != 0;  // a wave loads pieces of x and of W
  static_assert(STAGES >= 1 && STAGES * D < 64, "vmcnt range");
};

// Lane offset of load `inst` of a slice's B half, and the k that its piece starts
// at.  KC: [n][k] pieces, as the A half; else [k][n] rows of BN columns, read back
// transposed.
__device__ __forceinline__ int lora_chunk(int lane) { return (lane & 7) ^ ((lane >> 3) & 7); }
template <bool KC, int BN>
__device__ __forceinline__ uint32_t lora_b_off(int inst, int lane, int64_t sk, int64_t sn, int64_t cols) {
  if constexpr (KC) {
    const int n = inst * 8 + (lane >> 3);
    return n < cols ? (uint32_t)(n * sn * 2) + (uint32_t)lora_chunk(lane) * 16 + kLoraBack : kLoraOob;
  } else {
    constexpr int CPR = BN / 8;
    const int row = inst * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ tr_row_swz<CPR>(row);
    return c * 8 < cols ? (uint32_t)(row * sk * 2) + (uint32_t)c * 16 + kLoraBack : kLoraOob;
  }
}
template <bool KC, int BN>
__device__ __forceinline__ int lora_b_k(int inst, int lane) {
  constexpr int CPR = BN / 8;
  if constexpr (KC) return lora_chunk(lane) * 8;
  else return inst * (64 / CPR) + lane / CPR;
}

template <typename OpT, int MI, int NJ, int WMW, int WNW, int STAGES, bool WKC, bool BKC, bool SPLIT>
__global__ __launch_bounds__(256, (LoraTile<MI, NJ, WMW, WNW, STAGES>::OCC)) void lora_gemm_kernel(
    const LoraParams p, const LoraSplit sp) {
  using T = LoraTile<MI, NJ, WMW, WNW, STAGES>;
  constexpr int BM = T::BM, BN = T::BN, D = T::D, SLICE = T::SLICE;
  __shared__ __attribute__((aligned(1024))) char ring[STAGES * SLICE];
  __shared__ int32_t s_row[BM], s_id[BM];
  static_assert(BM <= 256, "a row per thread");

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
    k_lo = (int64_t)split * sp.slices * 64;
    k_hi = k_lo + (int64_t)sp.slices * 64 < p.K ? k_lo + (int64_t)sp.slices * 64 : p.K;
  }
  const int64_t m0 = (int64_t)(id / tiles_n) * BM, n0 = (int64_t)(id % tiles_n) * BN;

  // the tile's rows; their ids are in flight until the projection is done
  int64_t my_row = -1, my_id = -1;
  if (tid < BM) {
    const int64_t m = m0 + tid;
    my_row = m < p.rows ? (p.order != nullptr ? p.order[m] : m) : -1;
    if (my_row < 0 || my_row >= p.rows) my_row = -1;
    s_row[tid] = (int32_t)my_row;
    if (!SPLIT && my_row >= 0)
      my_id = p.ids_is_int64 ? ((const int64_t*)p.ids)[my_row] : (int64_t)((const int32_t*)p.ids)[my_row];
  }
  lds_barrier();

  // ---- sources of this wave's loads: instruction g = wave * D + j fills 1 KB of
  // the slice, A rows first
  // (without an order x is addressed from the tile's first row)
  const int64_t first = p.order != nullptr ? 0 : m0;
  const __amdgpu_buffer_rsrc_t ra = lora_rsrc(reinterpret_cast<const OpT*>(p.x) + first * p.x_ld + k_lo);
  const __amdgpu_buffer_rsrc_t rw = lora_rsrc(reinterpret_cast<const OpT*>(p.w) + n0 * p.w_sn + k_lo * p.w_sk);
  const int a_k = lora_chunk(lane) * 8;  // the k that a lane's pieces of x start at
  uint32_t off[D];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int g = wave * D + j;
    if (g < T::A_INSTS) {
      const int32_t row = s_row[g * 8 + (lane >> 3)];
      off[j] = row >= 0 ? (uint32_t)(((int64_t)row - first) * p.x_ld * 2) + (uint32_t)a_k * 2 + kLoraBack : kLoraOob;
    } else {
      off[j] = lora_b_off<WKC, BN>(g - T::A_INSTS, lane, p.w_sk, p.w_sn, p.N - n0);
    }
    if (off[j] != kLoraOob) off[j] -= 1024u * (uint32_t)(j & 3);
  }
  const int32_t kw = (int32_t)(k_hi - k_lo);
  const uint32_t b_step = (uint32_t)((WKC ? 1 : p.w_sk) * 128);  // bytes a slice moves W by
  auto issue_one = [&](auto jc, __amdgpu_buffer_rsrc_t rsa, __amdgpu_buffer_rsrc_t rsb, uint32_t o, uint32_t sa,
                       uint32_t sb, char* dst) {
    constexpr int J = decltype(jc)::value;
    const bool is_a = wave * D + (T::MIXED ? J : 0) < T::A_INSTS;
    buf_dma<16, (J & 3) * 1024>(is_a ? rsa : rsb, o, is_a ? sa : sb, dst + (wave * D + (J & ~3)) * 1024);
  };
  const int32_t S = (kw + 63) / 64;
  int32_t i_k = 0;  // k of the slice to be issued, and its offsets
  uint32_t i_a = 0, i_b = 0;
  auto issue_part = [&](auto jc, char* dst) { issue_one(jc, ra, rw, off[decltype(jc)::value], i_a, i_b, dst); };
  // before a slice is issued that k ends in, or past: its pieces from there on read zeros
  auto issue_mask = [&]() {
    if (i_k + 64 <= kw) return;
    static_for<D>([&](auto jc) {
      constexpr int J = decltype(jc)::value;
      const int g = wave * D + J;
      if (i_k + (g < T::A_INSTS ? a_k : lora_b_k<WKC, BN>(g - T::A_INSTS, lane)) >= kw) off[J] = kLoraOob;
    });
  };
  auto issue_next = [&]() {
    i_k += 64;
    i_a += 128;
    i_b += b_step;
    if (i_k >= kw) i_a = i_b = 0;  // (only offsets past the range from here on)
    issue_mask();
  };
  issue_mask();

  // ---- fragments of the two halves of a slice.  [row][k] rows of 128 bytes hold
  // chunk c at c ^ (row & 7); the second half's chunks are 4 on, bit 6 of the address
  const uint32_t st0 = lds_addr(ring);
  const uint32_t kc_lane = (uint32_t)(fr * 128 + ((fq ^ (fr & 7)) << 4));
  const uint32_t a_f = st0 + (uint32_t)(wm * MI * 2048) + kc_lane;
  const uint32_t kc_f = st0 + T::A_BYTES + (uint32_t)(wn * NJ * 2048) + kc_lane;
  uint32_t tr_f[NJ];
  {
    constexpr int CPR = BN / 8;
    const int r = fq * 8 + (fr >> 2);
    const int lo = ((fr & 1) << 3) + (((fr >> 1) & 1) << 4);
#pragma unroll
    for (int i = 0; i < NJ; ++i)
      tr_f[i] = st0 + T::A_BYTES + (uint32_t)(r * BN * 2 + lo + (((wn * NJ * 2 + 2 * i) ^ tr_row_swz<CPR>(r)) << 4));
  }
  // the R-th read of half H of the slice in buffer B: x's blocks, then W's
  auto read_one = [&](auto buf, auto half, auto rc, lds_u32x4 (&fa)[MI], auto& fb) {
    constexpr int B = decltype(buf)::value, H = decltype(half)::value, R = decltype(rc)::value;
    constexpr uint32_t at = (uint32_t)B * SLICE;
    if constexpr (R < MI) {
      fa[R] = lds_read128_at<R * 2048>((a_f ^ (H * 64)) + at);
    } else if constexpr (std::is_same_v<std::remove_reference_t<decltype(fb)>, lds_u32x4[NJ]>) {
      fb[R - MI] = lds_read128_at<(R - MI) * 2048>((kc_f ^ (H * 64)) + at);
    } else {
      constexpr int i = (R - MI) / 2, h = (R - MI) % 2;
      fb[i][h] = lds_read_tr<(H * 32 + h * 4) * BN * 2>(tr_f[i] + at);
    }
  };
  auto read_all = [&](auto buf, auto half, lds_u32x4 (&fa)[MI], auto& fb) {
    constexpr int R = std::is_same_v<std::remove_reference_t<decltype(fb)>, lds_u32x4[NJ]> ? MI + NJ : MI + 2 * NJ;
    static_for<R>([&](auto rc) { read_one(buf, half, rc, fa, fb); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    lora_wait(fa);
    lora_wait(fb);
  };

  // ---- accumulators: acc[j][i] holds columns 16 j + 4 fq + {0..3} of row 16 i + fr.
  // base's values of row block i:
  const int64_t nw = n0 + wn * NJ * 16;
  auto base_of = [&](int i, f32x4_t (&v)[NJ]) {
    const int64_t row = s_row[(wm * MI + i) * 16 + fr];
#pragma unroll
    for (int j = 0; j < NJ; ++j) v[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (p.base == nullptr) return;
    const int64_t at = (row >= 0 ? row : 0) * p.base_ld;  // (rows past the last are not stored)
    if (p.base_vec && nw + NJ * 16 <= p.n_out) {
      if (p.base_dtype == kF32) {
        const float* q = reinterpret_cast<const float*>(p.base) + at + nw + 4 * fq;
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] = *reinterpret_cast<const f32x4_t*>(q + j * 16);
      } else {
        // as the stores below write it, and the lane swaps backwards
        const OpT* q = reinterpret_cast<const OpT*>(p.base) + at + nw + 8 * fq;
        uint4 raw[NJ / 2];
#pragma unroll
        for (int j = 0; j < NJ / 2; ++j) raw[j] = *reinterpret_cast<const uint4*>(q + j * 32);
#pragma unroll
        for (int j = 0; j < NJ / 2; ++j) {
          const auto s0 = __builtin_amdgcn_permlane16_swap(raw[j].x, raw[j].z, false, false);
          const auto s1 = __builtin_amdgcn_permlane16_swap(raw[j].y, raw[j].w, false, false);
          const auto u0 = __builtin_amdgcn_permlane32_swap(s0[0], s0[1], false, false);
          const auto u1 = __builtin_amdgcn_permlane32_swap(s1[0], s1[1], false, false);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            union { uint32_t u[2]; OpT e[4]; } c;
            c.u[0] = u0[h];
            c.u[1] = u1[h];
            v[2 * j + h] = f32x4_t{to_f32(c.e[0]), to_f32(c.e[1]), to_f32(c.e[2]), to_f32(c.e[3])};
          }
        }
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t n = nw + j * 16 + 4 * fq + q;
        if (n < p.n_out) v[j][q] = load_as_f32(p.base, p.base_dtype, at + n);
      }
  };
  f32x4_t acc[NJ][MI];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if constexpr (!SPLIT && !T::AGPR) {
    if (p.base != nullptr)
      static_for<MI>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        f32x4_t v[NJ];
        base_of(i, v);
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j][i] = v[j];
      });
  }

  // ---- the shared weights
  using WFrag = std::conditional_t<WKC, lds_u32x4[NJ], lds_u32x2[NJ][2]>;
  if (STAGES > 1 && S > 0) {  // (one stage: calls without W)
    constexpr int kAhead = STAGES > 1 ? STAGES - 2 : 0;
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      static_for<D>([&](auto j) { issue_part(j, ring + s * SLICE); });
      issue_next();
      issue_fence();
    }
    lds_u32x4 a0[MI], a1[MI];
    WFrag b0, b1;
    vm_wait<(kAhead + 1) * D>();
    lds_barrier();
    read_all(std::integral_constant<int, 0>(), std::integral_constant<int, 0>(), a0, b0);
    // The products of a half of the slice in buffer B, with the next half's reads and
    // (LOAD) the loads of slice s + STAGES between them: the matrix unit is busy for
    // 16 cycles with each, in which up to three others issue.
    auto half = [&](auto bc, auto hc, lds_u32x4 (&ca)[MI], WFrag& cb, lds_u32x4 (&na)[MI], WFrag& nb) {
      constexpr int B = decltype(bc)::value, H = decltype(hc)::value;
      constexpr int P = MI * NJ, R = MI + (WKC ? NJ : 2 * NJ);
      using NB = std::integral_constant<int, H == 0 ? B : (B + 1) % STAGES>;
      using NH = std::integral_constant<int, 1 - H>;
      char* dst = ring + B * SLICE;
      lora_mfma_ready();
      static_for<P>([&](auto tc) {
        constexpr int t = decltype(tc)::value, jb = t / MI, i = t % MI;
        lora_mfma_one<OpT, T::AGPR>(acc[jb][i], lora_frag(cb[jb]), ca[i]);
        static_for<R>([&](auto rc) {
          if constexpr (decltype(rc)::value * (P - P / 4) / R == t) read_one(NB(), NH(), rc, na, nb);
        });
        if constexpr (H == 1)
          static_for<D>([&](auto j) {
            if constexpr (decltype(j)::value * P / D == t) issue_part(j, dst);
          });
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (H == 1) issue_next();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      lora_wait(na);
      lora_wait(nb);
    };
    // slice s: its first half is in (a0, b0).  After the first half's products every
    // wave has the second in registers, so that the buffer takes slice s + STAGES.
    auto slice = [&](auto bc) {
      half(bc, std::integral_constant<int, 0>(), a0, b0, a1, b1);
      vm_wait<kAhead * D>();  // slice s + 1 has landed
      lds_barrier();
      half(bc, std::integral_constant<int, 1>(), a1, b1, a0, b0);
    };
    // (the ring's slices at a time, zeros past the last: leaving within them made the
    // compiler spill the largest tile's registers)
    for (int32_t s = 0; s < S; s += STAGES)
      static_for<STAGES>([&](auto bc) {
        if (T::AGPR || s + decltype(bc)::value < S) slice(bc);
      });
    vm_wait<0>();
    if constexpr (T::AGPR) lora_mfma_done(acc);
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
  if (tid < BM) s_id[tid] = my_id >= 0 && my_id < p.n ? (int32_t)my_id : -1;
  lds_barrier();
  using BFrag = std::conditional_t<BKC, lds_u32x4[NJ], lds_u32x2[NJ][2]>;
  int32_t ids[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) ids[i] = s_id[(wm * MI + i) * 16 + fr];
  const __amdgpu_buffer_rsrc_t rh = lora_rsrc(reinterpret_cast<const OpT*>(p.h) + first * p.h_ld);
  uint32_t hoff[D];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    const int g = wave * D + j;
    if (g < T::A_INSTS) {
      const int32_t row = s_row[g * 8 + (lane >> 3)];
      hoff[j] = row >= 0 ? (uint32_t)(((int64_t)row - first) * p.h_ld * 2) + (uint32_t)a_k * 2 + kLoraBack : kLoraOob;
    } else {
      hoff[j] = lora_b_off<BKC, BN>(g - T::A_INSTS, lane, p.b_sr, p.b_sn, p.N - n0);
    }
    if (hoff[j] != kLoraOob) hoff[j] -= 1024u * (uint32_t)(j & 3);
  }
  const int32_t rank = (int32_t)p.rank;
  // one adapter, or none, for the whole tile?
  bool uniform = true;
#pragma unroll
  for (int i = 0; i < BM / 64; ++i) uniform &= s_id[i * 64 + lane] == s_id[0];
  uniform = __all(uniform);
  bool dropped = false;  // this lane left infinities or NaN out of an adapter's values
  const uint32_t hb_step = (uint32_t)((BKC ? 1 : p.b_sr) * 128);
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
    for (int32_t r0 = 0; r0 < rank; r0 += STAGES * 64) {  // the ring's slices at a time
      lds_barrier();                                        // the buffers' last reads
#pragma unroll
      for (int s = 0; s < STAGES; ++s) {
        const int32_t k = r0 + s * 64;
        if (k < rank)
          static_for<D>([&](auto j) {
            constexpr int J = decltype(j)::value;
            const int g = wave * D + J;
            const bool in = g < T::A_INSTS ? k + a_k < p.h_ld : k + lora_b_k<BKC, BN>(g - T::A_INSTS, lane) < rank;
            issue_one(j, rh, rb, in ? hoff[J] : kLoraOob, (uint32_t)k * 2,
                      (uint32_t)(k / 64) * hb_step, ring + s * SLICE);
          });
      }
      vm_wait<0>();
      lds_barrier();
      static_for<2 * STAGES>([&](auto sc) {
        constexpr int s = decltype(sc)::value;
        if (r0 + s * 32 >= rank) return;
        lds_u32x4 af[MI];
        BFrag bf;
        read_all(std::integral_constant<int, s / 2>(), std::integral_constant<int, s % 2>(), af, bf);
        if (!uniform) {
#pragma unroll
          for (int i = 0; i < MI; ++i)
            if (ids[i] != a) af[i] = lds_u32x4{0u, 0u, 0u, 0u};
          lora_finite<OpT>(bf, dropped);
        }
        uint4 w[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) w[j] = lora_frag(bf[j]);
        lora_operands(w, af);
        lora_mfma_ready();
        static_for<MI * NJ>([&](auto tc) {
          constexpr int j = decltype(tc)::value / MI, i = decltype(tc)::value % MI;
          lora_mfma_one<OpT, T::AGPR>(acc[j][i], w[j], af[i]);
        });
        if constexpr (T::AGPR) lora_mfma_done(acc);
      });
    }
  }

  // ---- the stores (the largest tile adds base here, a row block at a time: with the
  // loads of several in flight the compiler ran out of registers)
  static_for<MI>([&](auto ic) {
    constexpr int i = decltype(ic)::value;
    const int64_t row = s_row[(wm * MI + i) * 16 + fr];
    OpT* dst = reinterpret_cast<OpT*>(p.out) + row * p.out_ld;
    f32x4_t add[NJ];
    if constexpr (T::AGPR) base_of(i, add);
    static_for<NJ / 2>([&](auto pc) {
      constexpr int pr = decltype(pc)::value;
      uint32_t a[2], b[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        union { uint32_t u; OpT e[2]; } pa, pb;
        f32x4_t va = acc[2 * pr][i], vb = acc[2 * pr + 1][i];
        if constexpr (T::AGPR) va += add[2 * pr], vb += add[2 * pr + 1];
        pa.e[0] = from_f32<OpT>(va[2 * h]);
        pa.e[1] = from_f32<OpT>(va[2 * h + 1]);
        pb.e[0] = from_f32<OpT>(vb[2 * h]);
        pb.e[1] = from_f32<OpT>(vb[2 * h + 1]);
        a[h] = pa.u;
        b[h] = pb.u;
      }
      const auto s0 = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
      const auto s1 = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
      const auto u0 = __builtin_amdgcn_permlane16_swap(s0[0], s0[1], false, false);
      const auto u1 = __builtin_amdgcn_permlane16_swap(s1[0], s1[1], false, false);
      const int64_t n = nw + pr * 32 + 8 * fq;
      if (row >= 0 && n < p.n_out) {
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
    });
    __builtin_amdgcn_sched_barrier(0);
  });

  // ---- what was left out: added to the rows it belongs to, an element at a time
  if (__any(dropped)) {
    vm_wait<0>();  // the stores above
    // (The arguments are read again here: with those that only this part takes in registers
    // from the start the largest tile's prologue spilled scalars, and 16384 rows of
    // 2048 -> 2048 at rank 64 took 3-5 us more a call, of 152; so 1-3.)
    using Args = const __attribute__((address_space(4))) LoraParams;
    Args* q = (Args*)__builtin_amdgcn_kernarg_segment_ptr();  // (p is the first argument)
    asm volatile("" : "+s"(q));
    for (int i = 0; i < MI * 16; ++i) {
      const int64_t row = s_row[wm * MI * 16 + i];
      const int32_t a = s_id[wm * MI * 16 + i];
      if (a < 0) continue;
      const OpT* h = reinterpret_cast<const OpT*>(q->h) + row * q->h_ld;
      const OpT* b = reinterpret_cast<const OpT*>(q->b) + a * q->b_se;
      for (int64_t n = nw + lane; n < nw + NJ * 16 && n < q->n_out; n += 64) {
        float sum = 0.f;
        for (int32_t r = 0; r < rank; ++r) {
          const float v = to_f32(b[r * q->b_sr + n * q->b_sn]);
          if (!isfinite(v)) sum += to_f32(h[r]) * v;
        }
        if (isfinite(sum)) continue;
        OpT* at = reinterpret_cast<OpT*>(q->out) + row * q->out_ld + n;
        float rest = to_f32(*at);
        // An infinity against the sum's may have come of the output's rounding alone, and a
        // NaN of an infinite inner value times the zero of what was left out; then the terms
        // without those say what they are.
        if (isinf(sum) && !isfinite(rest) && rest != sum) {
          // (up to a NaN, or the other infinity, which makes one)
          rest = q->base != nullptr ? load_as_f32(q->base, q->base_dtype, row * q->base_ld + n) : 0.f;
#pragma unroll 1
          for (int32_t r = 0; r < rank && !isnan(rest + sum); ++r) {
            const float v = to_f32(b[r * q->b_sr + n * q->b_sn]);
            if (isfinite(v)) rest += to_f32(h[r]) * v;
          }
          const OpT* x = reinterpret_cast<const OpT*>(q->x) + row * q->x_ld;
          const OpT* w = reinterpret_cast<const OpT*>(q->w);
          const int64_t K = w != nullptr ? q->K : 0;
#pragma unroll 1
          for (int64_t k = 0; k < K && !isnan(rest + sum); ++k)
            rest += to_f32(x[k]) * to_f32(w[k * q->w_sk + n * q->w_sn]);
        }
        *at = from_f32<OpT>(rest + sum);
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
  auto go = [&](auto mi, auto nj, auto wm, auto wn, auto st) {
    constexpr int MI = decltype(mi)::value, NJ = decltype(nj)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    constexpr int ST = decltype(st)::value;
    using T = LoraTile<MI, NJ, WM, WN, ST>;
    const int64_t n = tiles(T::BM, T::BN);
    if (n > 0x7fffffffll) return hipErrorInvalidValue;
    hipLaunchKernelGGL((lora_gemm_kernel<OpT, MI, NJ, WM, WN, ST, WKC, BKC, false>), dim3((unsigned)n), dim3(256), 0, s, p,
                       LoraSplit{});
    return hipGetLastError();
  };
  using std::integral_constant;
  using i2 = integral_constant<int, 2>;
  using i4 = integral_constant<int, 4>;
  using i8 = integral_constant<int, 8>;
  // without W the reads of base and the stores are all there is: small tiles with one
  // buffer, so that a CU holds more of them (16384 rows of 1024 of base and 8 adapters of
  // rank 32: 24.7 us, 29 with a ring of two)
  if (p.w == nullptr) return go(i2(), i4(), i2(), i2(), integral_constant<int, 1>());
  // Otherwise the tile of least time, by rounds of tiles over the 256 CUs.  At 2048 k
  // a round took 53 us of 256 x 256 (one on a CU), 33 of 128 x 128 (two on a CU; 29 when
  // each has one) and 17 of 64 x 128 (one); at 1024 k in the same proportion.  Whole
  // calls of rank 32 in us, with 256 x 256 / 128 x 128 / 64 x 128 tiles:
  //   rows x k x columns  1024 x 2048 x 2048: 62 / 39 / 28.5;  4096 x 2048 x 2048: 61 / 47 / 76;
  //   12288 x 2048 x 2048: 124 / 120 / 207;  16384 x 2048 x 2048: 136 / 152 / 270;
  //   2560 x 1024 x 1024: 41 / 22 / 26;  12288 x 2048 x 1024: 71 / 76 / 109
  // (256 x 128 tiles in a ring of three were behind one of these at every size).
  auto rounds = [](int64_t t, int64_t per) { return (t + per - 1) / per; };
  const int64_t t128 = tiles(128, 128);
  const int64_t c256 = 53 * rounds(tiles(256, 256), 256), c64 = 17 * rounds(tiles(64, 128), 256);
  const int64_t c128 = 33 * rounds(t128, 512) - (t128 % 512 > 0 && t128 % 512 <= 256 ? 4 : 0);
  if (c256 <= c128 && c256 <= c64) return go(i8(), i8(), i2(), i2(), i2());
  if (c128 <= c64) return go(i4(), i4(), i2(), i2(), i2());
  return go(i2(), i4(), i2(), i2(), i4());
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
    const dim3 grid((unsigned)((p.rows + 64 / KW - 1) / (64 / KW) * kLoraInnerTurns));
    if (akc)
      hipLaunchKernelGGL((lora_inner_tile_kernel<OpT, RB, KW, true>), grid, dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((lora_inner_tile_kernel<OpT, RB, KW, false>), grid, dim3(256), 0, s, p);
  };
  auto by_rank = [&](auto kw) {
    using std::integral_constant;
    if (p.rank <= 16) go(integral_constant<int, 1>(), kw);
    else if (p.rank <= 32) go(integral_constant<int, 2>(), kw);
    else if (p.rank <= 64) go(integral_constant<int, 4>(), kw);
    else if (p.rank <= 128) go(integral_constant<int, 8>(), kw);
    else go(integral_constant<int, 16>(), kw);
  };
  // (whole calls of 2048 -> 1024 at rank 64 in us, k shared by 2 waves / 4: 4096 rows 45.7 /
  // 41.7, 8192 57.1 / 60.5, 16384 85.4 / 103.2: few rows need more workgroups, many fewer
  // readers of A)
  if (p.rows >= 8192) by_rank(std::integral_constant<int, 2>());
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
      hipLaunchKernelGGL((lora_gemm_kernel<OpT, 2, 4, 2, 2, 2, false, false, true>), grid, dim3(256), 0, s, p, sp);
    else
      hipLaunchKernelGGL((lora_gemm_kernel<OpT, 2, 4, 2, 2, 2, true, false, true>), grid, dim3(256), 0, s, p, sp);
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
