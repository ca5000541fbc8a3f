// The adapters' own products in 16-bit operands of whole 16-byte pieces
// (cvmm_lora.h): the inner rows, their gradients' twin, and calls of few rows.
#pragma once

#include "cvmm_gemm_panel.h"
#include "cvmm_lora.h"

namespace cvmm {

// Eight rows of eight values -> eight columns of eight values: the value pairs of
// rows 2 i and 2 i + 1 side by side, one permute per pair.
__device__ __forceinline__ void lora_transpose8(const uint4 (&r)[8], uint4 (&c)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // columns 2 j and 2 j + 1
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = reinterpret_cast<const uint32_t*>(&r[2 * i])[j];
      const uint32_t y = reinterpret_cast<const uint32_t*>(&r[2 * i + 1])[j];
      lo[i] = __builtin_amdgcn_perm(y, x, 0x05040100);
      hi[i] = __builtin_amdgcn_perm(y, x, 0x07060302);
    }
    c[2 * j] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    c[2 * j + 1] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  }
}

// v, or zeros: by bits, where a choice became a branch around a wait for v.
__device__ __forceinline__ uint4 keep_if(const uint4& v, bool keep) {
  const uint32_t m = keep ? ~0u : 0u;
  return make_uint4(v.x & m, v.y & m, v.z & m, v.w & m);
}

// ---------------------------------------------------------------------------
// (Loads at clamped places, zeroed where they are used: a guard around each made
// them wait for one another.)
//
// h of 64 / KW rows, 16 per wave, KW of the four waves sharing k.  A lane
// loads the pieces of x that its matrix operand holds straight from memory; A
// comes through LDS as [rank][k] rows, transposed on the way where it is stored
// [k][rank].  Bound by reading x once; each workgroup reads its adapters whole,
// from L2.  Measured: 16384 rows of 2048, rank 64: 29-32 us (67 MB at 2.2 TB/s: a
// stage's A waits for its LDS turn, and ranks 33-64 with k shared by two waves, in the
// 168 registers that three workgroups a CU leave, spill 40 bytes a lane); 8192 of 1024,
// rank 16: 11 (1.5 TB/s); 16384 of 128: 10, the chain order, id, row, store.
// ---------------------------------------------------------------------------
// Workgroups that share the adapters of a tile, in turns: nearly all tiles have one
// or two (a request ends within), and a second one, taken after the first, made the
// launch wait for the few tiles that have two (1999 rows of 2048 in runs of 8
// adapters of rank 32, whole call without W: 23.9 us, with four turns 17.5; 16384
// rows in runs that end with tiles: 30 either way).
constexpr int kLoraInnerTurns = 4;

template <int RB, int KW>
struct LoraInnerCfg {
  // k per LDS stage, a part of which each wave takes
  static constexpr int KS = RB >= 16 ? 128 : KW == 4 && RB <= 4 ? 512 : 256;
  static constexpr int KWAVE = KS / KW;        // k per wave and stage
  static constexpr int LDB = KS * 2 + 16;      // bytes per LDS row
  static constexpr int CHUNKS = RB * 16 * (KS / 8);  // 16-byte pieces of a stage
  static constexpr int PER = (CHUNKS / 8 + 255) / 256;  // blocks of 8 x 8 per thread
};

template <typename OpT, int RB, int KW, bool AKC>
__global__ __launch_bounds__(256, RB <= 4 ? 3 : 1) void lora_inner_tile_kernel(const LoraParams p) {
  using C = LoraInnerCfg<RB, KW>;
  constexpr int ROWS = 64 / KW;
  constexpr int XS = C::KWAVE / 32;  // 32-k steps of a wave per stage
  constexpr int RED = 4 * (KW - 1) / KW * RB * 64 * 16;
  constexpr int A_LDS = RB * 16 * C::LDB;
  __shared__ __attribute__((aligned(16))) char lds[A_LDS > RED ? A_LDS : RED];
  __shared__ int32_t s_row[ROWS], s_id[ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  // Tiles that stand together on one XCD, whose L2 then holds their adapters; the
  // first turns of all tiles before the second (mixed, the tiles with work came to
  // every fourth CU).
  const uint32_t tiles = gridDim.x / kLoraInnerTurns;
  const uint32_t tile = xcd_remap((uint32_t)blockIdx.x % tiles, tiles);
  const int my_turn = (int)(blockIdx.x / tiles);
  const int64_t m0 = (int64_t)tile * ROWS;
  const int32_t rank = (int32_t)p.rank;  // at most 16 RB
  if (tid < ROWS) {
    const int64_t m = m0 + tid;
    int64_t row = m < p.rows ? (p.order != nullptr ? p.order[m] : m) : -1;
    if (row < 0 || row >= p.rows) row = -1;
    s_row[tid] = (int32_t)row;
    s_id[tid] = row >= 0 ? lora_id(p, row) : -1;
  }
  __syncthreads();
  const int my = wave / KW * 16 + fr;  // the tile row of this lane's operand
  const int32_t row = s_row[my], my_id = s_id[my];
  const OpT* xrow = reinterpret_cast<const OpT*>(p.x) + (int64_t)(row >= 0 ? row : 0) * p.x_ld;
  const int k_part = wave % KW, k_wave = k_part * C::KWAVE;
  const int32_t K = (int32_t)p.K;

  f32x4_t res[RB];  // res[b]: rank 16 b + 4 fq + {0..3} of row `my`
#pragma unroll
  for (int b = 0; b < RB; ++b) res[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  bool made = my_id < 0 && my_turn == 0;  // the row is this workgroup's to write
  int turn = 0;
  for (int32_t cur = -1;;) {
    int32_t a = lane < ROWS ? s_id[lane % ROWS] : -1;
    a = wave_min_i32(a > cur ? a : INT32_MAX);
    if (a == INT32_MAX) break;
    cur = a;
    if (turn++ % kLoraInnerTurns != my_turn) continue;
    const bool mine = my_id == a;
    made |= mine;
    const bool any = __ballot(mine) != 0;  // (a wave without rows of it still stages A)
    const OpT* am = reinterpret_cast<const OpT*>(p.a) + a * p.a_se;
    uint4 xv[XS], av[C::PER][8];
    auto load_x = [&](int32_t k0) {
#pragma unroll
      for (int s = 0; s < XS; ++s) {
        const int32_t k = k0 + k_wave + s * 32 + fq * 8;
        xv[s] = *reinterpret_cast<const uint4*>(xrow + (k < K ? k : K - 8));
      }
    };
    // blocks of 8 k x 8 of the rank
    auto load_a = [&](int32_t k0) {
#pragma unroll
      for (int u = 0; u < C::PER; ++u) {
        const int i = u * 256 + tid;
        const int ro = AKC ? i / (C::KS / 8) : i % (RB * 2), ko = AKC ? i % (C::KS / 8) : i / (RB * 2);
        const int32_t k = k0 + ko * 8, r = ro * 8;
        if (C::CHUNKS / 8 % 256 != 0 && i >= C::CHUNKS / 8) break;  // (whole waves)
        const OpT* at = am + (int64_t)(r < rank ? r : 0) * p.a_sr + (int64_t)(k < K ? k : 0) * p.a_sk;
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          av[u][v] = *reinterpret_cast<const uint4*>(at + v * (AKC ? p.a_sr : p.a_sk));
        }
      }
    };
    auto store_a = [&](int32_t k0) {
#pragma unroll
      for (int u = 0; u < C::PER; ++u) {
        const int i = u * 256 + tid;
        if (i >= C::CHUNKS / 8) break;
        const int ro = AKC ? i / (C::KS / 8) : i % (RB * 2), ko = AKC ? i % (C::KS / 8) : i / (RB * 2);
        char* at = lds + ro * 8 * C::LDB + (ko ^ (ro & 7)) * 16;  // (8 threads' writes: 8 chunks)
#pragma unroll
        for (int v = 0; v < 8; ++v) av[u][v] = keep_if(av[u][v], k0 + ko * 8 < K && ro * 8 < rank);
        if constexpr (AKC) {
#pragma unroll
          for (int v = 0; v < 8; ++v) *reinterpret_cast<uint4*>(at + v * C::LDB) = av[u][v];
        } else {
          uint4 t[8];
          lora_transpose8(av[u], t);
#pragma unroll
          for (int v = 0; v < 8; ++v) *reinterpret_cast<uint4*>(at + v * C::LDB) = t[v];
        }
      }
    };
    f32x4_t acc[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    load_a(0);
    load_x(0);
    for (int32_t k0 = 0; k0 < K; k0 += C::KS) {
      __syncthreads();  // the last stage's reads
      store_a(k0);
      uint4 xc[XS];
#pragma unroll
      for (int s = 0; s < XS; ++s) xc[s] = keep_if(xv[s], k0 + k_wave + s * 32 + fq * 8 < K);
      lds_barrier();
      if (k0 + C::KS < K) {
        load_a(k0 + C::KS);
        load_x(k0 + C::KS);
      }
      if (any) {
        // (one step's operands are read while the last's products run)
        uint4 w[2][RB];
        auto read_w = [&](int s) {
#pragma unroll
          for (int b = 0; b < RB; ++b)
            w[s & 1][b] = *reinterpret_cast<const uint4*>(
                lds + (b * 16 + fr) * C::LDB + ((k_wave / 8 + s * 4 + fq) ^ ((b * 2 + fr / 8) & 7)) * 16);
        };
        read_w(0);
#pragma unroll
        for (int s = 0; s < XS; ++s) {
          if (s + 1 < XS) read_w(s + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int b = 0; b < RB; ++b) MfmaOp<OpT>::step(acc[b], w[s & 1][b], xc[s]);
        }
      }
    }
    if constexpr (KW > 1) {
      // the waves' sums, added in wave order by the first
      const int group = wave / KW * (KW - 1);
      __syncthreads();
      if (k_part > 0) {
#pragma unroll
        for (int b = 0; b < RB; ++b)
          *reinterpret_cast<f32x4_t*>(lds + (((group + k_part - 1) * RB + b) * 64 + lane) * 16) = acc[b];
      }
      __syncthreads();
      if (k_part == 0) {
#pragma unroll
        for (int w = 0; w < KW - 1; ++w)
#pragma unroll
          for (int b = 0; b < RB; ++b)
            acc[b] += *reinterpret_cast<const f32x4_t*>(lds + (((group + w) * RB + b) * 64 + lane) * 16);
      }
    }
    const float sc = lora_scale(p, a);
    if (mine) {
#pragma unroll
      for (int b = 0; b < RB; ++b) res[b] = sc * acc[b];
    }
  }
  if (!made || k_part != 0) return;
  OpT* h = reinterpret_cast<OpT*>(p.h);
  OpT* ht = reinterpret_cast<OpT*>(p.ht);
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int64_t r = b * 16 + 4 * fq;
    union { uint2 u; OpT e[4]; } o;
#pragma unroll
    // (an infinity of x times a copy's zeros would be NaN)
    for (int v = 0; v < 4; ++v) o.e[v] = from_f32<OpT>(r + v < p.rank_out ? res[b][v] : 0.f);
    if (row >= 0 && r < p.h_ld) *reinterpret_cast<uint2*>(h + row * p.h_ld + r) = o.u;
    if (ht != nullptr && m0 + my < p.rows) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (r + v < p.rank_out) ht[(r + v) * p.ht_ld + m0 + my] = o.e[v];
    }
  }
  // zeros up to the whole slices of 32 that the projection reads
  if (RB == 1 && row >= 0) *reinterpret_cast<uint2*>(h + row * p.h_ld + 16 + 4 * fq) = make_uint2(0, 0);
}

// ---------------------------------------------------------------------------
// Calls of few rows, most of them with an adapter of their own: plain 32-bit
// multiply-adds, each of a row's matrices read once and spread over many
// workgroups.  Nothing but the output is rounded.  First launch: shares of x A_i (here)
// beside shares of x W (the split GEMM); second: their sums, then h B_i
// (lora_join_kernel).  Bound by launches and the latency of one chain of loads each:
// 32 rows of 2048 -> 2048, rank 16, 64 adapters: 5.6 + 4.0 us, 12 MB, of which 2.4
// would be bandwidth; one row of 1024 -> 1024: 4.8 + 4.2.
// ---------------------------------------------------------------------------
constexpr int kLoraRowLds = 256 * 8 * 4;  // bytes of LDS that lora_inner_row uses

// Share `share` of the inner row of `row`, over k in [share * h_k, + h_k).
template <typename OpT>
__device__ __forceinline__ void lora_inner_row(const LoraParams& p, const LoraSplit& sp, uint32_t block, float* lds) {
  const int tid = threadIdx.x;
  const int64_t row = block / (uint32_t)sp.h_splits;
  const int32_t share = (int32_t)(block % (uint32_t)sp.h_splits), rank = (int32_t)p.rank;
  const int32_t a = lora_id(p, row);
  if (a < 0) return;  // the join reads no inner row there
  const int32_t k0 = share * sp.h_k, k1 = k0 + sp.h_k < p.K ? k0 + sp.h_k : (int32_t)p.K;
  const OpT* x = reinterpret_cast<const OpT*>(p.x) + row * p.x_ld;
  const OpT* am = reinterpret_cast<const OpT*>(p.a) + a * p.a_se;
  float* out = sp.h_part + ((int64_t)share * p.rows + row) * rank;
  if (p.a_sr == 1) {
    // [k][rank]: a thread takes 8 of the rank at every G-th k
    const int L = rank / 8, G = 256 / L, ro = tid % L, kk = tid / L;
    float acc[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) acc[v] = 0.f;
    if (kk < G) {
#pragma unroll 4
      for (int32_t k = k0 + kk; k < k1; k += G) {
        Chunk16 c;
        c.u = *reinterpret_cast<const uint4*>(am + (int64_t)k * p.a_sk + ro * 8);
        const float xv = to_f32(x[k]);
#pragma unroll
        for (int v = 0; v < 8; ++v) acc[v] += xv * to_f32(reinterpret_cast<const OpT*>(&c)[v]);
      }
#pragma unroll
      for (int v = 0; v < 8; ++v) lds[kk * rank + ro * 8 + v] = acc[v];
    }
    for (int n = G; n > 1; n = (n + 1) / 2) {  // entries [half, n) onto [0, ...)
      __syncthreads();
      const int half = (n + 1) / 2;
      for (int i = tid; i < (n - half) * rank; i += 256) lds[i] += lds[half * rank + i];
    }
    __syncthreads();
    if (tid < rank) out[tid] = lds[tid];
  } else {
    // [rank][k]: 16 threads along k per inner value
    for (int r = tid / 16; r < rank; r += 16) {
      float s = 0.f;
#pragma unroll 4
      for (int32_t k = k0 + (tid % 16) * 8; k < k1; k += 128) {
        Chunk16 c, d;
        c.u = *reinterpret_cast<const uint4*>(am + r * p.a_sr + k);
        d.u = *reinterpret_cast<const uint4*>(x + k);
#pragma unroll
        for (int v = 0; v < 8; ++v)
          s += to_f32(reinterpret_cast<const OpT*>(&c)[v]) * to_f32(reinterpret_cast<const OpT*>(&d)[v]);
      }
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) s += __shfl_xor(s, d, 64);
      if (tid % 16 == 0) out[r] = s;
    }
  }
}

template <typename OpT>
__global__ __launch_bounds__(256) void lora_inner_row_kernel(const LoraParams p, const LoraSplit sp) {
  __shared__ float lds[kLoraRowLds / 4];
  lora_inner_row<OpT>(p, sp, blockIdx.x, lds);
}

// out of one row, 4 columns a thread: base, the shares of x W in order, h B_i.
constexpr int kLoraJoinThreads = 128;
template <typename OpT>
__global__ __launch_bounds__(kLoraJoinThreads) void lora_join_kernel(const LoraParams p, const LoraSplit sp) {
  __shared__ float h[kLoraMaxRank];
  const int64_t row = blockIdx.y;
  const int32_t a = lora_id(p, row), rank = (int32_t)p.rank;
  if (a >= 0) {
    const float sc = lora_scale(p, a);
    for (int r = threadIdx.x; r < rank; r += kLoraJoinThreads) {
      float s = 0.f;
#pragma unroll 4
      for (int q = 0; q < sp.h_splits; ++q) s += sp.h_part[((int64_t)q * p.rows + row) * rank + r];
      h[r] = r < p.rank_out ? sc * s : 0.f;  // (an infinity of x times a copy's zeros would be NaN)
    }
  }
  __syncthreads();
  const int64_t n = ((int64_t)blockIdx.x * kLoraJoinThreads + threadIdx.x) * 4;
  if (n >= p.n_out) return;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (sp.part != nullptr) {
#pragma unroll 8
    for (int s = 0; s < sp.splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(sp.part + ((int64_t)s * p.rows + row) * sp.part_ld + n);
      acc[0] += v.x, acc[1] += v.y, acc[2] += v.z, acc[3] += v.w;
    }
  }
  if (a >= 0) {
    const OpT* bm = reinterpret_cast<const OpT*>(p.b) + a * p.b_se;
    if (p.b_sn == 1) {
#pragma unroll 8
      for (int r = 0; r < rank; ++r) {
        const uint2 raw = *reinterpret_cast<const uint2*>(bm + r * p.b_sr + n);
        const OpT* v = reinterpret_cast<const OpT*>(&raw);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += h[r] * to_f32(v[j]);
      }
    } else {
      for (int r = 0; r < rank; r += 8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          Chunk16 c;
          c.u = *reinterpret_cast<const uint4*>(bm + (n + j) * p.b_sn + r);
#pragma unroll
          for (int v = 0; v < 8; ++v) acc[j] += h[r + v] * to_f32(reinterpret_cast<const OpT*>(&c)[v]);
        }
      }
    }
  }
  OpT* out = reinterpret_cast<OpT*>(p.out) + row * p.out_ld + n;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j >= p.n_out) break;
    if (p.base != nullptr) acc[j] += load_as_f32(p.base, p.base_dtype, row * p.base_ld + n + j);
    out[j] = from_f32<OpT>(acc[j]);
  }
}

// ---------------------------------------------------------------------------
// The adapters' gradients (cvmm_lora_bwd_adapters): a wave takes 128 columns of x
// (of g) in steps of 32 sorted rows.  A lane loads 16 bytes of 8 rows -- 8 columns
// -- and turns the block round in registers (32 permutes), which makes it the
// matrix operands of 8 blocks of 16 columns; the inner rows lie transposed and are
// operands as they are.  No LDS in the loop; bound by reading x and g once.  The
// waves of a workgroup share its rows; an adapter's rows are dealt out to `shares`
// workgroups, whose partial sums the second launch adds in order.  Measured: 8192
// rows, 8 adapters of rank 16, 1024 -> 1024: 14.3 us (34 MB at 2.4 TB/s) and 4.5 for the
// sums; 16384 rows, 64 adapters, 128 -> 1024: 18.2 (38 MB at 2.1 TB/s): eight gathered
// rows in flight per lane.
// ---------------------------------------------------------------------------
template <typename OpT, int RB>
__global__ __launch_bounds__(256) void lora_wgrad_fast_kernel(const LoraWgradParams p) {
  __shared__ __attribute__((aligned(16))) f32x4_t red[2][8 * RB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int64_t bi = (p.d_in + 127) / 128;
  const bool in = (int64_t)blockIdx.x < bi;
  if ((in ? p.ga : p.gb) == nullptr) return;
  const int64_t c0 = (in ? blockIdx.x : blockIdx.x - bi) * 128 + fr * 8;
  const int64_t r0 = (int64_t)blockIdx.y * RB * 16;
  const int32_t e = (int32_t)(blockIdx.z / (uint32_t)p.shares), share = (int32_t)(blockIdx.z % (uint32_t)p.shares);
  // (32 bits: at most 2^31 - 1 rows)
  const int64_t lo64 = p.offsets[e > 0 ? e - 1 : 0], hi64 = p.offsets[e], rows64 = p.rows;
  const int32_t lo = e > 0 && lo64 > 0 ? (int32_t)(lo64 < rows64 ? lo64 : rows64) : 0;
  const int32_t hi = hi64 < 0 ? 0 : (int32_t)(hi64 < rows64 ? hi64 : rows64);
  // shares of whole steps (a power of two of them)
  const int32_t base = lo & ~31;
  const int32_t steps = hi > lo ? (hi - base + 31) / 32 : 0;
  const int sh = __builtin_ctz(p.shares);
  const int32_t s_from = (int32_t)(((int64_t)steps * share) >> sh), s_to = (int32_t)(((int64_t)steps * (share + 1)) >> sh);
  const OpT* rows = reinterpret_cast<const OpT*>(in ? p.x : p.g);
  const int64_t ld = in ? p.x_ld : p.g_ld, width = in ? p.d_in : p.d_out;
  const OpT* t = reinterpret_cast<const OpT*>(in ? p.ut : p.ht);
  f32x4_t acc[8][RB];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int b = 0; b < RB; ++b) acc[j][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const bool col_in = c0 < width;
  const OpT* col = rows + (col_in ? c0 : 0);
  uint4 xv[8], tv[RB];
  uint32_t x_in = 0;  // which of them count, as bits
  // the rows of the step after the one that is loaded: the order's loads do not stand
  // before the rows' own
  int64_t at[8];
  auto load_order = [&](int32_t s) {
#pragma unroll
    for (int v = 0; v < 8; ++v) {
      const int32_t q = base + s * 32 + fq * 8 + v;
      at[v] = p.order[q < lo ? lo : q < hi ? q : hi - 1];
    }
  };
  auto load = [&](int32_t s) {
    const int32_t q0 = base + s * 32 + fq * 8;
#pragma unroll
    for (int v = 0; v < 8; ++v) {
      const bool in = q0 + v >= lo && q0 + v < hi && at[v] >= 0 && at[v] < p.rows;
      xv[v] = *reinterpret_cast<const uint4*>(col + (in ? at[v] : 0) * ld);
      x_in = v == 0 ? (in ? 1u : 0u) : x_in | (in ? 1u << v : 0u);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int64_t r = r0 + b * 16 + fr;
      tv[b] = *reinterpret_cast<const uint4*>(t + (r < p.rank && q0 < hi ? r * p.t_ld + q0 : 0));
    }
    if (s + 4 < s_to) load_order(s + 4);
  };
  int32_t s = s_from + wave;
  if (s < s_to) {
    load_order(s);
    load(s);
  }
  for (; s < s_to; s += 4) {
    uint4 xc[8], xt[8], tc[RB];
    // the neighbours' rows: zeros, whatever they hold
#pragma unroll
    for (int v = 0; v < 8; ++v) xc[v] = keep_if(xv[v], (x_in >> v) & 1u);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      Chunk16 c;
      c.u = tv[b];
      const bool in = r0 + b * 16 + fr < p.rank;
#pragma unroll
      for (int v = 0; v < 8; ++v)
        if (!in || !((x_in >> v) & 1u)) c.s[v] = 0;
      tc[b] = c.u;
    }
    if (s + 4 < s_to) load(s + 4);
    lora_transpose8(xc, xt);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int b = 0; b < RB; ++b) MfmaOp<OpT>::step(acc[j][b], tc[b], xt[j]);
  }
  // the waves' sums: 2 and 3 to 0 and 1, then 1 to 0
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int b = 0; b < RB; ++b) red[wave - half][j * RB + b][lane] = acc[j][b];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[j][b] += red[wave][j * RB + b][lane];
    }
    __syncthreads();
  }
  if (wave != 0 || !col_in) return;
  // acc[j][b][v]: column c0 + j, rank r0 + 16 b + 4 fq + v
  const int64_t na = p.d_in * p.rank * p.n, total = na + p.d_out * p.rank * p.n;
  float* part = p.part + (int64_t)share * total + (in ? 0 : na);
  void* out = in ? p.ga : p.gb;
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t r = r0 + b * 16 + 4 * fq + v;
      if (r >= p.rank) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c0 + j >= width) continue;
        const int64_t at = in ? (e * p.d_in + c0 + j) * p.rank + r : (e * p.rank + r) * p.d_out + c0 + j;
        if (p.shares > 1) part[at] = acc[j][b][v];
        else store_from_f32(out, p.g_dtype, at, acc[j][b][v]);
      }
    }
}

}  // namespace cvmm
