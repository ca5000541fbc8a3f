// Low-rank adapters of many requests beside a shared projection, no counterpart
// in cvmm.py.  Rows of any order; any types, strides and widths.
//
// Two launches: the inner rows h = s x A_i, then the projection with h B_i added
// in its accumulators.  A tile holds rows of several adapters: it walks the
// adapters that occur in it, by rising id, forms each one's product for the whole
// tile and keeps it in that adapter's rows alone (selected, not multiplied by
// zero: an infinity or a NaN of one request's adapter stays with its rows).
// h is rounded to the op type, whose matrix instructions form h B_i: an error of
// at most half a step of each of its values, beside the one of the output's own
// rounding; kept in two 16-bit parts, h would take twice the adapters' slices.  (Calls
// of few rows form h B_i of 32-bit values, cvmm_lora_rows.h.)  All sums are 32-bit.
//
// The general kernels here are bound by their element loads and two barriers a slice of
// 128 bytes: fp32, rank 16, 8192 rows of 1024 -> 1024 330 us (the library's product alone
// 126), all gradients 749; 32 rows of 2048 -> 2048 820, in 32 workgroups that walk all of k.
#include "cvmm_common.h"
#include "cvmm_internal.h"
#include "cvmm_lora.h"
#include "cvmm_mfma.h"
#include "../../include/cvmm_hip.h"

namespace cvmm {

constexpr int kLoraTile = 64;

// LDS slice of 64 rows by BK values of k, 16 bytes of padding a row.
template <typename OpT>
struct LoraSlice {
  static constexpr int BK = 128 / sizeof(OpT);
  static constexpr int LD = BK + 16 / sizeof(OpT);
  static constexpr int PER = kLoraTile * BK / 256;  // values per thread
};

// A 64 x BK block src[r * sr + k * sk], zero from n_r and n_k on: consecutive
// threads along the unit stride.
template <typename OpT>
__device__ __forceinline__ void lora_load(const OpT* __restrict__ src, int64_t sr, int64_t sk, int64_t n_r,
                                          int64_t n_k, OpT (&v)[LoraSlice<OpT>::PER]) {
  using S = LoraSlice<OpT>;
  const bool along_k = sk == 1;
#pragma unroll
  for (int j = 0; j < S::PER; ++j) {
    const int i = j * 256 + (int)threadIdx.x;
    const int r = along_k ? i / S::BK : i % kLoraTile, k = along_k ? i % S::BK : i / kLoraTile;
    v[j] = r < n_r && k < n_k ? src[r * sr + k * sk] : from_f32<OpT>(0.f);
  }
}
template <typename OpT>
__device__ __forceinline__ void lora_store(OpT* __restrict__ dst, bool along_k, const OpT (&v)[LoraSlice<OpT>::PER]) {
  using S = LoraSlice<OpT>;
#pragma unroll
  for (int j = 0; j < S::PER; ++j) {
    const int i = j * 256 + (int)threadIdx.x;
    const int r = along_k ? i / S::BK : i % kLoraTile, k = along_k ? i % S::BK : i / kLoraTile;
    dst[r * S::LD + k] = v[j];
  }
}
// Rows gathered by an LDS table of row indices (or -1: zeros).
template <typename OpT>
__device__ __forceinline__ void lora_load_rows(const OpT* __restrict__ src, int64_t ld, const int64_t* rows,
                                               int64_t n_k, OpT (&v)[LoraSlice<OpT>::PER]) {
  using S = LoraSlice<OpT>;
#pragma unroll
  for (int j = 0; j < S::PER; ++j) {
    const int i = j * 256 + (int)threadIdx.x, r = i / S::BK, k = i % S::BK;
    const int64_t row = rows[r];
    v[j] = row >= 0 && k < n_k ? src[row * ld + k] : from_f32<OpT>(0.f);
  }
}

// acc[j] += 16 rows of this wave x 64 columns over one slice.
template <typename OpT>
__device__ __forceinline__ void lora_mfma(f32x4_t (&acc)[4], const OpT* as, const OpT* bs, int wave, int lane) {
  using S = LoraSlice<OpT>;
  constexpr int EPC = MfmaOp<OpT>::EPC;
  const int r = lane & 15, q = lane >> 4;
#pragma unroll
  for (int st = 0; st < S::BK / MfmaOp<OpT>::KSTEP; ++st) {
    const int k = st * MfmaOp<OpT>::KSTEP + q * EPC;
    const uint4 a = *reinterpret_cast<const uint4*>(as + (wave * 16 + r) * S::LD + k);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      MfmaOp<OpT>::step(acc[j], a, *reinterpret_cast<const uint4*>(bs + (j * 16 + r) * S::LD + k));
  }
}

// The product of 64 rows (gathered by `rows`) with src[k * sk + c * sc], c < n_c,
// over all K, into acc; every thread of the workgroup enters.
template <typename OpT>
__device__ __forceinline__ void lora_product(f32x4_t (&acc)[4], OpT* as, OpT* bs, const OpT* __restrict__ x,
                                             int64_t x_ld, const int64_t* rows, const OpT* __restrict__ src,
                                             int64_t sk, int64_t sc, int64_t n_c, int64_t K, int wave, int lane) {
  using S = LoraSlice<OpT>;
  OpT va[S::PER], vb[S::PER];
  lora_load_rows(x, x_ld, rows, K, va);
  lora_load(src, sc, sk, n_c, K, vb);
  for (int64_t k0 = 0; k0 < K; k0 += S::BK) {
    __syncthreads();  // the last slice's reads
    lora_store(as, true, va);
    lora_store(bs, sk == 1, vb);
    __syncthreads();
    if (k0 + S::BK < K) {
      lora_load_rows(x + k0 + S::BK, x_ld, rows, K - k0 - S::BK, va);
      lora_load(src + (k0 + S::BK) * sk, sc, sk, n_c, K - k0 - S::BK, vb);
    }
    lora_mfma(acc, as, bs, wave, lane);
  }
}

// The ids of the tile's rows and the rows' indices; rows past the last: -1.
__device__ __forceinline__ void lora_tile_rows(const LoraParams& p, int64_t m0, bool ordered, int32_t* ids,
                                               int64_t* rows) {
  if (threadIdx.x < kLoraTile) {
    const int64_t m = m0 + threadIdx.x;
    int64_t row = m < p.rows ? (ordered && p.order != nullptr ? p.order[m] : m) : -1;
    if (row < 0 || row >= p.rows) row = -1;  // (an order that is no permutation)
    ids[threadIdx.x] = row >= 0 ? lora_id(p, row) : -1;
    rows[threadIdx.x] = row;
  }
  __syncthreads();
}

// h of 64 rows and 64 columns of the rank.
template <typename OpT>
__global__ __launch_bounds__(256) void lora_inner_kernel(const LoraParams p) {
  using S = LoraSlice<OpT>;
  __shared__ __attribute__((aligned(16))) OpT as[kLoraTile * S::LD], bs[kLoraTile * S::LD];
  __shared__ int64_t rows[kLoraTile];
  __shared__ int32_t ids[kLoraTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t m0 = (int64_t)blockIdx.x * kLoraTile, c0 = (int64_t)blockIdx.y * kLoraTile;
  lora_tile_rows(p, m0, true, ids, rows);
  f32x4_t res[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) res[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int col = lane & 15, r0 = wave * 16 + (lane >> 4) * 4;
  const int32_t mine = ids[lane];
  for (int32_t cur = -1;;) {
    const int32_t a = wave_min_i32(mine > cur ? mine : INT32_MAX);  // the same in every wave
    if (a == INT32_MAX) break;
    cur = a;
    f32x4_t acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    lora_product<OpT>(acc, as, bs, (const OpT*)p.x, p.x_ld, rows,
                      (const OpT*)p.a + a * p.a_se + c0 * p.a_sr, p.a_sk, p.a_sr, p.rank - c0, p.K, wave, lane);
    const float s = lora_scale(p, a);
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (ids[r0 + v] == a) {
#pragma unroll
        for (int j = 0; j < 4; ++j) res[j][v] = s * acc[j][v];
      }
  }
  OpT* h = (OpT*)p.h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t c = c0 + j * 16 + col;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t row = rows[r0 + v];
      const OpT o = from_f32<OpT>(c < p.rank ? res[j][v] : 0.f);
      if (row >= 0 && c < p.h_ld) h[row * p.h_ld + c] = o;
      if (p.ht != nullptr && m0 + r0 + v < p.rows && c < p.rank) ((OpT*)p.ht)[c * p.ht_ld + m0 + r0 + v] = o;
    }
  }
}

// 64 x 64 of the output.
template <typename OpT>
__global__ __launch_bounds__(256) void lora_out_kernel(const LoraParams p) {
  using S = LoraSlice<OpT>;
  __shared__ __attribute__((aligned(16))) OpT as[kLoraTile * S::LD], bs[kLoraTile * S::LD];
  __shared__ int64_t rows[kLoraTile];
  __shared__ int32_t ids[kLoraTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tiles_n = (p.N + kLoraTile - 1) / kLoraTile;
  const int64_t id = xcd_remap((int64_t)blockIdx.x, (int64_t)gridDim.x);
  const int64_t m0 = (id / tiles_n) * kLoraTile, n0 = (id % tiles_n) * kLoraTile;
  lora_tile_rows(p, m0, false, ids, rows);
  f32x4_t res[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) res[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (p.w != nullptr)
    lora_product<OpT>(res, as, bs, (const OpT*)p.x, p.x_ld, rows, (const OpT*)p.w + n0 * p.w_sn, p.w_sk, p.w_sn,
                      p.N - n0, p.K, wave, lane);
  const int col = lane & 15, r0 = wave * 16 + (lane >> 4) * 4;
  const int32_t mine = ids[lane];
  for (int32_t cur = -1;;) {
    const int32_t a = wave_min_i32(mine > cur ? mine : INT32_MAX);
    if (a == INT32_MAX) break;
    cur = a;
    f32x4_t acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    lora_product<OpT>(acc, as, bs, (const OpT*)p.h, p.h_ld, rows,
                      (const OpT*)p.b + a * p.b_se + n0 * p.b_sn, p.b_sr, p.b_sn, p.N - n0, p.rank, wave, lane);
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (ids[r0 + v] == a) {
#pragma unroll
        for (int j = 0; j < 4; ++j) res[j][v] += acc[j][v];
      }
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int64_t row = rows[r0 + v];
    if (row < 0) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = n0 + j * 16 + col;
      if (c >= p.N) continue;
      float o = res[j][v];
      if (p.base != nullptr) o += load_as_f32(p.base, p.base_dtype, row * p.base_ld + c);
      ((OpT*)p.out)[row * p.out_ld + c] = from_f32<OpT>(o);
    }
  }
}

template <typename OpT>
static hipError_t launch_general(const LoraParams& p, hipStream_t s) {
  const int64_t tm = (p.rows + kLoraTile - 1) / kLoraTile, tn = (p.N + kLoraTile - 1) / kLoraTile;
  if (tm * tn > 0x7fffffffll) return hipErrorInvalidValue;
  hipLaunchKernelGGL((lora_inner_kernel<OpT>), dim3((unsigned)tm, (unsigned)((p.rank + kLoraTile - 1) / kLoraTile)),
                     dim3(256), 0, s, p);
  if (p.out == nullptr) return hipGetLastError();
  hipLaunchKernelGGL((lora_out_kernel<OpT>), dim3((unsigned)(tm * tn)), dim3(256), 0, s, p);
  return hipGetLastError();
}

template <typename OpT> hipError_t launch_lora_gemm_op(const LoraParams& p, hipStream_t s);
template <typename OpT> hipError_t launch_lora_inner_op(const LoraParams& p, hipStream_t s);
template <typename OpT> hipError_t launch_lora_few_op(const LoraParams& p, const LoraSplit& sp, hipStream_t s);
template <typename OpT> hipError_t launch_lora_wgrad_op(const LoraWgradParams& p, hipStream_t s);

namespace {
bool al16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

// A matrix [rows][cols] of aligned 16-byte pieces along the dimension of stride 1.
bool pieces(const void* q, int64_t se, int64_t sr, int64_t sc) {
  return al16(q) && se % 8 == 0 && ((sc == 1 && sr % 8 == 0) || (sr == 1 && sc % 8 == 0));
}

// What the 16-byte kernels take: whole pieces, and distances that their 32-bit
// offsets hold (a tile's rows and columns, a matrix along k).  A projection past them takes
// the general kernels: 1024 rows of 8192 -> 65536 959 us (the library's product alone 853),
// of 8192 -> 152064 46.6 ms (2.1).
bool fast_ok(const LoraParams& p, int32_t op) {
  constexpr int64_t kReach = (int64_t)1 << 30;  // elements below 2^31 bytes, the slack off
  auto reach = [&](int64_t k, int64_t sk, int64_t sn) { return k * sk + 256 * sn < kReach - 8192; };
  return op != kF32 && p.K % 8 == 0 && p.N % 8 == 0 && p.rank % 8 == 0 && al16(p.x) && p.x_ld % 8 == 0 &&
         p.x_ld < kReach / 512 && pieces(p.a, p.a_se, p.a_sk, p.a_sr) && pieces(p.b, p.b_se, p.b_sr, p.b_sn) &&
         reach(p.rank, p.b_sr, p.b_sn) &&
         (p.w == nullptr || (pieces(p.w, 0, p.w_sk, p.w_sn) && reach(p.K, p.w_sk, p.w_sn)));
}

// Calls that are two launches of plain multiply-adds beside a GEMM split along k:
// the tiles of the others take one adapter after the other, which rows of many
// adapters pay for.  Whole calls of 2048 -> 2048 in us, this way / by tiles:
//   rows of 32 adapters  rank 16: 256 20.1 / 88.9, 512 29.7 / 93.1, 768 38 / 93;
//                        rank 64: 256 36.3 / 126, 512 60.3 / 127
//   rows of one or two   rank 16: 256 20.0 / 25.4, 512 29.2 / 26.4, 768 37 / 27;
//                        rank 64: 256 35.4 / 31.1, 512 58.0 / 31.9
// The ids are not known here; the limits are where the second kind, a prompt's, loses
// a few us at most.  Above them rows of many adapters in mixed order would be better off
// this way (384 rows of 32 adapters at rank 128: 200 us by tiles, 62 this way); a
// selection, which sorts them, is their remedy (73 with the sort).
bool few_rows(int64_t rows, int64_t rank) { return rows <= (rank <= 16 ? 512 : 256); }

// Workgroups of the split GEMM (64 x 128 tiles): one per CU, with 256 k each where
// k allows (32 rows of 2048 -> 2048: 9.3 us, 11.2 with 128 each and 10.8 with 512; 8
// rows of 4096 -> 4096: 13.2 with 512 k each in 256 workgroups, 16.8 with 1024 in
// 128).  Shares of the inner rows: four loads a thread (32 rows: 11.2 us; one 12.1,
// sixteen 13.5).
LoraSplit few_split(int64_t rows, int64_t K, int64_t N, int64_t rank) {
  LoraSplit sp{};
  const int64_t tiles = ((rows + 63) / 64) * ((N + 127) / 128), all = (K + 63) / 64;
  int64_t splits = (256 + tiles - 1) / tiles;
  if (splits > all / 4) splits = all / 4;
  if (splits < 1) splits = 1;
  sp.slices = (int32_t)((all + splits - 1) / splits);
  sp.splits = (int32_t)((all + sp.slices - 1) / sp.slices);
  sp.gemm_blocks = (uint32_t)(tiles * sp.splits);
  sp.part_ld = (N + 7) / 8 * 8;
  const int64_t per = 4 * (256 / (rank / 8 > 0 ? rank / 8 : 1));  // k that a workgroup takes in four loads a thread
  int64_t shares = (K + per - 1) / per;
  if (shares > 16) shares = 16;
  sp.h_k = (int32_t)(((K + shares - 1) / shares + 7) / 8 * 8);
  sp.h_splits = (int32_t)((K + sp.h_k - 1) / sp.h_k);
  return sp;
}

size_t h_bytes(int64_t rows, int64_t rank, int32_t op) {
  return align_up((size_t)rows * (size_t)((rank + 31) / 32 * 32) * dtype_size(op), 256);
}

struct LoraCopies {
  size_t x, w, a, b;
  size_t total() const { return x + w + a + b; }
};
// which: CVMM_LORA_COPY_* of the operands that are copied
LoraCopies copies_bytes(int64_t rows, int64_t n, int64_t K, int64_t N, int64_t rank, int32_t which) {
  const size_t k8 = (size_t)pad8(K), n8 = (size_t)pad8(N), r8 = (size_t)pad8(rank);
  auto room = [&](int32_t bit, size_t values) { return which & bit ? align_up(values * 2, 256) : 0; };
  return {room(CVMM_LORA_COPY_X, (size_t)rows * k8), room(CVMM_LORA_COPY_WEIGHT, k8 * n8),
          room(CVMM_LORA_COPY_A, (size_t)n * k8 * r8), room(CVMM_LORA_COPY_B, (size_t)n * r8 * n8)};
}

// The operands of a call that are not whole pieces, by their widths or by themselves.
int32_t to_copy(const LoraParams& p) {
  const bool k = p.K % 8 != 0, n = p.N % 8 != 0, r = p.rank % 8 != 0;
  return (k || p.x_ld % 8 != 0 || !al16(p.x) ? CVMM_LORA_COPY_X : 0) |
         (p.w != nullptr && (k || n || !pieces(p.w, 0, p.w_sk, p.w_sn)) ? CVMM_LORA_COPY_WEIGHT : 0) |
         (k || r || !pieces(p.a, p.a_se, p.a_sk, p.a_sr) ? CVMM_LORA_COPY_A : 0) |
         (n || r || !pieces(p.b, p.b_se, p.b_sr, p.b_sn) ? CVMM_LORA_COPY_B : 0);
}

// Matrices [n][d_i][d_j] of any strides in 16-bit values -> whole pieces, zeros in
// the padding, the unit stride's dimension kept; all of a call in one launch (777 rows of
// 1000 -> 518: one launch of 3-4 us, three took 9.4; whole call 30.2 -> 25.3).
struct LoraPad {
  const uint16_t* src;
  uint4* dst;
  int64_t se, su, sv;       // element strides of the matrices, rows and values
  uint32_t n_u, n_v;        // rows and values of a row that there are
  uint32_t rows, pieces_v;  // rows of a copy, pieces of a row
  uint32_t pieces, end;     // pieces in all; the workgroup after the last
};
// Bytes of x up to which it joins that launch (whole calls of 1001 -> 1001, in it / in one
// of its own: 1999 rows 32.6 / 33.7 us, 4000 the same, 16384 102 / 96.5).
constexpr size_t kLoraPadRows = (size_t)6 << 20;
struct LoraPads {
  LoraPad of[4];
  int32_t n;
};

__global__ __launch_bounds__(256) void lora_pad_kernel(const LoraPads p) {
  int j = 0;
  while (j < p.n - 1 && blockIdx.x >= p.of[j].end) ++j;
  const LoraPad q = p.of[j];
  const uint32_t i = (blockIdx.x - (j > 0 ? p.of[j - 1].end : 0u)) * 256u + threadIdx.x;
  if (i >= q.pieces) return;
  const uint32_t row = i / q.pieces_v, v = (i % q.pieces_v) * 8u, u = row % q.rows, e = row / q.rows;
  Chunk16 c;
#pragma unroll
  for (uint32_t k = 0; k < 8; ++k)
    c.s[k] = u < q.n_u && v + k < q.n_v ? q.src[(int64_t)e * q.se + (int64_t)u * q.su + (int64_t)(v + k) * q.sv]
                                        : (uint16_t)0;
  q.dst[i] = c.u;
}

// One more matrix to copy, its pointer and strides those of the copy from here on.
// pad_i: rows of zeros behind the last, too.
void add_pad(LoraPads& all, const void*& q, int64_t& se, int64_t& si, int64_t& sj, int64_t n, int64_t d_i, int64_t d_j,
             char* at, bool pad_i = true) {
  const bool t = pad_i && si == 1 && sj != 1;
  const int64_t n_u = t ? d_j : d_i, n_v = t ? d_i : d_j;
  LoraPad& o = all.of[all.n];
  o.src = (const uint16_t*)q;
  o.dst = (uint4*)at;
  o.se = se;
  o.su = t ? sj : si;
  o.sv = t ? si : sj;
  o.n_u = (uint32_t)n_u;
  o.n_v = (uint32_t)n_v;
  o.rows = (uint32_t)(pad_i ? pad8(n_u) : n_u);
  o.pieces_v = (uint32_t)(pad8(n_v) / 8);
  o.pieces = (uint32_t)n * o.rows * o.pieces_v;
  o.end = (all.n > 0 ? all.of[all.n - 1].end : 0u) + (o.pieces + 255u) / 256u;
  ++all.n;
  q = at;
  se = pad8(d_i) * pad8(d_j);
  si = t ? 1 : pad8(d_j);
  sj = t ? pad8(d_i) : 1;
}

template <typename OpT>
hipError_t launch_fast(const LoraParams& q, void* ws, hipStream_t s) {
  LoraParams p = q;
  p.out_vec = al16(p.out) && p.out_ld % 8 == 0 && p.n_out % 8 == 0;
  p.base_vec = p.base != nullptr && al16(p.base) && p.base_ld % (p.base_dtype == kF32 ? 4 : 8) == 0;
  if (few_rows(p.rows, p.rank) && p.ht == nullptr) {
    LoraSplit sp = few_split(p.rows, p.K, p.N, p.rank);
    sp.h_part = (float*)ws;
    if (p.w != nullptr)
      sp.part = (float*)((char*)ws + align_up((size_t)sp.h_splits * (size_t)(p.rows * p.rank) * 4, 256));
    return launch_lora_few_op<OpT>(p, sp, s);
  }
  p.h = ws;
  const hipError_t e = launch_lora_inner_op<OpT>(p, s);
  if (e != hipSuccess || p.out == nullptr) return e;
  // the projection takes the rows by their order where 32-bit offsets reach them all
  const int64_t wide = p.x_ld > p.h_ld ? p.x_ld : p.h_ld;
  if (p.order != nullptr && p.rows * wide >= ((int64_t)1 << 30) - 8192) p.order = nullptr;
  return launch_lora_gemm_op<OpT>(p, s);
}
}  // namespace

size_t lora_workspace_bytes(int64_t rows, int32_t n, int64_t K, int64_t N, int64_t rank, int32_t op, bool weight,
                            int32_t copied) {
  size_t own = h_bytes(rows, rank, op);
  if (op == kF32) return own;
  if (few_rows(rows, pad8(rank))) {
    const LoraSplit sp = few_split(rows, pad8(K), pad8(N), pad8(rank));
    const size_t few = align_up((size_t)sp.h_splits * (size_t)(rows * pad8(rank)) * 4, 256) +
                       (weight ? (size_t)sp.splits * (size_t)rows * (size_t)sp.part_ld * 4 : 0);
    own = own > few ? own : few;
  }
  if (copied & CVMM_LORA_COPY_ALL) copied = ~0;
  return align_up(own, 256) + copies_bytes(rows, n, K, N, rank, weight ? copied : copied & ~CVMM_LORA_COPY_WEIGHT).total();
}

hipError_t launch_lora(const LoraParams& q, int32_t op, void* ws, size_t ws_bytes, hipStream_t s) {
  LoraParams p = q;
  p.n_out = p.N;
  p.rank_out = p.rank;
  LoraPads pads{};
  void* x_copy = nullptr;  // x's copy where it takes a launch of its own
  if (op != kF32 && !fast_ok(p, op)) {
    // copies of whole pieces, where there is room for them
    const size_t own = lora_workspace_bytes(p.rows, p.n, p.K, p.N, p.rank, op, p.w != nullptr, 0);
    const int32_t which = to_copy(p);
    const LoraCopies c = copies_bytes(p.rows, p.n, p.K, p.N, p.rank, which);
    // (what the copies' grids and 32-bit indices hold)
    constexpr size_t kMost = (size_t)1 << 34;
    if (c.x < kMost && c.w < kMost && c.a < kMost && c.b < kMost && ws_bytes >= own + c.total()) {
      char* at = (char*)ws + own;
      int64_t se = 0;
      if (which & CVMM_LORA_COPY_X) {
        if (c.x <= kLoraPadRows) {
          int64_t unit = 1;
          add_pad(pads, p.x, se, p.x_ld, unit, 1, p.rows, p.K, at, false);
        } else {
          p.x = x_copy = at;
          p.x_ld = pad8(p.K);
        }
      }
      at += c.x;
      se = 0;
      if (which & CVMM_LORA_COPY_WEIGHT) add_pad(pads, p.w, se, p.w_sk, p.w_sn, 1, p.K, p.N, at);
      at += c.w;
      if (which & CVMM_LORA_COPY_A) add_pad(pads, p.a, p.a_se, p.a_sk, p.a_sr, p.n, p.K, p.rank, at);
      at += c.a;
      if (which & CVMM_LORA_COPY_B) add_pad(pads, p.b, p.b_se, p.b_sr, p.b_sn, p.n, p.rank, p.N, at);
      p.K = pad8(p.K);
      p.N = pad8(p.N);
      p.rank = pad8(p.rank);
      p.h_ld = (p.rank + 31) / 32 * 32;
    }
  }
  if (!fast_ok(p, op)) {
    // (matrices past 32-bit offsets too, copied or not: the general kernels store up to N
    // and the rank, so they get the call's own sizes and operands, and nothing is copied)
    p = q;
    p.h = ws;
    if (op == kBF16) return launch_general<bf16_t>(p, s);
    if (op == kF16) return launch_general<f16_t>(p, s);
    return launch_general<float>(p, s);
  }
  if (x_copy != nullptr) {
    const hipError_t e = launch_pad_rows(q.x, op, q.x_ld, q.rows, q.K, nullptr, 0, op, x_copy, s);
    if (e != hipSuccess) return e;
  }
  if (pads.n > 0) {
    hipLaunchKernelGGL(lora_pad_kernel, dim3(pads.of[pads.n - 1].end), dim3(256), 0, s, pads);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return op == kBF16 ? launch_fast<bf16_t>(p, ws, s) : launch_fast<f16_t>(p, ws, s);
}

// ---------------------------------------------------------------------------
// The adapters' gradients: dA_i = sum_p x[p]^T u[p], dB_i = sum_p h[p]^T g[p]
// over the rows p of adapter i, in the sorted order in which u and h stand
// transposed.  One block of 64 x 64 values per workgroup and share of the
// adapter's rows; the shares are added in order by a second launch.
// ---------------------------------------------------------------------------
template <typename OpT>
__global__ __launch_bounds__(256) void lora_wgrad_kernel(const LoraWgradParams p) {
  using S = LoraSlice<OpT>;
  __shared__ __attribute__((aligned(16))) OpT as[kLoraTile * S::LD], bs[kLoraTile * S::LD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // dA's blocks, then dB's: wide dimension (columns of x or g) by rank
  const int64_t bi = (p.d_in + 63) / 64;
  const bool in = (int64_t)blockIdx.x < bi;
  const int64_t w0 = (in ? blockIdx.x : blockIdx.x - bi) * 64, r0 = (int64_t)blockIdx.y * 64;
  if ((in ? p.ga : p.gb) == nullptr) return;
  const int32_t e = blockIdx.z / p.shares, share = blockIdx.z % p.shares;
  const int64_t lo = e > 0 && p.offsets[e - 1] > 0 ? p.offsets[e - 1] : 0;
  const int64_t hi = p.offsets[e] < p.rows ? p.offsets[e] : p.rows;
  const int64_t len = hi > lo ? hi - lo : 0;
  const int64_t from = lo + len * share / p.shares, to = lo + len * (share + 1) / p.shares;
  const OpT* rows = (const OpT*)(in ? p.x : p.g);
  const int64_t ld = in ? p.x_ld : p.g_ld, width = in ? p.d_in : p.d_out;
  const OpT* t = (const OpT*)(in ? p.ut : p.ht) + r0 * p.t_ld;
  f32x4_t acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int64_t p0 = from; p0 < to; p0 += S::BK) {
    __syncthreads();
    // wide operand: as[c][k], k = sorted position; thin operand: bs[r][k]
#pragma unroll
    for (int j = 0; j < S::PER; ++j) {
      const int i = j * 256 + (int)threadIdx.x, c = i % 64, k = i / 64;
      OpT v = from_f32<OpT>(0.f);
      if (p0 + k < to && w0 + c < width) {
        const int64_t row = p.order[p0 + k];
        if (row >= 0 && row < p.rows) v = rows[row * ld + w0 + c];
      }
      as[c * S::LD + k] = v;
    }
    OpT vb[S::PER];
    lora_load(t + p0, p.t_ld, 1, p.rank - r0, to - p0, vb);
    lora_store(bs, true, vb);
    __syncthreads();
    lora_mfma(acc, as, bs, wave, lane);
  }
  const int64_t total = p.d_in * p.rank * p.n;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int64_t c = w0 + wave * 16 + (lane >> 4) * 4 + v, r = r0 + j * 16 + (lane & 15);
      if (c >= width || r >= p.rank) continue;
      const int64_t at = in ? (e * p.d_in + c) * p.rank + r : (e * p.rank + r) * p.d_out + c;
      if (p.shares > 1)
        p.part[(int64_t)share * (total + p.d_out * p.rank * p.n) + (in ? at : total + at)] = acc[j][v];
      else
        store_from_f32(in ? p.ga : p.gb, p.g_dtype, at, acc[j][v]);
    }
  }
}

__global__ __launch_bounds__(256) void lora_wgrad_sum_kernel(const LoraWgradParams p) {
  const int64_t na = p.d_in * p.rank * p.n, total = na + p.d_out * p.rank * p.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    if ((i < na ? p.ga : p.gb) == nullptr) continue;
    float s = 0.f;
#pragma unroll 4
    for (int32_t q = 0; q < p.shares; ++q) s += p.part[q * total + i];
    if (i < na) store_from_f32(p.ga, p.g_dtype, i, s);
    else store_from_f32(p.gb, p.g_dtype, i - na, s);
  }
}

static int32_t lora_wgrad_shares(int64_t rows, int32_t n, int64_t d_in, int64_t d_out, int64_t rank) {
  const int64_t blocks = ((d_in + 127) / 128 + (d_out + 127) / 128) * ((rank + 63) / 64) * n;
  // (8192 rows, 4 adapters of rank 32, 1024 -> 1024, forward and backward: 107 us; for
  // 128 workgroups 110, for 1024 119)
  int64_t s = 1;
  while (s < 64 && blocks * s < 256 && rows / (n * s) > 128) s *= 2;
  return (int32_t)s;
}

static size_t wgrad_part_bytes(int64_t rows, int32_t n, int64_t d_in, int64_t d_out, int64_t rank) {
  const int32_t s = lora_wgrad_shares(rows, n, d_in, d_out, rank);
  return s > 1 ? align_up((size_t)s * (size_t)n * (size_t)rank * (size_t)(d_in + d_out) * 4, 256) : 0;
}

size_t lora_wgrad_workspace_bytes(int64_t rows, int32_t n, int64_t d_in, int64_t d_out, int64_t rank, bool copied) {
  return wgrad_part_bytes(rows, n, d_in, d_out, rank) +
         (copied ? align_up((size_t)rows * (size_t)pad8(d_in) * 2, 256) + (size_t)rows * (size_t)pad8(d_out) * 2 : 0);
}

hipError_t launch_lora_wgrad(const LoraWgradParams& q, int32_t op, size_t ws_bytes, hipStream_t s) {
  LoraWgradParams p = q;
  p.shares = lora_wgrad_shares(p.rows, p.n, p.d_in, p.d_out, p.rank);
  auto rows_ok = [&] {
    return (p.ga == nullptr || (al16(p.x) && p.x_ld % 8 == 0 && p.d_in % 8 == 0)) &&
           (p.gb == nullptr || (al16(p.g) && p.g_ld % 8 == 0 && p.d_out % 8 == 0));
  };
  bool fast = op != kF32 && p.t_ld % 8 == 0 && al16(p.ht) && al16(p.ut);
  if (fast && !rows_ok()) {
    // rows of whole pieces, where there is room for the copies
    fast = ws_bytes >= lora_wgrad_workspace_bytes(p.rows, p.n, p.d_in, p.d_out, p.rank, true) &&
           p.rows * ((p.d_in > p.d_out ? p.d_in : p.d_out) + 8) < ((int64_t)1 << 33);
    char* at = (char*)p.part + wgrad_part_bytes(p.rows, p.n, p.d_in, p.d_out, p.rank);
    if (fast && p.ga != nullptr) {
      const hipError_t e = launch_pad_rows(p.x, op, p.x_ld, p.rows, p.d_in, nullptr, 0, op, at, s);
      if (e != hipSuccess) return e;
      p.x = at;
      p.x_ld = pad8(p.d_in);
    }
    at += align_up((size_t)p.rows * (size_t)pad8(p.d_in) * 2, 256);
    if (fast && p.gb != nullptr) {
      const hipError_t e = launch_pad_rows(p.g, op, p.g_ld, p.rows, p.d_out, nullptr, 0, op, at, s);
      if (e != hipSuccess) return e;
      p.g = at;
      p.g_ld = pad8(p.d_out);
    }
  }
  const int64_t bx = (p.d_in + 63) / 64 + (p.d_out + 63) / 64, by = (p.rank + 63) / 64, bz = (int64_t)p.n * p.shares;
  if (bx > 0x7fffffffll || bz > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)bx, (unsigned)by, (unsigned)bz);
  if (fast) {
    const hipError_t e = op == kBF16 ? launch_lora_wgrad_op<bf16_t>(p, s) : launch_lora_wgrad_op<f16_t>(p, s);
    if (e != hipSuccess) return e;
  } else if (op == kBF16) hipLaunchKernelGGL((lora_wgrad_kernel<bf16_t>), grid, dim3(256), 0, s, p);
  else if (op == kF16) hipLaunchKernelGGL((lora_wgrad_kernel<f16_t>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((lora_wgrad_kernel<float>), grid, dim3(256), 0, s, p);
  if (p.shares > 1) {
    const int64_t total = (p.d_in + p.d_out) * p.rank * p.n;
    const int64_t wg = (total + 1023) / 1024;
    hipLaunchKernelGGL(lora_wgrad_sum_kernel, dim3((unsigned)(wg < 4096 ? wg : 4096)), dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

}  // namespace cvmm
