// Dense product with an epilogue:
//   v[m, n] = sum over k of A[m, k] * B[n, k] (int8: times As[m] * Bs[n]) + bias[n]
//   C[m, n] = scale * act(v[m, n]) + R[m, n];  gated: scale * act(v[m, n]) * v[m, N + n] + R[m, n].
// Sums, and everything behind them, are fp32 (int8: the sum is int32 and exact); a result is rounded once.  A K block is 128 bytes of a row,
// 64 values of 16 bits or 128 of int8, two matrix instructions of every 16 x 16 sums.  B (the weight) is the instructions' first
// operand: a lane holds four neighbouring columns of C for one token.
#pragma once
#include <type_traits>

#include "fp8.h"
#include "gemm.h"
#include "tiles.h"

namespace lo {

struct DenseArgs {
  const int8_t *A, *B;
  const float *As, *Bs;
  const void *bias, *R;
  void *C;
  void *part;        // [splits][M][pitch] sums over parts of K, fp32 or int32; gated: the other projection's half a pitch on
  int64_t M, N, rs;  // rs: R's row stride, in values
  int32_t lda, ldb;  // bytes
  int32_t K;         // bytes of a row, a multiple of 16
  int32_t act, gated, bias_f32, out;
  float scale;
  int32_t KB, m_tiles, n_tiles, splits, pitch;
};
constexpr int kBlockK = 128; // bytes

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// The operands' types and the matrix instructions: sixteen bytes a lane of 16 rows of either operand, 64 bytes of K, into the 16 x 16 sums.
template <int DT> struct Operand {
  typedef v4f Acc;
  typedef float Sum;
  static __device__ __forceinline__ Acc mfma(const v4i a, const v4i b, const Acc c) {
    if constexpr (DT == LO_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <> struct Operand<LO_I8> {
  typedef v4i Acc;
  typedef int Sum;
  static __device__ __forceinline__ Acc mfma(const v4i a, const v4i b, const Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float load_value(const void *p, int type, int64_t at) {
  if (type == LO_F32) return static_cast<const float *>(p)[at];
  const uint16_t h = static_cast<const uint16_t *>(p)[at];
  return type == LO_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}
// The same in two halves, the load and what needs its value.
__device__ __forceinline__ uint32_t value_bits(const void *p, int type, int64_t at) {
  return type == LO_F32 ? static_cast<const uint32_t *>(p)[at] : static_cast<const uint16_t *>(p)[at];
}
__device__ __forceinline__ float value_of(uint32_t v, int type) {
  return type == LO_F32 ? __builtin_bit_cast(float, v) : type == LO_BF16 ? bf16_to_f32(static_cast<uint16_t>(v)) : f16_to_f32(static_cast<uint16_t>(v));
}
__device__ __forceinline__ uint16_t to_half(int type, float v) { return type == LO_BF16 ? f32_to_bf16(v) : f32_to_f16(v); }
__device__ __forceinline__ void store_value(void *p, int type, int64_t at, float v) {
  if (type == LO_F32) static_cast<float *>(p)[at] = v;
  else static_cast<uint16_t *>(p)[at] = to_half(type, v);
}
__device__ __forceinline__ float activate(int act, float v) { return act == LO_ACT_SILU ? silu_f32(v) : act == LO_ACT_GELU ? gelu_f32(v) : v; }
// A sum's value before the activation; n counts B's rows.
template <class T> __device__ __forceinline__ float dense_value(const DenseArgs &a, T sum, int64_t m, int64_t n) {
  float v = static_cast<float>(sum);
  if (a.As) v = v * a.As[m] * a.Bs[n];
  return a.bias ? v + load_value(a.bias, a.bias_f32 ? LO_F32 : a.out, n) : v;
}
__device__ __forceinline__ float dense_result(const DenseArgs &a, float v, int64_t m, int64_t n) {
  return a.R ? __builtin_fmaf(a.scale, v, load_value(a.R, a.out, m * a.rs + n)) : a.scale * v;
}

// ---- up to 16 tokens ---------------------------------------------------------------------------------------------------------
// A workgroup takes 16 / C rows of B (gated: half of them of either projection) and all tokens, at most 16 / C; its waves share K and add
// their sums up through LDS, in the same order every time.  With C > 1 the 16 rows of a matrix instruction's operands are C K blocks of the
// workgroup's rows, and of the tokens; of its 16 x 16 sums those on the diagonal of C x C squares count, and are added up with the waves'.
// Weights are read once, straight into registers, U K blocks of a wave in flight.  HBM bounds it where there are rows enough (one token, gated 2048 x 7168 bf16:
// 59 MB in 14.4 us; int8 29 MB in 8.8; 7168 x 2048 bf16 29 MB in 8.6), else the launch and one round trip (256 x 7168 bf16 4.3 us, 128 x 2048 3.5).
template <int DT, int U>
__global__ __launch_bounds__(512) void gemm_dense_few_kernel(const DenseArgs a, int lg) {
  typedef Operand<DT> Op;
  __shared__ __attribute__((aligned(16))) int red[8][256]; // [wave][16 of tokens][16 of B's rows]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int C = 1 << lg, width = 16 >> lg, half = a.gated ? width >> 1 : width; // rows of B; columns of the result
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * half;
  const int row = r & (width - 1), block = r >> (4 - lg); // of the workgroup, of the C
  int64_t nb = n0 + (row < half ? row : row - half);
  nb = (nb < a.N ? nb : a.N - 1) + (row < half ? 0 : a.N); // (rows and tokens past the end: the last one again, not stored)
  const int at0 = block * kBlockK + q * 16;
  const int8_t *const pb = a.B + nb * a.ldb + at0;
  const int8_t *const pa = a.A + (row < a.M ? row : a.M - 1) * a.lda + at0;
  // What a result takes beside the sums, the thread's first one's in front of the K blocks.
  struct Beside {
    float as, bs[2];
    uint32_t bias[2], add;
  };
  const int count = static_cast<int>(a.M) * half, lgh = 4 - lg - (a.gated ? 1 : 0);
  const auto fetch = [&](int i) __attribute__((always_inline)) {
    Beside b = {};
    const int64_t m = i >> lgh, n = n0 + (i & (half - 1));
    if (i >= count || n >= a.N) return b;
    if constexpr (DT == LO_I8) b.as = a.As[m], b.bs[0] = a.Bs[n];
    if (a.bias) b.bias[0] = value_bits(a.bias, a.bias_f32 ? LO_F32 : a.out, n);
    if (a.gated) {
      if constexpr (DT == LO_I8) b.bs[1] = a.Bs[n + a.N];
      if (a.bias) b.bias[1] = value_bits(a.bias, a.bias_f32 ? LO_F32 : a.out, n + a.N);
    }
    if (a.R) b.add = value_bits(a.R, a.out, m * a.rs + n);
    return b;
  };
  Beside beside = fetch(threadIdx.x);
  typename Op::Acc acc = {};
  const int step = C * kBlockK;
  for (int k0 = wave * step; k0 < a.K; k0 += waves * U * step) {
    v4i w[U][2], x[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + u * waves * step + h * 64, at = k + at0 < a.K ? k : -at0; // past the row's end: its first bytes, cleared below
        w[u][h] = __builtin_nontemporal_load(reinterpret_cast<const v4i *>(pb + at));
        x[u][h] = *reinterpret_cast<const v4i *>(pa + at);
      }
    }
    __builtin_amdgcn_sched_barrier(0); // (all of them asked for)
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = k0 + u * waves * step + h * 64 + at0 < a.K;
        acc = Op::mfma(in ? w[u][h] : v4i{}, in ? x[u][h] : v4i{}, acc);
      }
    }
  }
  *reinterpret_cast<v4i *>(&red[wave][r * 16 + 4 * q]) = __builtin_bit_cast(v4i, acc);
  __syncthreads();
  for (int i = threadIdx.x; i < count;) {
    const int m = i >> lgh, c = i & (half - 1);
    const int64_t n = n0 + c;
    const auto value = [&](int col, int p) __attribute__((always_inline)) {
      typename Op::Sum sum = 0;
      for (int j = 0; j < waves; ++j)
        for (int k = 0; k < C; ++k) sum += __builtin_bit_cast(typename Op::Sum, red[j][(k * width + m) * 16 + k * width + col]);
      float v = static_cast<float>(sum);
      if constexpr (DT == LO_I8) v = v * beside.as * beside.bs[p];
      return a.bias ? v + value_of(beside.bias[p], a.bias_f32 ? LO_F32 : a.out) : v;
    };
    if (n < a.N) {
      float v = activate(a.act, value(c, 0));
      if (a.gated) v *= value(c + half, 1);
      store_value(a.C, a.out, m * a.N + n, a.R ? __builtin_fmaf(a.scale, v, value_of(beside.add, a.out)) : a.scale * v);
    }
    i += blockDim.x;
    if (i < count) beside = fetch(i);
  }
}

// ---- tiles -----------------------------------------------------------------------------------------------------------------
// Both operands go to LDS by direct loads, a K block to a stage of a ring; 16-byte pieces of a row are swizzled by the row.  A gated
// product's fragments of 16 rows hold eight of either projection, so that the epilogue finds both values of a column in one wave.
//
// What bounds them: the largest sizes the matrix cores and the clock under their load (8192 x 4096 x 7168 bf16 with bias and residual 348 to 367 us, 1.31 to
// 1.38 PFLOP/s; the library's plain product 365; int8 4096 x 4096 x 7168 87 to 91 us, 2.7 POP/s, library 105); all others the copies, which bring a CU 65 to 70 bytes a ns
// whatever the ring's depth (the products or the LDS reads taken away, a K block of 128 x 128 takes 0.45 to 0.50 us in place of 0.53), since operands come into
// each XCD's L2 once and several CUs wait for the same lines: copies of lines that are there run at 130.  Larger tiles copy less and fill
// fewer CUs; K in another order for each tile gained nothing, nor did one sharer's reading ahead into L2 (96 x 96: a K block 0.40 us, with all
// operands there 0.33, which is the LDS's).  32 x 32 instructions (400 / 364 us for the largest size), waves of 128 x 128 (438) and a third
// place for the tokens' part (379) were slower.
constexpr int dense_staging(int tn, int wm, int wn, int rows) { return wm * wn * rows * (tn / wn * 4 + 16); } // bytes
// Token fragments of a wave that the epilogue turns around at a time: all of them, or half where they do not fit into the ring.
constexpr int dense_round(int tm, int tn, int wm, int wn, int ring) {
  return (dense_staging(tn, wm, wn, tm / wm) <= ring || tm / wm / 16 % 2 ? tm : tm / 2) / wm / 16;
}
constexpr int dense_lds(int tm, int tn, int wm, int wn, int ring, bool part) {
  const int staging = part ? 0 : dense_staging(tn, wm, wn, dense_round(tm, tn, wm, wn, ring) * 16);
  return ring > staging ? ring : staging;
}

// What a workgroup multiplies, and how its waves' copies find it.
template <int TM, int TN, int WM, int WN, bool PART> struct DenseTileOf {
  static constexpr int kWaves = WM * WN, kA = TM / 8 / kWaves, kB = TN / 8 / kWaves; // 1 KB copies of a K block, of a wave
  static_assert(TM / 8 % kWaves == 0 && TN / 8 % kWaves == 0 && TM / WM % 16 == 0 && TN / WN % 16 == 0, "tile");
  int lane, r, q, wave, wm, wn, split, rows, cols, KB, tail;
  int64_t m0, n0;
  brsrc A, B[2]; // B's rows; gated: of the two projections
  int voff[kA + kB];
  int lds[2]; // the lane's pieces of a fragment
  __device__ __forceinline__ bool start(const DenseArgs &a, int group_m) {
    int mt, nt;
    split = PART ? blockIdx.y : 0;
    if (!dense_tile(blockIdx.x, a.m_tiles, a.n_tiles, group_m, mt, nt)) return false;
    mt = __builtin_amdgcn_readfirstlane(mt), nt = __builtin_amdgcn_readfirstlane(nt); // (a division's results: the descriptors go to scalar registers)
    lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const int first = PART ? static_cast<int>(static_cast<int64_t>(a.KB) * split / a.splits) : 0;
    KB = (PART ? static_cast<int>(static_cast<int64_t>(a.KB) * (split + 1) / a.splits) : a.KB) - first;
    const int width = a.gated ? TN / 2 : TN; // columns of C
    m0 = static_cast<int64_t>(mt) * TM, n0 = static_cast<int64_t>(nt) * width;
    rows = static_cast<int>(a.M - m0 < TM ? a.M - m0 : TM), cols = static_cast<int>(a.N - n0 < width ? a.N - n0 : width);
    const int left = a.K - first * kBlockK; // bytes of a row from this part on
    A = make_rsrc(a.A + m0 * a.lda + first * kBlockK, static_cast<uint32_t>((rows - 1) * a.lda + left));
#pragma unroll
    for (int p = 0; p < 2; ++p) B[p] = make_rsrc(a.B + (n0 + (a.gated && p ? a.N : 0)) * a.ldb + first * kBlockK, static_cast<uint32_t>((cols - 1) * a.ldb + left));
    const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
    for (int j = 0; j < kA; ++j) voff[j] = ((wave * kA + j) * 8 + (lane >> 3)) * a.lda + piece;
#pragma unroll
    for (int j = 0; j < kB; ++j) {
      const int g = wave * kB + j; // eight rows; a fragment is two of them
      voff[kA + j] = ((a.gated ? g >> 1 : g) * 8 + (lane >> 3)) * a.ldb + piece;
    }
    // Past a row's end (in its last K block, where K is no multiple of 128 bytes) a piece's offset is past the extents, which end at 2^30 at the most.
    tail = (KB - 1) * kBlockK + piece < left ? 0 : 1 << 30;
#pragma unroll
    for (int h = 0; h < 2; ++h) lds[h] = r * kBlockK + (((h * 4 + q) ^ (r & 7)) * 16);
    return true;
  }
  // Copy c of K block kb.  What lies past the extents is written as zero: rows past the end, and past the last K block all of it (the copies,
  // which the waits count, fetch nothing).
  __device__ __forceinline__ void copy(int c, int kb, int8_t *to_a, int8_t *to_b) const {
    const int at = voff[c] + (kb < KB - 1 ? 0 : kb == KB - 1 ? tail : 1 << 30), soff = kb < KB ? kb * kBlockK : 0;
    if (c < kA) copy16(A, to_a + (wave * kA + c) * 1024, at, soff);
    else copy16((wave * kB + c - kA) & 1 ? B[1] : B[0], to_b + (wave * kB + c - kA) * 1024, at, soff);
  }
};

// Rows of COLS fp32 values in a wave's LDS, COLS * 4 + 16 bytes apart.  Gated: eights of either projection in turn.
// Activates them where they lie (gated: the gate's, times the other's).
template <int ROWS, int COLS, bool GATED> __device__ __forceinline__ void dense_activate(int act, int8_t *stg, int lane) {
  constexpr int kFours = COLS / (GATED ? 8 : 4); // of a row
#pragma unroll 2
  for (int i = lane; i < ROWS * kFours; i += 64) {
    const int k = i % kFours, slot = GATED ? (k >> 1) * 16 + (k & 1) * 4 : k * 4;
    v4f *const p = reinterpret_cast<v4f *>(stg + i / kFours * (COLS * 4 + 16) + slot * 4);
    v4f v = *p;
    if (act == LO_ACT_SILU) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = silu_f32(v[j]);
    } else if (act == LO_ACT_GELU) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = gelu_f32(v[j]);
    }
    if constexpr (GATED) v = v * p[2];
    *p = v;
  }
  lds_order();
}
// Stores them, scaled and the residual added, in whole pieces of 16 bytes: `in` rows of C from value c0 on (of R from r0), `left` columns.
// EARLY: so many of a lane's first pieces of R are in `early`.
template <int ROWS, int COLS, bool GATED, int OUT, int EARLY>
__device__ __forceinline__ void dense_rows(const DenseArgs &a, const int8_t *stg, int lane, int64_t c0, int64_t r0, int in, int left, const v4i *early) {
  constexpr int V = OUT == LO_F32 ? 4 : 8, kLanes = (GATED ? COLS / 2 : COLS) / V, kTurns = (ROWS * kLanes + 63) / 64, U = kTurns < 4 ? kTurns : 4;
  typedef std::conditional_t<OUT == LO_F32, v4f, v8u16> Piece;
  typedef std::conditional_t<OUT == LO_F32, float, uint16_t> Value;
#pragma unroll 1
  for (int first = 0; first < kTurns; first += U) {
    Piece add[U] = {};
    if (a.R) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = (first + u) * 64 + lane, row = i / kLanes, c = i % kLanes * V;
        if (u < EARLY && first == 0) add[u] = __builtin_bit_cast(Piece, early[u]);
        else if (row < in && c < left) add[u] = *reinterpret_cast<const Piece *>(static_cast<const Value *>(a.R) + r0 + row * a.rs + c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (first + u) * 64 + lane, row = i / kLanes, c = i % kLanes * V;
      if (row >= in || c >= left) continue;
      const v4f *const p = reinterpret_cast<const v4f *>(stg + row * (COLS * 4 + 16) + (GATED ? (c >> 3) * 16 + (c & 7) : c) * 4);
      Piece o;
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const v4f v = p[j / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (OUT == LO_F32) o[j + k] = a.R ? __builtin_fmaf(a.scale, v[k], add[u][j + k]) : a.scale * v[k];
          else o[j + k] = from_f32<OUT>(a.R ? __builtin_fmaf(a.scale, v[k], to_f32<OUT>(add[u][j + k])) : a.scale * v[k]);
        }
      }
      *reinterpret_cast<Piece *>(static_cast<Value *>(a.C) + c0 + row * a.N + c) = o;
    }
  }
}

// Whether rows of C, and of R, begin on 16 bytes.
__device__ __forceinline__ bool dense_whole(const DenseArgs &a) {
  const int size = a.out == LO_F32 ? 4 : 2;
  return ((a.N * size | (a.R ? a.rs * size : 0) | static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.C) | reinterpret_cast<uintptr_t>(a.R))) & 15) == 0;
}

// What the epilogue reads beside the sums, as it lies, so that small tiles ask for it in front of the K blocks and save its round trip (int8 24 x 7168 x 2048 with
// a residual 7.3 -> 7.0 us; 96 x 96 and more gain nothing).
// ADD: pieces of the residual that a lane adds first, in dense_rows' order, of the ROWS rows that the epilogue turns around first.
template <int DT, int FM, int FN, int ADD, int ROWS> struct DenseBeside {
  float as[FM], bs[FN][4];
  uint32_t bias[FN][4];
  v4i add[ADD > 0 ? ADD : 1];
  template <class TILE> __device__ __forceinline__ void load(const DenseArgs &a, const TILE &t) {
    const int64_t nw = t.n0 + t.wn * (a.gated ? FN * 8 : FN * 16);
    const auto columns = [&](auto &&f) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t c = nw + (a.gated ? n * 8 + 4 * (t.q & 1) : n * 16 + 4 * t.q) + i;
          f(n, i, (c < a.N ? c : a.N - 1) + (a.gated && t.q >= 2 ? a.N : 0));
        }
    };
    if constexpr (DT == LO_I8) columns([&](int n, int i, int64_t at) __attribute__((always_inline)) { bs[n][i] = a.Bs[at]; });
    if (!a.bias) columns([&](int n, int i, int64_t) __attribute__((always_inline)) { bias[n][i] = 0; });
    else if (a.bias_f32 || a.out == LO_F32) columns([&](int n, int i, int64_t at) __attribute__((always_inline)) { bias[n][i] = value_bits(a.bias, LO_F32, at); });
    else columns([&](int n, int i, int64_t at) __attribute__((always_inline)) { bias[n][i] = value_bits(a.bias, LO_BF16, at); });
    if constexpr (DT == LO_I8) {
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        const int row = (t.wm * FM + m) * 16 + t.r;
        as[m] = a.As[t.m0 + (row < t.rows ? row : t.rows - 1)];
      }
    }
    if constexpr (ADD > 0) {
      if (!a.R || a.gated || !dense_whole(a)) return;
      const int row0 = t.wm * FM * 16, in = t.rows - row0, left = t.cols - t.wn * FN * 16;
      const int64_t r0 = (t.m0 + row0) * a.rs + nw;
      const auto pieces = [&](auto values) __attribute__((always_inline)) {
        constexpr int V = decltype(values)::value, kLanes = FN * 16 / V;
#pragma unroll
        for (int u = 0; u < ADD; ++u) {
          const int i = u * 64 + t.lane, row = i / kLanes, c = i % kLanes * V;
          add[u] = v4i{};
          if (row < ROWS && row < in && c < left) add[u] = *reinterpret_cast<const v4i *>(static_cast<const int8_t *>(a.R) + (r0 + row * a.rs + c) * (16 / V));
        }
      };
      if (a.out == LO_F32) pieces(std::integral_constant<int, 4>{});
      else pieces(std::integral_constant<int, 8>{});
    }
  }
};

// What becomes of a workgroup's sums.  PART: they go to a.part.  RING: bytes of LDS that are free by now.
template <int DT, int TM, int TN, int WM, int WN, bool PART, int RING, int FM, int FN, int ADD, int ROWS>
__device__ __forceinline__ void dense_finish(const DenseArgs &a, const DenseTileOf<TM, TN, WM, WN, PART> &t, typename Operand<DT>::Acc (&acc)[FM][FN],
                                             const DenseBeside<DT, FM, FN, ADD, ROWS> &b, int8_t *smem) {
  constexpr int kCols = TN / WN; // B's rows of a wave
  if constexpr (PART) {
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int mr = t.wm * (TM / WM) + m * 16 + t.r;
      int *const row = static_cast<int *>(a.part) + (t.split * a.M + t.m0 + mr) * a.pitch + t.n0;
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const int c = a.gated ? (t.wn * kCols + n * 16) / 2 + 4 * (t.q & 1) : t.wn * kCols + n * 16 + 4 * t.q;
        if (mr < t.rows && c < t.cols) *reinterpret_cast<v4i *>(row + c + (a.gated && t.q >= 2 ? a.pitch / 2 : 0)) = __builtin_bit_cast(v4i, acc[m][n]);
      }
    }
  } else {
    // A wave turns its tokens around in LDS, kRound fragments of them at a time, in fp32 (its own part; LDS operations of a wave execute in
    // order), and stores whole pieces of rows, activated and the residual added: 16 bytes a lane, or, where rows of either do not begin on 16
    // bytes, a value a lane, which takes a round of 256 x 256 tiles 15 to 25 us more (8192 x 4095 x 7168 bf16 389 us, x 4096 354; 4779 x 3354 x 768 71, x 3360 40;
    // int8 8005 x 3861 x 512 79, x 3864 38; gated 1531 x 767 x 2048 fp16 27.6, x 768 21.3; nothing in parts of K, 333 x 577 x 7168 16.0 and x 576 16.0).
    constexpr int kPitch = kCols * 4 + 16, kRound = dense_round(TM, TN, WM, WN, RING), kRows = kRound * 16;
    int8_t *const stg = smem + t.wave * kRows * kPitch;
    const bool whole = dense_whole(a);
    const int of_c = t.wn * (a.gated ? kCols / 2 : kCols); // this wave's first column of C
    const int64_t nw = t.n0 + of_c;
    const int left = t.cols - of_c;
    float bias[FN][4];
    const auto convert = [&](auto type) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) bias[n][i] = value_of(b.bias[n][i], decltype(type)::value);
    };
    if (a.bias_f32 || a.out == LO_F32) convert(std::integral_constant<int, LO_F32>{});
    else if (a.out == LO_BF16) convert(std::integral_constant<int, LO_BF16>{});
    else convert(std::integral_constant<int, LO_F16>{});
    const auto each = [&](auto gated, auto early, auto type, int64_t c0, int64_t r0, int in) __attribute__((always_inline)) {
      constexpr bool kGated = decltype(gated)::value;
      dense_rows<kRows, kCols, kGated, decltype(type)::value, !kGated && decltype(early)::value ? ADD : 0>(a, stg, t.lane, c0, r0, in, left, b.add);
    };
    const auto of_type = [&](auto gated, auto early, int64_t c0, int64_t r0, int in) __attribute__((always_inline)) {
      if (a.out == LO_BF16) each(gated, early, std::integral_constant<int, LO_BF16>{}, c0, r0, in);
      else if (a.out == LO_F16) each(gated, early, std::integral_constant<int, LO_F16>{}, c0, r0, in);
      else each(gated, early, std::integral_constant<int, LO_F32>{}, c0, r0, in);
    };
    static_assert(ADD == 0 || (FM == kRound && ROWS == kRows), "the residual's first pieces are of the only round");
#pragma unroll
    for (int round = 0; round < FM / kRound; ++round) {
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        if (m / kRound != round) continue;
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          v4f o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[i] = static_cast<float>(acc[m][n][i]);
            if constexpr (DT == LO_I8) o[i] = o[i] * b.as[m] * b.bs[n][i];
            if (a.bias) o[i] += bias[n][i];
          }
          *reinterpret_cast<v4f *>(stg + (m % kRound * 16 + t.r) * kPitch + (n * 16 + 4 * t.q) * 4) = o;
        }
      }
      lds_order();
      const int row0 = t.wm * (TM / WM) + round * kRows, in = t.rows - row0 < kRows ? t.rows - row0 : kRows;
      const int64_t c0 = (t.m0 + row0) * a.N + nw, r0 = (t.m0 + row0) * a.rs + nw;
      if (a.gated) dense_activate<kRows, kCols, true>(a.act, stg, t.lane);
      else if (a.act != LO_ACT_NONE) dense_activate<kRows, kCols, false>(a.act, stg, t.lane);
      if (whole && a.gated) {
        of_type(std::true_type{}, std::false_type{}, c0, r0, in);
      } else if (whole) {
        of_type(std::false_type{}, std::integral_constant<bool, (ADD > 0)>{}, c0, r0, in);
      } else {
#pragma unroll 1
        for (int i = t.lane; i < kRows * kCols; i += 64) {
          const int row = i / kCols, slot = i % kCols, c = a.gated ? (slot >> 4) * 8 + (slot & 7) : slot;
          if (row >= in || c >= left || (a.gated && (slot & 8))) continue;
          const float v = *reinterpret_cast<const float *>(stg + row * kPitch + slot * 4);
          store_value(a.C, a.out, c0 + row * a.N + c, dense_result(a, v, t.m0 + row0 + row, nw + c));
        }
      }
      lds_order();
    }
  }
}

// A wave holds its fragments of a whole K block in registers, and the next one's are read while they are multiplied: the workgroup meets once a
// K block, when the next one has landed and everybody's reads of this one are done, so that the ring is refilled from there on and an LDS
// round trip lies under a K block's products.
template <int DT, int TM, int TN, int WM, int WN, int ST, bool PART>
__global__ __launch_bounds__(WM * WN * 64) void gemm_dense_ring_kernel(const DenseArgs a, int group_m) {
  typedef Operand<DT> Op;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16; // fragments of a wave: tokens, weights
  constexpr int kStage = (TM + TN) * kBlockK;
  DenseTileOf<TM, TN, WM, WN, PART> t;
  constexpr int kCopies = t.kA + t.kB; // of a stage
  static_assert(ST >= 2, "ring");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  if (!t.start(a, group_m)) return;
  auto copy = [&](int c, int kb, int stage) __attribute__((always_inline)) { t.copy(c, kb, smem + stage * kStage, smem + stage * kStage + TM * kBlockK); };
  const int8_t *const sa = smem + t.wm * (TM / WM) * kBlockK, *const sb = smem + (TM + t.wn * (TN / WN)) * kBlockK;
  struct Fragments {
    v4i x[2][FM], w[2][FN]; // [half of the K block]
  };
  auto read = [&](Fragments &f, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int m = 0; m < FM; ++m) f.x[h][m] = *reinterpret_cast<const v4i *>(sa + stage * kStage + m * 2048 + t.lds[h]);
#pragma unroll
      for (int n = 0; n < FN; ++n) f.w[h][n] = *reinterpret_cast<const v4i *>(sb + stage * kStage + n * 2048 + t.lds[h]);
    }
  };
  typename Op::Acc acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[m][n] = typename Op::Acc{};
  constexpr bool kEarly = !PART && FM * FN <= 4; // (larger tiles gain nothing by it)
  constexpr int kRows = dense_round(TM, TN, WM, WN, ST * kStage) * 16, kTurns = (FM * FN + 1) / 2; // (turns of 16-bit pieces)
  DenseBeside<DT, FM, FN, kEarly && kRows == FM * 16 ? kTurns : 0, kRows> beside;
  if constexpr (kEarly) beside.load(a, t);
#pragma unroll
  for (int i = 0; i < ST; ++i)
#pragma unroll
    for (int c = 0; c < kCopies; ++c) copy(c, i, i);
  Fragments f[2];
  wait_barrier<(ST - 1) * kCopies>();
  read(f[0], 0);
  int stage = 0;
  auto step = [&](const Fragments &now, Fragments &then, int kb) __attribute__((always_inline)) {
    const int next = stage == ST - 1 ? 0 : stage + 1;
    wait_barrier<(ST - 2) * kCopies>();
    read(then, next);
#pragma unroll
    for (int c = 0; c < kCopies; ++c) copy(c, kb + ST, stage);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int n = 0; n < FN; ++n) acc[m][n] = Op::mfma(now.w[h][n], now.x[h][m], acc[m][n]);
    constexpr int kProducts = 2 * FM * FN, kReads = 2 * (FM + FN);
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if (i < kCopies) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    if constexpr (kReads > kProducts) __builtin_amdgcn_sched_group_barrier(0x100, kReads - kProducts, 0);
    __builtin_amdgcn_sched_barrier(0);
    stage = next;
  };
  for (int kb = 0; kb < t.KB; kb += 2) {
    step(f[0], f[1], kb);
    if (kb + 1 < t.KB) step(f[1], f[0], kb + 1);
  }
  wait_barrier<0>(); // no copy lands in what the epilogue uses, or outlives the workgroup
  if constexpr (!PART && !kEarly) beside.load(a, t);
  dense_finish<DT, TM, TN, WM, WN, PART, ST * kStage>(a, t, acc, beside, smem);
}

// The largest tiles, whose fragments of a K block do not fit into the registers twice.  A wave keeps its weight fragments of a K block in registers and
// walks through its token fragments, a step each: the next token fragment is read while this one is multiplied.  The workgroup meets in front of
// the last step, when nobody reads the K block's place any more and the next one has landed: behind the barrier its first operands are read under
// the step's products.  The weights' half of a place is free long before the tokens', once every wave has its fragments: the workgroup
// meets in front of step kMid too, and from there on the next but one K block's weights are asked for, its tokens behind the last barrier.
template <int DT, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void gemm_dense_step_kernel(const DenseArgs a, int group_m) {
  typedef Operand<DT> Op;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16; // fragments of a wave: tokens, weights
  constexpr int kStage = (TM + TN) * kBlockK;
  DenseTileOf<TM, TN, WM, WN, false> t;
  constexpr int kA = t.kA, kB = t.kB, kMid = kA - 1;
  static_assert(kMid >= 1 && kMid < FM - 1 && FM % 2 == 0, "steps for the copies");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  if (!t.start(a, group_m)) return;
  const int8_t *const sa = smem + t.wm * (TM / WM) * kBlockK, *const sb = smem + (TM + t.wn * (TN / WN)) * kBlockK;
  auto copy = [&](int c, int kb, int place) __attribute__((always_inline)) { t.copy(c, kb, smem + place * kStage, smem + place * kStage + TM * kBlockK); };
  auto read = [&](const int8_t *base, int f, int h, int place) __attribute__((always_inline)) {
    return *reinterpret_cast<const v4i *>(base + place * kStage + f * 2048 + t.lds[h]);
  };
  typename Op::Acc acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[m][n] = typename Op::Acc{};
#pragma unroll
  for (int c = 0; c < kA + kB; ++c) copy(c, 0, 0);
#pragma unroll
  for (int c = kA; c < kA + kB; ++c) copy(c, 1, 1);
  copy(0, 1, 1);
  wait_barrier<kB + 1>();
  v4i w[2][FN], x[2][2]; // [half of the K block][fragment], [step][half]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int n = 0; n < FN; ++n) w[h][n] = read(sb, n, h, 0);
    x[0][h] = read(sa, 0, h, 0);
  }
  int place = 0;
  for (int kb = 0; kb < t.KB; ++kb) {
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int cur = m & 1;
      const bool over = m + 1 == FM;
      if (over) wait_barrier<kB>();
#pragma unroll
      for (int h = 0; h < 2; ++h) x[cur ^ 1][h] = read(sa, over ? 0 : m + 1, h, over ? place ^ 1 : place);
      if (m == kMid) asm volatile("s_barrier" ::: "memory"); // (every wave has used its weights: they are in registers)
      if (over) copy(0, kb + 2, place);
      else if (m < kMid) copy(m + 1, kb + 1, place ^ 1);
#pragma unroll
      for (int c = 0; c < kB; ++c)
        if (!over && kMid + c * (FM - 1 - kMid) / kB == m) copy(kA + c, kb + 2, place);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          acc[m][n] = Op::mfma(w[h][n], x[cur][h], acc[m][n]);
          if (over) w[h][n] = read(sb, n, h, place ^ 1);
        }
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int n = 0; n < 2 * FN; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (n < 2) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        if (over) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    place ^= 1;
  }
  wait_barrier<0>(); // no copy lands in what the epilogue uses, or outlives the workgroup
  DenseBeside<DT, FM, FN, 0, 0> beside;
  beside.load(a, t);
  dense_finish<DT, TM, TN, WM, WN, false, 2 * kStage>(a, t, acc, beside, smem);
}

// The parts of K added up in their order, and the epilogue.
template <int DT> __global__ __launch_bounds__(256) void gemm_dense_join_kernel(const DenseArgs a) {
  typedef typename Operand<DT>::Sum T;
  const int half = a.gated ? a.pitch / 2 : a.pitch;
  const int64_t quads = a.M * (half / 4), step = a.M * a.pitch;
  // whole quads are stored where rows begin on a quad: c may begin on any value
  const bool whole = (a.N & 3) == 0 && (reinterpret_cast<uintptr_t>(a.C) & (a.out == LO_F32 ? 15 : 7)) == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < quads; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t m = i / (half / 4), n = (i - m * (half / 4)) * 4;
    auto sum = [&](int64_t at, T (&v)[4]) __attribute__((always_inline)) {
      const int *const p = static_cast<const int *>(a.part) + m * a.pitch + at;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = 0;
      for (int k = 0; k < a.splits; k += 4) { // (four parts asked for at a time: int8 333 x 576 x 7168 12.0 -> 11.6 us)
        typename Operand<DT>::Acc d[4];
#pragma unroll
        for (int l = 0; l < 4; ++l) d[l] = *reinterpret_cast<const typename Operand<DT>::Acc *>(p + (k + l < a.splits ? k + l : k) * step);
#pragma unroll
        for (int l = 0; l < 4; ++l)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = k + l < a.splits ? v[j] + d[l][j] : v[j];
      }
    };
    T g[4], u[4];
    float v[4];
    sum(n, g);
    if (a.gated) sum(n + half, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = n + j < a.N ? n + j : a.N - 1;
      v[j] = activate(a.act, dense_value(a, g[j], m, c));
      if (a.gated) v[j] *= dense_value(a, u[j], m, c + a.N);
      v[j] = dense_result(a, v[j], m, c);
    }
    if (whole && a.out == LO_F32) {
      *reinterpret_cast<v4f *>(static_cast<float *>(a.C) + m * a.N + n) = v4f{v[0], v[1], v[2], v[3]};
    } else if (whole) {
      *reinterpret_cast<v4u16 *>(static_cast<uint16_t *>(a.C) + m * a.N + n) =
          v4u16{to_half(a.out, v[0]), to_half(a.out, v[1]), to_half(a.out, v[2]), to_half(a.out, v[3])};
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) store_value(a.C, a.out, m * a.N + n + j, v[j]);
    }
  }
}

template <class K> static int launch_dense_kernel(const DenseArgs &a, K kernel, int lds, int threads, unsigned long long *done, hipStream_t stream) {
  const int rc = reserve_lds_once(reinterpret_cast<const void *>(kernel), lds, done);
  if (rc) return rc;
  const int group_m = a.m_tiles < 4 ? a.m_tiles : 4; // (2, 4, 8 and 16 are within 3 % of each other: 8192 x 4096 x 7168 bf16 360, 354, 352, 356 us, 2048 x 4096 x 4096 70, 69, 69, 69)
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((a.m_tiles * a.n_tiles + 7) / 8 * 8), a.splits), dim3(threads), lds, stream, a, group_m);
  return LO_OK;
}
constexpr int64_t kMostTiles = 1 << 22; // (512 threads of each are below a grid's 2^32)
static int64_t dense_tiles(int64_t M, int64_t N, int tm, int tn, bool gated) {
  const int64_t width = gated ? tn / 2 : tn;
  return (M + tm - 1) / tm * ((N + width - 1) / width);
}
static int set_dense_tiles(DenseArgs &a, int tm, int tn) {
  const int64_t width = a.gated ? tn / 2 : tn, m_tiles = (a.M + tm - 1) / tm, n_tiles = (a.N + width - 1) / width;
  LO_REQUIRE(m_tiles * n_tiles < kMostTiles, LO_ENOTSUP, "gemm_bias_act: %lld x %lld outputs", (long long)a.M, (long long)a.N);
  a.m_tiles = static_cast<int32_t>(m_tiles);
  a.n_tiles = static_cast<int32_t>(n_tiles);
  return LO_OK;
}
template <int DT, int TM, int TN, int WM, int WN> static int launch_dense_step(DenseArgs a, hipStream_t stream) {
  constexpr int ring = 2 * (TM + TN) * kBlockK, lds = dense_lds(TM, TN, WM, WN, ring, false);
  static_assert(lds <= 160 * 1024, "LDS");
  static unsigned long long done = 0;
  const int rc = set_dense_tiles(a, TM, TN);
  return rc ? rc : launch_dense_kernel(a, gemm_dense_step_kernel<DT, TM, TN, WM, WN>, lds, WM * WN * 64, &done, stream);
}
template <int DT, int TM, int TN, int WM, int WN, int ST> static int launch_dense_ring(DenseArgs a, int parts, hipStream_t stream) {
  constexpr int ring = ST * (TM + TN) * kBlockK, lds = dense_lds(TM, TN, WM, WN, ring, false);
  static_assert(lds <= 160 * 1024, "LDS");
  static unsigned long long done[2] = {0, 0};
  int rc = set_dense_tiles(a, TM, TN);
  if (rc) return rc;
  if (parts <= 1) return launch_dense_kernel(a, gemm_dense_ring_kernel<DT, TM, TN, WM, WN, ST, false>, lds, WM * WN * 64, &done[0], stream);
  a.splits = parts;
  rc = launch_dense_kernel(a, gemm_dense_ring_kernel<DT, TM, TN, WM, WN, ST, true>, ring, WM * WN * 64, &done[1], stream);
  if (rc) return rc;
  const int64_t blocks = (a.M * ((a.gated ? a.pitch / 2 : a.pitch) / 4) + 255) / 256;
  hipLaunchKernelGGL((gemm_dense_join_kernel<DT>), dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, a);
  return LO_OK;
}
// C (as a power of two) and the waves: see the kernel.
template <int DT> static int launch_dense_few(const DenseArgs &a, int lg, int waves, int u, hipStream_t stream) {
  const int64_t width = (16 >> lg) / (a.gated ? 2 : 1);
  const dim3 grid(static_cast<unsigned>((a.N + width - 1) / width)), block(waves * 64);
  switch (u) {
  case 1: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 1>), grid, block, 0, stream, a, lg); break;
  case 2: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 2>), grid, block, 0, stream, a, lg); break;
  case 3: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 3>), grid, block, 0, stream, a, lg); break;
  case 4: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 4>), grid, block, 0, stream, a, lg); break;
  case 5: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 5>), grid, block, 0, stream, a, lg); break;
  case 6: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 6>), grid, block, 0, stream, a, lg); break;
  case 7: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 7>), grid, block, 0, stream, a, lg); break;
  default: hipLaunchKernelGGL((gemm_dense_few_kernel<DT, 8>), grid, block, 0, stream, a, lg);
  }
  return LO_OK;
}

enum { kD256, kD192, kD128x256, kD128x192, kD128, kD96, kD64x128, kD64, kD64x32, kD32, kDenseTiles };
constexpr int kDenseFew = -1; // in a tile's place: up to 16 tokens, gemm_dense_few_kernel
// One operand type's kernels (gemm_dense_*.hip).  parts: of K; of the kernel of few tokens lg + 8 * waves.
template <int DT> int launch_dense(const DenseArgs &a, int tile, int parts, hipStream_t stream);
template <> int launch_dense<LO_BF16>(const DenseArgs &a, int tile, int parts, hipStream_t stream);
template <> int launch_dense<LO_F16>(const DenseArgs &a, int tile, int parts, hipStream_t stream);
template <> int launch_dense<LO_I8>(const DenseArgs &a, int tile, int parts, hipStream_t stream);
#define LO_DENSE_LAUNCHERS(DT)                                                                   \
  template <> int launch_dense<DT>(const DenseArgs &a, int tile, int parts, hipStream_t stream) { \
    switch (tile) {                                                                               \
    case kD256: return launch_dense_step<DT, 256, 256, 2, 4>(a, stream);                          \
    case kD192: return launch_dense_step<DT, 192, 256, 2, 4>(a, stream);                          \
    case kD128x256: return launch_dense_ring<DT, 128, 256, 2, 4, 3>(a, parts, stream);            \
    case kD128x192: return launch_dense_ring<DT, 128, 192, 2, 4, 3>(a, parts, stream);            \
    case kD128: return launch_dense_ring<DT, 128, 128, 2, 4, 4>(a, parts, stream);                \
    case kD96: return launch_dense_ring<DT, 96, 96, 2, 2, 3>(a, parts, stream);                   \
    case kD64x128: return launch_dense_ring<DT, 64, 128, 2, 4, 4>(a, parts, stream);              \
    case kD64: return launch_dense_ring<DT, 64, 64, 2, 2, 4>(a, parts, stream);                   \
    case kD64x32: return launch_dense_ring<DT, 64, 32, 2, 2, 6>(a, parts, stream);                \
    case kD32: return launch_dense_ring<DT, 32, 32, 1, 2, 8>(a, parts, stream);                   \
    default: return launch_dense_few<DT>(a, parts & 7, parts >> 3 & 15, parts >> 7, stream);                       \
    }                                                                                             \
  }

} // namespace lo
