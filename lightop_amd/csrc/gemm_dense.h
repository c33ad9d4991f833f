// Dense product with an epilogue:
//   v[m, n] = sum over k of A[m, k] * B[n, k] (int8: times As[m] * Bs[n]) + bias[n]
//   C[m, n] = scale * act(v[m, n]) + R[m, n];  gated: scale * act(v[m, n]) * v[m, N + n] + R[m, n].
// Sums, and everything behind them, are fp32 (int8: the sum is int32 and exact); a result is rounded once.  A K block is 128 bytes of a row,
// 64 values of 16 bits or 128 of int8, two matrix instructions of every 16 x 16 sums.  B (the weight) is the instructions' first
// operand: a lane holds four neighbouring columns of C for one token.
#pragma once
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

// The operands' types: sixteen bytes a lane of 16 rows of either operand, 64 bytes of K, into the 16 x 16 sums.
template <int DT> struct Operand {
  typedef v4f Acc;
  static __device__ __forceinline__ Acc mfma(const v4i a, const v4i b, const Acc c) {
    if constexpr (DT == LO_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <> struct Operand<LO_I8> {
  typedef v4i Acc;
  static __device__ __forceinline__ Acc mfma(const v4i a, const v4i b, const Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float load_value(const void *p, int type, int64_t at) {
  if (type == LO_F32) return static_cast<const float *>(p)[at];
  const uint16_t h = static_cast<const uint16_t *>(p)[at];
  return type == LO_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
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
// A workgroup takes 16 rows of B (gated: eight of either projection) and all tokens; its waves share the K blocks and add their sums up through
// LDS, in the same order every time.  Weights are read once, straight into registers, four K blocks of a wave in flight.
template <int DT>
__global__ __launch_bounds__(1024) void gemm_dense_few_kernel(const DenseArgs a) {
  typedef Operand<DT> Op;
  typedef typename Op::Acc Acc;
  __shared__ __attribute__((aligned(16))) int red[16][256]; // [wave][token][B's row]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (a.gated ? 8 : 16);
  int64_t nb = n0 + (a.gated ? r & 7 : r);
  nb = (nb < a.N ? nb : a.N - 1) + (a.gated && r >= 8 ? a.N : 0); // (rows and tokens past the end: the last one again, not stored)
  const int8_t *const pb = a.B + nb * a.ldb + q * 16;
  const int8_t *const pa = a.A + (r < a.M ? r : a.M - 1) * a.lda + q * 16;
  Acc acc = {};
  constexpr int U = 4;
  for (int kb0 = wave; kb0 < a.KB; kb0 += waves * U) {
    v4i w[U][2], x[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * waves, kc = (kb < a.KB ? kb : kb0) * kBlockK; // past the end: this one again, left out below
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = kc + q * 16 + h * 64 < a.K ? kc + h * 64 : -q * 16; // past the row's end: its first bytes, cleared below
        w[u][h] = __builtin_nontemporal_load(reinterpret_cast<const v4i *>(pb + at));
        x[u][h] = *reinterpret_cast<const v4i *>(pa + at);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * waves;
      if (kb >= a.KB) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = kb * kBlockK + q * 16 + h * 64 < a.K;
        acc = Op::mfma(in ? w[u][h] : v4i{}, in ? x[u][h] : v4i{}, acc);
      }
    }
  }
  *reinterpret_cast<v4i *>(&red[wave][r * 16 + 4 * q]) = __builtin_bit_cast(v4i, acc);
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int64_t m = threadIdx.x >> 4;
  const int c = threadIdx.x & 15;
  const int64_t n = n0 + c;
  if (m >= a.M || n >= a.N || (a.gated && c >= 8)) return;
  typedef decltype(Acc{}[0] + Acc{}[0]) T;
  auto sum = [&](int at) __attribute__((always_inline)) {
    T v = __builtin_bit_cast(T, red[0][at]);
    for (int i = 1; i < waves; ++i) v += __builtin_bit_cast(T, red[i][at]);
    return v;
  };
  float v = activate(a.act, dense_value(a, sum(threadIdx.x), m, n));
  if (a.gated) v *= dense_value(a, sum(threadIdx.x + 8), m, n + a.N);
  store_value(a.C, a.out, m * a.N + n, dense_result(a, v, m, n));
}

// ---- tiles -----------------------------------------------------------------------------------------------------------------
// Both operands go to LDS by direct loads, a K block to a stage of a ring of ST; 16-byte pieces of a row are swizzled by the row.  A wave keeps its
// weight fragments of a K block in registers and walks through its token fragments, a step each: the next token fragment is read while this
// one is multiplied.  The workgroup meets in front of the last step, when nobody reads the K block's stage any more: behind the barrier the
// next block's first operands are read under the step's products, and the copies of the block that takes the stage over are asked
// for, a few a step.  A gated product's fragments hold eight weight rows of either projection.
//
// PART: this workgroup's part of K only, its sums to a.part.
constexpr int dense_staging(int tn, int wm, int wn, int round) { return wm * wn * round * 16 * (tn / wn * 4 + 16); } // bytes
// Token fragments of a wave that the epilogue turns around at a time: all of them, or half where they do not fit.
constexpr int dense_round(int tm, int tn, int wm, int wn) { return dense_staging(tn, wm, wn, tm / wm / 16) <= 160 * 1024 ? tm / wm / 16 : tm / wm / 32; }
constexpr int dense_lds(int tm, int tn, int wm, int wn, int st, bool part) {
  const int ring = st * (tm + tn) * kBlockK, staging = part ? 0 : dense_staging(tn, wm, wn, dense_round(tm, tn, wm, wn));
  return ring > staging ? ring : staging;
}
template <int DT, int TM, int TN, int WM, int WN, int ST, bool PART>
__global__ __launch_bounds__(WM * WN * 64) void gemm_dense_tile_kernel(const DenseArgs a, int group_m) {
  typedef Operand<DT> Op;
  typedef typename Op::Acc Acc;
  constexpr int kWaves = WM * WN;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16;            // fragments of a wave: tokens, weights
  constexpr int kA = TM / 8 / kWaves, kB = TN / 8 / kWaves, kCopies = kA + kB; // 1 KB copies of a stage, of a wave
  constexpr int kStep = (kCopies + FM - 1) / FM;                               // copies of a step
  constexpr int kStage = (TM + TN) * kBlockK;
  // Two stages leave a copy little time.  The weights' part of a stage is free long before the tokens', once every wave has its fragments:
  // the workgroup meets in front of step kMid too, and from there on the next but one K block's weights are asked for, its tokens
  // behind the last step's barrier.
  constexpr bool kApart = ST == 2;
  constexpr int kMid = kA - 1;
  static_assert(!kApart || (kA >= 2 && kMid < FM - 1), "steps for the copies");
  static_assert(TM / 8 % kWaves == 0 && TN / 8 % kWaves == 0 && (TM / WM) % 16 == 0 && (TN / WN) % 16 == 0 && FM % 2 == 0, "tile");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  int mt, nt;
  const int split = PART ? blockIdx.y : 0;
  if (!dense_tile(blockIdx.x, a.m_tiles, a.n_tiles, group_m, mt, nt)) return;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int first = PART ? static_cast<int>(static_cast<int64_t>(a.KB) * split / a.splits) : 0;
  const int KB = (PART ? static_cast<int>(static_cast<int64_t>(a.KB) * (split + 1) / a.splits) : a.KB) - first;
  const bool gated = a.gated;
  const int width = gated ? TN / 2 : TN; // columns of C
  const int64_t m0 = static_cast<int64_t>(mt) * TM, n0 = static_cast<int64_t>(nt) * width;
  const int rows = static_cast<int>(a.M - m0 < TM ? a.M - m0 : TM), cols = static_cast<int>(a.N - n0 < width ? a.N - n0 : width);
  const int8_t *const pa = a.A + m0 * a.lda + first * kBlockK;
  const int8_t *pb[kB]; // of the projection that a copy's eight rows belong to
  const uint32_t endA = static_cast<uint32_t>((rows - 1) * a.lda + a.K - first * kBlockK), endB = static_cast<uint32_t>((cols - 1) * a.ldb + a.K - first * kBlockK);
  int voff[kA + kB];
  const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
#pragma unroll
  for (int j = 0; j < kA; ++j) voff[j] = ((wave * kA + j) * 8 + (lane >> 3)) * a.lda + piece;
#pragma unroll
  for (int j = 0; j < kB; ++j) {
    const int g = wave * kB + j; // eight rows; a fragment is two of them
    pb[j] = a.B + (n0 + (gated && (g & 1) ? a.N : 0)) * a.ldb + first * kBlockK;
    voff[kA + j] = ((gated ? g >> 1 : g) * 8 + (lane >> 3)) * a.ldb + piece;
  }
  // Past a row's end (in its last K block, where K is no multiple of 128 bytes) a piece's offset is past the extents, which end below 2^30.
  const int last = a.KB - 1 - first, tail = last * kBlockK + piece < a.K - first * kBlockK ? 0 : 1 << 30;
  // Copy c of K block kb.  What lies past the extents is written as zero: rows past the end, and past the last K block, where the extents are
  // empty, all of it (the copies, which the waits count, fetch nothing).
  auto copy = [&](int c, int kb, int stage) __attribute__((always_inline)) {
    const bool in = kb < KB;
    const int at = voff[c] + (kb == last ? tail : 0), soff = in ? kb * kBlockK : 0;
    if (c < kA) copy16(make_rsrc(pa, in ? endA : 0u), smem + stage * kStage + (wave * kA + c) * 1024, at, soff);
    else copy16(make_rsrc(pb[c - kA], in ? endB : 0u), smem + stage * kStage + TM * kBlockK + (wave * kB + c - kA) * 1024, at, soff);
  };
  const int lds[2] = {r * kBlockK + ((q ^ (r & 7)) * 16), r * kBlockK + (((q + 4) ^ (r & 7)) * 16)};
  const int8_t *const sa = smem + wm * (TM / WM) * kBlockK, *const sb = smem + (TM + wn * (TN / WN)) * kBlockK;
  auto read = [&](const int8_t *base, int f, int h, int stage) __attribute__((always_inline)) {
    return *reinterpret_cast<const v4i *>(base + stage * kStage + f * 2048 + lds[h]);
  };
  Acc acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[m][n] = Acc{};

  if constexpr (kApart) {
#pragma unroll
    for (int c = 0; c < kCopies; ++c) copy(c, 0, 0);
#pragma unroll
    for (int c = kA; c < kCopies; ++c) copy(c, 1, 1);
    copy(0, 1, 1);
    wait_barrier<kB + 1>();
  } else {
#pragma unroll
    for (int i = 0; i < ST; ++i)
#pragma unroll
      for (int c = 0; c < (i < ST - 1 ? kCopies : kStep); ++c) copy(c, i, i);
    wait_barrier<(ST - 2) * kCopies + kStep>();
  }
  v4i w[2][FN], x[2][2]; // [half of the K block][fragment], [step][half]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int n = 0; n < FN; ++n) w[h][n] = read(sb, n, h, 0);
    x[0][h] = read(sa, 0, h, 0);
  }
  int stage = 0;
  for (int kb = 0; kb < KB; ++kb) {
    const int next = stage == ST - 1 ? 0 : stage + 1, prev = stage == 0 ? ST - 1 : stage - 1;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int cur = m & 1;
      if (m + 1 < FM) {
#pragma unroll
        for (int h = 0; h < 2; ++h) x[cur ^ 1][h] = read(sa, m + 1, h, stage);
      } else {
        wait_barrier<kApart ? kB : (ST - 2) * kCopies>();
#pragma unroll
        for (int h = 0; h < 2; ++h) x[cur ^ 1][h] = read(sa, 0, h, next);
      }
      if constexpr (kApart) {
        if (m == kMid) asm volatile("s_barrier" ::: "memory"); // (every wave has used its weights: they are in registers)
        if (m + 1 == FM) {
          copy(0, kb + 2, stage);
        } else if (m < kMid) {
          copy(m + 1, kb + 1, next);
        } else {
#pragma unroll
          for (int c = 0; c < kB; ++c)
            if (c * (FM - 1 - kMid) / kB == m - kMid) copy(kA + c, kb + 2, stage);
        }
      } else { // the stage that the last barrier freed
#pragma unroll
        for (int c = 0; c < kStep; ++c) {
          const int at = (m + 1 == FM ? 0 : m + 1) * kStep + c;
          if (at < kCopies) copy(at, m + 1 == FM ? kb + ST : kb + ST - 1, m + 1 == FM ? stage : prev);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          acc[m][n] = Op::mfma(w[h][n], x[cur][h], acc[m][n]);
          if (m + 1 == FM) w[h][n] = read(sb, n, h, next);
        }
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int n = 0; n < 2 * FN; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (n < 2) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        if (m + 1 == FM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    stage = next;
  }
  wait_barrier<0>(); // no copy lands in what the epilogue uses, or outlives the workgroup

  constexpr int kCols = TN / WN; // B's rows of a wave
  if constexpr (PART) {
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int mr = wm * (TM / WM) + m * 16 + r;
      int *const row = static_cast<int *>(a.part) + (split * a.M + m0 + mr) * a.pitch + n0;
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const int c = gated ? (wn * kCols + n * 16) / 2 + 4 * (q & 1) : wn * kCols + n * 16 + 4 * q;
        if (mr < rows && c < cols) *reinterpret_cast<v4i *>(row + c + (gated && q >= 2 ? a.pitch / 2 : 0)) = __builtin_bit_cast(v4i, acc[m][n]);
      }
    }
  } else {
    // A wave turns its tokens around in LDS, kRound fragments of them at a time, in fp32 (its own part; LDS operations of a wave execute in
    // order), and stores whole pieces of rows, activated and the residual added: 16 bytes a lane, or, where rows of either do not begin on 16
    // bytes, a value a lane.
    constexpr int kPitch = kCols * 4 + 16, kRound = dense_round(TM, TN, WM, WN), kRows = kRound * 16;
    int8_t *const stg = smem + wave * kRows * kPitch;
    const int size = a.out == LO_F32 ? 4 : 2;
    const bool whole = ((a.N * size | (a.R ? a.rs * size : 0) | static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.C) | reinterpret_cast<uintptr_t>(a.R))) & 15) == 0;
    const int out_cols = gated ? kCols / 2 : kCols; // of C, of this wave
    const int64_t nw = n0 + wn * out_cols;
    const int left = cols - wn * out_cols; // of them in C
    float bs[FN][4], bias[FN][4], as[FM];
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t c = nw + (gated ? n * 8 + 4 * (q & 1) : n * 16 + 4 * q) + i;
        const int64_t at = (c < a.N ? c : a.N - 1) + (gated && q >= 2 ? a.N : 0);
        if constexpr (DT == LO_I8) bs[n][i] = a.Bs[at];
        bias[n][i] = a.bias ? load_value(a.bias, a.bias_f32 ? LO_F32 : a.out, at) : 0.0f;
      }
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int row = wm * (TM / WM) + m * 16 + r;
      if constexpr (DT == LO_I8) as[m] = a.As[m0 + (row < rows ? row : rows - 1)];
    }
    // a row's values from column c: of the gate (or of C), and of the other projection
    auto place = [&](int row, int c) __attribute__((always_inline)) {
      return reinterpret_cast<const float *>(stg + row * kPitch) + (gated ? (c >> 3) * 16 + (c & 7) : c);
    };
    auto four = [&](int row, int c, float *v) __attribute__((always_inline)) {
      const float *const p = place(row, c);
      const v4f g = *reinterpret_cast<const v4f *>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = activate(a.act, g[i]);
      if (gated) {
        const v4f u = *reinterpret_cast<const v4f *>(p + 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= u[i];
      }
    };
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
            if constexpr (DT == LO_I8) o[i] = o[i] * as[m] * bs[n][i];
            if (a.bias) o[i] += bias[n][i];
          }
          *reinterpret_cast<v4f *>(stg + (m % kRound * 16 + r) * kPitch + (n * 16 + 4 * q) * 4) = o;
        }
      }
      lds_order();
      const int row0 = wm * (TM / WM) + round * kRows, in = rows - row0 < kRows ? rows - row0 : kRows;
      const int64_t c0 = (m0 + row0) * a.N + nw, r0 = (m0 + row0) * a.rs + nw;
      if (whole && a.out != LO_F32) {
        const int lanes = out_cols / 8; // of a row
#pragma unroll 1
        for (int i = lane; i < kRows * lanes; i += 64) {
          const int row = i / lanes, c = i % lanes * 8;
          if (row >= in || c >= left) continue;
          v8u16 o, add = {};
          if (a.R) add = *reinterpret_cast<const v8u16 *>(static_cast<const uint16_t *>(a.R) + r0 + row * a.rs + c);
          float v[8];
          four(row, c, v);
          four(row, c + 4, v + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = a.R ? __builtin_fmaf(a.scale, v[i], a.out == LO_BF16 ? bf16_to_f32(add[i]) : f16_to_f32(add[i])) : a.scale * v[i];
            o[i] = to_half(a.out, v[i]);
          }
          *reinterpret_cast<v8u16 *>(static_cast<uint16_t *>(a.C) + c0 + row * a.N + c) = o;
        }
      } else if (whole) {
        const int lanes = out_cols / 4;
#pragma unroll 1
        for (int i = lane; i < kRows * lanes; i += 64) {
          const int row = i / lanes, c = i % lanes * 4;
          if (row >= in || c >= left) continue;
          v4f add = {0.0f, 0.0f, 0.0f, 0.0f}, o;
          if (a.R) add = *reinterpret_cast<const v4f *>(static_cast<const float *>(a.R) + r0 + row * a.rs + c);
          float v[4];
          four(row, c, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = a.R ? __builtin_fmaf(a.scale, v[i], add[i]) : a.scale * v[i];
          *reinterpret_cast<v4f *>(static_cast<float *>(a.C) + c0 + row * a.N + c) = o;
        }
      } else {
#pragma unroll 1
        for (int i = lane; i < kRows * out_cols; i += 64) {
          const int row = i / out_cols, c = i % out_cols;
          if (row >= in || c >= left) continue;
          const float *const p = place(row, c);
          const float v = activate(a.act, p[0]) * (gated ? p[8] : 1.0f);
          store_value(a.C, a.out, c0 + row * a.N + c, dense_result(a, v, m0 + row0 + row, nw + c));
        }
      }
      lds_order();
    }
  }
}

// The parts of K added up in their order, and the epilogue.
template <int DT> __global__ __launch_bounds__(256) void gemm_dense_join_kernel(const DenseArgs a) {
  typedef decltype(typename Operand<DT>::Acc{}[0] + typename Operand<DT>::Acc{}[0]) T;
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
      for (int k = 0; k < a.splits; ++k) {
        const auto d = *reinterpret_cast<const typename Operand<DT>::Acc *>(p + k * step);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += d[j];
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

template <int DT, int TM, int TN, int WM, int WN, int ST, bool PART> static int launch_dense_parts(const DenseArgs &a, hipStream_t stream) {
  constexpr int lds = dense_lds(TM, TN, WM, WN, ST, PART);
  static_assert(lds <= 160 * 1024, "LDS");
  const auto kernel = gemm_dense_tile_kernel<DT, TM, TN, WM, WN, ST, PART>;
  static unsigned long long done = 0;
  const int rc = reserve_lds_once(reinterpret_cast<const void *>(kernel), lds, &done);
  if (rc) return rc;
  const int group_m = a.m_tiles < 4 ? a.m_tiles : 4;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((a.m_tiles * a.n_tiles + 7) / 8 * 8), PART ? a.splits : 1), dim3(WM * WN * 64), lds,
                     stream, a, group_m);
  return LO_OK;
}
template <int DT, int TM, int TN, int WM, int WN, int ST, bool SPLIT> static int launch_dense_tile(DenseArgs a, int parts, hipStream_t stream) {
  const int64_t width = a.gated ? TN / 2 : TN, m_tiles = (a.M + TM - 1) / TM, n_tiles = (a.N + width - 1) / width;
  LO_REQUIRE(m_tiles * n_tiles < (1 << 22), LO_ENOTSUP, "gemm_bias_act: %lld x %lld outputs", (long long)a.M, (long long)a.N);
  a.m_tiles = static_cast<int32_t>(m_tiles);
  a.n_tiles = static_cast<int32_t>(n_tiles);
  if constexpr (SPLIT) {
    if (parts > 1) {
      a.splits = parts;
      const int rc = launch_dense_parts<DT, TM, TN, WM, WN, ST, true>(a, stream);
      if (rc) return rc;
      const int64_t blocks = (a.M * ((a.gated ? a.pitch / 2 : a.pitch) / 4) + 255) / 256;
      hipLaunchKernelGGL((gemm_dense_join_kernel<DT>), dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, a);
      return LO_OK;
    }
  }
  return launch_dense_parts<DT, TM, TN, WM, WN, ST, false>(a, stream);
}

enum { kD256, kD192, kD128x256, kD128, kD64, kD64x32, kDenseTiles };
constexpr int kDenseFew = -1; // in a tile's place: up to 16 tokens, gemm_dense_few_kernel
// One operand type's kernels (gemm_dense_*.hip).
template <int DT> int launch_dense(const DenseArgs &a, int tile, int parts, hipStream_t stream);
template <> int launch_dense<LO_BF16>(const DenseArgs &a, int tile, int parts, hipStream_t stream);
template <> int launch_dense<LO_F16>(const DenseArgs &a, int tile, int parts, hipStream_t stream);
template <> int launch_dense<LO_I8>(const DenseArgs &a, int tile, int parts, hipStream_t stream);
#define LO_DENSE_LAUNCHERS(DT)                                                                                                    \
  template <> int launch_dense<DT>(const DenseArgs &a, int tile, int parts, hipStream_t stream) {                                  \
    switch (tile) {                                                                                                                \
    case kD256: return launch_dense_tile<DT, 256, 256, 2, 4, 2, false>(a, parts, stream);                                          \
    case kD192: return launch_dense_tile<DT, 192, 256, 2, 4, 2, false>(a, parts, stream);                                          \
    case kD128x256: return launch_dense_tile<DT, 128, 256, 2, 4, 3, true>(a, parts, stream);                                       \
    case kD128: return launch_dense_tile<DT, 128, 128, 2, 4, 4, true>(a, parts, stream);                                           \
    case kD64: return launch_dense_tile<DT, 64, 64, 2, 2, 4, true>(a, parts, stream);                                              \
    case kD64x32: return launch_dense_tile<DT, 64, 32, 2, 2, 4, true>(a, parts, stream);                                           \
    default: {                                                                                                                     \
      const int waves = a.KB >= 16 ? 16 : a.KB >= 8 ? 8 : 4;                                                                       \
      const int64_t width = a.gated ? 8 : 16;                                                                                      \
      hipLaunchKernelGGL((gemm_dense_few_kernel<DT>), dim3(static_cast<unsigned>((a.N + width - 1) / width)), dim3(waves * 64), 0, \
                         stream, a);                                                                                               \
      return LO_OK;                                                                                                                \
    }                                                                                                                              \
    }                                                                                                                              \
  }

} // namespace lo
