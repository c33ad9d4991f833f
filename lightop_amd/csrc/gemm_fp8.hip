// Dense product of e4m3 operands with a scale for each block of 128:
//   C[m, n] = sum over kb of (A[m, kb] . B[n, kb]) * As[m, kb] * Bs[n / 128, kb],
// A [M, K] rows with one scale for 128 values, B [N, K] a weight with one for 128 x 128.  A K block's 128 products are one MFMA
// (v_mfma_f32_16x16x128_f8f6f4, which starts from zero), its fp32 result is folded into the fp32 sum with the scales' product.
// (An fp32 output and up to 16 tokens take the exact form of it, fp8.h.)  Weights are the A operand: a lane holds four neighbouring columns of C for one token,
// whose scale it carries.
#include "gemm.h"
#include "fp8.h"

namespace lo {

struct Fp8GemmArgs {
  const int8_t *A, *B;
  const float *As, *Bs;
  void *C;
  float *part; // [splits][M][pitch] sums over parts of K
  int64_t M, N, K;
  int32_t KB, m_tiles, n_tiles, splits, pitch;
};

template <int DT> __device__ __forceinline__ void store_c(void *c, int64_t at, float v) {
  if constexpr (DT == LO_F32) static_cast<float *>(c)[at] = v;
  else static_cast<uint16_t *>(c)[at] = from_f32<DT>(v);
}

// ---- up to 16 tokens ---------------------------------------------------------------------------------------------------------
// A workgroup takes 16 columns and all tokens; its waves share the K blocks and add their sums up through LDS, in the same order every time.
// Weights are read once, straight into registers, four K blocks of a wave in flight: HBM and the launch bound it (1 x 4096 x 7168: 29 MB in
// 8.5 us), where N is narrow the few workgroups (1 x 576 x 7168, 36 of them, 7.6 us; 16 rows 10.7).  Rows past the tokens are past the extents and read as zeros.
template <int DT>
__global__ __launch_bounds__(1024) void gemm_fp8_few_kernel(const Fp8GemmArgs a) {
  __shared__ __attribute__((aligned(16))) float red[16][256]; // [wave][token][column]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int K = static_cast<int>(a.K), KB = a.KB;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t cols = a.N - n0 < 16 ? a.N - n0 : 16;
  const brsrc rB = make_rsrc(a.B + n0 * K, static_cast<uint32_t>(cols * K));
  const brsrc rA = make_rsrc(a.A, static_cast<uint32_t>(a.M * K));
  const brsrc rS = make_rsrc(a.As, static_cast<uint32_t>(a.M * KB * 4));
  const float *const bs = a.Bs + (n0 >> 7) * KB;
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = 4;
  for (int kb0 = wave; kb0 < KB; kb0 += waves * U) {
    v8i w[U], x[U];
    float s[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * waves, kc = kb < KB ? kb : kb0; // past the end: this one again, left out below
      const int at = r * K + q * 16 + kc * kGroup;
      w[u] = join(bld16<kCacheStream>(rB, at, 0), bld16<kCacheStream>(rB, at + 64, 0));
      b[u] = bs[kc];
      x[u] = join(bld16(rA, at, 0), bld16(rA, at + 64, 0));
      s[u] = bld_f32(rS, (r * KB + kc) * 4, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb0 + u * waves >= KB) break;
      const v4f d = mfma_e4m3_exact(w[u], x[u]);
      const float sc = s[u] * b[u];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], sc, acc[i]);
    }
  }
  *reinterpret_cast<v4f *>(&red[wave][r * 16 + 4 * q]) = acc;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int64_t m = threadIdx.x >> 4, n = n0 + (threadIdx.x & 15);
  if (m >= a.M || n >= a.N) return;
  float v = red[0][threadIdx.x];
  for (int i = 1; i < waves; ++i) v += red[i][threadIdx.x];
  store_c<DT>(a.C, m * a.N + n, v);
}

// Workgroups are dealt round-robin to the 8 XCDs: each takes a range of tiles of its own, in groups of G token tiles by all columns, so that
// tiles at work at one time share rows and columns in its L2.
__device__ __forceinline__ bool dense_tile(int bid, int m_tiles, int n_tiles, int G, int &mt, int &nt) {
  const int total = m_tiles * n_tiles, per = (total + 7) / 8, id = (bid & 7) * per + (bid >> 3);
  if ((bid >> 3) >= per || id >= total) return false;
  const int first = id / (G * n_tiles) * G, in = id - first * n_tiles;
  const int size = m_tiles - first < G ? m_tiles - first : G;
  nt = in / size;
  mt = first + in - nt * size;
  return true;
}

// ---- tiles -----------------------------------------------------------------------------------------------------------------
// Both operands go to LDS by direct loads, a K block to a stage of a ring of ST; 16-byte pieces of a row are swizzled by the row.  The rows'
// scales go there four K blocks at a time (a scale is a line of its own to the texture path, whatever it fetches of it).  A wave keeps its
// weight fragments of a K block in registers and walks through its token fragments, a step each: the next token fragment is read while this
// one is multiplied and the one before is folded.  The workgroup meets in front of the last step, when nobody reads the K block's stage any
// more: behind the barrier the next block's first operands are read under the step's products, and the copies of the block that takes the
// stage over are asked for, a few a step.
//
// 8192 x 4096 x 7168 in 256 x 256 tiles, two stages: 199 us, 2.4 PFLOP/s (the library's product of 8192^3 without block scales 2.78).  The K
// loop is bound by the MFMAs with the fold's vector instructions between them, and by the clock, 1.7 GHz under that load.  Freeing the
// weights' and the tokens' half of a stage apart took it from 217 us; other orders of the copies, s_setprio and groups of 8 token tiles to an
// XCD gained nothing.  Middle sizes lose to their last round of workgroups, narrow ones to a step's latency: rings of six and eight stages
// (64 x 64, 64 x 32) and an XCD to each part of K are no faster (each pair of one run, so / as it is: 333 x 576 x 7168 13.1 / 13.3 us, 48 x 7168 x 2048 8.0 / 8.0; by themselves 12.3 and 7.7).
// An fp32 output's exact products take their time in large sizes: 8192 x 4096 x 7168 510 us, 1531 x 7168 x 2048 59, 333 x 576 x 7168 15.0, 48 x 7168 x
// 2048 10.0.
__device__ __forceinline__ void copy16(brsrc r, int8_t *lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, voff, soff, 0, 0);
}
// All but this wave's newest N copies have landed and what it has read from LDS is there, and the workgroup meets.
template <int N> __device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// PART: this workgroup's part of K only, its fp32 sums to a.part.
template <int DT, int TM, int TN, int WM, int WN, int ST, bool PART>
__global__ __launch_bounds__(WM * WN * 64) void gemm_fp8_tile_kernel(const Fp8GemmArgs a, int group_m) {
  constexpr int kWaves = WM * WN;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16;             // fragments of a wave: tokens, weights
  constexpr int kA = TM / 8 / kWaves, kB = TN / 8 / kWaves, kCopies = 1 + kA + kB; // 1 KB copies of a stage, of a wave, and its scales
  constexpr int kStep = (kCopies + FM - 1) / FM;                                   // copies of a step
  constexpr int kStage = (TM + TN) * kGroup;
  // Two stages leave a copy little time.  The weights' part of a stage is free long before the tokens', once every wave has its fragments:
  // the workgroup meets in front of step kMid too, and from there on the next but one K block's weights are asked for, its tokens
  // behind the last step's barrier.
  constexpr bool kApart = ST == 2;
  constexpr int kMid = kA - 1;
  static_assert(!kApart || (kA >= 2 && kMid < FM - 2), "steps for the copies");
  static_assert(TM / 8 % kWaves == 0 && TN / 8 % kWaves == 0 && TM % 64 == 0 && TM / 64 <= kWaves && (TN / WN) % 16 == 0 && 128 % (TN / WN) == 0 &&
                    FM % 2 == 0 && ST <= 5, "tile");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  int8_t *const sS = smem + ST * kStage; // [K blocks / 4, odd or even][token][4] scales
  int mt, nt;
  const int split = PART ? blockIdx.y : 0;
  if (!dense_tile(blockIdx.x, a.m_tiles, a.n_tiles, group_m, mt, nt)) return;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int K = static_cast<int>(a.K), allKB = a.KB;
  const int first = PART ? static_cast<int>(static_cast<int64_t>(allKB) * split / a.splits) : 0;
  const int KB = (PART ? static_cast<int>(static_cast<int64_t>(allKB) * (split + 1) / a.splits) : allKB) - first;
  const int64_t m0 = static_cast<int64_t>(mt) * TM, n0 = static_cast<int64_t>(nt) * TN;
  const int rows = static_cast<int>(a.M - m0 < TM ? a.M - m0 : TM), cols = static_cast<int>(a.N - n0 < TN ? a.N - n0 : TN);
  const int8_t *const pa = a.A + m0 * K + first * kGroup, *const pb = a.B + n0 * K + first * kGroup;
  const float *const ps = a.As + m0 * allKB + first;
  const int ends = (rows * allKB - first) * 4;
  int voff[kA + kB];
#pragma unroll
  for (int j = 0; j < kA + kB; ++j) {
    const int row = (j < kA ? wave * kA + j : wave * kB + j - kA) * 8 + (lane >> 3);
    voff[j] = row * K + (((lane & 7) ^ (row & 7)) * 16);
  }
  const int sgrp = wave % (TM / 64), soff = (sgrp * 64 + lane) * allKB * 4;
  // Copy c of K block kb.  Rows past the end are past the extents and read as zero; past the last K block the extents are empty, and the
  // copies (which the waits count) fetch nothing.
  auto copy_scales = [&](int four, bool in) __attribute__((always_inline)) { // of K blocks 4 * four ..
    // (what is past the extents is written as zero: the empty copies go where nobody reads)
    copy16(make_rsrc(ps, in ? static_cast<uint32_t>(ends) : 0u), sS + (in ? (four & 1) * TM + sgrp * 64 : 2 * TM) * 16, soff,
           four * 16);
  };
  auto copy = [&](int c, int kb, int stage) __attribute__((always_inline)) {
    const bool in = kb < KB;
    if (c == 0) { // once in four: those behind the ones that K block kb - 1 (two stages), kb - ST + 1 begins
      const int at = kb - ST + 1;
      copy_scales((at >> 2) + 1, (at & 3) == 0 && at > 0);
    } else if (c <= kA) {
      copy16(make_rsrc(pa, in ? static_cast<uint32_t>(rows * K - first * kGroup) : 0u), smem + stage * kStage + (wave * kA + c - 1) * 1024,
             voff[c - 1], kb * kGroup);
    } else {
      copy16(make_rsrc(pb, in ? static_cast<uint32_t>(cols * K - first * kGroup) : 0u),
             smem + stage * kStage + TM * kGroup + (wave * kB + c - 1 - kA) * 1024, voff[c - 1], kb * kGroup);
    }
  };
  int64_t nblk = (n0 + wn * (TN / WN)) >> 7;
  const int64_t last = (a.N - 1) >> 7;
  nblk = nblk < last ? nblk : last;
  const float *const bs = a.Bs + nblk * allKB + first;
  float bvec = 0.0f; // weight scales of 64 K blocks, one a lane
  const int lds0 = r * kGroup + ((q ^ (r & 7)) * 16), lds1 = r * kGroup + (((q + 4) ^ (r & 7)) * 16);
  const int8_t *const sa = smem + wm * (TM / WM) * kGroup, *const sb = smem + (TM + wn * (TN / WN)) * kGroup;
  const float *const ss = reinterpret_cast<const float *>(sS) + (wm * (TM / WM) + r) * 4;
  auto scale = [&](int m, int kb) __attribute__((always_inline)) { return ss[((kb >> 2) & 1) * TM * 4 + m * 64 + (kb & 3)]; };
  auto read = [&](const int8_t *base, int f, int stage) __attribute__((always_inline)) {
    const int8_t *const p = base + stage * kStage + f * 2048;
    return join(*reinterpret_cast<const v4i *>(p + lds0), *reinterpret_cast<const v4i *>(p + lds1));
  };
  v4f acc[FM][FN], dprev[FN];
#pragma unroll
  for (int n = 0; n < FN; ++n) {
    dprev[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int m = 0; m < FM; ++m) acc[m][n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  float sprev = 0.0f;

  copy_scales(0, true);
  copy_scales(1, true);
  if constexpr (kApart) {
#pragma unroll
    for (int c = 1; c < kCopies; ++c) copy(c, 0, 0);
#pragma unroll
    for (int c = 1 + kA; c < kCopies; ++c) copy(c, 1, 1);
    copy(0, 1, 1);
    copy(1, 1, 1);
    wait_barrier<kB + 2>();
  } else {
#pragma unroll
    for (int i = 0; i < ST; ++i)
#pragma unroll
      for (int c = 0; c < (i < ST - 1 ? kCopies : kStep); ++c) copy(c, i, i);
    wait_barrier<(ST - 2) * kCopies + kStep>();
  }
  v8i w[FN], x[2];
  float s[2];
#pragma unroll
  for (int n = 0; n < FN; ++n) w[n] = read(sb, n, 0);
  x[0] = read(sa, 0, 0);
  s[0] = scale(0, 0);
  auto fold = [&](int m) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = __builtin_fmaf(dprev[n][i], sprev, acc[m][n][i]);
  };
  int stage = 0;
  for (int kb = 0; kb < KB; ++kb) {
    if ((kb & 63) == 0) { // (its wait, here and not at the use, is one for every copy asked for before: once in 64 K blocks)
      const int at = kb + lane;
      bvec = bs[at < KB ? at : KB - 1];
      asm volatile("" : "+v"(bvec));
    }
    const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bvec), kb & 63));
    const int next = stage == ST - 1 ? 0 : stage + 1, prev = stage == 0 ? ST - 1 : stage - 1;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int cur = m & 1;
      if (m + 1 < FM) {
        x[cur ^ 1] = read(sa, m + 1, stage);
        s[cur ^ 1] = scale(m + 1, kb);
      } else {
        wait_barrier<kApart ? kB : (ST - 2) * kCopies>();
        x[cur ^ 1] = read(sa, 0, next);
        s[cur ^ 1] = scale(0, kb + 1);
      }
      if constexpr (kApart) {
        if (m == kMid) asm volatile("s_barrier" ::: "memory"); // (every wave has used its weights: they are in registers)
        if (m + 1 == FM) {
          copy(0, kb + 2, stage);
          copy(1, kb + 2, stage);
        } else if (m < kMid) {
          if (m + 2 <= kA) copy(m + 2, kb + 1, next);
        } else {
#pragma unroll
          for (int c = 0; c < kB; ++c)
            if (c * (FM - 1 - kMid) / kB == m - kMid) copy(1 + kA + c, kb + 2, stage);
        }
      } else { // the stage that the last barrier freed
#pragma unroll
        for (int c = 0; c < kStep; ++c) {
          const int at = (m + 1 == FM ? 0 : m + 1) * kStep + c;
          if (at < kCopies) copy(at, m + 1 == FM ? kb + ST : kb + ST - 1, m + 1 == FM ? stage : prev);
        }
      }
      v4f d[FN];
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        d[n] = mfma_e4m3_as<DT == LO_F32>(w[n], x[cur]);
        if (m + 1 == FM) w[n] = read(sb, n, next);
      }
      fold(m == 0 ? FM - 1 : m - 1);
#pragma unroll
      for (int n = 0; n < FN; ++n) dprev[n] = d[n];
      sprev = s[cur] * b;
      if constexpr (DT != LO_F32) {
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int n = 0; n < FN; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          if (kApart ? n + 2 == FN || (n + 1 == FN && m + 1 == FM) : n < kStep) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
          if (m + 1 == FM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    stage = next;
  }
  fold(FM - 1);
  wait_barrier<0>(); // no copy lands in what the epilogue uses, or outlives the workgroup

  constexpr int kCols = TN / WN;
  if constexpr (PART) {
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int mr = wm * (TM / WM) + m * 16 + r;
      float *const row = a.part + (split * a.M + m0 + mr) * a.pitch + n0 + wn * kCols + 4 * q;
#pragma unroll
      for (int n = 0; n < FN; ++n)
        if (mr < rows && wn * kCols + n * 16 + 4 * q < cols) *reinterpret_cast<v4f *>(row + n * 16) = acc[m][n];
    }
  } else {
    // A wave turns 16 tokens x its columns around in LDS (its own part; LDS operations of a wave execute in order) and stores whole pieces of
    // rows: 16 bytes a lane, or, where rows do not begin on 16 bytes, a value a lane.
    constexpr int kSize = DT == LO_F32 ? 4 : 2, kPitch = kCols * kSize + 16, kLanes = kCols * kSize / 16; // lanes of a row
    static_assert(kWaves * 16 * kPitch <= ST * kStage, "staging");
    int8_t *const stg = smem + wave * 16 * kPitch;
    const bool whole = (a.N * kSize & 15) == 0 && (reinterpret_cast<uintptr_t>(a.C) & 15) == 0;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        if constexpr (DT == LO_F32) {
          *reinterpret_cast<v4f *>(stg + r * kPitch + (n * 16 + 4 * q) * 4) = acc[m][n];
        } else {
          v4u16 o;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = from_f32<DT>(acc[m][n][i]);
          *reinterpret_cast<v4u16 *>(stg + r * kPitch + (n * 16 + 4 * q) * 2) = o;
        }
      }
      lds_order();
      const int row0 = wm * (TM / WM) + m * 16;
      if (whole) {
#pragma unroll
        for (int j = 0; j < (16 * kLanes + 63) / 64; ++j) {
          const int row = (lane + 64 * j) / kLanes, c = (lane + 64 * j) % kLanes * 16;
          if (16 * kLanes < 64 && row >= 16) break;
          const v4i v = *reinterpret_cast<const v4i *>(stg + row * kPitch + c);
          if (row0 + row < rows && wn * kCols + c / kSize < cols)
            *reinterpret_cast<v4i *>(static_cast<int8_t *>(a.C) + ((m0 + row0 + row) * a.N + n0 + wn * kCols) * kSize + c) = v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16 * kCols / 64; ++j) {
          const int row = (lane + 64 * j) / kCols, c = (lane + 64 * j) % kCols;
          if (row0 + row < rows && wn * kCols + c < cols) {
            const int64_t at = (m0 + row0 + row) * a.N + n0 + wn * kCols + c;
            if constexpr (DT == LO_F32) static_cast<float *>(a.C)[at] = *reinterpret_cast<const float *>(stg + row * kPitch + c * 4);
            else static_cast<uint16_t *>(a.C)[at] = *reinterpret_cast<const uint16_t *>(stg + row * kPitch + c * 2);
          }
        }
      }
      lds_order();
    }
  }
}

// The parts of K added up in their order.
template <int DT> __global__ __launch_bounds__(256) void gemm_fp8_join_kernel(const Fp8GemmArgs a) {
  const int64_t quads = a.M * (a.pitch / 4), step = a.M * a.pitch;
  // whole quads are stored where rows begin on a quad: c may begin on any value
  const bool whole = (a.N & 3) == 0 && (reinterpret_cast<uintptr_t>(a.C) & (DT == LO_F32 ? 15 : 7)) == 0;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < quads; i += static_cast<int64_t>(gridDim.x) * 256) {
    const float *const p = a.part + i * 4;
    v4f v = *reinterpret_cast<const v4f *>(p);
    for (int k = 1; k < a.splits; ++k) v += *reinterpret_cast<const v4f *>(p + k * step);
    const int64_t m = i / (a.pitch / 4), n = (i - m * (a.pitch / 4)) * 4;
    if (whole) {
      if constexpr (DT == LO_F32) {
        *reinterpret_cast<v4f *>(static_cast<float *>(a.C) + m * a.N + n) = v;
      } else {
        v4u16 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = from_f32<DT>(v[j]);
        *reinterpret_cast<v4u16 *>(static_cast<uint16_t *>(a.C) + m * a.N + n) = o;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < a.N) store_c<DT>(a.C, m * a.N + n + j, v[j]);
    }
  }
}

template <int DT, int TM, int TN, int WM, int WN, int ST, bool PART> static int launch_tile_parts(const Fp8GemmArgs &a, hipStream_t stream) {
  constexpr int lds = ST * (TM + TN) * kGroup + (2 * TM + 64) * 16;
  static_assert(lds <= 160 * 1024, "LDS");
  const auto kernel = gemm_fp8_tile_kernel<DT, TM, TN, WM, WN, ST, PART>;
  static unsigned long long done = 0;
  const int rc = reserve_lds_once(reinterpret_cast<const void *>(kernel), lds, &done);
  if (rc) return rc;
  const int group_m = a.m_tiles < 4 ? a.m_tiles : 4;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((a.m_tiles * a.n_tiles + 7) / 8 * 8), PART ? a.splits : 1), dim3(WM * WN * 64), lds,
                     stream, a, group_m);
  return LO_OK;
}
template <int DT> static int join_parts(const Fp8GemmArgs &a, hipStream_t stream) {
  const int64_t blocks = (a.M * (a.pitch / 4) + 255) / 256;
  hipLaunchKernelGGL((gemm_fp8_join_kernel<DT>), dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, a);
  return LO_OK;
}

// Which tile, and how many parts of K: the smallest estimate of the time.  A K block takes a CU t1 us with one workgroup of the tile on it and
// tn_us with as many as it holds (LDS); a workgroup starts and ends in `start` us; the parts are joined by a launch of kJoinUs that moves
// them twice at kJoinBytes a us.  The figures are fitted to 16-bit outputs of 67 sizes (17 to 8192 tokens, N 576 to 7168, K 256 to 7168), each timed with
// every tile and 1 to 8 parts: the choice is 0.1 % off the fastest on average, 2.4 % at the most.  For fp32 outputs, whose products take four times as
// long, the same figures only order the tiles and parts: they are not fitted, and how far that choice is off is not measured.  us, by another tile / by the choice: 1531 x
// 7168 x 2048 28.9 (256 x 256) / 25.0 (192 x 256), 726 x 7168 x 2048 22.6 (192 x 256) / 17.9 (128 x 256), 490 x 7168 x 2048 22.1 (192 x
// 256) / 14.2 (128 x 128), 333 x 576 x 7168 18.9 (64 x 32, whole) / 12.9 (64 x 64, four parts), 48 x 7168 x 2048 9.4 (64 x 64) / 7.6 (64 x 32).
struct Fp8Tile {
  int tm, tn, held;
  float t1, tn_us, start;
};
enum { kT256, kT192, kT128x256, kT128, kT64, kT64x32, kFp8Tiles };
constexpr Fp8Tile kFp8Tile[kFp8Tiles] = {{256, 256, 1, 1.55f, 1.55f, 3.0f}, {192, 256, 1, 1.30f, 1.30f, 3.0f}, {128, 256, 1, 0.93f, 0.93f, 2.0f},
                                         {128, 128, 1, 0.60f, 0.60f, 2.0f}, {64, 64, 2, 0.30f, 0.54f, 1.9f},   {64, 32, 3, 0.23f, 0.60f, 1.2f}};
constexpr float kJoinUs = 3.2f, kJoinBytes = 4.7e6f;
constexpr int kMostParts = 8, kLeastBlocks = 4; // of K, in a part
struct Fp8Plan {
  int tile, parts;
};
static int64_t part_pitch(int64_t N) { return (N + 3) / 4 * 4; }
static Fp8Plan plan_gemm_fp8(int64_t M, int64_t N, int64_t KB, bool exact, bool may_split) {
  Fp8Plan best{-1, 1};
  float least = 0.0f;
  for (int i = exact ? kT128 : 0; i < kFp8Tiles; ++i) { // (an fp32 output's products take four times as long: tiles that leave room for them)
    const Fp8Tile &t = kFp8Tile[i];
    const int64_t tiles = ((M + t.tm - 1) / t.tm) * ((N + t.tn - 1) / t.tn);
    for (int parts = 1; parts <= (may_split && i >= kT128x256 ? kMostParts : 1); parts += parts < 4 ? 1 : 2) {
      const int64_t bytes = parts * M * part_pitch(N) * 4;
      if (parts > 1 && KB / parts < kLeastBlocks) break;
      const int64_t each = (tiles * parts + 255) / 256; // workgroups of a CU
      const float blocks = static_cast<float>((KB + parts - 1) / parts);
      const int64_t rounds = each / t.held, rest = each % t.held;
      float us = static_cast<float>(rounds) * (t.start + blocks * t.tn_us);
      if (rest) us += t.start + blocks * (t.t1 + (t.held > 1 ? (t.tn_us - t.t1) * static_cast<float>(rest - 1) / static_cast<float>(t.held - 1) : 0.0f));
      if (parts > 1) us += kJoinUs + 2.0f * static_cast<float>(bytes) / kJoinBytes;
      if (best.tile < 0 || us < least) best = {i, parts}, least = us;
    }
  }
  return best;
}

template <int DT, int TM, int TN, int WM, int WN, int ST> static int launch_tile(Fp8GemmArgs a, int parts, hipStream_t stream) {
  const int64_t m_tiles = (a.M + TM - 1) / TM, n_tiles = (a.N + TN - 1) / TN;
  LO_REQUIRE(m_tiles * n_tiles < (1 << 22), LO_ENOTSUP, "gemm_w8a8_fp8_block: %lld x %lld outputs", (long long)a.M, (long long)a.N);
  a.m_tiles = static_cast<int32_t>(m_tiles);
  a.n_tiles = static_cast<int32_t>(n_tiles);
  if constexpr (TM >= 192) {
    return launch_tile_parts<DT, TM, TN, WM, WN, ST, false>(a, stream);
  } else {
    if (parts <= 1) return launch_tile_parts<DT, TM, TN, WM, WN, ST, false>(a, stream);
    a.splits = parts;
    a.pitch = static_cast<int32_t>(part_pitch(a.N));
    // (parts are fp32: of a 16-bit output by one kernel for both types)
    const int rc = launch_tile_parts<DT == LO_F32 ? LO_F32 : LO_BF16, TM, TN, WM, WN, ST, true>(a, stream);
    return rc ? rc : join_parts<DT>(a, stream);
  }
}
constexpr int64_t kFp8FewTokens = 16; // gemm_fp8_few_kernel
template <int DT> static int launch_gemm_fp8(const Fp8GemmArgs &a, int64_t part_bytes, hipStream_t stream) {
  // us, this / the tiles: 1 x 4096 x 7168 9.1 / 11.5, 16: 11.2 / 12.1, 16 x 7168 x 2048 7.4 / 7.4; 32 tokens in two fragments 15.7 / 12.3
  if (a.M <= kFp8FewTokens) {
    const int waves = a.KB >= 16 ? 16 : a.KB >= 8 ? 8 : 4;
    hipLaunchKernelGGL((gemm_fp8_few_kernel<DT>), dim3(static_cast<unsigned>((a.N + 15) / 16)), dim3(waves * 64), 0, stream, a);
    return LO_OK;
  }
  // (with less room than the parts take K stays whole: the order of the sum goes by whether there is a workspace, not by its size)
  Fp8Plan p = plan_gemm_fp8(a.M, a.N, a.KB, DT == LO_F32, true);
  if (p.parts * a.M * part_pitch(a.N) * 4 > part_bytes && p.parts > 1) p = plan_gemm_fp8(a.M, a.N, a.KB, DT == LO_F32, false);
  if constexpr (DT != LO_F32) {
    if (p.tile == kT256) return launch_tile<DT, 256, 256, 2, 4, 2>(a, 1, stream);
    if (p.tile == kT192) return launch_tile<DT, 192, 256, 2, 4, 2>(a, 1, stream);
    if (p.tile == kT128x256) return launch_tile<DT, 128, 256, 2, 4, 3>(a, p.parts, stream);
  }
  if (p.tile == kT128) return launch_tile<DT, 128, 128, 2, 4, 4>(a, p.parts, stream);
  if (p.tile == kT64) return launch_tile<DT, 64, 64, 2, 2, 4>(a, p.parts, stream);
  return launch_tile<DT, 64, 32, 2, 2, 4>(a, p.parts, stream);
}

static int check_gemm_fp8_sizes(int64_t M, int64_t N, int64_t K, int out_dtype) {
  LO_REQUIRE(M >= 0 && N >= 0, LO_EINVAL, "gemm_w8a8_fp8_block: bad sizes %lld x %lld", (long long)M, (long long)N);
  LO_REQUIRE(K > 0 && K % kGroup == 0, LO_EINVAL, "gemm_w8a8_fp8_block: K (%lld) must be a multiple of 128", (long long)K);
  LO_REQUIRE(K <= (1 << 22), LO_ENOTSUP, "gemm_w8a8_fp8_block: K (%lld) is at most %d", (long long)K, 1 << 22);
  LO_REQUIRE(M <= (1 << 24) && N <= (1 << 24), LO_ENOTSUP, "gemm_w8a8_fp8_block: M and N are at most 2^24");
  LO_REQUIRE(out_dtype == LO_BF16 || out_dtype == LO_F16 || out_dtype == LO_F32, LO_ENOTSUP, "gemm_w8a8_fp8_block: the output is bf16, fp16 or fp32");
  return LO_OK;
}

} // namespace lo

extern "C" int64_t lo_gemm_w8a8_fp8_block_workspace_bytes(int64_t M, int64_t N, int64_t K, int out_dtype) {
  using namespace lo;
  const int rc = check_gemm_fp8_sizes(M, N, K, out_dtype);
  if (rc) return rc;
  if (M <= kFp8FewTokens || N == 0) return 0;
  const Fp8Plan p = plan_gemm_fp8(M, N, K / kGroup, out_dtype == LO_F32, true);
  return p.parts > 1 ? p.parts * M * part_pitch(N) * 4 : 0;
}

extern "C" int lo_gemm_w8a8_fp8_block_tile_query(int64_t M, int64_t N, int64_t K, int out_dtype, int has_workspace, int32_t *tile_m, int32_t *tile_n,
                                                 int32_t *parts) {
  using namespace lo;
  const int rc = check_gemm_fp8_sizes(M, N, K, out_dtype);
  if (rc) return rc;
  LO_REQUIRE(tile_m && tile_n && parts, LO_EINVAL, "gemm_w8a8_fp8_block_tile_query: null pointer");
  const bool few = M <= kFp8FewTokens;
  const Fp8Plan p = few || N == 0 ? Fp8Plan{kT64x32, 1} : plan_gemm_fp8(M, N, K / kGroup, out_dtype == LO_F32, has_workspace != 0);
  *tile_m = few ? 16 : kFp8Tile[p.tile].tm;
  *tile_n = few ? 16 : kFp8Tile[p.tile].tn;
  *parts = p.parts;
  return LO_OK;
}

extern "C" int lo_gemm_w8a8_fp8_block(const void *a, const float *a_scale, const void *b, const float *b_scale, void *c, int out_dtype,
                                      int64_t M, int64_t N, int64_t K, void *workspace, int64_t workspace_bytes, lo_stream_t stream) {
  using namespace lo;
  const int bad = check_gemm_fp8_sizes(M, N, K, out_dtype);
  if (bad) return bad;
  if (M == 0 || N == 0) return LO_OK;
  LO_REQUIRE(a && a_scale && b && b_scale && c, LO_EINVAL, "gemm_w8a8_fp8_block: null pointer");
  const auto off = [](const void *p, unsigned al) { return (reinterpret_cast<uintptr_t>(p) & (al - 1)) != 0; };
  LO_REQUIRE(!off(a, 16) && !off(b, 16) && !off(a_scale, 4) && !off(b_scale, 4) && !off(c, out_dtype == LO_F32 ? 4 : 2), LO_EINVAL,
             "gemm_w8a8_fp8_block: operands must be 16-byte aligned");
  LO_REQUIRE(!off(workspace, 16) && workspace_bytes >= 0, LO_EINVAL, "gemm_w8a8_fp8_block: the workspace must be 16-byte aligned");
  const int64_t room = workspace ? workspace_bytes : 0;
  const Fp8GemmArgs args{static_cast<const int8_t *>(a), static_cast<const int8_t *>(b), a_scale, b_scale, c, static_cast<float *>(workspace), M, N, K,
                         static_cast<int32_t>(K / kGroup), 0, 0, 1, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = out_dtype == LO_BF16 ? launch_gemm_fp8<LO_BF16>(args, room, s)
                 : out_dtype == LO_F16 ? launch_gemm_fp8<LO_F16>(args, room, s)
                                          : launch_gemm_fp8<LO_F32>(args, room, s);
  return rc ? rc : check_launch("gemm_w8a8_fp8_block");
}
