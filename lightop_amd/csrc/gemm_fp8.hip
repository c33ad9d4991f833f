// Dense product of e4m3 operands with a scale for each block of 128:
//   C[m, n] = sum over kb of (A[m, kb] . B[n, kb]) * As[m, kb] * Bs[n / 128, kb],
// A [M, K] rows with one scale for 128 values, B [N, K] a weight with one for 128 x 128.  A K block's 128 products are one MFMA
// (v_mfma_f32_16x16x128_f8f6f4, which starts from zero), its fp32 result is folded into the fp32 sum with the scales' product.
// (An fp32 output takes the exact form of it, fp8.h.)  Weights are the A operand: a lane holds four neighbouring columns of C for one token, whose scale it carries.
#include "gemm.h"
#include "fp8.h"

namespace lo {

struct Fp8GemmArgs {
  const int8_t *A, *B;
  const float *As, *Bs;
  void *C;
  int64_t M, N, K;
  int32_t KB, m_tiles, n_tiles;
};

template <int DT> __device__ __forceinline__ void store_c(void *c, int64_t at, float v) {
  if constexpr (DT == LO_F32) static_cast<float *>(c)[at] = v;
  else static_cast<uint16_t *>(c)[at] = from_f32<DT>(v);
}

// ---- few tokens ------------------------------------------------------------------------------------------------------------
// A workgroup takes 16 columns and all tokens; its waves share the K blocks and add their sums up through LDS, in the same order every time.
// Weights are read once, straight into registers.
template <int DT, int NF>
__global__ __launch_bounds__(1024) void gemm_fp8_few_kernel(const Fp8GemmArgs a) {
  extern __shared__ float red[]; // [wave][token][column]
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int K = static_cast<int>(a.K), KB = a.KB;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t cols = a.N - n0 < 16 ? a.N - n0 : 16;
  const brsrc rB = make_rsrc(a.B + n0 * K, static_cast<uint32_t>(cols * K));
  const brsrc rA = make_rsrc(a.A, static_cast<uint32_t>(a.M * K));
  const brsrc rS = make_rsrc(a.As, static_cast<uint32_t>(a.M * KB * 4));
  const float *const bs = a.Bs + (n0 >> 7) * KB;
  v4f acc[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) acc[f] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = NF == 1 ? 4 : NF == 2 ? 3 : 2; // K blocks in flight
  for (int kb0 = wave; kb0 < KB; kb0 += waves * U) {
    v8i w[U], x[U][NF];
    float s[U][NF], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * waves;
      const int kc = kb < KB ? kb : kb0; // past the end: this one again, left out below
      const int at = r * K + q * 16 + kc * kGroup;
      w[u] = join(bld16<kCacheStream>(rB, at, 0), bld16<kCacheStream>(rB, at + 64, 0));
      b[u] = bs[kc];
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        x[u][f] = join(bld16(rA, at + f * 16 * K, 0), bld16(rA, at + f * 16 * K + 64, 0));
        s[u][f] = bld_f32(rS, ((f * 16 + r) * KB + kc) * 4, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb0 + u * waves >= KB) break;
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const v4f d = mfma_e4m3_for<DT>(w[u], x[u][f]);
        const float sc = s[u][f] * b[u];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][i] = __builtin_fmaf(d[i], sc, acc[f][i]);
      }
    }
  }
#pragma unroll
  for (int f = 0; f < NF; ++f) *reinterpret_cast<v4f *>(red + ((wave * NF + f) * 16 + r) * 16 + 4 * q) = acc[f];
  __syncthreads();
  for (int o = threadIdx.x; o < NF * 256; o += blockDim.x) {
    const int64_t m = o >> 4, n = n0 + (o & 15);
    if (m >= a.M || n >= a.N) continue;
    float v = red[o];
    for (int i = 1; i < waves; ++i) v += red[i * NF * 256 + o];
    store_c<DT>(a.C, m * a.N + n, v);
  }
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
// Both operands go to LDS by direct loads, a K block at a time in two stages; 16-byte pieces of a row are swizzled by the row.
__device__ __forceinline__ void copy16(brsrc r, int8_t *lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, voff, soff, 0, 0);
}
template <int N> __device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int DT, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void gemm_fp8_tile_kernel(const Fp8GemmArgs a, int group_m) {
  constexpr int kWaves = WM * WN, kThreads = kWaves * 64;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16; // fragments of a wave: tokens, weights
  constexpr int kPieces = (TM + TN) / 8, kPer = kPieces / kWaves; // 1 KB copies of a stage, of a wave
  constexpr int kStage = (TM + TN) * kGroup;
  static_assert(kPieces % kWaves == 0 && TM % 8 == 0 && (TN / WN) % 16 == 0 && 128 % (TN / WN) == 0 && TM <= kThreads, "tile");
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  float *const sS = reinterpret_cast<float *>(smem + 2 * kStage); // [stage][token]
  int mt, nt;
  if (!dense_tile(blockIdx.x, a.m_tiles, a.n_tiles, group_m, mt, nt)) return;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
  const int K = static_cast<int>(a.K), KB = a.KB;
  const int64_t m0 = static_cast<int64_t>(mt) * TM, n0 = static_cast<int64_t>(nt) * TN;
  const int rows = static_cast<int>(a.M - m0 < TM ? a.M - m0 : TM), cols = static_cast<int>(a.N - n0 < TN ? a.N - n0 : TN);
  // rows past the end are past the extents, and read as zero
  const brsrc rA = make_rsrc(a.A + m0 * K, static_cast<uint32_t>(rows * K));
  const brsrc rB = make_rsrc(a.B + n0 * K, static_cast<uint32_t>(cols * K));
  const brsrc rS = make_rsrc(a.As + m0 * KB, static_cast<uint32_t>(rows * KB * 4));
  int voff[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int p = wave * kPer + j, row = (p < TM / 8 ? p : p - TM / 8) * 8 + (lane >> 3);
    voff[j] = row * K + (((lane & 7) ^ (row & 7)) * 16);
  }
  auto copy = [&](int kb) __attribute__((always_inline)) {
    const int soff = kb * kGroup;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int p = wave * kPer + j;
      int8_t *const to = smem + (kb & 1) * kStage + p * 1024;
      if (p < TM / 8) copy16(rA, to, voff[j], soff);
      else copy16(rB, to, voff[j], soff);
    }
  };
  int64_t nblk = (n0 + wn * (TN / WN)) >> 7;
  const int64_t last = (a.N - 1) >> 7;
  nblk = nblk < last ? nblk : last;
  const float *const bs = a.Bs + nblk * KB;
  const int lds0 = r * kGroup + ((q ^ (r & 7)) * 16), lds1 = r * kGroup + (((q + 4) ^ (r & 7)) * 16);
  v4f acc[FM][FN];
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[m][n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  auto load_s = [&](int kb) __attribute__((always_inline)) { return bld_f32(rS, (tid < TM ? tid : 0) * KB * 4, (kb < KB ? kb : KB - 1) * 4); };

  copy(0);
  float s = load_s(0);
  if (tid < TM) sS[tid] = s;
  s = load_s(1);
  for (int kb = 0; kb < KB; ++kb) {
    wait_barrier<0>(); // this K block is in LDS, and nobody reads the one before any more
    if (kb + 1 < KB) copy(kb + 1);
    if (tid < TM) sS[((kb + 1) & 1) * TM + tid] = s;
    s = load_s(kb + 2);
    const int8_t *const sa = smem + (kb & 1) * kStage + wm * (TM / WM) * kGroup;
    const int8_t *const sb = smem + (kb & 1) * kStage + TM * kGroup + wn * (TN / WN) * kGroup;
    const float *const ss = sS + (kb & 1) * TM + wm * (TM / WM);
    const float b = bs[kb];
    v8i w[FN];
#pragma unroll
    for (int n = 0; n < FN; ++n)
      w[n] = join(*reinterpret_cast<const v4i *>(sb + n * 2048 + lds0), *reinterpret_cast<const v4i *>(sb + n * 2048 + lds1));
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const v8i x = join(*reinterpret_cast<const v4i *>(sa + m * 2048 + lds0), *reinterpret_cast<const v4i *>(sa + m * 2048 + lds1));
      const float sc = ss[m * 16 + r] * b;
#pragma unroll
      for (int n = 0; n < FN; ++n) {
        const v4f d = mfma_e4m3_for<DT>(w[n], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][n][i] = __builtin_fmaf(d[i], sc, acc[m][n][i]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < FM; ++m) {
    const int mr = wm * (TM / WM) + m * 16 + r;
    if (mr >= rows) continue;
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int nc = wn * (TN / WN) + n * 16 + 4 * q + i;
        if (nc < cols) store_c<DT>(a.C, (m0 + mr) * a.N + n0 + nc, acc[m][n][i]);
      }
  }
}

template <int DT, int TM, int TN, int WM, int WN> static int launch_tile(Fp8GemmArgs a, hipStream_t stream) {
  constexpr int lds = 2 * (TM + TN) * kGroup + 2 * TM * 4;
  const auto kernel = gemm_fp8_tile_kernel<DT, TM, TN, WM, WN>;
  static unsigned long long done = 0;
  const int rc = reserve_lds_once(reinterpret_cast<const void *>(kernel), lds, &done);
  if (rc) return rc;
  a.m_tiles = static_cast<int32_t>((a.M + TM - 1) / TM);
  a.n_tiles = static_cast<int32_t>((a.N + TN - 1) / TN);
  const int group_m = a.m_tiles < 4 ? a.m_tiles : 4;
  const int64_t tiles = static_cast<int64_t>(a.m_tiles) * a.n_tiles;
  LO_REQUIRE(tiles < (1 << 22), LO_ENOTSUP, "gemm_w8a8_fp8_block: %lld x %lld outputs", (long long)a.M, (long long)a.N);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((tiles + 7) / 8 * 8)), dim3(WM * WN * 64), lds, stream, a, group_m);
  return LO_OK;
}
template <int DT, int NF> static int launch_few(const Fp8GemmArgs &a, hipStream_t stream) {
  const int waves = a.KB >= 16 ? 16 : a.KB >= 8 ? 8 : 4;
  hipLaunchKernelGGL((gemm_fp8_few_kernel<DT, NF>), dim3(static_cast<unsigned>((a.N + 15) / 16)), dim3(waves * 64), waves * NF * 1024,
                     stream, a);
  return LO_OK;
}
template <int DT> static int launch_gemm_fp8(const Fp8GemmArgs &a, hipStream_t stream) {
  if (a.M <= 16) return launch_few<DT, 1>(a, stream);
  if (a.M <= 32) return launch_few<DT, 2>(a, stream);
  if (a.M <= 64) return launch_few<DT, 4>(a, stream);
  return launch_tile<DT, 128, 128, 2, 2>(a, stream);
}

} // namespace lo

extern "C" int lo_gemm_w8a8_fp8_block(const void *a, const float *a_scale, const void *b, const float *b_scale, void *c, int out_dtype,
                                      int64_t M, int64_t N, int64_t K, lo_stream_t stream) {
  using namespace lo;
  LO_REQUIRE(M >= 0 && N >= 0, LO_EINVAL, "gemm_w8a8_fp8_block: bad sizes %lld x %lld", (long long)M, (long long)N);
  LO_REQUIRE(K > 0 && K % kGroup == 0, LO_EINVAL, "gemm_w8a8_fp8_block: K (%lld) must be a multiple of 128", (long long)K);
  LO_REQUIRE(K <= (1 << 22), LO_ENOTSUP, "gemm_w8a8_fp8_block: K (%lld) is at most %d", (long long)K, 1 << 22);
  LO_REQUIRE(M <= (1 << 24) && N <= (1 << 24), LO_ENOTSUP, "gemm_w8a8_fp8_block: M and N are at most 2^24");
  LO_REQUIRE(out_dtype == LO_BF16 || out_dtype == LO_F16 || out_dtype == LO_F32, LO_ENOTSUP, "gemm_w8a8_fp8_block: the output is bf16, fp16 or fp32");
  if (M == 0 || N == 0) return LO_OK;
  LO_REQUIRE(a && a_scale && b && b_scale && c, LO_EINVAL, "gemm_w8a8_fp8_block: null pointer");
  const auto off = [](const void *p, unsigned al) { return (reinterpret_cast<uintptr_t>(p) & (al - 1)) != 0; };
  LO_REQUIRE(!off(a, 16) && !off(b, 16) && !off(a_scale, 4) && !off(b_scale, 4) && !off(c, out_dtype == LO_F32 ? 4 : 2), LO_EINVAL,
             "gemm_w8a8_fp8_block: operands must be 16-byte aligned");
  const Fp8GemmArgs args{static_cast<const int8_t *>(a), static_cast<const int8_t *>(b), a_scale, b_scale, c, M, N, K,
                         static_cast<int32_t>(K / kGroup), 0, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = out_dtype == LO_BF16 ? launch_gemm_fp8<LO_BF16>(args, s)
                 : out_dtype == LO_F16 ? launch_gemm_fp8<LO_F16>(args, s) : launch_gemm_fp8<LO_F32>(args, s);
  return rc ? rc : check_launch("gemm_w8a8_fp8_block");
}
