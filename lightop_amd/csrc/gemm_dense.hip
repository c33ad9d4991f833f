// Entry points of the dense product with an epilogue (gemm_dense.h).
#include "gemm_dense.h"

namespace lo {

// A wave takes 16 rows of A and 16 columns of C (gated: of both halves), operands straight from memory.
template <int DT> __global__ __launch_bounds__(256) void gemm_dense_simple_kernel(const DenseArgs a) {
  typedef Operand<DT> Op;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, wave = threadIdx.x >> 6;
  const int columns = static_cast<int>((a.N + 15) / 16);
  const int64_t m = (static_cast<int64_t>(blockIdx.x / columns) * 4 + wave) * 16 + r, n0 = static_cast<int64_t>(blockIdx.x % columns) * 16;
  const int64_t ma = m < a.M ? m : a.M - 1, nb = n0 + r < a.N ? n0 + r : a.N - 1;
  const int8_t *const pa = a.A + ma * a.lda, *const pb = a.B + nb * a.ldb, *const pu = a.B + (nb + a.N) * a.ldb;
  typename Op::Acc g = {}, u = {};
  for (int k = 0; k < a.K; k += 64) {
    const int at = k + q * 16;
    v4i x = {}, w = {}, y = {};
    if (at < a.K) {
      x = *reinterpret_cast<const v4i *>(pa + at);
      w = *reinterpret_cast<const v4i *>(pb + at);
      if (a.gated) y = *reinterpret_cast<const v4i *>(pu + at);
    }
    g = Op::mfma(w, x, g);
    if (a.gated) u = Op::mfma(y, x, u);
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + 4 * q + i;
    if (m >= a.M || n >= a.N) continue;
    float v = activate(a.act, dense_value(a, g[i], m, n));
    if (a.gated) v *= dense_value(a, u[i], m, n + a.N);
    dense_store(a, v, m, n);
  }
}

constexpr int64_t kMostStride = 4 << 20; // bytes: 256 rows of a tile stay within 2^30
static int check_dense_sizes(int dtype, int64_t M, int64_t N, int64_t K) {
  LO_REQUIRE(dtype == LO_BF16 || dtype == LO_F16 || dtype == LO_I8, LO_ENOTSUP, "gemm_bias_act: operands are bf16, fp16 or int8");
  LO_REQUIRE(M >= 0 && N >= 0, LO_EINVAL, "gemm_bias_act: bad sizes %lld x %lld", (long long)M, (long long)N);
  const int64_t unit = dtype == LO_I8 ? 16 : 8, most = dtype == LO_I8 ? 131056 : kMostStride / 2; // (sums of int8 products stay below 2^31)
  LO_REQUIRE(K > 0 && K % unit == 0, LO_EINVAL, "gemm_bias_act: K (%lld) must be a multiple of %lld", (long long)K, (long long)unit);
  LO_REQUIRE(K <= most, LO_ENOTSUP, "gemm_bias_act: K (%lld) is at most %lld", (long long)K, (long long)most);
  LO_REQUIRE(M <= (1 << 24) && N <= (1 << 23), LO_ENOTSUP, "gemm_bias_act: %lld x %lld outputs (at most 2^24 x 2^23)", (long long)M, (long long)N);
  return LO_OK;
}

} // namespace lo

extern "C" int64_t lo_gemm_bias_act_workspace_bytes(int dtype, int gated, int64_t M, int64_t N, int64_t K) {
  using namespace lo;
  (void)gated;
  const int rc = check_dense_sizes(dtype, M, N, K);
  return rc;
}

extern "C" int lo_gemm_bias_act(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int dtype, const float *a_scale, const float *b_scale,
                                const void *bias, int bias_dtype, int activation, int gated, float scale, const void *residual, int64_t residual_stride,
                                void *c, int out_dtype, int64_t M, int64_t N, int64_t K, void *workspace, int64_t workspace_bytes, lo_stream_t stream) {
  using namespace lo;
  const int bad = check_dense_sizes(dtype, M, N, K);
  if (bad) return bad;
  LO_REQUIRE(out_dtype == LO_BF16 || out_dtype == LO_F16 || out_dtype == LO_F32, LO_ENOTSUP, "gemm_bias_act: the output is bf16, fp16 or fp32");
  LO_REQUIRE(activation == LO_ACT_NONE || activation == LO_ACT_SILU || activation == LO_ACT_GELU, LO_EINVAL, "gemm_bias_act: unknown activation %d",
             activation);
  LO_REQUIRE(!bias || bias_dtype == out_dtype || bias_dtype == LO_F32, LO_ENOTSUP, "gemm_bias_act: the bias has the output's type or is fp32");
  if (M == 0 || N == 0) return LO_OK;
  const bool i8 = dtype == LO_I8;
  const int64_t size = i8 ? 1 : 2, out_size = out_dtype == LO_F32 ? 4 : 2, rows = gated ? 2 * N : N;
  LO_REQUIRE(a && b && c && i8 == (a_scale != nullptr) && i8 == (b_scale != nullptr), LO_EINVAL,
             "gemm_bias_act: null pointer, or scales of 16-bit operands");
  LO_REQUIRE((M == 1 || a_stride >= K) && (rows == 1 || b_stride >= K) && (!residual || M == 1 || residual_stride >= N), LO_EINVAL,
             "gemm_bias_act: rows overlap (strides %lld, %lld, %lld)", (long long)a_stride, (long long)b_stride, (long long)residual_stride);
  const int64_t lda = (M == 1 ? K : a_stride) * size, ldb = (rows == 1 ? K : b_stride) * size;
  LO_REQUIRE(lda <= kMostStride && ldb <= kMostStride, LO_ENOTSUP, "gemm_bias_act: rows are at most 4 MiB apart");
  const auto off = [](const void *p, int64_t al) { return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(al - 1)) != 0; };
  LO_REQUIRE(!off(a, 16) && !off(b, 16) && lda % 16 == 0 && ldb % 16 == 0, LO_EINVAL, "gemm_bias_act: operands' rows must be 16-byte aligned");
  LO_REQUIRE(!off(a_scale, 4) && !off(b_scale, 4) && !off(c, out_size) && !off(residual, out_size) &&
                 !off(bias, bias_dtype == LO_F32 ? 4 : out_size),
             LO_EINVAL, "gemm_bias_act: a pointer is not aligned to its type");
  LO_REQUIRE(!off(workspace, 16) && workspace_bytes >= 0, LO_EINVAL, "gemm_bias_act: the workspace must be 16-byte aligned");
  const uintptr_t c0 = reinterpret_cast<uintptr_t>(c), c1 = c0 + M * N * out_size;
  const auto meets = [&](const void *p, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return p && at < c1 && c0 < at + bytes;
  };
  LO_REQUIRE(!meets(a, (M - 1) * lda + K * size) && !meets(b, (rows - 1) * ldb + K * size) && !meets(a_scale, 4 * M) && !meets(b_scale, 4 * rows) &&
                 !meets(bias, rows * (bias_dtype == LO_F32 ? 4 : out_size)) &&
                 !(meets(residual, ((M - 1) * residual_stride + N) * out_size) && !(residual == c && (M == 1 || residual_stride == N))),
             LO_EINVAL, "gemm_bias_act: the output overlaps an input");
  DenseArgs args{static_cast<const int8_t *>(a), static_cast<const int8_t *>(b), a_scale, b_scale, bias, residual, c, M, N, M == 1 ? N : residual_stride,
                 static_cast<int32_t>(lda), static_cast<int32_t>(ldb), static_cast<int32_t>(K * size), activation, gated != 0, bias_dtype == LO_F32,
                 out_dtype, scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t workgroups = (N + 15) / 16 * ((M + 63) / 64);
  LO_REQUIRE(workgroups < (1 << 24), LO_ENOTSUP, "gemm_bias_act: %lld x %lld outputs", (long long)M, (long long)N);
  const dim3 grid(static_cast<unsigned>(workgroups));
  if (dtype == LO_BF16) hipLaunchKernelGGL((gemm_dense_simple_kernel<LO_BF16>), grid, dim3(256), 0, s, args);
  else if (dtype == LO_F16) hipLaunchKernelGGL((gemm_dense_simple_kernel<LO_F16>), grid, dim3(256), 0, s, args);
  else hipLaunchKernelGGL((gemm_dense_simple_kernel<LO_I8>), grid, dim3(256), 0, s, args);
  return check_launch("gemm_bias_act");
}
