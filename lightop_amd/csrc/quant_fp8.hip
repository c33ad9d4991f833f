// e4m3 quantisation of rows in groups of 128, plain or of a gated activation: act(x[:, :I]) * x[:, I:] in fp32.  16 lanes hold a group,
// eight values each: a 16-byte load of either half, a maximum over four lane steps, an 8-byte store, no LDS.  HBM bounds it, GELU aside: in a
// captured graph, over inputs of more than the caches hold, plain rows of 8192 x 7168 bf16 37.5 us (4.75 TB/s), fp32 53.6 (5.5); SiLU of 8192 x 4096
// bf16 38.2 (4.4), of 4096 x 2048 11.9 (3.6; 9.5 with the inputs in the caches); 333 x 7168 plain 3.1, the launch.  GELU's complement of the error function
// is vector work: 8192 x 4096 57.2 us (3.0 TB/s), 4096 x 2048 15.9.
#include "fp8.h"

namespace lo {

// ACT: -1 plain, else the activation.  per_row: groups of a row of the output.
template <int DT, int ACT>
__global__ __launch_bounds__(256) void group_quant_fp8_kernel(const void *__restrict__ x, int64_t groups, int64_t per_row, float floor,
                                                              int8_t *__restrict__ q, float *__restrict__ s) {
  const int sub = threadIdx.x & 15;
  for (int64_t g = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4); g < groups; g += static_cast<int64_t>(gridDim.x) * 16) {
    float v[8];
    if constexpr (ACT < 0) {
      load8<DT>(x, g * kGroup + sub * 8, v);
    } else {
      const int64_t at = (g + g / per_row * per_row) * kGroup + sub * 8; // a row of the input is gate and up
      float u[8];
      load8<DT>(x, at, v);
      load8<DT>(x, at + per_row * kGroup, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_mul_f32<ACT>(v[i], u[i]);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    float sc;
    const Fp8Group grp = fp8_group(fmaxf(top, floor), sc);
    *reinterpret_cast<v2i *>(q + g * kGroup + sub * 8) = v2i{fp8_pack4(&v[0], grp), fp8_pack4(&v[4], grp)};
    if (sub == 0) s[g] = sc;
  }
}

template <int ACT>
static void launch_group_quant_fp8(const void *x, int dtype, int64_t rows, int64_t cols, float floor, int8_t *q, float *s,
                                   hipStream_t stream) {
  const int64_t per_row = cols / kGroup, groups = rows * per_row, blocks = (groups + 15) / 16;
  const dim3 grid(static_cast<unsigned>(blocks < 65536 ? blocks : 65536));
  if (dtype == LO_BF16)
    hipLaunchKernelGGL((group_quant_fp8_kernel<LO_BF16, ACT>), grid, dim3(256), 0, stream, x, groups, per_row, floor, q, s);
  else if (dtype == LO_F16)
    hipLaunchKernelGGL((group_quant_fp8_kernel<LO_F16, ACT>), grid, dim3(256), 0, stream, x, groups, per_row, floor, q, s);
  else
    hipLaunchKernelGGL((group_quant_fp8_kernel<LO_F32, ACT>), grid, dim3(256), 0, stream, x, groups, per_row, floor, q, s);
}

static int check_group_quant_fp8(const char *what, const void *x, int dtype, int64_t rows, int64_t cols, const void *q, const void *s) {
  LO_REQUIRE(dtype == LO_BF16 || dtype == LO_F16 || dtype == LO_F32, LO_ENOTSUP, "%s: bf16, fp16 or fp32", what);
  LO_REQUIRE(rows >= 0 && cols > 0 && cols % kGroup == 0, LO_EINVAL, "%s: the output width (%lld) must be a multiple of 128", what,
             (long long)cols);
  LO_REQUIRE(rows == 0 || (x && q && s), LO_EINVAL, "%s: null pointer", what);
  LO_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0 &&
                 (reinterpret_cast<uintptr_t>(s) & 3) == 0,
             LO_EINVAL, "%s: input must be 16-byte and q 8-byte aligned", what);
  return LO_OK;
}

} // namespace lo

extern "C" int lo_per_token_group_quant_fp8(const void *x, int dtype, int64_t rows, int64_t cols, float eps, void *q, float *s,
                                            lo_stream_t stream) {
  using namespace lo;
  const int rc = check_group_quant_fp8("per_token_group_quant_fp8", x, dtype, rows, cols, q, s);
  if (rc) return rc;
  // (a smaller floor lets a group's reciprocal leave the normal range)
  LO_REQUIRE(eps >= 1e-30f && eps < __builtin_inff(), LO_EINVAL, "per_token_group_quant_fp8: eps (%g) must be from 1e-30 up and finite", eps);
  if (rows == 0) return LO_OK;
  launch_group_quant_fp8<-1>(x, dtype, rows, cols, eps, static_cast<int8_t *>(q), s, static_cast<hipStream_t>(stream));
  return check_launch("per_token_group_quant_fp8");
}

extern "C" int lo_act_mul_group_quant_fp8(const void *c1, int dtype, int activation, int64_t rows, int64_t I, void *q, float *s,
                                          lo_stream_t stream) {
  using namespace lo;
  const int rc = check_group_quant_fp8("act_mul_group_quant_fp8", c1, dtype, rows, I, q, s);
  if (rc) return rc;
  LO_REQUIRE(activation == LO_ACT_SILU || activation == LO_ACT_GELU, LO_EINVAL, "act_mul_group_quant_fp8: unknown activation %d", activation);
  if (rows == 0) return LO_OK;
  if (activation == LO_ACT_GELU)
    launch_group_quant_fp8<LO_ACT_GELU>(c1, dtype, rows, I, 1e-10f, static_cast<int8_t *>(q), s, static_cast<hipStream_t>(stream));
  else
    launch_group_quant_fp8<LO_ACT_SILU>(c1, dtype, rows, I, 1e-10f, static_cast<int8_t *>(q), s, static_cast<hipStream_t>(stream));
  return check_launch("act_mul_group_quant_fp8");
}
