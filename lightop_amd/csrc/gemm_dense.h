// Dense product with an epilogue:
//   v[m, n] = sum over k of A[m, k] * B[n, k] (int8: times As[m] * Bs[n]) + bias[n]
//   C[m, n] = scale * act(v[m, n]) + R[m, n];  gated: scale * act(v[m, n]) * v[m, N + n] + R[m, n].
// Sums, and everything behind them, are fp32 (int8: the sum is int32 and exact); a result is rounded once.
#pragma once
#include "fp8.h"
#include "gemm.h"

namespace lo {

struct DenseArgs {
  const int8_t *A, *B;
  const float *As, *Bs;
  const void *bias, *R;
  void *C;
  int64_t M, N, rs;  // rs: R's row stride, in values
  int32_t lda, ldb;  // bytes
  int32_t K;         // bytes of a row, a multiple of 16
  int32_t act, gated, bias_f32, out;
  float scale;
};

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// The operands' types: sixteen bytes a lane of 16 rows of either operand, 64 bytes of K, into the 16 x 16 sums.
template <int DT> struct Operand {
  static constexpr int kSize = 2;
  typedef v4f Acc;
  static __device__ __forceinline__ Acc mfma(const v4i a, const v4i b, const Acc c) {
    if constexpr (DT == LO_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <> struct Operand<LO_I8> {
  static constexpr int kSize = 1;
  typedef v4i Acc;
  static __device__ __forceinline__ Acc mfma(const v4i a, const v4i b, const Acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float load_value(const void *p, int type, int64_t at) {
  if (type == LO_F32) return static_cast<const float *>(p)[at];
  const uint16_t h = static_cast<const uint16_t *>(p)[at];
  return type == LO_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}
__device__ __forceinline__ void store_value(void *p, int type, int64_t at, float v) {
  if (type == LO_F32) static_cast<float *>(p)[at] = v;
  else static_cast<uint16_t *>(p)[at] = type == LO_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
}
__device__ __forceinline__ float activate(int act, float v) { return act == LO_ACT_SILU ? silu_f32(v) : act == LO_ACT_GELU ? gelu_f32(v) : v; }
// A row's value before the activation; n counts B's rows.
template <class T> __device__ __forceinline__ float dense_value(const DenseArgs &a, T sum, int64_t m, int64_t n) {
  float v = static_cast<float>(sum);
  if (a.As) v = v * a.As[m] * a.Bs[n];
  return a.bias ? v + load_value(a.bias, a.bias_f32 ? LO_F32 : a.out, n) : v;
}
__device__ __forceinline__ void dense_store(const DenseArgs &a, float v, int64_t m, int64_t n) {
  store_value(a.C, a.out, m * a.N + n, a.R ? __builtin_fmaf(a.scale, v, load_value(a.R, a.out, m * a.rs + n)) : a.scale * v);
}

} // namespace lo
