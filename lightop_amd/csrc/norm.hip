// RMS norm with the residual's addition, ending in 8 bits: what stands in front of a quantised layer.
//   z = x + r,  y = z * (mean(z^2) + eps)^-1/2 * w,  and y's codes and scales,
// everything in fp32 between the inputs and the outputs; z and, where it is asked for, y are rounded once to the rows' type.  The 8-bit
// rules are the package's: int8 per token (reference: int8_utils.py:20-44), int8 per 128 values (int8_utils.py:74-122), e4m3 per
// 128 values (fp8.h).
//
// One pass: a row stays in registers between its sum of squares and its codes (and, per token, its maximum), so a value is read once and
// every output written once.  A workgroup a row: the row's two reductions then meet in LDS, and thousands of rows fill the card; rows that
// several workgroups shared would need a second launch.  What bounds it is HBM (with a residual, e4m3 codes: 8192 x 7168 bf16, 413 MB in 79-82 us,
// 5.0-5.2 TB/s, what a copy reaches; fp32, 765 MB in 140 us, 5.5 TB/s; 4096 x 4096 fp32 42 us), for a few hundred rows the chain of load, barrier and
// store (700 x 4096 bf16 6.2 us, fp16 with int8 groups and the normed rows 7.3), for one row the launch (2.8 us).  The weight asked for in
// front of the first barrier gained nothing.  (Times in a captured graph, over inputs of more than the caches hold.)
#include "fp8.h"

namespace lo {

constexpr int64_t kNormMaxH = 65536;
// Up to so many rows a thread takes one piece (a row's steps, one behind the other, are what counts), beyond as many as fill 256 threads.  us (inputs in the caches), so /
// with 256 threads, bf16 rows with a residual, e4m3: 512 x 7168 7.6 / 8.7, 700 x 4096 6.2 / 6.6, 1000 x 7168 12.6 / 11.8, 2048 x 7168 21.1 / 19.9.
constexpr int64_t kNormFew = 768;

struct NormArgs {
  const void *x, *r, *w;
  void *z, *y;
  int8_t *q;
  float *s;
  int64_t xs, rs; // row strides, in values
  int32_t H;
  int32_t w_f32;
  int64_t row0; // of the launch's first workgroup
  float eps;
};

// The sum, or the maximum, over the workgroup's waves of values that its lanes have already reduced.
template <bool MAX> __device__ __forceinline__ float across_waves(float v, float *red, int waves) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float o = __shfl_xor(v, d);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < waves; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  return v;
}

// A workgroup a row; CH pieces of eight values a thread.
template <int DT, int FORM, int CH>
__global__ __launch_bounds__(1024) void rms_norm_quant_kernel(const NormArgs a) {
  __shared__ float red[2][16];
  const int tid = threadIdx.x, threads = blockDim.x, waves = threads >> 6;
  const int pieces = a.H / 8;
  const int64_t row = a.row0 + blockIdx.x, base = row * a.H;
  float v[CH][8];
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int p = tid + j * threads;
    if (p < pieces) {
      load8<DT>(a.x, row * a.xs + p * 8, v[j]);
      if (a.r) {
        float r[8];
        load8<DT>(a.r, row * a.rs + p * 8, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] += r[i];
        store8<DT>(a.z, base + p * 8, v[j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[j][i], v[j][i], ss);
  }
  ss = across_waves<false>(ss, red[0], waves);
  const float rstd = 1.0f / sqrtf(ss / static_cast<float>(a.H) + a.eps);

  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int p = tid + j * threads;
    if (p < pieces) {
      float w[8];
      if (a.w_f32) load8<LO_F32>(a.w, p * 8, w);
      else load8<DT>(a.w, p * 8, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rstd * w[i];
      if (a.y) store8<DT>(a.y, base + p * 8, v[j]);
    }
    if constexpr (FORM == LO_Q_INT8_ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[j][i]));
    } else if (p < pieces) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[j][i]));
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d)); // 16 lanes hold a group, all of them in the row or none
      top = fmaxf(top, 1e-10f);
      float s;
      v2i packed;
      if constexpr (FORM == LO_Q_FP8_GROUPS) {
        const Fp8Group g = fp8_group(top, s);
        packed = v2i{fp8_pack4(&v[j][0], g), fp8_pack4(&v[j][4], g)};
      } else {
        s = top / 127.0f;
        const float y = 1.0f / s;
        packed = v2i{static_cast<int>(quant4(&v[j][0], s, y)), static_cast<int>(quant4(&v[j][4], s, y))};
      }
      *reinterpret_cast<v2i *>(a.q + base + p * 8) = packed;
      if ((tid & 15) == 0) a.s[(base >> 7) + (p >> 4)] = s;
    }
  }
  if constexpr (FORM == LO_Q_INT8_ROWS) {
    amax = fmaxf(across_waves<true>(amax, red[1], waves), 1e-10f);
    const float inv = 127.0f / amax;
    if (tid == 0) a.s[row] = amax / 127.0f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int p = tid + j * threads;
      if (p >= pieces) continue;
      int b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = rne_i8(v[j][i] * inv);
      *reinterpret_cast<v2i *>(a.q + base + p * 8) =
          v2i{static_cast<int>(pack4_i8(b[0], b[1], b[2], b[3])), static_cast<int>(pack4_i8(b[4], b[5], b[6], b[7]))};
    }
  }
}

template <int DT, int FORM> static void launch_norm(NormArgs a, int64_t M, hipStream_t stream) {
  const bool few = M <= kNormFew;
  // (a thread holds at most eight pieces; short rows take fewer threads)
  const int pieces = a.H / 8;
  int threads = pieces > 8 * 256 || few ? 1024 : 256;
  while (threads > 64 && threads / 2 >= pieces) threads /= 2;
  const int ch = (pieces + threads - 1) / threads;
  constexpr int64_t kRows = 1 << 21; // of one launch: a grid holds fewer than 2^32 threads
  for (; a.row0 < M; a.row0 += kRows) {
    const dim3 grid(static_cast<unsigned>(M - a.row0 < kRows ? M - a.row0 : kRows)), block(static_cast<unsigned>(threads));
    if (ch <= 1) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 1>), grid, block, 0, stream, a);
    else if (ch <= 2) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 2>), grid, block, 0, stream, a);
    else if (ch <= 4) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 4>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 8>), grid, block, 0, stream, a);
  }
}
template <int DT> static void launch_norm_form(int form, const NormArgs &a, int64_t M, hipStream_t stream) {
  if (form == LO_Q_INT8_ROWS) launch_norm<DT, LO_Q_INT8_ROWS>(a, M, stream);
  else if (form == LO_Q_INT8_GROUPS) launch_norm<DT, LO_Q_INT8_GROUPS>(a, M, stream);
  else launch_norm<DT, LO_Q_FP8_GROUPS>(a, M, stream);
}

} // namespace lo

extern "C" int lo_rms_norm_quant(const void *x, int dtype, int64_t x_stride, const void *residual, int64_t residual_stride,
                                 const void *weight, int weight_dtype, int64_t M, int64_t H, float eps, int q_form,
                                 void *residual_out, void *normed_out, void *q, float *scale, lo_stream_t stream) {
  using namespace lo;
  LO_REQUIRE(M >= 0, LO_EINVAL, "rms_norm_quant: %lld rows", (long long)M);
  LO_REQUIRE(dtype == LO_BF16 || dtype == LO_F16 || dtype == LO_F32, LO_ENOTSUP, "rms_norm_quant: rows are bf16, fp16 or fp32");
  LO_REQUIRE(weight_dtype == dtype || weight_dtype == LO_F32, LO_ENOTSUP, "rms_norm_quant: the weight has the rows' type or is fp32");
  LO_REQUIRE(q_form == LO_Q_INT8_ROWS || q_form == LO_Q_INT8_GROUPS || q_form == LO_Q_FP8_GROUPS, LO_EINVAL,
             "rms_norm_quant: unknown output form %d", q_form);
  LO_REQUIRE(H > 0 && H % (q_form == LO_Q_INT8_ROWS ? 8 : kGroup) == 0, LO_EINVAL,
             "rms_norm_quant: the hidden size (%lld) must be a multiple of %d", (long long)H, q_form == LO_Q_INT8_ROWS ? 8 : kGroup);
  LO_REQUIRE(H <= kNormMaxH, LO_ENOTSUP, "rms_norm_quant: rows of %lld values (at most %lld)", (long long)H, (long long)kNormMaxH);
  LO_REQUIRE(eps >= 0.0f, LO_EINVAL, "rms_norm_quant: eps must not be negative");
  if (M == 0) return LO_OK;
  LO_REQUIRE(x && weight && q && scale && (!residual || residual_out), LO_EINVAL, "rms_norm_quant: null pointer");
  LO_REQUIRE((x_stride >= H || M == 1) && (!residual || residual_stride >= H || M == 1), LO_EINVAL,
             "rms_norm_quant: rows overlap (stride below %lld)", (long long)H);
  const int64_t piece = dtype == LO_F32 ? 4 : 8;
  LO_REQUIRE(x_stride % piece == 0 && (!residual || residual_stride % piece == 0), LO_EINVAL,
             "rms_norm_quant: row strides must keep rows 16-byte aligned");
  const auto off = [](const void *p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; };
  LO_REQUIRE(!off(x, 16) && !off(residual, 16) && !off(weight, 16) && !off(residual_out, 16) && !off(normed_out, 16) && !off(q, 8) &&
                 !off(scale, 4),
             LO_EINVAL, "rms_norm_quant: rows and weight must be 16-byte, q 8-byte aligned");
  // the sum may take the place of a whole input, row by row; a row of it over another input row would be read too late
  const int64_t size = dtype == LO_F32 ? 4 : 2;
  const auto over = [&](const void *in, int64_t stride) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(in), z = reinterpret_cast<uintptr_t>(residual_out);
    return residual && !(p == z && (stride == H || M == 1)) && p < z + M * H * size && z < p + ((M - 1) * stride + H) * size;
  };
  LO_REQUIRE(!over(x, x_stride) && !over(residual, residual_stride), LO_EINVAL,
             "rms_norm_quant: residual_out overlaps an input without being it");
  NormArgs a{x, residual, weight, residual_out, normed_out, static_cast<int8_t *>(q), scale, x_stride, residual_stride,
             static_cast<int32_t>(H), weight_dtype == LO_F32, 0, eps};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == LO_BF16) launch_norm_form<LO_BF16>(q_form, a, M, s);
  else if (dtype == LO_F16) launch_norm_form<LO_F16>(q_form, a, M, s);
  else launch_norm_form<LO_F32>(q_form, a, M, s);
  return check_launch("rms_norm_quant");
}
