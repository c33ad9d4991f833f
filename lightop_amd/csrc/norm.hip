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

// Codes of a thread's eight values, of a group that it shares with the 15 lanes around it (all of them in the row or none).
template <int FORM> __device__ __forceinline__ void group_codes(const float (&v)[8], int8_t *q, float *scale) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  top = fmaxf(top, 1e-10f);
  float s;
  v2i packed;
  if constexpr (FORM == LO_Q_FP8_GROUPS) {
    const Fp8Group g = fp8_group(top, s);
    packed = v2i{fp8_pack4(&v[0], g), fp8_pack4(&v[4], g)};
  } else {
    s = top / 127.0f;
    const float y = 1.0f / s;
    packed = v2i{static_cast<int>(quant4(&v[0], s, y)), static_cast<int>(quant4(&v[4], s, y))};
  }
  *reinterpret_cast<v2i *>(q) = packed;
  if ((threadIdx.x & 15) == 0) *scale = s;
}
// Codes of a row whose largest magnitude is amax.
template <int CH> __device__ __forceinline__ void row_codes(const float (&v)[CH][8], float amax, int8_t *q, float *scale, int pieces) {
  amax = fmaxf(amax, 1e-10f);
  const float inv = 127.0f / amax;
  if (threadIdx.x == 0) *scale = amax / 127.0f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int p = threadIdx.x + j * blockDim.x;
    if (p >= pieces) continue;
    int b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = rne_i8(v[j][i] * inv);
    *reinterpret_cast<v2i *>(q + p * 8) =
        v2i{static_cast<int>(pack4_i8(b[0], b[1], b[2], b[3])), static_cast<int>(pack4_i8(b[4], b[5], b[6], b[7]))};
  }
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
      group_codes<FORM>(v[j], a.q + base + p * 8, a.s + (base >> 7) + (p >> 4));
    }
  }
  if constexpr (FORM == LO_Q_INT8_ROWS) row_codes<CH>(v, across_waves<true>(amax, red[1], waves), a.q + base, a.s + row, pieces);
}

struct NormGrid {
  static constexpr int64_t kRows = 1 << 21; // of one launch: a grid holds fewer than 2^32 threads
  int threads, ch;
  NormGrid(int H, int64_t M, int many = 256) {
    // (a thread holds at most eight pieces; short rows take fewer threads)
    const int pieces = H / 8;
    threads = pieces > 8 * 256 || M <= kNormFew ? 1024 : many;
    while (threads > 64 && threads / 2 >= pieces) threads /= 2;
    ch = (pieces + threads - 1) / threads;
  }
  dim3 rows(int64_t left) const { return dim3(static_cast<unsigned>(left < kRows ? left : kRows)); }
};
template <int DT, int FORM> static void launch_norm(NormArgs a, int64_t M, hipStream_t stream) {
  const NormGrid g(a.H, M);
  for (; a.row0 < M; a.row0 += NormGrid::kRows) {
    const dim3 grid = g.rows(M - a.row0), block(static_cast<unsigned>(g.threads));
    if (g.ch <= 1) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 1>), grid, block, 0, stream, a);
    else if (g.ch <= 2) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 2>), grid, block, 0, stream, a);
    else if (g.ch <= 4) hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 4>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((rms_norm_quant_kernel<DT, FORM, 8>), grid, block, 0, stream, a);
  }
}
template <int DT> static void launch_norm_form(int form, const NormArgs &a, int64_t M, hipStream_t stream) {
  if (form == LO_Q_INT8_ROWS) launch_norm<DT, LO_Q_INT8_ROWS>(a, M, stream);
  else if (form == LO_Q_INT8_GROUPS) launch_norm<DT, LO_Q_INT8_GROUPS>(a, M, stream);
  else launch_norm<DT, LO_Q_FP8_GROUPS>(a, M, stream);
}

// ---- the norms behind and in front of a block ---------------------------------------------------------------------------------
//   h = x * (mean(x^2) + eps)^-1/2 * post,  z = residual_scale * r + scale * act(gate) * h,  y = z * (mean(z^2) + eps)^-1/2 * w
// and y's codes; in fp32 between the inputs and the outputs, as above.  A workgroup a row, x and r read once and both asked for in front of
// the first sum, where the registers hold them (fp32 rows 205 -> 188 us).  HBM bounds it: 8192 x 7168 bf16, norms on both sides with a gate of channels, 470 MB in
// 91 to 94 us (5.0 to 5.2 TB/s, a copy's rate), without the norm behind 84.5 (5.6); a sigmoid of channels or 8-bit codes add vector work a value (int8 rows 86 us for
// 411 MB, with both 103); for one row the launch and two sums across the workgroup (2048 values 4.0 us).  Two rows a workgroup, so that the weights and the gate serve both,
// were slower (100 / 91).
constexpr int kNoCodes = -1;
struct NormBlockArgs {
  const void *x, *r, *post, *w, *gate;
  void *z, *y;
  int8_t *q;
  float *s;
  int64_t xs, rs, gs; // row strides, in values
  int64_t row0;       // of the launch's first workgroup
  uint32_t gate_rows; // rows that share a row of the gate
  int32_t H;
  int32_t post_f32, w_f32, gate_f32, gate_channels, gate_sigmoid;
  float eps, scale, residual_scale;
};

// Eight values as they lie, for a use further on.
template <int DT> struct Eight {
  v4i at[DT == LO_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *x, int64_t i) {
    const v4i *const p = reinterpret_cast<const v4i *>(static_cast<const char *>(x) + i * (DT == LO_F32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < (DT == LO_F32 ? 2 : 1); ++j) at[j] = p[j];
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (DT == LO_F32) return __builtin_bit_cast(v4f, at[i >> 2])[i & 3];
    else return to_f32<DT>(__builtin_bit_cast(v8u16, at[0])[i]);
  }
};
template <int DT> __device__ __forceinline__ void load8_as(const void *x, int f32, int64_t at, float (&v)[8]) {
  if (f32) load8<LO_F32>(x, at, v);
  else load8<DT>(x, at, v);
}

template <int DT, int FORM, int CH>
__global__ __launch_bounds__(1024) void rms_norm_block_kernel(const NormBlockArgs a) {
  __shared__ float red[3][16];
  const int tid = threadIdx.x, threads = blockDim.x, waves = threads >> 6;
  const int pieces = a.H / 8;
  const int64_t row = a.row0 + blockIdx.x, base = row * a.H;
  constexpr bool kEarly = CH <= 4; // the residual is asked for in front of the first sum, where the registers hold it
  Eight<DT> x[CH], res[kEarly ? CH : 1];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int p = tid + j * threads;
    x[j] = Eight<DT>{};
    if (p < pieces) {
      x[j].load(a.x, row * a.xs + p * 8);
      if constexpr (kEarly) res[j].load(a.r, row * a.rs + p * 8);
    }
  }
  const int64_t gate0 = a.gate ? static_cast<uint32_t>(row) / a.gate_rows * a.gs : 0;
  float token = 1.0f;
  if (a.gate && !a.gate_channels) {
    token = a.gate_f32 ? static_cast<const float *>(a.gate)[gate0]
            : DT == LO_F32 ? static_cast<const float *>(a.gate)[gate0] : to_f32<DT>(static_cast<const uint16_t *>(a.gate)[gate0]);
    if (a.gate_sigmoid) token = sigmoid_f32(token);
  }
  float rstd = 1.0f;
  if (a.post) {
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[j][i], x[j][i], ss);
    rstd = 1.0f / sqrtf(across_waves<false>(ss, red[0], waves) / static_cast<float>(a.H) + a.eps);
  }
  float v[CH][8];
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int p = tid + j * threads;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = x[j][i];
    if (p < pieces) {
      float w[8];
      Eight<DT> r;
      if constexpr (kEarly) r = res[j];
      else r.load(a.r, row * a.rs + p * 8);
      if (a.post) {
        load8_as<DT>(a.post, a.post_f32, p * 8, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rstd * w[i];
      }
      if (a.gate_channels) {
        load8_as<DT>(a.gate, a.gate_f32, gate0 + p * 8, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] *= a.gate_sigmoid ? sigmoid_f32(w[i]) : w[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] *= token;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = a.residual_scale * r[i] + a.scale * v[j][i];
      store8<DT>(a.z, base + p * 8, v[j]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[j][i], v[j][i], ss);
  }
  if (!a.w) return;
  rstd = 1.0f / sqrtf(across_waves<false>(ss, red[1], waves) / static_cast<float>(a.H) + a.eps);
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int p = tid + j * threads;
    if (p < pieces) {
      float w[8];
      load8_as<DT>(a.w, a.w_f32, p * 8, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * rstd * w[i];
      if (a.y) store8<DT>(a.y, base + p * 8, v[j]);
    }
    if constexpr (FORM == LO_Q_INT8_ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[j][i]));
    } else if constexpr (FORM != kNoCodes) {
      if (p < pieces) group_codes<FORM>(v[j], a.q + base + p * 8, a.s + (base >> 7) + (p >> 4));
    }
  }
  if constexpr (FORM == LO_Q_INT8_ROWS) row_codes<CH>(v, across_waves<true>(amax, red[2], waves), a.q + base, a.s + row, pieces);
}

template <int DT, int FORM> static void launch_norm_block(NormBlockArgs a, int64_t M, hipStream_t stream) {
  // us, 256 threads / 512, 8192 rows bf16: without codes 7168 89.8 / 87.7 (a gate of channels 93.9 / 90.3), 5120 64.6 / 65.7, 4096 45.3 / 51.7, 2560 32.6 / 41.8; with
  // e4m3 codes 7168 85.8 / 87.3, 4096 46.7 / 54.8.  128 / 256: rows of 2048 with int8 codes, 8192 26.6 / 28.8, 4096 14.9 / 17.0, 1000 7.1 / 6.9
  const NormGrid g(a.H, M, FORM == kNoCodes && a.H > 5120 ? 512 : a.H <= 2048 && M >= 2048 ? 128 : 256);
  for (; a.row0 < M; a.row0 += NormGrid::kRows) {
    const dim3 grid = g.rows(M - a.row0), block(static_cast<unsigned>(g.threads));
    if (g.ch <= 1) hipLaunchKernelGGL((rms_norm_block_kernel<DT, FORM, 1>), grid, block, 0, stream, a);
    else if (g.ch <= 2) hipLaunchKernelGGL((rms_norm_block_kernel<DT, FORM, 2>), grid, block, 0, stream, a);
    else if (g.ch <= 4) hipLaunchKernelGGL((rms_norm_block_kernel<DT, FORM, 4>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((rms_norm_block_kernel<DT, FORM, 8>), grid, block, 0, stream, a);
  }
}
template <int DT> static void launch_norm_block_form(int form, const NormBlockArgs &a, int64_t M, hipStream_t stream) {
  if (form == LO_Q_INT8_ROWS) launch_norm_block<DT, LO_Q_INT8_ROWS>(a, M, stream);
  else if (form == LO_Q_INT8_GROUPS) launch_norm_block<DT, LO_Q_INT8_GROUPS>(a, M, stream);
  else if (form == LO_Q_FP8_GROUPS) launch_norm_block<DT, LO_Q_FP8_GROUPS>(a, M, stream);
  else launch_norm_block<DT, kNoCodes>(a, M, stream);
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

extern "C" int lo_rms_norm_block(const void *x, int dtype, int64_t x_stride, const void *residual, int64_t residual_stride, const void *post_weight,
                                 int post_weight_dtype, const void *gate, int gate_dtype, int64_t gate_stride, int64_t gate_rows, int gate_channels,
                                 int gate_sigmoid, const void *weight, int weight_dtype, float scale, float residual_scale, int64_t M, int64_t H,
                                 float eps, int q_form, void *residual_out, void *normed_out, void *q, float *q_scale, lo_stream_t stream) {
  using namespace lo;
  LO_REQUIRE(M >= 0, LO_EINVAL, "rms_norm_block: %lld rows", (long long)M);
  LO_REQUIRE(M <= INT32_MAX, LO_ENOTSUP, "rms_norm_block: %lld rows (at most 2^31 - 1)", (long long)M);
  LO_REQUIRE(dtype == LO_BF16 || dtype == LO_F16 || dtype == LO_F32, LO_ENOTSUP, "rms_norm_block: rows are bf16, fp16 or fp32");
  LO_REQUIRE((!weight || weight_dtype == dtype || weight_dtype == LO_F32) && (!post_weight || post_weight_dtype == dtype || post_weight_dtype == LO_F32) &&
                 (!gate || gate_dtype == dtype || gate_dtype == LO_F32),
             LO_ENOTSUP, "rms_norm_block: weights and gate have the rows' type or are fp32");
  LO_REQUIRE(q_form == LO_Q_NONE || q_form == LO_Q_INT8_ROWS || q_form == LO_Q_INT8_GROUPS || q_form == LO_Q_FP8_GROUPS, LO_EINVAL,
             "rms_norm_block: unknown output form %d", q_form);
  const bool groups = q_form == LO_Q_INT8_GROUPS || q_form == LO_Q_FP8_GROUPS;
  LO_REQUIRE(H > 0 && H % (groups ? kGroup : 8) == 0, LO_EINVAL, "rms_norm_block: the hidden size (%lld) must be a multiple of %d", (long long)H,
             groups ? kGroup : 8);
  LO_REQUIRE(H <= kNormMaxH, LO_ENOTSUP, "rms_norm_block: rows of %lld values (at most %lld)", (long long)H, (long long)kNormMaxH);
  LO_REQUIRE(eps >= 0.0f, LO_EINVAL, "rms_norm_block: eps must not be negative");
  LO_REQUIRE(weight || (q_form == LO_Q_NONE && !normed_out), LO_EINVAL, "rms_norm_block: normed rows and codes need the weight of the norm");
  LO_REQUIRE(!gate || (gate_rows > 0 && gate_stride >= 0), LO_EINVAL, "rms_norm_block: rows of the gate: stride %lld, each for %lld rows",
             (long long)gate_stride, (long long)gate_rows);
  if (M == 0) return LO_OK;
  LO_REQUIRE(x && residual && residual_out && (q_form == LO_Q_NONE || (q && q_scale)) && (!weight || normed_out || q_form != LO_Q_NONE), LO_EINVAL,
             "rms_norm_block: null pointer");
  LO_REQUIRE(M == 1 || (x_stride >= H && residual_stride >= H), LO_EINVAL, "rms_norm_block: rows overlap (stride below %lld)", (long long)H);
  const int64_t piece = dtype == LO_F32 ? 4 : 8, size = dtype == LO_F32 ? 4 : 2, gate_size = gate_dtype == LO_F32 ? 4 : 2;
  LO_REQUIRE(x_stride % piece == 0 && residual_stride % piece == 0 && (!gate || !gate_channels || gate_stride * gate_size % 16 == 0), LO_EINVAL,
             "rms_norm_block: row strides must keep rows 16-byte aligned");
  const auto off = [](const void *p, unsigned al) { return (reinterpret_cast<uintptr_t>(p) & (al - 1)) != 0; };
  LO_REQUIRE(!off(x, 16) && !off(residual, 16) && !off(weight, 16) && !off(post_weight, 16) && !off(residual_out, 16) && !off(normed_out, 16) &&
                 !off(q, 8) && !off(q_scale, 4) && !off(gate, gate_channels ? 16 : static_cast<unsigned>(gate_size)),
             LO_EINVAL, "rms_norm_block: rows, weights and a gate of channels must be 16-byte, q 8-byte aligned");
  // the sum may take the place of a whole input, row by row; a row of it over another input row would be read too late
  const uintptr_t z = reinterpret_cast<uintptr_t>(residual_out), z_end = z + M * H * size;
  const auto meets = [&](const void *p, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return p && at < z_end && z < at + bytes;
  };
  const auto over = [&](const void *in, int64_t stride) {
    return !(reinterpret_cast<uintptr_t>(in) == z && (stride == H || M == 1)) && meets(in, ((M - 1) * stride + H) * size);
  };
  LO_REQUIRE(!over(x, x_stride) && !over(residual, residual_stride) &&
                 !meets(gate, (gate ? (M - 1) / gate_rows * gate_stride + (gate_channels ? H : 1) : 0) * gate_size) &&
                 !meets(weight, H * (weight_dtype == LO_F32 ? 4 : 2)) && !meets(post_weight, H * (post_weight_dtype == LO_F32 ? 4 : 2)),
             LO_EINVAL, "rms_norm_block: residual_out overlaps an input without being it");
  const NormBlockArgs a{x, residual, post_weight, weight, gate, residual_out, normed_out, static_cast<int8_t *>(q), q_scale, x_stride, residual_stride,
                        gate_stride, 0, gate ? static_cast<uint32_t>(gate_rows < M ? gate_rows : M) : 1u, static_cast<int32_t>(H), post_weight_dtype == LO_F32, weight_dtype == LO_F32,
                        gate_dtype == LO_F32, gate && gate_channels, gate_sigmoid != 0, eps, scale, residual_scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == LO_BF16) launch_norm_block_form<LO_BF16>(q_form, a, M, s);
  else if (dtype == LO_F16) launch_norm_block_form<LO_F16>(q_form, a, M, s);
  else launch_norm_block_form<LO_F32>(q_form, a, M, s);
  return check_launch("rms_norm_block");
}
