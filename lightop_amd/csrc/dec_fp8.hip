// The experts of a few tokens with e4m3 weights (128 x 128 blocks) in two launches:
//   h = xq w1[e]^T,  v = act(h[:I]) * h[I:],  y = vq w2[e]^T,  out[t] = factor * sum_j w[t, j] * y[t, e_j] (+ shared[t]),
// xq and vq the e4m3 codes of rows in groups of 128 (fp8.h).  At these sizes the layer is a stream of the hit experts' weights:
//   up     one workgroup per (expert hit, 16 columns of I).  It finds the slots of its expert, its waves share the K blocks of the 16 gate
//          and 16 up rows and quantise their part of the token rows into LDS while the weights are on their way, and the sums meet in
//          LDS.  v goes to the workspace in fp32: rounded on the way it would move codes of the second quantisation.
//   down   one workgroup per 16 columns of the output.  Its waves share (expert hit, part of K) and leave each slot's 16 values in LDS;
//          then every token's slots are added up in their order.  No atomics: the order of every sum is fixed.
// Both products are the exact ones (fp8.h): the matrix cores have time, and an error of 1e-5 moves codes of the second quantisation.
// Ids that no expert of this rank answers to (out of range, or -1 in the map) add nothing.  An id that a token has twice is computed once
// and counted with both weights.
#include "gemm.h"
#include "fp8.h"

namespace lo {

constexpr int kFewTokens = 64;  // one expert's list
constexpr int kFewSlots = 1024; // of a call
constexpr int kUpU = 3, kDownU = 2; // K blocks of a wave in flight
constexpr int kFewWaves = 8;

struct Fp8ExpertsArgs {
  const void *x, *ids, *shared;
  const int8_t *w1, *w2;
  const float *w1s, *w2s, *topk_w;
  const int32_t *map;
  void *out;
  float *act;       // [slots, I]
  int32_t *counts;  // [units] tokens of the unit's expert
  int32_t *lists;   // [units, kFewTokens] their slots
  int32_t S, H, I, E, Eg, top_k, units, parts;
  float factor;
  bool ids64, by_slot;
};

__device__ __forceinline__ int local_expert(const Fp8ExpertsArgs &a, int s) {
  const int64_t id = a.ids64 ? static_cast<const int64_t *>(a.ids)[s] : static_cast<const int32_t *>(a.ids)[s];
  if (id < 0 || id >= a.Eg) return -1;
  const int e = a.map ? a.map[id] : static_cast<int>(id);
  return e >= 0 && e < a.E ? e : -1;
}

// A group's codes and scale from eight values on each of 16 lanes, to a row of 128 bytes whose 16-byte pieces are swizzled by the row.
__device__ __forceinline__ void codes_to_lds(const float (&v)[8], int sub, int row, int8_t *rows, float *scales) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  float s;
  const Fp8Group g = fp8_group(fmaxf(top, 1e-10f), s);
  *reinterpret_cast<v2i *>(rows + row * kGroup + (((sub >> 1) ^ (row & 7)) * 16) + (sub & 1) * 8) = v2i{fp8_pack4(&v[0], g), fp8_pack4(&v[4], g)};
  if (sub == 0) scales[row] = s;
}
// Operand of row r from such rows.
__device__ __forceinline__ v8i codes_from_lds(const int8_t *rows, int r, int q) {
  return join(*reinterpret_cast<const v4i *>(rows + r * kGroup + ((q ^ (r & 7)) * 16)),
              *reinterpret_cast<const v4i *>(rows + r * kGroup + (((q + 4) ^ (r & 7)) * 16)));
}

template <int DT, int ACT>
__global__ __launch_bounds__(kFewWaves * 64) void experts_fp8_up_kernel(const Fp8ExpertsArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t codes[kFewWaves][kUpU][16 * kGroup];
  __shared__ float scales[kFewWaves][kUpU][16];
  __shared__ int16_t key[kFewSlots];
  __shared__ int16_t list[kFewWaves][kFewTokens];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int u = blockIdx.y, n0 = blockIdx.x * 16, H = a.H, I = a.I, KB = H / kGroup;
  for (int s = tid; s < a.S; s += kFewWaves * 64) key[s] = static_cast<int16_t>(local_expert(a, s));
  __syncthreads();
  // the expert's slots in their order, one a token; every wave has its own list
  const int e = __builtin_amdgcn_readfirstlane(a.by_slot ? key[u] : u);
  int count = 0;
  if (e >= 0)
    for (int base = 0; base < a.S; base += 64) {
      const int s = base + lane;
      bool hit = s < a.S && key[s] == e;
      if (hit)
        for (int j = s / a.top_k * a.top_k; j < s; ++j) hit = hit && key[j] != e;
      const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
      if (hit) list[wave][count + __popcll(hits & ((1ull << lane) - 1))] = static_cast<int16_t>(s);
      count += __popcll(hits);
    }
  lds_order();
  if (a.by_slot && count && list[wave][0] != u) count = 0; // an earlier slot's workgroups have this expert
  count = __builtin_amdgcn_readfirstlane(count);
  if (n0 == 0 && wave == 0) {
    if (lane == 0) a.counts[u] = count;
    if (lane < count) a.lists[u * kFewTokens + lane] = list[0][lane];
  }
  if (!count) return;

  const int8_t *const w = a.w1 + static_cast<int64_t>(e) * 2 * I * H;
  const brsrc rG = make_rsrc(w + static_cast<int64_t>(n0) * H, static_cast<uint32_t>(16 * H));
  const brsrc rU = make_rsrc(w + static_cast<int64_t>(I + n0) * H, static_cast<uint32_t>(16 * H));
  const float *const sg = a.w1s + (static_cast<int64_t>(e) * (2 * I / kGroup) + n0 / kGroup) * KB;
  const float *const su = sg + static_cast<int64_t>(I / kGroup) * KB;
  for (int f = 0; f < count; f += 16) {
    const int n = count - f < 16 ? count - f : 16;
    v4f acc[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int kb0 = wave; kb0 < KB; kb0 += kFewWaves * kUpU) {
      v8i wg[kUpU], wu[kUpU];
#pragma unroll
      for (int k = 0; k < kUpU; ++k) {
        const int kb = kb0 + k * kFewWaves, at = r * H + q * 16 + (kb < KB ? kb : kb0) * kGroup;
        wg[k] = join(bld16(rG, at, 0), bld16(rG, at + 64, 0));
        wu[k] = join(bld16(rU, at, 0), bld16(rU, at + 64, 0));
      }
      for (int g = q; g < n * kUpU; g += 4) { // 16 lanes a group
        const int row = g / kUpU, k = g % kUpU, kb = kb0 + k * kFewWaves;
        if (kb >= KB) continue;
        float v[8];
        load8<DT>(a.x, static_cast<int64_t>(list[wave][f + row] / a.top_k) * H + kb * kGroup + r * 8, v);
        codes_to_lds(v, r, row, codes[wave][k], scales[wave][k]);
      }
      lds_order();
#pragma unroll
      for (int k = 0; k < kUpU; ++k) {
        const int kb = kb0 + k * kFewWaves;
        if (kb >= KB) break;
        const v8i x = codes_from_lds(codes[wave][k], r, q); // (rows from n on hold anything: columns that are not kept)
        const float s = scales[wave][k][r], s0 = s * sg[kb], s1 = s * su[kb];
        const v4f d0 = mfma_e4m3_exact(wg[k], x), d1 = mfma_e4m3_exact(wu[k], x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[0][i] = __builtin_fmaf(d0[i], s0, acc[0][i]);
          acc[1][i] = __builtin_fmaf(d1[i], s1, acc[1][i]);
        }
      }
      lds_order();
    }
    // [gate, up][token][column] of the wave, over its codes
    const auto red = [&](int w) { return reinterpret_cast<float *>(codes[w][0]); };
    lds_order();
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<v4f *>(red(wave) + h * 256 + r * 16 + 4 * q) = acc[h];
    __syncthreads();
    if (tid < n * 16) {
      float g = 0.0f, up = 0.0f;
#pragma unroll
      for (int i = 0; i < kFewWaves; ++i) g += red(i)[tid], up += red(i)[256 + tid];
      a.act[static_cast<int64_t>(list[0][f + (tid >> 4)]) * I + n0 + (tid & 15)] = act_mul_f32<ACT>(g, up);
    }
    __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(kFewWaves * 64) void experts_fp8_down_kernel(const Fp8ExpertsArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t codes[kFewWaves][kDownU][16 * kGroup];
  __shared__ float scales[kFewWaves][kDownU][16];
  __shared__ int16_t key[kFewSlots];
  __shared__ int16_t unit[kFewSlots]; // units with tokens
  __shared__ int units;
  extern __shared__ __attribute__((aligned(16))) float ys[]; // [part][slot][column]
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, I = a.I, KB = I / kGroup;
  for (int s = tid; s < a.S; s += kFewWaves * 64) key[s] = static_cast<int16_t>(local_expert(a, s));
  if (wave == 0) {
    int found = 0;
    for (int base = 0; base < a.units; base += 64) {
      const bool hit = base + lane < a.units && a.counts[base + lane] > 0;
      const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
      if (hit) unit[found + __popcll(hits & ((1ull << lane) - 1))] = static_cast<int16_t>(base + lane);
      found += __popcll(hits);
    }
    if (lane == 0) units = found;
  }
  __syncthreads();
  const int items = units * a.parts;
  for (int it = wave; it < items; it += kFewWaves) {
    const int part = it % a.parts, u = __builtin_amdgcn_readfirstlane(unit[it / a.parts]);
    const int count = a.counts[u];
    const int32_t *const list = a.lists + u * kFewTokens;
    const int e = __builtin_amdgcn_readfirstlane(key[list[0]]);
    const int lo = KB * part / a.parts, hi = KB * (part + 1) / a.parts;
    const brsrc rW = make_rsrc(a.w2 + (static_cast<int64_t>(e) * a.H + n0) * I, static_cast<uint32_t>(16 * I));
    const float *const sw = a.w2s + (static_cast<int64_t>(e) * (a.H / kGroup) + n0 / kGroup) * KB;
    for (int f = 0; f < count; f += 16) {
      const int n = count - f < 16 ? count - f : 16;
      v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int kb0 = lo; kb0 < hi; kb0 += kDownU) {
        v8i w[kDownU];
#pragma unroll
        for (int k = 0; k < kDownU; ++k) {
          const int at = r * I + q * 16 + (kb0 + k < hi ? kb0 + k : kb0) * kGroup;
          w[k] = join(bld16(rW, at, 0), bld16(rW, at + 64, 0));
        }
        for (int g = q; g < n * kDownU; g += 4) {
          const int row = g / kDownU, k = g % kDownU, kb = kb0 + k;
          if (kb >= hi) continue;
          float v[8];
          load8<LO_F32>(a.act, static_cast<int64_t>(list[f + row]) * I + kb * kGroup + r * 8, v);
          codes_to_lds(v, r, row, codes[wave][k], scales[wave][k]);
        }
        lds_order();
#pragma unroll
        for (int k = 0; k < kDownU; ++k) {
          if (kb0 + k >= hi) break;
          const v4f d = mfma_e4m3_exact(w[k], codes_from_lds(codes[wave][k], r, q));
          const float s = scales[wave][k][r] * sw[kb0 + k];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], s, acc[i]);
        }
        lds_order();
      }
      if (r < n) *reinterpret_cast<v4f *>(ys + (part * a.S + list[f + r]) * 16 + 4 * q) = acc;
    }
  }
  __syncthreads();
  const int M = a.S / a.top_k;
  for (int o = tid; o < M * 16; o += kFewWaves * 64) {
    const int t = o >> 4, c = o & 15, s0 = t * a.top_k;
    float v = 0.0f;
    for (int j = 0; j < a.top_k; ++j) {
      const int e = key[s0 + j];
      if (e < 0) continue;
      int from = 0;
      while (key[s0 + from] != e) ++from; // the slot that holds the token's result of this expert
      float y = 0.0f;
      for (int p = 0; p < a.parts; ++p) y += ys[(p * a.S + s0 + from) * 16 + c];
      v = __builtin_fmaf(a.topk_w[s0 + j], y, v);
    }
    v *= a.factor;
    const int64_t at = static_cast<int64_t>(t) * a.H + n0 + c;
    if (a.shared) v += to_f32<DT>(static_cast<const uint16_t *>(a.shared)[at]);
    static_cast<uint16_t *>(a.out)[at] = from_f32<DT>(v);
  }
}

static int64_t few_units(int64_t S, int64_t E) { return S < E ? S : E; }

template <int DT> static int launch_experts_fp8(const Fp8ExpertsArgs &a, int activation, hipStream_t stream) {
  const dim3 up(static_cast<unsigned>(a.I / 16), static_cast<unsigned>(a.units)), down(static_cast<unsigned>(a.H / 16));
  if (activation == LO_ACT_GELU) hipLaunchKernelGGL((experts_fp8_up_kernel<DT, LO_ACT_GELU>), up, dim3(kFewWaves * 64), 0, stream, a);
  else hipLaunchKernelGGL((experts_fp8_up_kernel<DT, LO_ACT_SILU>), up, dim3(kFewWaves * 64), 0, stream, a);
  const int rc = check_launch("fused_experts_fp8");
  if (rc) return rc;
  const auto kernel = experts_fp8_down_kernel<DT>;
  static unsigned long long done = 0;
  const int rc2 = reserve_lds_once(reinterpret_cast<const void *>(kernel), kFewSlots * 64, &done);
  if (rc2) return rc2;
  hipLaunchKernelGGL(kernel, down, dim3(kFewWaves * 64), a.parts * a.S * 64, stream, a);
  return check_launch("fused_experts_fp8");
}

} // namespace lo

extern "C" int64_t lo_fused_experts_fp8_workspace_bytes(int64_t M, int32_t top_k, int64_t I, int32_t E) {
  using namespace lo;
  if (M < 0 || top_k < 1 || I < kGroup || E < 1) return LO_EINVAL;
  return M * top_k * I * 4 + few_units(M * top_k, E) * (kFewTokens + 1) * 4;
}

extern "C" int lo_fused_experts_fp8(const void *x, int dtype, int64_t M, int64_t H, int64_t I, int32_t E, int32_t num_experts,
                                    int32_t top_k, const void *w1, const float *w1s, const void *w2, const float *w2s,
                                    const float *topk_w, const void *topk_ids, int ids_dtype, const int32_t *expert_map, int activation,
                                    float routed_scaling_factor, const void *shared_output, void *out, void *workspace,
                                    int64_t workspace_bytes, lo_stream_t stream) {
  using namespace lo;
  LO_REQUIRE(dtype == LO_BF16 || dtype == LO_F16, LO_ENOTSUP, "fused_experts_fp8: activations are bf16 or fp16");
  LO_REQUIRE(ids_dtype == LO_I32 || ids_dtype == LO_I64, LO_EINVAL, "fused_experts_fp8: ids are int32 or int64");
  LO_REQUIRE(activation == LO_ACT_SILU || activation == LO_ACT_GELU, LO_EINVAL, "fused_experts_fp8: unknown activation %d", activation);
  LO_REQUIRE(M >= 0 && H >= kGroup && H % kGroup == 0 && I >= kGroup && I % kGroup == 0, LO_EINVAL,
             "fused_experts_fp8: hidden (%lld) and intermediate (%lld) sizes must be multiples of 128", (long long)H, (long long)I);
  LO_REQUIRE(H <= (1 << 20) && I <= (1 << 20), LO_ENOTSUP, "fused_experts_fp8: hidden and intermediate sizes are at most 2^20");
  LO_REQUIRE(E >= 1 && E <= 2048 && num_experts >= E && top_k >= 1, LO_EINVAL, "fused_experts_fp8: bad expert counts");
  LO_REQUIRE(num_experts == E || expert_map, LO_EINVAL, "fused_experts_fp8: %d experts routed over, %d here, and no expert_map", num_experts, E);
  LO_REQUIRE(M <= kFewTokens && M * top_k <= kFewSlots, LO_ENOTSUP,
             "fused_experts_fp8: %lld tokens of %d slots (at most %d tokens and %d slots)", (long long)M, top_k, kFewTokens, kFewSlots);
  if (M == 0) return LO_OK;
  LO_REQUIRE(x && w1 && w1s && w2 && w2s && topk_w && topk_ids && out && workspace, LO_EINVAL, "fused_experts_fp8: null pointer");
  const auto off = [](const void *p, unsigned al) { return (reinterpret_cast<uintptr_t>(p) & (al - 1)) != 0; };
  LO_REQUIRE(!off(x, 16) && !off(w1, 16) && !off(w2, 16) && !off(workspace, 16) && !off(out, 2) && !off(shared_output, 2), LO_EINVAL,
             "fused_experts_fp8: rows, weights and workspace must be 16-byte aligned");
  const int64_t need = lo_fused_experts_fp8_workspace_bytes(M, top_k, I, E);
  LO_REQUIRE(workspace_bytes >= need, LO_ENOSPC, "fused_experts_fp8: workspace holds %lld bytes, needs %lld", (long long)workspace_bytes,
             (long long)need);
  Fp8ExpertsArgs a{};
  a.x = x; a.ids = topk_ids; a.shared = shared_output;
  a.w1 = static_cast<const int8_t *>(w1); a.w2 = static_cast<const int8_t *>(w2);
  a.w1s = w1s; a.w2s = w2s; a.topk_w = topk_w; a.map = expert_map; a.out = out;
  a.S = static_cast<int32_t>(M * top_k); a.H = static_cast<int32_t>(H); a.I = static_cast<int32_t>(I);
  a.E = E; a.Eg = num_experts; a.top_k = top_k; a.factor = routed_scaling_factor;
  a.ids64 = ids_dtype == LO_I64;
  a.units = static_cast<int32_t>(few_units(a.S, E));
  a.by_slot = a.S < E;
  a.act = static_cast<float *>(workspace);
  a.counts = reinterpret_cast<int32_t *>(a.act + static_cast<int64_t>(a.S) * I);
  a.lists = a.counts + a.units;
  // parts of K: enough for every wave where few experts are hit, and their results fit LDS
  const int KB = a.I / kGroup;
  a.parts = 8;
  while (a.parts > 1 && (a.parts > KB || a.parts * a.S > kFewSlots)) a.parts /= 2;
  return dtype == LO_F16 ? launch_experts_fp8<LO_F16>(a, activation, static_cast<hipStream_t>(stream))
                         : launch_experts_fp8<LO_BF16>(a, activation, static_cast<hipStream_t>(stream));
}
