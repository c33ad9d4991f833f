// The experts of a few tokens with e4m3 weights (128 x 128 blocks) in two launches, or in four:
//   h = xq w1[e]^T,  v = act(h[:I]) * h[I:],  y = vq w2[e]^T,  out[t] = factor * sum_j w[t, j] * y[t, e_j] (+ shared[t]),
// xq and vq the e4m3 codes of rows in groups of 128 (fp8.h).  At these sizes the layer is a stream of the hit experts' weights:
//   up     one workgroup per (expert hit, 16 columns of I).  Its waves share the K blocks of the 16 gate and 16 up rows and quantise their part
//          of the token rows into LDS while the weights are on their way; the sums meet in LDS.  v goes to the workspace in fp32: rounded
//          on the way it would move codes of the second quantisation.
//   down   one workgroup per 16 columns of the output.  Its waves share (expert hit, part of K) and leave each slot's 16 values in LDS;
//          then every token's slots are added up in their order, by the experts' halves where two workgroups share them (few_split).  No
//          atomics on results: the order of every sum is fixed.
// Both find the experts hit from the ids by themselves.  The first product is the exact one (fp8.h): the matrix cores have time, and an error
// of 1e-5 moves codes of the second quantisation.  So is the second one in the four launches; in the two its rounding to 16 bits follows the e4m3 instruction.
//
// HBM bounds them once many experts are hit (64 tokens of a DeepSeek-V3 share of 32 experts: 1.23 GB in 245 us, 5.0 TB/s, a copy's rate; of
// Qwen3-30B-A3B 0.59 GB in 132 us), the two launches' dependent round trips with a few (one token of Qwen3-30B-A3B 18 us: ids, rows and
// weights, activations, weights).  Weights go straight to registers: every byte of them is used by one wave only, and what it would wait for
// at a barrier it has in flight instead.  16 columns a workgroup of `down`: eight gained nothing.
// Ids that no expert of this rank answers to (out of range, or -1 in the map) add nothing.  An id that a token has twice is computed once
// and counted with both weights.
#include "gemm.h"
#include "fp8.h"

namespace lo {

constexpr int kFewTokens = 64;   // of a call
constexpr int kFewSlots = 1024;
constexpr int kFewExperts = 2048;
constexpr int kFewU = 4;         // K blocks of a wave in flight
constexpr int kFewMaxWaves = 16; // (down)
constexpr int kFewGroup = 8;     // tokens of a workgroup (down), at the most
constexpr int kFewParts = 4;     // of the second product's K, at the most

// In two launches, every workgroup quantising the rows that it needs, or in four: a launch in front of either product does it once, and the
// second product goes over all tokens at a time.  Two where few experts are hit (for ids that spread evenly: slots that stay here, at the most
// every expert once), as far as a wave holds the slots in its lanes.  Two / four in us: Qwen3-30B-A3B, 16 experts hit 26 / 28, 24: 39 / 37,
// 32: 49 / 43, 64: 78 / 61; a DeepSeek-V3 share (one of 8), 64 slots of which 8 stay 76 / 80.
constexpr int kFewTwo = 24;
// Where the four launches' second product has fewer workgroups of 16 columns than there are CUs, two share a column block's experts and a fifth
// launch joins them: 64 tokens of Qwen3-30B-A3B (H 2048) 132 us, with one workgroup 159, with three 151, with four 142 (one fits a CU).
static int few_split(int64_t H) { return H / 16 < 256 ? 2 : 1; }
static bool few_in_two(int64_t slots, int64_t experts, int64_t routed) {
  const int64_t here = slots * experts / routed;
  return slots <= 64 && (here < experts ? here : experts) < kFewTwo;
}

struct Fp8ExpertsArgs {
  const void *x, *ids, *shared;
  const int8_t *w1, *w2;
  const float *w1s, *w2s, *topk_w;
  const int32_t *map;
  void *out;
  float *act;       // [slots, I]
  const int8_t *xq, *aq; // CODES: rows of x [tokens, H] and of act [slots, I], and their scales
  const float *xs, *as;
  float *part;           // [split, tokens, H]: outputs, of the experts of one of `split` workgroups each (down)
  int32_t S, H, I, E, Eg, top_k, units, parts;
  int32_t rows;     // of a wave's codes: tokens that an expert may have at a time
  int32_t group;    // tokens of a workgroup (down)
  int32_t split;    // workgroups that share the experts of 16 columns (down, with codes)
  float factor;
  bool ids64, by_slot;
};

__device__ __forceinline__ int local_expert(const Fp8ExpertsArgs &a, int s) {
  const int64_t id = a.ids64 ? static_cast<const int64_t *>(a.ids)[s] : static_cast<const int32_t *>(a.ids)[s];
  if (id < 0 || id >= a.Eg) return -1;
  const int e = a.map ? a.map[id] : static_cast<int>(id);
  return e >= 0 && e < a.E ? e : -1;
}

// ---- which experts are hit, and by which slots --------------------------------------------------------------------------------
// SMALL (up to 64 slots): a wave has a slot a lane and needs nobody.  Else the slots' experts are in LDS.
template <bool SMALL> struct Route {
  const Fp8ExpertsArgs &a;
  int16_t *keys; // LDS, [slots]: expert, -1 for none here
  int lane, S;
  int key = -1;  // SMALL: expert of slot `lane`

  // S slots from slot0 on, which begins a token
  __device__ __forceinline__ Route(const Fp8ExpertsArgs &args, int16_t *k, int ln, int slot0, int slots) : a(args), keys(k), lane(ln), S(slots) {
    if constexpr (SMALL) {
      if (lane < S) key = local_expert(a, slot0 + lane);
    } else {
      for (int s = threadIdx.x; s < S; s += blockDim.x) keys[s] = static_cast<int16_t>(local_expert(a, slot0 + s));
      __syncthreads();
    }
  }
  __device__ __forceinline__ int slot_expert(int s) const {
    return SMALL ? __builtin_amdgcn_readlane(key, s) : __builtin_amdgcn_readfirstlane(keys[s]);
  }
  // The expert's slots, one a token, into the wave's list, and how many; none if `lead` is not negative and not the first of them.
  __device__ __forceinline__ int slots(int e, int lead, int16_t *list) const {
    int count = 0;
    for (int base = 0; base < (SMALL ? 1 : S); base += 64) {
      const int s = base + lane;
      bool hit = SMALL ? key == e : s < S && keys[s] == e;
      const uint64_t all = __builtin_amdgcn_ballot_w64(hit);
      if (!all) continue;
      if (lead >= 0 && count == 0 && base + __builtin_ctzll(all) != lead) return 0;
      if constexpr (SMALL) { // (not a token's later slots with this expert)
        hit = hit && !(all & earlier_of_token());
      } else if (hit) {
        for (int j = s / a.top_k * a.top_k; j < s; ++j) hit = hit && keys[j] != e;
      }
      const uint64_t hits = __builtin_amdgcn_ballot_w64(hit);
      if (hit) list[count + __popcll(hits & ((1ull << lane) - 1))] = static_cast<int16_t>(s);
      count += __popcll(hits);
    }
    lds_order();
    return __builtin_amdgcn_readfirstlane(count);
  }
  // SMALL: lanes of the token's slots before this one
  __device__ __forceinline__ uint64_t earlier_of_token() const { return (1ull << lane) - (1ull << lane / a.top_k * a.top_k); }
};

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

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// LDS of a wave: codes of kFewU K blocks, their scales, two lists of slots
__host__ __device__ constexpr int few_wave_lds(int rows) { return kFewU * (rows * kGroup + 64) + 2 * kFewTokens * 2; }
constexpr int kFewRed = 2048; // gate and up sums of a wave (up)
constexpr int kFewSums = 2048; // slots' sums of parts of K (down, with codes)
// K blocks of a wave at a time (down; with codes, rows and weights take registers alike)
__host__ __device__ constexpr int few_down_blocks(bool codes) { return codes ? 2 : kFewU; }
// where `ends` is in LDS (down, with codes), behind everything else
__host__ __device__ constexpr int few_down_ends(int waves, int per_wave, int parts, int slots, int units, int E) {
  return (waves * per_wave + slots * (parts * 64 + 4 + 3 * 2) + (units + E) * 2 + 15) / 16 * 16;
}
// the sum of the lanes' numbers up to this one
__device__ __forceinline__ int upto_lane(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// A unit is a slot where there are fewer slots than experts (the first of its expert's; the others' workgroups end), else an expert.
template <int DT, int ACT, bool SMALL, bool CODES>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(4))) void experts_fp8_up_kernel(const Fp8ExpertsArgs a) {
  extern __shared__ __attribute__((aligned(16))) int8_t smem[]; // [wave] codes, scales, list; [wave] sums; slots' experts
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, u = blockIdx.y, H = a.H, I = a.I, KB = H / kGroup, R = a.rows, per = few_wave_lds(R);
  int8_t *const codes = smem + wave * per;
  float *const scales = reinterpret_cast<float *>(codes + kFewU * R * kGroup);
  int16_t *const list = reinterpret_cast<int16_t *>(scales + kFewU * 16);
  float *const red = reinterpret_cast<float *>(smem + waves * per); // [wave][gate, up][token][column]
  const Route<SMALL> route(a, reinterpret_cast<int16_t *>(smem + waves * (per + kFewRed)), lane, 0, a.S);
  const int e = a.by_slot ? route.slot_expert(u) : u;
  if (e < 0) return;
  const int count = route.slots(e, a.by_slot ? u : -1, list);
  if (!count) return;

  const int8_t *const w = a.w1 + static_cast<int64_t>(e) * 2 * I * H;
  const brsrc rG = make_rsrc(w + static_cast<int64_t>(n0) * H, static_cast<uint32_t>(16 * H));
  const brsrc rU = make_rsrc(w + static_cast<int64_t>(I + n0) * H, static_cast<uint32_t>(16 * H));
  const float *const sg = a.w1s + (static_cast<int64_t>(e) * (2 * I / kGroup) + n0 / kGroup) * KB;
  const float *const su = sg + static_cast<int64_t>(I / kGroup) * KB;
  for (int f = 0; f < count; f += 16) { // (more than 16 tokens of one expert read its weights again, out of L2)
    const int n = count - f < 16 ? count - f : 16;
    v4f acc[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int kb0 = wave; kb0 < KB; kb0 += waves * kFewU) {
      // the rows in front of the weights: what is asked for first comes first, and they are quantised meanwhile
      float v[8], sx[kFewU];
      v8i x[kFewU];
      const int row = r < n ? r : 0; // (columns from n on are not kept)
      auto rows_at = [&](int g) __attribute__((always_inline)) { // of group g: 16 lanes, eight values each
        const int kb = kb0 + g % kFewU * waves;
        load8<DT>(a.x, static_cast<int64_t>(list[f + g / kFewU] / a.top_k) * H + (kb < KB ? kb : kb0) * kGroup + r * 8, v);
      };
      if constexpr (CODES) {
        const int token = list[f + row] / a.top_k;
#pragma unroll
        for (int k = 0; k < kFewU; ++k) {
          const int kb = kb0 + k * waves, kc = kb < KB ? kb : kb0;
          const int8_t *const at = a.xq + static_cast<int64_t>(token) * H + kc * kGroup + q * 16;
          x[k] = join(*reinterpret_cast<const v4i *>(at), *reinterpret_cast<const v4i *>(at + 64));
          sx[k] = a.xs[token * KB + kc];
        }
      } else if (q < n * kFewU) {
        rows_at(q);
      }
      v8i wg[kFewU], wu[kFewU];
#pragma unroll
      for (int k = 0; k < kFewU; ++k) {
        const int kb = kb0 + k * waves, kc = kb < KB ? kb : kb0, at = r * H + q * 16 + kc * kGroup;
        wg[k] = join(bld16(rG, at, 0), bld16(rG, at + 64, 0));
        wu[k] = join(bld16(rU, at, 0), bld16(rU, at + 64, 0));
      }
      const int mine = kb0 + lane % kFewU * waves; // scales of the weights, a K block a lane
      const float bg = sg[mine < KB ? mine : kb0], bu = su[mine < KB ? mine : kb0];
      if constexpr (!CODES) {
        for (int g = q; g < n * kFewU; g += 4) {
          if (g >= 4) rows_at(g);
          codes_to_lds(v, r, g / kFewU, codes + g % kFewU * R * kGroup, scales + g % kFewU * 16);
        }
        lds_order();
      }
#pragma unroll
      for (int k = 0; k < kFewU; ++k) {
        if (kb0 + k * waves >= KB) break;
        if constexpr (!CODES) {
          x[k] = codes_from_lds(codes + k * R * kGroup, row, q);
          sx[k] = scales[k * 16 + row];
        }
        const float s0 = sx[k] * lane_value(bg, k), s1 = sx[k] * lane_value(bu, k);
        const v4f d0 = mfma_e4m3_exact(wg[k], x[k]), d1 = mfma_e4m3_exact(wu[k], x[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[0][i] = __builtin_fmaf(d0[i], s0, acc[0][i]);
          acc[1][i] = __builtin_fmaf(d1[i], s1, acc[1][i]);
        }
      }
      lds_order();
    }
    if (f) __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) *reinterpret_cast<v4f *>(red + wave * 512 + h * 256 + r * 16 + 4 * q) = acc[h];
    __syncthreads();
    for (int o = tid; o < n * 16; o += blockDim.x) {
      float g = 0.0f, up = 0.0f;
      for (int i = 0; i < waves; ++i) g += red[i * 512 + o], up += red[i * 512 + 256 + o];
      a.act[static_cast<int64_t>(list[f + (o >> 4)]) * I + n0 + (o & 15)] = act_mul_f32<ACT>(g, up);
    }
  }
}

// Without codes: tokens in groups of up to 64 slots, one to blockIdx.y; a wave holds the group's routing in its lanes, and an expert has
// 16 tokens at the most.  With them: all tokens (read by groups, weights that several of them hit came from HBM more than once: 64 tokens of
// a DeepSeek-V3 share 165 us), the routing in LDS.
template <int DT, bool CODES>
__global__ __launch_bounds__(1024) void experts_fp8_down_kernel(const Fp8ExpertsArgs a) {
  constexpr int U = few_down_blocks(CODES);
  // [wave] codes, scales, lists; [part][slot][column] results; [slot] weight; [slot] the token's first one with this expert, -1: none here;
  // with codes: [slot] expert; the slots by expert; the experts hit; an expert's place among them; where the slots of each end
  extern __shared__ __attribute__((aligned(16))) int8_t smem[];
  __shared__ uint32_t present[CODES ? kFewExperts / 32 : 1];
  __shared__ int number;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, I = a.I, KB = I / kGroup, R = a.rows, per = few_wave_lds(R), parts = a.parts;
  const int share = blockIdx.y, first = CODES ? 0 : blockIdx.y * a.group, M = a.S / a.top_k - first < a.group ? a.S / a.top_k - first : a.group;
  const int S = M * a.top_k, slot0 = first * a.top_k, pitch = CODES ? S : 64; // of the group
  int8_t *const codes = smem + wave * per;
  float *const scales = reinterpret_cast<float *>(codes + kFewU * R * kGroup);
  int16_t *const lists = reinterpret_cast<int16_t *>(scales + kFewU * 16);
  float *const ys = reinterpret_cast<float *>(smem + waves * per), *const weight = ys + parts * pitch * 16;
  int16_t *const from = reinterpret_cast<int16_t *>(weight + pitch), *const keys = from + pitch, *const sorted = keys + pitch;
  int16_t *const hit = sorted + pitch, *const place = hit + a.units;
  int32_t *const ends = reinterpret_cast<int32_t *>(smem + few_down_ends(waves, per, parts, pitch, a.units, a.E));
  if constexpr (CODES)
    for (int i = tid; i < kFewExperts / 32; i += blockDim.x) present[i] = 0;
  const Route<!CODES> route(a, keys, lane, slot0, S);
  // (asked for here, not behind the last product)
  for (int s = tid; s < S; s += blockDim.x) weight[s] = a.topk_w[slot0 + s];
  float shared = 0.0f;
  if (a.shared && tid < M * 16)
    shared = to_f32<DT>(static_cast<const uint16_t *>(a.shared)[static_cast<int64_t>(first + (tid >> 4)) * a.H + n0 + (tid & 15)]);
  uint64_t leaders = 0; // without codes: first slots of the experts hit
  int experts = 0;
  if constexpr (!CODES) {
    int mine = -1;
    for (uint64_t left = __builtin_amdgcn_ballot_w64(route.key >= 0); left; ++experts) { // an expert at a time
      const int s = __builtin_ctzll(left);
      const uint64_t same = __builtin_amdgcn_ballot_w64(route.key == __builtin_amdgcn_readlane(route.key, s));
      if (same >> lane & 1) {
        const uint64_t before = same & route.earlier_of_token();
        mine = before ? __builtin_ctzll(before) : lane;
      }
      left &= ~same;
      leaders |= 1ull << s;
    }
    if (wave == 0) from[lane] = static_cast<int16_t>(mine);
  } else {
    // every expert's slots, one a token, side by side (a slot a thread; their order within an expert, which the atomics leave open, says only
    // which column of a product a token takes)
    static_assert(kFewSlots <= kFewMaxWaves * 64, "a slot a thread");
    const int e = tid < S ? keys[tid] : -1;
    int j = tid / a.top_k * a.top_k;
    if (e >= 0) {
      while (keys[j] != e) ++j;
      atomicOr(&present[e >> 5], 1u << (e & 31));
    }
    if (tid < S) from[tid] = static_cast<int16_t>(e < 0 ? -1 : j);
    __syncthreads();
    if (wave == 0) {
      static_assert(kFewExperts / 32 == 64, "a word a lane");
      uint32_t left = present[lane];
      const int own = __popc(left), upto = upto_lane(own, lane);
      for (int at = upto - own; left; left &= left - 1, ++at) {
        const int x = lane * 32 + __builtin_ctz(left);
        hit[at] = static_cast<int16_t>(x);
        place[x] = static_cast<int16_t>(at);
        ends[at] = 0;
      }
      if (lane == 63) number = upto;
    }
    __syncthreads();
    experts = (number - share + a.split - 1) / a.split; // every split-th of those hit
    const bool counts = e >= 0 && j == tid;
    const int at = e >= 0 ? place[e] : 0, rank = counts ? atomicAdd(&ends[at], 1) : 0;
    if (e >= 0 && at % a.split != share) from[tid] = -1;
    __syncthreads();
    if (wave == 0)
      for (int base = 0, before = 0; base < number; base += 64) {
        const int own = base + lane < number ? ends[base + lane] : 0, upto = before + upto_lane(own, lane);
        if (base + lane < number) ends[base + lane] = upto;
        before = __builtin_amdgcn_readlane(upto, 63);
      }
    __syncthreads();
    if (counts) sorted[(at ? ends[at - 1] : 0) + rank] = static_cast<int16_t>(tid);
    __syncthreads();
  }

  // The wave's work: (expert, part of K), of every `waves`-th, 16 of the expert's tokens at a time; up to U K blocks of them at a time, the next
  // ones' weights and rows asked for before these are used.
  const int items = experts * parts;
  struct Piece {
    int it, e, part, count, f, kb, hi;
    int list; // with codes where its slots begin in `sorted`, else which of the wave's lists
  };
  auto begin = [&](int it, int list) __attribute__((always_inline)) {
    Piece p{it, 0, 0, 0, 0, 0, 1, list};
    if (it >= items) return p; // (loads of nothing, below)
    int at = it / parts;
    p.part = it - at * parts;
    if constexpr (CODES) {
      at = at * a.split + share;
      p.e = __builtin_amdgcn_readfirstlane(hit[at]);
      p.list = at ? __builtin_amdgcn_readfirstlane(ends[at - 1]) : 0;
      p.count = __builtin_amdgcn_readfirstlane(ends[at]) - p.list;
    } else {
      uint64_t left = leaders;
      for (; at > 0; --at) left &= left - 1;
      p.e = route.slot_expert(__builtin_ctzll(left));
      p.list = list;
      p.count = route.slots(p.e, -1, lists + list * kFewTokens);
    }
    p.kb = KB * p.part / parts;
    p.hi = KB * (p.part + 1) / parts;
    return p;
  };
  auto next = [&](Piece p) __attribute__((always_inline)) {
    if (p.kb + U < p.hi) {
      p.kb += U;
    } else if (CODES && p.f + 16 < p.count) {
      p.f += 16;
      p.kb = KB * p.part / parts;
    } else {
      p = begin(p.it + waves, p.list ^ 1);
    }
    return p;
  };
  v8i w[2][U];
  float b[2], v[8]; // scales of the weights, a K block a lane; activations
  v8i x[2][U];
  float sx[2][U];
  auto acts_at = [&](const Piece &p, int g) __attribute__((always_inline)) { // of group g: 16 lanes, eight values each
    const int kb = p.kb + g % U;
    load8<LO_F32>(a.act, static_cast<int64_t>(slot0 + lists[p.list * kFewTokens + g / U]) * I + (kb < p.hi ? kb : p.hi - 1) * kGroup + r * 8, v);
  };
  // With codes the same number of loads on every path, past the last piece too (there the extents are empty): a wait for what was asked for a
  // piece ago must not become one for what was asked for just now.
  auto load = [&](const Piece &p, int at) __attribute__((always_inline)) {
    if (!CODES && p.it >= items) return;
    if constexpr (CODES) {
      const int64_t slot = p.count > 0 ? sorted[p.list + (p.f + r < p.count ? p.f + r : 0)] : 0;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int kc = p.kb + k < p.hi ? p.kb + k : p.hi - 1;
        const int8_t *const row = a.aq + slot * I + kc * kGroup + q * 16;
        x[at][k] = join(*reinterpret_cast<const v4i *>(row), *reinterpret_cast<const v4i *>(row + 64));
        sx[at][k] = a.as[slot * KB + kc];
      }
    } else if (q < p.count * U) {
      acts_at(p, q);
    }
    const brsrc rW = make_rsrc(a.w2 + (static_cast<int64_t>(p.e) * a.H + n0) * I, p.it < items ? static_cast<uint32_t>(16 * I) : 0u);
    const float *const sw = a.w2s + (static_cast<int64_t>(p.e) * (a.H / kGroup) + n0 / kGroup) * KB;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int kc = p.kb + k < p.hi ? p.kb + k : p.hi - 1, off = r * I + q * 16 + kc * kGroup;
      w[at][k] = join(bld16(rW, off, 0), bld16(rW, off + 64, 0));
    }
    const int mine = p.kb + lane % U;
    b[at] = sw[mine < p.hi ? mine : p.hi - 1];
  };
  v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
  auto quantise = [&](const Piece &p) __attribute__((always_inline)) {
    if constexpr (CODES) return;
    for (int g = q; g < p.count * U; g += 4) {
      if (g >= 4) acts_at(p, g);
      codes_to_lds(v, r, g / U, codes + g % U * R * kGroup, scales + g % U * 16);
    }
    lds_order();
  };
  auto work = [&](const Piece &p, int at) __attribute__((always_inline)) {
    if (p.kb == KB * p.part / parts) acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int row = r < p.count ? r : 0; // (columns past the tokens are not kept)
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (p.kb + k >= p.hi) break;
      if constexpr (!CODES) {
        x[at][k] = codes_from_lds(codes + k * R * kGroup, row, q);
        sx[at][k] = scales[k * 16 + row];
      }
      const v4f d = mfma_e4m3_as<CODES>(w[at][k], x[at][k]);
      const float s = sx[at][k] * lane_value(b[at], k);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(d[i], s, acc[i]);
    }
    if (p.kb + U >= p.hi && p.f + r < p.count) {
      const int slot = CODES ? sorted[p.list + p.f + r] : lists[p.list * kFewTokens + r];
      *reinterpret_cast<v4f *>(ys + (p.part * pitch + slot) * 16 + 4 * q) = acc;
    }
    lds_order();
  };
  Piece p = begin(wave, 0);
  load(p, 0);
  while (p.it < items) { // two at a time, so that the buffers' names stand
    quantise(p);
    const Piece p1 = next(p);
    load(p1, 1);
    work(p, 0);
    if (p1.it >= items) break;
    quantise(p1);
    p = next(p1);
    load(p, 0);
    work(p1, 1);
  }
  __syncthreads();
  for (int o = tid; o < M * 16; o += blockDim.x) {
    const int t = o >> 4, c = o & 15, s0 = t * a.top_k;
    float sum = 0.0f;
    for (int j = 0; j < a.top_k; ++j) {
      const int s = from[s0 + j];
      if (s < 0) continue;
      float y = 0.0f;
      for (int k = 0; k < parts; ++k) y += ys[(k * pitch + s) * 16 + c];
      sum = __builtin_fmaf(weight[s0 + j], y, sum);
    }
    if (CODES && a.split > 1) {
      a.part[(static_cast<int64_t>(share) * M + t) * a.H + n0 + c] = sum;
      continue;
    }
    sum *= a.factor;
    const int64_t at = static_cast<int64_t>(first + t) * a.H + n0 + c;
    if (a.shared) sum += o == tid ? shared : to_f32<DT>(static_cast<const uint16_t *>(a.shared)[at]);
    static_cast<uint16_t *>(a.out)[at] = from_f32<DT>(sum);
  }
}

template <int DT> __global__ __launch_bounds__(256) void experts_fp8_join_kernel(const Fp8ExpertsArgs a, int64_t pieces) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= pieces) return;
  float sum[8], v[8];
  load8<LO_F32>(a.part, i * 8, sum);
  for (int k = 1; k < a.split; ++k) {
    load8<LO_F32>(a.part, (k * pieces + i) * 8, v);
#pragma unroll
    for (int n = 0; n < 8; ++n) sum[n] += v[n];
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    sum[n] *= a.factor;
    if (a.shared) sum[n] += to_f32<DT>(static_cast<const uint16_t *>(a.shared)[i * 8 + n]);
    static_cast<uint16_t *>(a.out)[i * 8 + n] = from_f32<DT>(sum[n]);
  }
}

template <int DT, int ACT, bool SMALL, bool CODES> static int launch_up(const Fp8ExpertsArgs &a, hipStream_t stream) {
  // waves that have kFewU K blocks each, in as few rounds as eight of them need
  const int KB = a.H / kGroup, rounds = (KB + 8 * kFewU - 1) / (8 * kFewU), waves = (KB + rounds * kFewU - 1) / (rounds * kFewU);
  const int lds = waves * (few_wave_lds(a.rows) + kFewRed) + (SMALL ? 0 : a.S * 2);
  const auto kernel = experts_fp8_up_kernel<DT, ACT, SMALL, CODES>;
  static unsigned long long done = 0;
  const int rc = reserve_lds_once(reinterpret_cast<const void *>(kernel), 8 * (few_wave_lds(16) + kFewRed) + kFewSlots * 2, &done);
  if (rc) return rc;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.I / 16), static_cast<unsigned>(a.units)), dim3(waves * 64), lds, stream, a);
  return check_launch("fused_experts_fp8");
}
template <int DT, bool CODES> static int launch_down(Fp8ExpertsArgs a, hipStream_t stream) {
  const int M = a.S / a.top_k, KB = a.I / kGroup;
  a.group = CODES ? M : 64 / a.top_k < kFewGroup ? 64 / a.top_k : kFewGroup;
  a.rows = CODES ? 0 : M < a.group ? M : a.group;
  // parts of K: what a wave has in flight at once, while the results fit LDS
  constexpr int U = few_down_blocks(CODES);
  a.parts = (KB + U - 1) / U < kFewParts ? (KB + U - 1) / U : kFewParts;
  while (CODES && a.parts * a.S > kFewSums) --a.parts;
  const int per = few_wave_lds(a.rows), units = a.S < a.E ? a.S : a.E; // experts hit, at the most
  a.units = units;
  const int lds = CODES ? few_down_ends(kFewMaxWaves, per, a.parts, a.S, units, a.E) + units * 4 : kFewMaxWaves * per + 64 * (a.parts * 64 + 6);
  constexpr int most = CODES ? few_down_ends(kFewMaxWaves, few_wave_lds(0), kFewSums / kFewSlots, kFewSlots, kFewSlots, kFewExperts) + kFewSlots * 4
                             : kFewMaxWaves * few_wave_lds(kFewGroup) + 64 * (kFewParts * 64 + 6);
  static_assert(most <= 160 * 1024 - 512, "LDS");
  const auto kernel = experts_fp8_down_kernel<DT, CODES>;
  static unsigned long long done = 0;
  const int rc = reserve_lds_once(reinterpret_cast<const void *>(kernel), most, &done);
  if (rc) return rc;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.H / 16), static_cast<unsigned>(CODES ? a.split : (M + a.group - 1) / a.group)),
                     dim3(kFewMaxWaves * 64), lds, stream, a);
  if (CODES && a.split > 1) {
    const int rc = check_launch("fused_experts_fp8");
    if (rc) return rc;
    const int64_t pieces = static_cast<int64_t>(M) * a.H / 8;
    hipLaunchKernelGGL(experts_fp8_join_kernel<DT>, dim3(static_cast<unsigned>((pieces + 255) / 256)), dim3(256), 0, stream, a, pieces);
  }
  return check_launch("fused_experts_fp8");
}
template <int DT> static int launch_experts_fp8(Fp8ExpertsArgs a, int activation, hipStream_t stream) {
  const int M = a.S / a.top_k;
  const bool gelu = activation == LO_ACT_GELU, small = few_in_two(a.S, a.E, a.Eg);
  // (rows that come as codes take no LDS)
  a.rows = !small ? 0 : M < 16 ? M : 16;
  int rc;
  if (small) {
    rc = gelu ? launch_up<DT, LO_ACT_GELU, true, false>(a, stream) : launch_up<DT, LO_ACT_SILU, true, false>(a, stream);
  } else {
    rc = lo_per_token_group_quant_fp8(a.x, DT, M, a.H, 1e-10f, const_cast<int8_t *>(a.xq), const_cast<float *>(a.xs), stream);
    if (rc) return rc;
    rc = gelu ? launch_up<DT, LO_ACT_GELU, false, true>(a, stream) : launch_up<DT, LO_ACT_SILU, false, true>(a, stream);
    if (rc) return rc;
    // (rows of slots without an expert here hold anything, and are not read)
    rc = lo_per_token_group_quant_fp8(a.act, LO_F32, a.S, a.I, 1e-10f, const_cast<int8_t *>(a.aq), const_cast<float *>(a.as), stream);
  }
  if (rc) return rc;
  return small ? launch_down<DT, false>(a, stream) : launch_down<DT, true>(a, stream);
}

} // namespace lo

namespace lo {
struct FewLayout { // of the workspace: activations; beyond two launches codes and scales of the rows and of the activations
  int64_t xq, xs, aq, as, part, total;
};
static FewLayout few_layout(int64_t M, int32_t top_k, int64_t H, int64_t I) {
  const int64_t S = M * top_k;
  FewLayout l{};
  l.total = S * I * 4;
  if (S < kFewTwo) return l; // (two launches, whatever the experts)
  const auto take = [&](int64_t bytes) {
    const int64_t at = l.total;
    l.total += (bytes + 15) / 16 * 16;
    return at;
  };
  l.xq = take(M * H);
  l.xs = take(M * (H / kGroup) * 4);
  l.aq = take(S * I);
  l.as = take(S * (I / kGroup) * 4);
  l.part = take(few_split(H) > 1 ? few_split(H) * M * H * 4 : 0);
  return l;
}
static int check_few_sizes(int64_t M, int32_t top_k, int64_t H, int64_t I) {
  LO_REQUIRE(M >= 0 && H >= kGroup && H % kGroup == 0 && I >= kGroup && I % kGroup == 0, LO_EINVAL,
             "fused_experts_fp8: hidden (%lld) and intermediate (%lld) sizes must be multiples of 128", (long long)H, (long long)I);
  LO_REQUIRE(H <= (1 << 20) && I <= (1 << 20), LO_ENOTSUP, "fused_experts_fp8: hidden and intermediate sizes are at most 2^20");
  LO_REQUIRE(top_k >= 1, LO_EINVAL, "fused_experts_fp8: top_k (%d) must be positive", top_k);
  LO_REQUIRE(top_k <= 64, LO_ENOTSUP, "fused_experts_fp8: top_k (%d) is at most 64", top_k);
  LO_REQUIRE(M <= kFewTokens && M * top_k <= kFewSlots, LO_ENOTSUP,
             "fused_experts_fp8: %lld tokens of %d slots (at most %d tokens and %d slots)", (long long)M, top_k, kFewTokens, kFewSlots);
  return LO_OK;
}
} // namespace lo

extern "C" int64_t lo_fused_experts_fp8_workspace_bytes(int64_t M, int32_t top_k, int64_t H, int64_t I) {
  using namespace lo;
  const int rc = check_few_sizes(M, top_k, H, I); // (what the call refuses takes no memory first)
  return rc ? rc : few_layout(M, top_k, H, I).total;
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
  LO_REQUIRE(E >= 1 && E <= kFewExperts && num_experts >= E, LO_EINVAL, "fused_experts_fp8: bad expert counts");
  LO_REQUIRE(num_experts == E || expert_map, LO_EINVAL, "fused_experts_fp8: %d experts routed over, %d here, and no expert_map", num_experts, E);
  const int bad = check_few_sizes(M, top_k, H, I);
  if (bad) return bad;
  if (M == 0) return LO_OK;
  LO_REQUIRE(x && w1 && w1s && w2 && w2s && topk_w && topk_ids && out && workspace, LO_EINVAL, "fused_experts_fp8: null pointer");
  const auto off = [](const void *p, unsigned al) { return (reinterpret_cast<uintptr_t>(p) & (al - 1)) != 0; };
  LO_REQUIRE(!off(x, 16) && !off(w1, 16) && !off(w2, 16) && !off(workspace, 16) && !off(out, 2) && !off(shared_output, 2), LO_EINVAL,
             "fused_experts_fp8: rows, weights and workspace must be 16-byte aligned");
  // (x has been read when the first output is stored; shared rows are read as they are added)
  const uintptr_t o = reinterpret_cast<uintptr_t>(out), sh = reinterpret_cast<uintptr_t>(shared_output), size = static_cast<uintptr_t>(M * H) * 2;
  LO_REQUIRE(!sh || sh == o || sh + size <= o || o + size <= sh, LO_EINVAL, "fused_experts_fp8: out overlaps shared_output without being it");
  const FewLayout layout = few_layout(M, top_k, H, I);
  const int64_t need = layout.total;
  LO_REQUIRE(workspace_bytes >= need, LO_ENOSPC, "fused_experts_fp8: workspace holds %lld bytes, needs %lld", (long long)workspace_bytes,
             (long long)need);
  Fp8ExpertsArgs a{};
  a.x = x; a.ids = topk_ids; a.shared = shared_output;
  a.w1 = static_cast<const int8_t *>(w1); a.w2 = static_cast<const int8_t *>(w2);
  a.w1s = w1s; a.w2s = w2s; a.topk_w = topk_w; a.map = expert_map; a.out = out;
  char *const ws = static_cast<char *>(workspace);
  a.act = reinterpret_cast<float *>(ws);
  a.xq = reinterpret_cast<int8_t *>(ws + layout.xq);
  a.xs = reinterpret_cast<float *>(ws + layout.xs);
  a.aq = reinterpret_cast<int8_t *>(ws + layout.aq);
  a.as = reinterpret_cast<float *>(ws + layout.as);
  a.part = reinterpret_cast<float *>(ws + layout.part);
  a.split = few_split(H);
  a.S = static_cast<int32_t>(M * top_k); a.H = static_cast<int32_t>(H); a.I = static_cast<int32_t>(I);
  a.E = E; a.Eg = num_experts; a.top_k = top_k; a.factor = routed_scaling_factor;
  a.ids64 = ids_dtype == LO_I64;
  a.by_slot = a.S < E;
  a.units = a.by_slot ? a.S : E;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == LO_F16 ? launch_experts_fp8<LO_F16>(a, activation, s) : launch_experts_fp8<LO_BF16>(a, activation, s);
}
