// Entry points of the dense product with an epilogue (gemm_dense.h), and which of its kernels a call takes.
#include "gemm_dense.h"

namespace lo {

static int64_t k_blocks(int dtype, int64_t K) { return (K * (dtype == LO_I8 ? 1 : 2) + kBlockK - 1) / kBlockK; }

// Which tile, and how many parts of K: the smallest estimate of the time.  A K block takes a CU t1 us with one workgroup of the tile on it and
// tn_us with as many as it holds (LDS); workgroups start and end in `start` us, those of each further round in `again`; the parts are joined by a launch
// of kJoinUs, and kPartUs for each, that moves them twice at kJoinBytes a us.  The figures are fitted to bf16 and int8 products of 968 sizes (5 to 16384
// tokens, N 20 to 160000, K 128 to 16384 bytes, plain and gated), each timed with every tile and 1 to 8 parts: the choice is 0.5 % off the fastest on average, 27 % at
// the most (52 x 2652 x 6656 bf16, gated; three sizes are over 20 %); fits without 200 of the sizes are 0.8 to 1.2 % off for these.  Sizes whose rows of C begin
// on 16 bytes and ones whose rows do not are fitted together, though a round of the two largest tiles ends faster with the former (beside its K blocks 8 to 10 us
// against 24 to 36, where K has up to 20 of them): `again` lies between.  us, by another tile / by the
// choice: 2003 x 1536 x 4096 int8, gated 37.2 (128 x 256) / 32.4 (128 x 192), 1531 x 768 x 2048 bf16, gated 23.4 (128 x 128) / 20.6 (96 x 96), 700 x 2048 x 2048 bf16 22.0
// (128 x 128) / 17.2 (64 x 128), 24 x 7168 x 2048 int8 9.8 (64 x 64) / 7.3 (32 x 32).
struct DenseTile {
  int tm, tn, held;
  float t1, tn_us, start, again;
};
constexpr DenseTile kDenseTile[kDenseTiles] = {{256, 256, 1, 1.532f, 1.532f, 3.14f, 10.00f}, {192, 256, 1, 1.254f, 1.254f, 3.69f, 7.57f}, {128, 256, 1, 1.012f, 1.012f, 2.70f, 4.97f},
                                               {128, 192, 1, 0.743f, 0.743f, 3.26f, 7.65f}, {128, 128, 1, 0.587f, 0.587f, 2.21f, 2.84f}, {96, 96, 2, 0.574f, 0.912f, 1.29f, 0.47f},
                                               {64, 128, 1, 0.540f, 0.540f, 0.83f, 0.38f}, {64, 64, 2, 0.370f, 0.648f, 0.69f, 0.12f}, {64, 32, 2, 0.277f, 0.496f, 0.01f, 0.32f},
                                               {32, 32, 2, 0.179f, 0.347f, 0.55f, 2.20f}};
constexpr float kJoinUs = 3.02f, kPartUs = 0.48f, kJoinBytes = 2.48e6f;
constexpr int kMostParts = 8, kLeastBlocks = 4; // of K, in a part
struct DensePlan {
  int tile, parts; // of K
  int few;         // gemm_dense_few_kernel: C, as a power of two, + 8 * waves + 128 * U
};
// Values of a row of the parts.
static int64_t part_pitch(int64_t N, bool gated) { return (N + 3) / 4 * 4 * (gated ? 2 : 1); }
// Whether gemm_dense_few_kernel takes a call: up to 16 tokens, where K is short enough for them.  It reads weights as they are needed and is through sooner, the tiles'
// copies run ahead of the products and stream long rows faster.  us, it / the best tile: bf16, 1 token 2048 x 7168 9.1 / 11.2, 7168 x 2048 8.6 / 9.0, but 16384 x
// 7168 45.9 / 41.7 and 65536 x 14336 358 / 307; 8 tokens 4096 x 2048 6.8 / 8.6, but x 7168 16.0 / 15.9, 7168 x 7168 28.5 / 20.1; 16 tokens 2048 x 2048 7.1 / 7.9, but
// x 7168 17.9 / 12.0; int8, 8 tokens 4096 x 7168 9.5 / 11.7, 16 11.1 / 12.0.
static bool few_tokens(int64_t M, int64_t rows, int64_t KB) {
  return M <= 16 && (rows <= 4096 ? M * KB <= (rows <= 2560 ? 600 : 900) : (M + 2) * KB <= 150);
}
static DensePlan plan_dense(int dtype, int64_t M, int64_t N, int64_t K, bool gated, bool may_split) {
  const int64_t KB = k_blocks(dtype, K);
  if (few_tokens(M, gated ? 2 * N : N, KB)) {
    // C: the fewest rounds of 256 workgroups, a larger C where that takes a twenty-fifth off (tokens are read C times), and four steps at the least.
    // Waves, and K blocks in flight of each (U): below 512 workgroups all steps at once on as many waves as that takes, from 36 steps on eight waves, one each; between,
    // as many as fit on the card at a time and share its bandwidth evenly, less than 4096 of both; beyond, all steps at once again.  More waves for the results of
    // many tokens.  U divides a wave's steps evenly.  Over 2900 sizes (1 to 16 tokens, 100 to 60000 rows, K 512 to 14336) that were timed with every C, waves and U:
    // 3.1 % over the fastest on average, tiles included; 20 sizes are over 20 %, 16 of them of over 10000 rows, 13 x 29696 x 640 bf16 the most (33 %, 14.3 us
    // against 10.7 by a tile; 1 x 38987 x 768 16.7 against 13.5 by C = 4; these were timed again, as single figures of the 2900 are up to 80 % too high).  The
    // borders are where the figures change; nothing in the mechanism says where they lie.  us, by this / one K block in flight: bf16, 1 token 256 x 7168 4.3 / 5.0, 7168 x 2048 8.6 / 9.2, gated 2048 x 7168 14.4 / 14.8.
    const int most = gated ? 3 : 4;
    const int64_t rows = gated ? 2 * N : N;
    int lg = 0, waves = 1;
    float least = 0.0f;
    for (int i = 0; i <= most && (i == 0 || (M <= 16 >> i && KB >> i >= 4)); ++i) {
      const int64_t workgroups = ((rows << i) + 15) / 16, rounds = (workgroups + 255) / 256;
      const float time = static_cast<float>(rounds) / static_cast<float>(workgroups) * (1.0f + 0.04f * static_cast<float>(i));
      if (i == 0 || time < least) lg = i, least = time;
    }
    const int64_t workgroups = ((rows << lg) + 15) / 16, steps = (KB + (1 << lg) - 1) >> lg, results = M * (16 >> lg) / (gated ? 2 : 1);
    int64_t flight = 8;
    if (workgroups < 512) {
      waves = steps < 8 ? 1 : steps < 20 ? 2 : steps < 36 ? 4 : 8;
      flight = steps < 36 ? 8 : 1;
      while (waves < 8 && results > 64 * waves && steps >= 2 * waves) waves *= 2;
    } else if (workgroups >= 2600) {
      waves = steps < 10 ? 1 : steps < 20 ? 2 : 4;
    } else if (workgroups >= 1024 || steps >= 10) {
      waves = workgroups < 1536 ? 2 : 1;
      flight = workgroups < 1024 || (workgroups >= 1536 && workgroups < 2048) ? 2 : 1;
    }
    while (waves > steps) waves /= 2;
    const int64_t each = (steps + waves - 1) / waves, passes = (each + flight - 1) / flight;
    return {kDenseFew, 1, lg + 8 * waves + 128 * static_cast<int>((each + passes - 1) / passes)};
  }
  DensePlan best{kDenseFew, 1, 0};
  float least = 0.0f;
  for (int i = M <= 16 ? kD32 : 0; i < kDenseTiles; ++i) { // (up to 16 tokens the smallest: 2.7 % over the fastest tile, 29 % at the most; by the estimate of all 2.9 and 76)
    const DenseTile &t = kDenseTile[i];
    const int64_t tiles = dense_tiles(M, N, t.tm, t.tn, gated);
    if (tiles >= kMostTiles) continue; // (never the largest tile: see check_dense_sizes)
    for (int parts = 1; parts <= (may_split && i >= kD128x256 ? kMostParts : 1); parts += parts < 4 ? 1 : 2) {
      const int64_t bytes = parts * M * part_pitch(N, gated) * 4;
      if (parts > 1 && KB / parts < kLeastBlocks) break;
      const int64_t each = (tiles * parts + 255) / 256; // workgroups of a CU
      const float blocks = static_cast<float>((KB + parts - 1) / parts);
      const int64_t rounds = each / t.held, rest = each % t.held;
      float us = static_cast<float>(rounds) * blocks * t.tn_us + t.start + t.again * static_cast<float>(rounds + (rest > 0) - 1);
      if (rest) us += blocks * (t.t1 + (t.held > 1 ? (t.tn_us - t.t1) * static_cast<float>(rest - 1) / static_cast<float>(t.held - 1) : 0.0f));
      if (parts > 1) us += kJoinUs + kPartUs * static_cast<float>(parts) + 2.0f * static_cast<float>(bytes) / kJoinBytes;
      if (best.tile < 0 || us < least) best = {i, parts, 0}, least = us;
    }
  }
  return best;
}

constexpr int64_t kMostStride = 4 << 20; // bytes: 256 rows of a tile stay within 2^30
static int check_dense_sizes(int dtype, int gated, int64_t M, int64_t N, int64_t K) {
  LO_REQUIRE(dtype == LO_BF16 || dtype == LO_F16 || dtype == LO_I8, LO_ENOTSUP, "gemm_bias_act: operands are bf16, fp16 or int8");
  LO_REQUIRE(M >= 0 && N >= 0, LO_EINVAL, "gemm_bias_act: bad sizes %lld x %lld", (long long)M, (long long)N);
  const int64_t unit = dtype == LO_I8 ? 16 : 8, most = dtype == LO_I8 ? 131056 : kMostStride / 2; // (sums of int8 products stay below 2^31)
  LO_REQUIRE(K > 0 && K % unit == 0, LO_EINVAL, "gemm_bias_act: K (%lld) must be a multiple of %lld", (long long)K, (long long)unit);
  LO_REQUIRE(K <= most, LO_ENOTSUP, "gemm_bias_act: K (%lld) is at most %lld", (long long)K, (long long)most);
  LO_REQUIRE(M <= (1 << 24) && N <= (1 << 23), LO_ENOTSUP, "gemm_bias_act: %lld x %lld outputs (at most 2^24 x 2^23)", (long long)M, (long long)N);
  LO_REQUIRE(dense_tiles(M, N, kDenseTile[kD256].tm, kDenseTile[kD256].tn, gated != 0) < kMostTiles, LO_ENOTSUP,
             "gemm_bias_act: %lld x %lld outputs (fewer than 2^22 tiles of 256 x %d)", (long long)M, (long long)N, gated ? 128 : 256);
  return LO_OK;
}

} // namespace lo

extern "C" int64_t lo_gemm_bias_act_workspace_bytes(int dtype, int gated, int64_t M, int64_t N, int64_t K) {
  using namespace lo;
  const int rc = check_dense_sizes(dtype, gated, M, N, K);
  if (rc) return rc;
  if (N == 0) return 0;
  const DensePlan p = plan_dense(dtype, M, N, K, gated != 0, true);
  return p.parts > 1 ? p.parts * M * part_pitch(N, gated != 0) * 4 : 0;
}

extern "C" int lo_gemm_bias_act_tile_query(int dtype, int gated, int64_t M, int64_t N, int64_t K, int has_workspace, int32_t *tile_m,
                                           int32_t *tile_n, int32_t *parts) {
  using namespace lo;
  const int rc = check_dense_sizes(dtype, gated, M, N, K);
  if (rc) return rc;
  LO_REQUIRE(tile_m && tile_n && parts, LO_EINVAL, "gemm_bias_act_tile_query: null pointer");
  const DensePlan p = plan_dense(dtype, M, N, K, gated != 0, has_workspace != 0);
  *tile_m = p.tile == kDenseFew ? 16 : kDenseTile[p.tile].tm;
  *tile_n = p.tile == kDenseFew ? 16 : kDenseTile[p.tile].tn;
  *parts = p.parts;
  return LO_OK;
}

extern "C" int lo_gemm_bias_act(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int dtype, const float *a_scale, const float *b_scale,
                                const void *bias, int bias_dtype, int activation, int gated, float scale, const void *residual, int64_t residual_stride,
                                void *c, int out_dtype, int64_t M, int64_t N, int64_t K, void *workspace, int64_t workspace_bytes, lo_stream_t stream) {
  using namespace lo;
  const int bad = check_dense_sizes(dtype, gated, M, N, K);
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
  const DenseArgs args{static_cast<const int8_t *>(a), static_cast<const int8_t *>(b), a_scale, b_scale, bias, residual, c, workspace, M, N,
                 M == 1 ? N : residual_stride, static_cast<int32_t>(lda), static_cast<int32_t>(ldb), static_cast<int32_t>(K * size), activation,
                 gated != 0, bias_dtype == LO_F32, out_dtype, scale, static_cast<int32_t>(k_blocks(dtype, K)), 0, 0, 1,
                 static_cast<int32_t>(part_pitch(N, gated != 0))};
  // (with less room than the parts take K stays whole: the order of the sum goes by whether there is a workspace, not by its size)
  DensePlan p = plan_dense(dtype, M, N, K, gated != 0, true);
  if (p.parts > 1 && p.parts * M * args.pitch * 4 > (workspace ? workspace_bytes : 0)) p = plan_dense(dtype, M, N, K, gated != 0, false);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int parts = p.tile == kDenseFew ? p.few : p.parts;
  const int rc = dtype == LO_BF16 ? launch_dense<LO_BF16>(args, p.tile, parts, s)
                 : dtype == LO_F16 ? launch_dense<LO_F16>(args, p.tile, parts, s)
                                   : launch_dense<LO_I8>(args, p.tile, parts, s);
  return rc ? rc : check_launch("gemm_bias_act");
}
