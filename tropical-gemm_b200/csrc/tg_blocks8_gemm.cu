// Products of matrices in 8-bit floating point with a scale for each block of 128.
#include <algorithm>
#include <cmath>
#include "tg_blocks8_umma.cuh"
#include "tg_operand8.cuh"

namespace tgi {

using tgb::ProductArgs8;

namespace {

// How a product is done, and what it is expected to take (us, on a B200).  The
// few-token kernel reads 128 rows of B per CTA and block, at the rate of one SM's
// way from L2.  The paired kernel does 256 x 256 in the time that an SM's tensor
// core needs, but its call is two launches (packing the scales and the product),
// three where a sum is split.  Measured (bf16 outputs, operands in L2, us, few /
// pairs): 333 x 1531 x 1111 5.6 / 16.3, 256 x 4096 x 4096 15.6 / 21.3,
// 1024 x 1024 x 4096 15.7 / 21.1, 512 x 4096 x 4096 30 / 20.6; the constants are fitted
// to such pairs and choose the faster of each.  Operands that come from memory have
// no term of their own.
// us per launch and per block of 16, 32 and 64 tokens
constexpr double kFewBase[] = {2.3, 2.8, 4.2}, kFewBlock[] = {0.22, 0.245, 0.34};
// us per call (two launches; kJoin is the third) and per block of the paired kernel
constexpr double kPairBase = 9.0, kPairBlock = 0.28, kPairTile = 0.5, kJoin = 2.5;
struct Plan {
  int tokens = 0;   // per tile of the few-token kernel, 0: pairs
  int split = 1;    // parts of a sum: CTAs of a cluster, or pairs
  double us = 1e30;
};

Plan pair_plan(int64_t m, int64_t n, int blocks) {
  const int half_n = n <= 128 ? 64 : 128, most = std::max(1, sm_count() / 2);
  const double tiles = double((m + 255) / 256) * double((n + 2 * half_n - 1) / (2 * half_n));
  Plan best;
  best.us = kPairBase + std::ceil(tiles / most) * (blocks * kPairBlock + kPairTile);
  // few tiles and a long sum: several pairs share a tile's sum and a second kernel joins the parts
  for (int split = 2; split * tiles <= most && blocks >= 8 * split; split++) {
    const int per = int(round_up((blocks + split - 1) / split, 4));
    if ((blocks + per - 1) / per != split) continue;
    const double us = kPairBase + kJoin + per * kPairBlock + kPairTile + 2e-6 * split * double(m) * double(n);
    if (us < best.us) { best.us = us; best.split = split; }
  }
  return best;
}

// What the few-token kernel's shapes would take, the paired one's plan given.
template <typename CLUSTERS> Plan few_plan(int64_t m, int64_t n, int blocks, Plan best, CLUSTERS&& clusters) {
  const int64_t tiles = (n + 127) / 128;
  if (tiles > 4096 || m > 16384) return best;   // far beyond what it is for
  for (int t = 0; t < 3; t++) {
    const int nt = 16 << t;
    if (t && m <= nt / 2) break;   // half of the tile would be empty
    const int64_t ctas = tiles * ((m + nt - 1) / nt), sms = sm_count();
    if (ctas > 16 * sms) continue;
    for (int split = 1; split <= 8; split *= 2) {
      if (split > 1 && blocks < 2 * split) break;
      const int steps = (blocks + split - 1) / split;
      const int64_t at_once = split == 1 ? sms : clusters(split);
      if (!at_once) break;
      const int64_t rounds = (ctas + at_once - 1) / at_once;
      // short sums leave room for two CTAs on an SM, which share the way from L2
      const bool two = split == 1 && size_t(steps) * size_t(16384 + nt * 128) < 108 * 1024;
      const double us = (two ? (rounds + 1) / 2 : rounds) * kFewBase[t] + rounds * steps * kFewBlock[t] + (split > 1 ? 0.3 : 0.0);
      if (us < best.us) { best.us = us; best.tokens = nt; best.split = split; }
    }
  }
  return best;
}

template <typename T, bool ROWS>
tg_status launch_pairs(const CUtensorMap& a, const CUtensorMap& b, ProductArgs8 p, int split, cudaStream_t st) {
  using S = tgb::PairShape;
  p.half_n = p.n <= 128 ? 64 : 128;   // narrow outputs: half the products are not wasted
  const int64_t tm = (p.m + 255) / 256, tn = (p.n + 2 * p.half_n - 1) / (2 * p.half_n);
  if (tm * tn > 0x3fffffff) return fail(TG_ERR_UNSUPPORTED, "%lld x %lld outputs", (long long)p.m, (long long)p.n);
  p.tiles_m = int(tm);
  p.tiles_n = int(tn);
  p.vec = aligned(p.c, 16) && (p.ldc * int64_t(sizeof(T))) % 16 == 0;
  p.splits = split;
  p.split_blocks = int(round_up((p.blocks + split - 1) / split, 4));
  const int pairs = split > 1 ? int(tm * tn) * split : int(std::min<int64_t>(tm * tn, std::max(1, sm_count() / 2)));
  // Blocks that the tensor core may sum (norm of the error over that of the result, sums of 65536 normal / positive
  // terms: 8 blocks 1.0e-7 / 1.9e-7, 32 2.3e-7 / 1.5e-6, 64 5.0e-7 / 3.9e-6; the plain f32 product 4.9e-7 / 4.7e-6).
  // 16-bit outputs round at 2^-11 at best.
  p.chunk = sizeof(T) == 4 ? 16 : 64;
  Scratch scratch(st);
  p.ldp = round_up(p.n, 4);
  const size_t parts = split > 1 ? size_t(split) * size_t(p.m) * size_t(p.ldp) : 0, groups = size_t(p.blocks + 3) / 4;
  p.pitch_a = tm * 256;
  p.pitch_b = tn * 2 * p.half_n;
  const size_t words_a = groups * size_t(p.pitch_a), words_b = groups * size_t(p.pitch_b);
  const cudaError_t e = scratch.reserve(Scratch::size_of<float>(parts) + Scratch::size_of<uint32_t>(words_a) + Scratch::size_of<uint32_t>(words_b) +
                                        Scratch::size_of<int>(tgb::kPackBlocks));
  if (e != cudaSuccess) return fail(TG_ERR_CUDA, "blocks8 product scratch: %s", cudaGetErrorString(e));
  p.part = scratch.take<float>(parts);
  p.words_a = scratch.take<uint32_t>(words_a);
  p.words_b = scratch.take<uint32_t>(words_b);
  p.other = scratch.take<int>(tgb::kPackBlocks);
  auto kern = tgb::blocks_pair_kernel<T, ROWS>;
  const void* entry = reinterpret_cast<const void*>(kern);
  // the epilogue's registers come from what the block was launched with
  if (kernel_regs(entry) * S::kThreads < 256 * S::kLow + (S::kThreads - 256) * S::kHigh)
    return fail(TG_ERR_UNSUPPORTED, "blocks8 product: built with too few registers");
  const tg_status s = ensure_smem(entry, S::kSmem);
  if (s != TG_OK) return s;
  launch_kernel(tgb::pack_scales_kernel, tgb::kPackBlocks, 256, 0, 0, st, p, ROWS ? 1 : 128);
  launch_kernel(kern, 2 * pairs, S::kThreads, S::kSmem, 0, st, a, b, p);
  if (split > 1)
    launch_kernel(tgb::blocks_join_kernel<T>, dim3(unsigned((p.n + 1023) / 1024), unsigned(std::min<int64_t>(p.m, 16384))), 256, 0, 0, st, p);
  return check_launch("blocks8 product");
}

template <int NT, typename T, bool ROWS>
tg_status launch_few(const CUtensorMap& tokens, const CUtensorMap& weights, ProductArgs8 p, int split, cudaStream_t st) {
  using S = tgb::FewShape<NT>;
  const int64_t tiles = (p.n + 127) / 128, tt = (p.m + NT - 1) / NT;
  auto kern = tgb::blocks_few_kernel<NT, T, ROWS>;
  const tg_status s = ensure_smem(reinterpret_cast<const void*>(kern), size_t(S::kMost) * S::kStage + S::kExchange + 1024);
  if (s != TG_OK) return s;
  p.split_blocks = (p.blocks + split - 1) / split;
  const int stages = std::min(S::kMost, p.split_blocks);
  size_t smem = size_t(stages) * S::kStage + (split > 1 ? S::kExchange : 0) + 1024;
  if (split > 1) smem = std::max<size_t>(smem, S::kAlone);
  launch_kernel(kern, dim3(unsigned(tiles * split), unsigned(tt)), S::kThreads, smem, split, st, tokens, weights, p, split, stages);
  return check_launch("blocks8 product");
}

}  // namespace
}  // namespace tgi

using namespace tgi;

extern "C" tg_status tg_blocks8_gemm(tg_dtype dtype, int64_t m, int64_t n, int64_t k, const void* a, int64_t lda,
                                     const float* a_scale, int64_t a_scale_row, int64_t a_scale_block, const void* b, int64_t ldb,
                                     int b_tall, const float* b_scale, int64_t b_scale_row, int64_t b_scale_block,
                                     const void* bias, void* c, int64_t ldc, void* stream) {
  clear_error();
  if (!elem8_size(dtype)) return fail(TG_ERR_INVALID_ARGUMENT, "8-bit blocks need f32, f16 or bf16, got dtype %d", int(dtype));
  if (m < 0 || n < 0 || k < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (m=%lld n=%lld k=%lld)", (long long)m, (long long)n, (long long)k);
  if (b_tall != 1 && b_tall != 128) return fail(TG_ERR_INVALID_ARGUMENT, "blocks are 1 or 128 rows tall, got %d", b_tall);
  if (m == 0 || n == 0) return TG_OK;
  if (m > kMostOutputs || n > kMostOutputs || k > kMostOutputs) return fail(TG_ERR_UNSUPPORTED, "m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k);
  if (!c || (k && (!a || !b || !a_scale || !b_scale))) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (lda < k) return fail(TG_ERR_DIMENSION_MISMATCH, "lda=%lld < %lld", (long long)lda, (long long)k);
  if (ldb < k) return fail(TG_ERR_DIMENSION_MISMATCH, "ldb=%lld < %lld", (long long)ldb, (long long)k);
  if (ldc < n) return fail(TG_ERR_DIMENSION_MISMATCH, "ldc=%lld < %lld", (long long)ldc, (long long)n);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProductArgs8 p{};
  p.m = m; p.n = n; p.ldc = ldc; p.c = c; p.bias = bias;
  p.a_scale = a_scale; p.a_row = a_scale_row; p.a_block = a_scale_block;
  p.b_scale = b_scale; p.b_row = b_scale_row; p.b_block = b_scale_block;
  if (k == 0)
    return with_type8(dtype, [&](auto t) {
      launch_kernel(tgb::blocks_bias_kernel<decltype(t)>, dim3(unsigned((n + 255) / 256), unsigned(std::min<int64_t>(m, 16384))), 256, 0, 0, st, p);
      return check_launch("blocks8 product");
    });
  Operand8 oa(static_cast<const int8_t*>(a), lda, m, k), ob(static_cast<const int8_t*>(b), ldb, n, k);
  Scratch scratch(st);
  if (const size_t need = oa.scratch() + ob.scratch()) {
    const cudaError_t e = scratch.reserve(need);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "blocks8 product scratch: %s", cudaGetErrorString(e));
  }
  tg8::PadArgs pads{};
  int padded = 0;
  oa.place(scratch, pads, padded);
  ob.place(scratch, pads, padded);
  pad_operands(pads, padded, st);
  p.blocks = int((k + 127) / 128);
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto rows) -> tg_status {
      constexpr bool R = decltype(rows)::value;
      // a CTA with all its stages takes an SM: the same number of clusters for every shape
      using F = tgb::FewShape<16>;
      const void* few = reinterpret_cast<const void*>(tgb::blocks_few_kernel<16, T, R>);
      const tg_status sized = ensure_smem(few, size_t(F::kMost) * F::kStage + F::kExchange + 1024);
      if (sized != TG_OK) return sized;
      auto clusters = [&](int split) { return int64_t(clusters_at_once(few, split)); };
      const Plan plan = few_plan(m, n, p.blocks, pair_plan(m, n, p.blocks), clusters);
      CUtensorMap ma, mb;
      if (!oa.map(128, plan.tokens ? plan.tokens : 128, &ma) || !ob.map(128, 128, &mb)) return fail(TG_ERR_CUDA, "blocks8 product: tensor map encoding failed");
      switch (plan.tokens) {
        case 16: return launch_few<16, T, R>(ma, mb, p, plan.split, st);
        case 32: return launch_few<32, T, R>(ma, mb, p, plan.split, st);
        case 64: return launch_few<64, T, R>(ma, mb, p, plan.split, st);
        default: return launch_pairs<T, R>(ma, mb, p, plan.split, st);
      }
    };
    return b_tall == 1 ? go(std::true_type{}) : go(std::false_type{});
  });
}
