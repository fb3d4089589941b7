// Products of matrices in 8-bit floating point with a scale for each block of 128.
#include <algorithm>
#include "tg_blocks8_umma.cuh"
#include "tg_operand8.cuh"

namespace tgi {

using tgb::ProductArgs8;

namespace {

template <typename T, bool ROWS>
tg_status launch_pairs(const CUtensorMap& a, const CUtensorMap& b, ProductArgs8 p, cudaStream_t st) {
  using S = tgb::PairShape;
  using X = tgb::ScaledShape;
  p.half_n = p.n <= 128 ? 64 : 128;   // narrow outputs: half the products are not wasted
  const int64_t tm = (p.m + 255) / 256, tn = (p.n + 2 * p.half_n - 1) / (2 * p.half_n);
  if (tm * tn > 0x3fffffff) return fail(TG_ERR_UNSUPPORTED, "%lld x %lld outputs", (long long)p.m, (long long)p.n);
  p.tiles_m = int(tm);
  p.tiles_n = int(tn);
  p.vec = aligned(p.c, 16) && (p.ldc * int64_t(sizeof(T))) % 16 == 0;
  const int most = std::max(1, sm_count() / 2);
  p.splits = 1;
  // few tiles and a long sum: several pairs share a tile's sum and a second kernel joins the parts
  if (tm * tn * 2 <= most) {
    const int split_blocks = std::max<int>(8, int((p.blocks * tm * tn + most - 1) / most + 3) / 4 * 4);
    const int splits = (p.blocks + split_blocks - 1) / split_blocks;
    const double saved = 0.35 * (p.blocks - split_blocks), cost = 5.0 + 8e-6 * splits * double(p.m) * double(p.n) / 4.0;   // us
    if (splits > 1 && saved > cost) {
      p.split_blocks = split_blocks;
      p.splits = splits;
    }
  }
  const int pairs = p.splits > 1 ? int(tm * tn) * p.splits : int(std::min<int64_t>(tm * tn, most));
  p.chunk = sizeof(T) == 4 ? 8 : 64;
  Scratch scratch(st);
  const size_t parts = p.splits > 1 ? size_t(p.splits) * size_t(p.m) * size_t(round_up(p.n, 4)) : 0;
  const size_t groups = size_t(p.blocks + 3) / 4;
  p.pitch_a = tm * 256;
  p.pitch_b = tn * 2 * p.half_n;
  const size_t words_a = groups * size_t(p.pitch_a), words_b = groups * size_t(p.pitch_b);
  const cudaError_t e = scratch.reserve(Scratch::size_of<float>(parts) + Scratch::size_of<uint32_t>(words_a) + Scratch::size_of<uint32_t>(words_b) +
                                        Scratch::size_of<int>(tgb::kPackBlocks));
  if (e != cudaSuccess) return fail(TG_ERR_CUDA, "blocks8 product scratch: %s", cudaGetErrorString(e));
  p.ldp = round_up(p.n, 4);
  p.part = scratch.take<float>(parts);
  p.words_a = scratch.take<uint32_t>(words_a);
  p.words_b = scratch.take<uint32_t>(words_b);
  p.other = scratch.take<int>(tgb::kPackBlocks);
  auto scaled = tgb::blocks_scaled_kernel<T>;
  auto any = tgb::blocks_pair_kernel<T, ROWS>;
  const void *scaled_entry = reinterpret_cast<const void*>(scaled), *any_entry = reinterpret_cast<const void*>(any);
  // the epilogue's registers come from what the block was launched with
  if (kernel_regs(any_entry) * S::kThreads < 128 * S::kLow + (S::kThreads - 128) * S::kHigh ||
      kernel_regs(scaled_entry) * X::kThreads < 256 * X::kLow + (X::kThreads - 256) * X::kHigh)
    return fail(TG_ERR_UNSUPPORTED, "blocks8 product: built with too few registers");
  tg_status s = ensure_smem(scaled_entry, X::kSmem);
  if (s == TG_OK) s = ensure_smem(any_entry, S::kSmem);
  if (s != TG_OK) return s;
  // The scales decide on the device which of the two kernels does the product; the other one returns at once.
  launch_kernel(tgb::pack_scales_kernel, tgb::kPackBlocks, 256, 0, 0, st, p, ROWS ? 1 : 128);
  launch_kernel(scaled, 2 * pairs, X::kThreads, X::kSmem, 0, st, a, b, p);
  launch_kernel(any, 2 * pairs, S::kThreads, S::kSmem, 0, st, a, b, p);
  if (p.splits > 1)
    launch_kernel(tgb::blocks_join_kernel<T>, dim3(unsigned((p.n + 1023) / 1024), unsigned(std::min<int64_t>(p.m, 16384))), 256, 0, 0, st, p);
  return check_launch("blocks8 product");
}

// Tokens per tile of the few-token kernel, or 0 for the paired one.
int few_tokens(int64_t m, int64_t n, int blocks) {
  if (m > 64) return m <= 512 && blocks >= 24 && (n + 127) / 128 * ((m + 127) / 128) * 2 <= sm_count() ? 128 : 0;
  return m <= 16 ? 16 : m <= 32 ? 32 : 64;
}

template <int NT, typename T, bool ROWS>
tg_status launch_few(const CUtensorMap& tokens, const CUtensorMap& weights, ProductArgs8 p, cudaStream_t st) {
  using S = tgb::FewShape<NT>;
  const int64_t tiles = (p.n + 127) / 128, tt = (p.m + NT - 1) / NT;
  auto kern = tgb::blocks_few_kernel<NT, T, ROWS>;
  const tg_status s = ensure_smem(reinterpret_cast<const void*>(kern), size_t(S::kMost) * S::kStage + S::kExchange + 1024);
  if (s != TG_OK) return s;
  // as many CTAs of a cluster per tile as run at once, each with at least two blocks of the sum
  int split = 1;
  while (split < 8 && tiles * tt <= clusters_at_once(reinterpret_cast<const void*>(kern), 2 * split) && p.blocks >= 4 * split) split *= 2;
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
  CUtensorMap ma, mb;
  const int nt = few_tokens(m, n, p.blocks);
  if (!oa.map(128, nt ? nt : 128, &ma) || !ob.map(128, 128, &mb)) return fail(TG_ERR_CUDA, "blocks8 product: tensor map encoding failed");
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto rows) {
      constexpr bool R = decltype(rows)::value;
      switch (nt) {
        case 16: return launch_few<16, T, R>(ma, mb, p, st);
        case 32: return launch_few<32, T, R>(ma, mb, p, st);
        case 64: return launch_few<64, T, R>(ma, mb, p, st);
        case 128: return launch_few<128, T, R>(ma, mb, p, st);
        default: return launch_pairs<T, R>(ma, mb, p, st);
      }
    };
    return b_tall == 1 ? go(std::true_type{}) : go(std::false_type{});
  });
}
