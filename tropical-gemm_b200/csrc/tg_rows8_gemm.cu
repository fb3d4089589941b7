// Products of matrices held in 8-bit rows: the forward product in 8-bit
// integers and the products of its backward.
#include <algorithm>
#include "tg_rows8.cuh"
#include "tg_operand8.cuh"
#include "tg_rows8_umma.cuh"

namespace tgi {

using tg8::ProductArgs;

dim3 row_grid(int64_t cols_per_block, int64_t cols, int64_t rows) {
  return dim3(unsigned((cols + cols_per_block - 1) / cols_per_block), unsigned(std::min<int64_t>(rows, 16384)));
}

template <int MODE, typename T>
tg_status launch_product(const CUtensorMap& a, const CUtensorMap& b, ProductArgs p, cudaStream_t st) {
  p.half_n = p.n <= 128 ? 64 : 128;   // narrow outputs: half the products and expansions are not wasted
  const int64_t tm = (p.m + tg8::kTile - 1) / tg8::kTile, tn = (p.n + 2 * p.half_n - 1) / (2 * p.half_n);
  if (tm * tn > 0x3fffffff)
    return fail(TG_ERR_UNSUPPORTED, "%lld x %lld outputs", (long long)p.m, (long long)p.n);
  p.tiles_m = int(tm);
  p.tiles_n = int(tn);
  p.vec = aligned(p.c, 16) && (p.ldc * int64_t(sizeof(T))) % 16 == 0;
  using S = tg8::ProductShape<MODE>;
  const int most = std::max(1, sm_count() / 2);
  p.splits = 1;
  // Few tiles and a long sum: several pairs share a tile's sum and a second
  // kernel joins the parts.  A stage takes about 0.35 us (backward 0.5) when few
  // pairs run; the parts cost their write and read and a launch.  Of 26 shapes
  // measured both ways this takes the slower way in two, by 9 and 15 %.
  if (tm * tn * 2 <= most) {
    const int split_blocks = std::max<int>((8 + p.planes - 1) / p.planes, int((p.blocks * tm * tn + most - 1) / most));
    const int splits = (p.blocks + split_blocks - 1) / split_blocks;
    const double saved = (S::kBack ? 0.5 : 0.35) * (p.blocks - split_blocks) * p.planes, cost = 5.0 + 8e-6 * splits * double(p.m) * double(p.n) / 4.0;
    if (splits > 1 && saved > cost) {
      p.split_blocks = split_blocks;
      p.splits = splits;
    }
  }
  // stages whose sum the tensor core may keep (see Walk); integer sums are exact
  p.chunk = p.planes == 3 ? 16 : S::kBack ? 256 / p.planes : std::max(1, p.blocks);
  const bool chunked = p.chunk < (p.splits > 1 ? p.split_blocks : p.blocks);
  const int pairs = p.splits > 1 ? int(tm * tn) * p.splits : int(std::min<int64_t>(tm * tn, most));
  const int64_t couples = (tm / 2) * tn;
  // with chunks one tile at a time: its sums are read out under the next ones
  // (8192 x 8192 x 4096 f32: 1.63 ms, two tiles at a time 1.97)
  p.doubles = S::kHalves == 2 && p.planes < 3 && p.splits == 1 ? int(couples / pairs * pairs) : 0;
  p.singles = int(tm * tn - 2 * int64_t(p.doubles));
  Scratch scratch(st);
  p.ldp = round_up(p.n, 4);
  const size_t parts = p.splits > 1 ? size_t(p.splits) * size_t(p.m) * size_t(p.ldp) : 0;
  const size_t sums = chunked ? size_t(pairs) * 4 * tg8::kEpiWarps * 1024 : 0;   // two tiles of a pair
  if (parts || sums) {
    const cudaError_t e = scratch.reserve(Scratch::size_of<uint32_t>(parts) + Scratch::size_of<float4>(sums));
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "rows8 product scratch: %s", cudaGetErrorString(e));
    p.part = scratch.take<uint32_t>(parts);
    p.work = scratch.take<float4>(sums);
  }
  auto run = [&](auto kern) {
    const tg_status s = ensure_smem(reinterpret_cast<const void*>(kern), S::kSmem);
    if (s == TG_OK) launch_kernel(kern, 2 * pairs, S::kThreads, S::kSmem, 0, st, a, b, p);
    return s;
  };
  tg_status launched;
  if constexpr (S::kBack) launched = chunked ? run(tg8::product_kernel<MODE, T, true>) : run(tg8::product_kernel<MODE, T, false>);
  else launched = run(tg8::product_kernel<MODE, T, false>);
  if (launched != TG_OK) return launched;
  if (p.splits > 1) launch_kernel(tg8::join_kernel<MODE == tg8::kForward, T>, row_grid(1024, p.n, p.m), 256, 0, 0, st, p);
  return check_launch("rows8 product");
}

// Tokens per tile of the few-token kernel, or 0 for the paired one.  Up to 64
// tokens the weights' read decides (4096 x 4096: one token 6.3 us, paired 13.0; 64
// tokens 9.0, 14.1; 8192 x 8192, 64 tokens 16.5, 28.1; 512 x 512, 64 tokens 6.5, 5.7).
// Above, what the few-token kernel has to offer is its split sum: it is taken for
// long sums of so few tiles that two CTAs or more share one.  us, few-token /
// paired, tokens x channels:
//   sums of 8192    128 x 2048 14.0 / 16.4, 128 x 4096 15.6 / 25.9, 256 x 4096 19.8 / 26.9,
//                   512 x 2048 19.0 / 26.0, 128 x 8192 22.8 / 31.0
//   of 4096         128 x 2048 10.4 / 12.4, 128 x 4096 12.1 / 14.7, 256 x 4096 15.3 / 14.8,
//                   512 x 2048 14.2 / 14.7, 128 x 8192 16.7 / 15.2
//   of 2048         128 x 2048 9.6 / 9.7, 128 x 4096 10.0 / 9.9, 256 x 4096 12.0 / 9.9
//   without a split (8192)   512 x 4096 25.8 / 24.1, 256 x 8192 28.6 / 24.4, 512 x 8192 54 / 27, 512 x 16384 125 / 51
int token_tile(int64_t m, int64_t n, int blocks) {
  if (m > 64) return m <= 512 && blocks >= 24 && (n + 127) / 128 * ((m + 127) / 128) * 2 <= sm_count() ? 128 : 0;
  return m <= 16 ? 16 : m <= 32 ? 32 : 64;
}

template <int NT, typename T>
tg_status launch_tokens(const CUtensorMap& tokens, const CUtensorMap& weights, ProductArgs p, cudaStream_t st) {
  using S = tg8::TokensShape<NT>;
  const int64_t tiles = (p.n + 127) / 128, tt = (p.m + NT - 1) / NT;
  auto kern = tg8::tokens_kernel<NT, T>;
  const tg_status s = ensure_smem(reinterpret_cast<const void*>(kern), size_t(S::kMost) * S::kStage + S::kExchange + 1024);
  if (s != TG_OK) return s;
  // as many CTAs of a cluster per tile as run at once, each with at least two
  // stages of the sum.  15 clusters of 8 and 33 of 4 do: one more is a second
  // round (us, split in 8 / 4 / 2, sums of 8192: 1 x 1920 6.2 / 6.9 / 9.0,
  // 1 x 2048 10.4 / 7.0 / 9.1, 128 x 2048 22.5 / 14.0 / 18.7; in 4 / 2: 1 x 4096
  // 9.4 / 9.8, 1 x 4352 13.9 / 9.9, 128 x 4608 28.2 / 19.9).
  int split = 1;
  while (split < 8 && tiles * tt <= clusters_at_once(reinterpret_cast<const void*>(kern), 2 * split) && p.blocks >= 4 * split) split *= 2;
  p.split_blocks = (p.blocks + split - 1) / split;
  const int stages = std::min(S::kMost, p.split_blocks);
  const size_t smem = size_t(stages) * S::kStage + (split > 1 ? S::kExchange : 0) + 1024;
  launch_kernel(kern, dim3(unsigned(tiles * split), unsigned(tt)), 128, smem, split, st, tokens, weights, p, split, stages);
  return check_launch("rows8 gemm");
}

}  // namespace tgi

using namespace tgi;

extern "C" {

tg_status tg_rows8_gemm(tg_dtype dtype, int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t lda,
                        const float* a_scale, const int8_t* b, int64_t ldb, const float* b_scale, const void* bias,
                        void* c, int64_t ldc, void* stream) {
  clear_error();
  if (!elem8_size(dtype)) return fail(TG_ERR_INVALID_ARGUMENT, "8-bit rows need f32, f16 or bf16, got dtype %d", int(dtype));
  if (m < 0 || n < 0 || k < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (m=%lld n=%lld k=%lld)", (long long)m, (long long)n, (long long)k);
  if (m == 0 || n == 0) return TG_OK;
  if (m > kMostOutputs || n > kMostOutputs) return fail(TG_ERR_UNSUPPORTED, "%lld x %lld outputs", (long long)m, (long long)n);
  if (k >= (int64_t(1) << 17)) return fail(TG_ERR_UNSUPPORTED, "k=%lld: 32-bit sums of 8-bit products are exact below 131072", (long long)k);
  if (!c || !a_scale || !b_scale || (k && (!a || !b))) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (lda < k) return fail(TG_ERR_DIMENSION_MISMATCH, "lda=%lld < %lld", (long long)lda, (long long)k);
  if (ldb < k) return fail(TG_ERR_DIMENSION_MISMATCH, "ldb=%lld < %lld", (long long)ldb, (long long)k);
  if (ldc < n) return fail(TG_ERR_DIMENSION_MISMATCH, "ldc=%lld < %lld", (long long)ldc, (long long)n);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Operand8 oa(a, lda, m, k), ob(b, ldb, n, k);
  Scratch scratch(st);
  if (const size_t need = oa.scratch() + ob.scratch()) {
    const cudaError_t e = scratch.reserve(need);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "rows8 gemm scratch: %s", cudaGetErrorString(e));
  }
  tg8::PadArgs pads{};
  int padded = 0;
  oa.place(scratch, pads, padded);
  ob.place(scratch, pads, padded);
  pad_operands(pads, padded, st);
  ProductArgs p{};
  p.m = m; p.n = n; p.ldc = ldc; p.c = c; p.row_scale = a_scale; p.col_scale = b_scale; p.bias = bias;
  p.sum = int(k);
  p.planes = 1;
  p.blocks = std::max(1, int((k + 127) / 128));
  CUtensorMap ma, mb;
  const int nt = token_tile(m, n, p.blocks);
  if (!oa.map(128, nt ? nt : 128, &ma) || !ob.map(128, 128, &mb)) return fail(TG_ERR_CUDA, "rows8 gemm: tensor map encoding failed");
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    switch (nt) {
      case 16: return launch_tokens<16, T>(ma, mb, p, st);
      case 32: return launch_tokens<32, T>(ma, mb, p, st);
      case 64: return launch_tokens<64, T>(ma, mb, p, st);
      case 128: return launch_tokens<128, T>(ma, mb, p, st);
      default: return launch_product<tg8::kForward, T>(ma, mb, p, st);
    }
  });
}

tg_status tg_rows8_gemm_backward(tg_dtype grad_dtype, tg_dtype out_dtype, int transposed, int64_t p, int64_t cols,
                                 int64_t r, const void* g, int64_t ldg, const int8_t* q, int64_t ldq,
                                 const float* scale, void* out, int64_t ldo, void* stream) {
  clear_error();
  if (!elem8_size(grad_dtype) || !elem8_size(out_dtype))
    return fail(TG_ERR_INVALID_ARGUMENT, "8-bit rows need f32, f16 or bf16, got dtypes %d and %d", int(grad_dtype), int(out_dtype));
  if (p < 0 || cols < 0 || r < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (p=%lld cols=%lld r=%lld)", (long long)p, (long long)cols, (long long)r);
  if (p == 0 || cols == 0) return TG_OK;
  if (!out || (r && (!g || !q || !scale))) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  const int64_t need = transposed ? p : r;
  if (r && ldg < need) return fail(TG_ERR_DIMENSION_MISMATCH, "ldg=%lld < %lld", (long long)ldg, (long long)need);
  if (r && ldq < cols) return fail(TG_ERR_DIMENSION_MISMATCH, "ldq=%lld < %lld", (long long)ldq, (long long)cols);
  if (ldo < cols) return fail(TG_ERR_DIMENSION_MISMATCH, "ldo=%lld < %lld", (long long)ldo, (long long)cols);
  if (p > kMostOutputs || cols > kMostOutputs || r > 0x3ffffc00)
    return fail(TG_ERR_UNSUPPORTED, "p=%lld cols=%lld r=%lld", (long long)p, (long long)cols, (long long)r);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (r == 0) {   // a sum of nothing
    const size_t e = elem8_size(out_dtype);
    const cudaError_t err = cudaMemset2DAsync(out, size_t(ldo) * e, 0, size_t(cols) * e, size_t(p), st);
    return err == cudaSuccess ? TG_OK : fail(TG_ERR_CUDA, "memset: %s", cudaGetErrorString(err));
  }
  const int64_t g_rows = transposed ? r : p, g_cols = transposed ? p : r;
  // bf16 goes to the tensor core as it is, with the scale in the 8-bit
  // operand's expansion (one rounding to bf16); f16 and f32 as the parts of
  // g * scale, with the 8-bit operand's integers exact.
  const int planes = grad_dtype == TG_BF16 ? 1 : grad_dtype == TG_F16 ? 2 : 3;
  const bool direct = grad_dtype == TG_BF16 && aligned(g, 16) && (ldg % 8 == 0 || g_rows == 1);
  const int64_t ldp = round_up(g_cols, 8);
  const size_t part_count = direct ? 0 : size_t(planes) * size_t(g_rows) * size_t(ldp);
  Operand8 oq(q, ldq, r, cols);
  Scratch scratch(st);
  if (const size_t need = oq.scratch() + Scratch::size_of<tg8::bf16>(part_count)) {
    const cudaError_t e = scratch.reserve(need);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "rows8 gemm backward scratch: %s", cudaGetErrorString(e));
  }
  tg8::PadArgs pads{};
  int padded = 0;
  oq.place(scratch, pads, padded);
  pad_operands(pads, padded, st);
  if (!direct) {
    tg8::bf16* parts = scratch.take<tg8::bf16>(part_count);
    const tg_status s = with_type8(grad_dtype, [&](auto t) {
      using T = decltype(t);
      launch_kernel(tg8::split_kernel<T>, row_grid(2048, ldp, g_rows), 256, 0, 0, st, g_rows, g_cols, static_cast<const T*>(g), ldg,
                                                                        planes > 1 ? scale : nullptr, transposed != 0, parts, ldp, planes, int(aligned(g, 16) && (ldg * int64_t(sizeof(T))) % 16 == 0));
      return check_launch("rows8 gemm backward");
    });
    if (s != TG_OK) return s;
    g = parts;
    ldg = ldp;
  } else if (g_rows == 1) {
    ldg = ldp;
  }
  ProductArgs a{};
  a.m = p; a.n = cols; a.ldc = ldo; a.c = out;
  a.sum_scale = planes == 1 ? scale : nullptr;
  a.sum = int(r);
  a.planes = planes;
  a.blocks = int((r + 63) / 64);
  CUtensorMap ma, mb;
  if (!encode_tma(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g, g_cols, g_rows, ldg, planes, g_rows * ldg, 64, transposed ? 64 : 128, &ma) ||
      !oq.map(128, 64, &mb))
    return fail(TG_ERR_CUDA, "rows8 gemm backward: tensor map encoding failed");
  return with_type8(out_dtype, [&](auto t) {
    using T = decltype(t);
    return transposed ? launch_product<tg8::kBackCols, T>(ma, mb, a, st) : launch_product<tg8::kBackRows, T>(ma, mb, a, st);
  });
}

}  // extern "C"
