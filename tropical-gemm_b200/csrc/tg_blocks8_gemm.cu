// Products of matrices in 8-bit floating point with a scale for each block of
// 128:
//   C[i,j] = sum_b a_scale(i,b) b_scale(j,b) sum_{k in b} A[i,k] B[j,k] + bias[j]
#include <algorithm>
#include "tg_blocks8.cuh"

namespace tgb {

struct GemmArgs {
  int64_t m, n, k, lda, ldb, ldc;
  const uint8_t *a, *b;
  const float *a_scale, *b_scale;
  int64_t a_scale_row, a_scale_block, b_scale_row, b_scale_block;
  int b_tall;
  const void* bias;
  void* c;
};

// 64 x 64 outputs per thread block, 4 x 4 per thread, codes expanded to f32 in
// shared memory 32 of the sum at a time.
template <typename T>
__global__ void __launch_bounds__(256) blocks_gemm_kernel(const GemmArgs p) {
  __shared__ float sa[32][65], sb[32][65];
  after_previous_kernel();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t n0 = int64_t(blockIdx.x) * 64, m0 = int64_t(blockIdx.y) * 64;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += 32) {
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int r = i >> 5, k = i & 31;
      const bool in = k0 + k < p.k;
      const int64_t b = (k0 + k) / kBlock, ra = m0 + r, rb = n0 + r;
      sa[k][r] = in && ra < p.m ? values2(p.a[ra * p.lda + k0 + k]).x * p.a_scale[ra * p.a_scale_row + b * p.a_scale_block] : 0.f;
      sb[k][r] = in && rb < p.n ? values2(p.b[rb * p.ldb + k0 + k]).x * p.b_scale[rb / p.b_tall * p.b_scale_row + b * p.b_scale_block] : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < 32; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t row = m0 + ty * 4 + i, col = n0 + tx * 4 + j;
      if (row >= p.m || col >= p.n) continue;
      const float z = acc[i][j] + (p.bias ? to_f32(static_cast<const T*>(p.bias)[col]) : 0.f);
      static_cast<T*>(p.c)[row * p.ldc + col] = from_f32<T>(z);
    }
}

}  // namespace tgb

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
  if (m > 0x7ffffc00 || n > 0x7ffffc00 || k > 0x7ffffc00) return fail(TG_ERR_UNSUPPORTED, "m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k);
  if (!c || (k && (!a || !b || !a_scale || !b_scale))) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (lda < k) return fail(TG_ERR_DIMENSION_MISMATCH, "lda=%lld < %lld", (long long)lda, (long long)k);
  if (ldb < k) return fail(TG_ERR_DIMENSION_MISMATCH, "ldb=%lld < %lld", (long long)ldb, (long long)k);
  if (ldc < n) return fail(TG_ERR_DIMENSION_MISMATCH, "ldc=%lld < %lld", (long long)ldc, (long long)n);
  tgb::GemmArgs p{m, n, k, lda, ldb, ldc, static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(b), a_scale, b_scale,
                  a_scale_row, a_scale_block, b_scale_row, b_scale_block, b_tall, bias, c};
  const int64_t tn = (n + 63) / 64, tm = (m + 63) / 64;
  if (tm > 65535) return fail(TG_ERR_UNSUPPORTED, "%lld rows", (long long)m);
  return with_type8(dtype, [&](auto t) {
    launch_kernel(tgb::blocks_gemm_kernel<decltype(t)>, dim3(unsigned(tn), unsigned(tm)), 256, 0, 0, static_cast<cudaStream_t>(stream), p);
    return check_launch("blocks8 gemm");
  });
}
