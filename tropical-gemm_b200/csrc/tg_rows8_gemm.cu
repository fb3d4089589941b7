// Products of matrices held in 8-bit rows: the forward product in 8-bit
// integers and the products of its backward.
#include <algorithm>
#include "tg_rows8.cuh"

namespace tg8 {

struct GemmArgs8 {
  int64_t m, n, k;
  const int8_t *a, *b;
  const float *a_scale, *b_scale;
  const void* bias;
  void* c;
  int64_t lda, ldb, ldc;
};

constexpr int kST = 64;   // tile edge of the simple kernels
constexpr int kSK = 32;   // bytes (forward) or rows (backward) of the sum per step

// 64 x 64 tile, 256 threads, 4 x 4 outputs each, four products per dp4a; any
// alignment.
template <typename T>
__global__ void __launch_bounds__(256) gemm8_simple_kernel(GemmArgs8 p) {
  __shared__ __align__(16) int8_t as[kST][kSK + 4], bs[kST][kSK + 4];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t m0 = int64_t(blockIdx.y) * kST, n0 = int64_t(blockIdx.x) * kST;
  int acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kSK) {
    for (int i = tid; i < kST * kSK; i += 256) {
      const int r = i / kSK, c = i % kSK;
      const bool in = k0 + c < p.k;
      as[r][c] = in && m0 + r < p.m ? p.a[(m0 + r) * p.lda + k0 + c] : 0;
      bs[r][c] = in && n0 + r < p.n ? p.b[(n0 + r) * p.ldb + k0 + c] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kSK; c += 4) {
      int av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        av[i] = *reinterpret_cast<const int*>(&as[ty * 4 + i][c]);
        bv[i] = *reinterpret_cast<const int*>(&bs[tx + 16 * i][c]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t r = m0 + ty * 4 + i, c = n0 + tx + 16 * j;
      if (r < p.m && c < p.n) {
        float z = float(acc[i][j]) * p.a_scale[r] * p.b_scale[c];
        if (p.bias) z += to_f32(static_cast<const T*>(p.bias)[c]);
        static_cast<T*>(p.c)[r * p.ldc + c] = from_f32<T>(z);
      }
    }
}

struct BackGemmArgs {
  int64_t p, cols, r;
  const void* g;
  const int8_t* q;
  const float* scale;
  void* out;
  int64_t ldg, ldq, ldo;
  int transposed;
};

template <typename GT, typename T>
__global__ void __launch_bounds__(256) gemm8_backward_simple_kernel(BackGemmArgs a) {
  __shared__ float gs[kSK][kST + 1], qs[kSK][kST];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t p0 = int64_t(blockIdx.y) * kST, c0 = int64_t(blockIdx.x) * kST;
  const GT* g = static_cast<const GT*>(a.g);
  float acc[4][4] = {};
  for (int64_t r0 = 0; r0 < a.r; r0 += kSK) {
    for (int i = tid; i < kST * kSK; i += 256) {
      int rr = i / kST, pp = i % kST;
      if (!a.transposed) { rr = i % kSK; pp = i / kSK; }
      const bool in = r0 + rr < a.r && p0 + pp < a.p;
      gs[rr][pp] = in ? to_f32(a.transposed ? g[(r0 + rr) * a.ldg + p0 + pp] : g[(p0 + pp) * a.ldg + r0 + rr]) : 0.f;
      const int r = i / kST, c = i % kST;
      qs[r][c] = r0 + r < a.r && c0 + c < a.cols ? float(a.q[(r0 + r) * a.ldq + c0 + c]) * a.scale[r0 + r] : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int r = 0; r < kSK; r++) {
      float gv[4], qv[4];
#pragma unroll
      for (int i = 0; i < 4; i++) { gv[i] = gs[r][ty * 4 + i]; qv[i] = qs[r][tx + 16 * i]; }
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = fmaf(gv[i], qv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t r = p0 + ty * 4 + i, c = c0 + tx + 16 * j;
      if (r < a.p && c < a.cols) static_cast<T*>(a.out)[r * a.ldo + c] = from_f32<T>(acc[i][j]);
    }
}

}  // namespace tg8

using namespace tgi;

extern "C" {

tg_status tg_rows8_gemm(tg_dtype dtype, int64_t m, int64_t n, int64_t k, const int8_t* a, int64_t lda,
                        const float* a_scale, const int8_t* b, int64_t ldb, const float* b_scale, const void* bias,
                        void* c, int64_t ldc, void* stream) {
  clear_error();
  if (!elem8_size(dtype)) return fail(TG_ERR_INVALID_ARGUMENT, "8-bit rows need f32, f16 or bf16, got dtype %d", int(dtype));
  if (m < 0 || n < 0 || k < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (m=%lld n=%lld k=%lld)", (long long)m, (long long)n, (long long)k);
  if (m == 0 || n == 0) return TG_OK;
  if (k >= (int64_t(1) << 17)) return fail(TG_ERR_UNSUPPORTED, "k=%lld: 32-bit sums of 8-bit products are exact below 131072", (long long)k);
  if (!c || !a_scale || !b_scale || (k && (!a || !b))) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (lda < k) return fail(TG_ERR_DIMENSION_MISMATCH, "lda=%lld < %lld", (long long)lda, (long long)k);
  if (ldb < k) return fail(TG_ERR_DIMENSION_MISMATCH, "ldb=%lld < %lld", (long long)ldb, (long long)k);
  if (ldc < n) return fail(TG_ERR_DIMENSION_MISMATCH, "ldc=%lld < %lld", (long long)ldc, (long long)n);
  if (m > 65535ll * tg8::kST || n > 0x7fffffff) return fail(TG_ERR_UNSUPPORTED, "m=%lld n=%lld", (long long)m, (long long)n);
  const tg8::GemmArgs8 p{m, n, k, a, b, a_scale, b_scale, bias, c, lda, ldb, ldc};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type8(dtype, [&](auto t) {
    tg8::gemm8_simple_kernel<decltype(t)><<<dim3(unsigned((n + 63) / 64), unsigned((m + 63) / 64)), 256, 0, st>>>(p);
    return check_launch("rows8 gemm");
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
  if (p > 65535ll * tg8::kST || cols > 0x7fffffff || r > 0x7fffffff)
    return fail(TG_ERR_UNSUPPORTED, "p=%lld cols=%lld r=%lld", (long long)p, (long long)cols, (long long)r);
  const tg8::BackGemmArgs a{p, cols, r, g, q, scale, out, ldg, ldq, ldo, transposed};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type8(grad_dtype, [&](auto gt) {
    return with_type8(out_dtype, [&](auto t) {
      tg8::gemm8_backward_simple_kernel<decltype(gt), decltype(t)><<<dim3(unsigned((cols + 63) / 64), unsigned((p + 63) / 64)), 256, 0, st>>>(a);
      return check_launch("rows8 gemm backward");
    });
  });
}

}  // extern "C"
