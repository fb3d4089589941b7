/*
 * tropical_gemm_b200.h -- C ABI of the B200-native tropical GEMM engine.
 *
 * C = A (x) B over a tropical semiring, optionally with the argmax index of
 * the winning k for every output, plus the argmax-scatter backward pass.
 *
 * Conventions shared by every entry point
 *   - All pointers are device pointers (cudaMalloc / torch CUDA storage),
 *     except where a comment says otherwise.  The library never allocates
 *     outputs: the caller passes C, argmax and gradient buffers.
 *   - `stream` is a cudaStream_t passed as void*; NULL means the legacy
 *     default stream.  Every call is stream-ordered and asynchronous: no
 *     host synchronisation happens inside the library.
 *   - Leading dimensions (lda/ldb/ldc) are in elements.  For TG_ROW_MAJOR
 *     A is M x K with A[i,k] at a[i*lda + k]; for TG_COL_MAJOR A[i,k] is at
 *     a[k*lda + i] (the column-major convention of the reference's Rust
 *     GPU API).  The same layout applies to B, C and argmax.
 *   - argmax is int32 with the same leading dimension as C; NULL selects
 *     the plain (value-only) GEMM.
 *   - Semantics follow the reference bit for bit: k is visited in
 *     ascending order, the accumulator starts at the semiring zero with
 *     index 0, and a product replaces it only when strictly better, so the
 *     lowest k among ties wins and outputs that nothing beats keep index 0.
 *     Integer MaxPlus/MinPlus use the sentinels -46340/+46340 (i32) and
 *     -3037000499/+3037000499 (i64) with the reference's saturating add.
 *   - Return value: TG_OK or an error code; tg_last_error() gives a
 *     human-readable message for the calling thread.
 */
#ifndef TROPICAL_GEMM_B200_H
#define TROPICAL_GEMM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { TG_MAXPLUS = 0, TG_MINPLUS = 1, TG_MAXMUL = 2 } tg_semiring;
/* TG_BF16 and TG_F16 are element types of the tg_rows8_* calls only. */
typedef enum { TG_F32 = 0, TG_F64 = 1, TG_I32 = 2, TG_I64 = 3, TG_BF16 = 4, TG_F16 = 5 } tg_dtype;
typedef enum { TG_ROW_MAJOR = 0, TG_COL_MAJOR = 1 } tg_layout;

typedef enum {
  TG_OK = 0,
  TG_ERR_INVALID_ARGUMENT = 1,  /* null pointer, negative size, bad enum   */
  TG_ERR_DIMENSION_MISMATCH = 2,/* leading dimension too small, etc.       */
  TG_ERR_UNSUPPORTED = 3,       /* combination not provided (e.g. int grad) */
  TG_ERR_CUDA = 4,              /* a CUDA runtime call failed              */
  TG_ERR_NO_DEVICE = 5          /* no CUDA device visible                  */
} tg_status;

/* Library version string, e.g. "0.2.0-b200". */
const char* tg_version(void);

/* Message describing the last failing call on this thread ("" if none). */
const char* tg_last_error(void);

/* Number of visible CUDA devices (0 when none); never fails.
 * Replaces cuda_device_count (crates/tropical-gemm-cuda/src/lib.rs:63). */
int tg_device_count(void);

/* C = A (x) B, optionally with argmax.
 * Replaces CudaKernel::launch_gemm and CudaKernelWithArgmax::launch_gemm_with_argmax
 * (crates/tropical-gemm-cuda/src/kernels.rs:22-27, :202-207), the free functions
 * tropical_matmul_gpu[_with_argmax] / tropical_gemm_gpu[_with_argmax]
 * (crates/tropical-gemm-cuda/src/lib.rs:221, :256, :354, :392), and the DLPack
 * launchers launch_gemm_external[_with_argmax]_f32 (kernels.rs:388-473).
 * M, N or K equal to 0 is accepted: with K == 0 every output is the semiring
 * zero with index 0; with M or N == 0 nothing is written. */
tg_status tg_gemm(tg_semiring semiring, tg_dtype dtype, tg_layout layout,
                  int64_t m, int64_t n, int64_t k,
                  const void* a, int64_t lda,
                  const void* b, int64_t ldb,
                  void* c, int64_t ldc,
                  int32_t* argmax,
                  void* stream);

/* Strided batched GEMM: for p in [0, batch) computes
 * C[p] = A[p] (x) B[p] with A[p] = a + p*stride_a (elements), etc.;
 * argmax uses stride_c.  One launch for the whole batch.
 * Replaces launch_gemm_external_batched_with_argmax_f32 (kernels.rs:498-550)
 * and tropical_matmul_gpu_strided_batched[_with_argmax]
 * (crates/tropical-gemm-cuda/src/lib.rs:486, :563, :1007). */
tg_status tg_gemm_strided_batched(tg_semiring semiring, tg_dtype dtype, tg_layout layout,
                                  int64_t batch, int64_t m, int64_t n, int64_t k,
                                  const void* a, int64_t lda, int64_t stride_a,
                                  const void* b, int64_t ldb, int64_t stride_b,
                                  void* c, int64_t ldc, int64_t stride_c,
                                  int32_t* argmax,
                                  void* stream);

/* Accumulating f32 GEMM over one K slice: every output starts from its
 * current value in C (and keeps its argmax) unless a product of this slice
 * strictly beats it; a winning k is written as k_offset + k.  Computing
 * K = [0, k1) with tg_gemm and then [k1, k2), ... with this call (A's and
 * B's slices, k_offset = slice start) gives results identical to one
 * tg_gemm over the whole K, so a caller can overlap the transfer of B's next
 * K slice with the arithmetic of the current one.  f32 only (others:
 * TG_ERR_UNSUPPORTED); argmax may be null (values only).  No reference
 * counterpart: the reference computes whole products in one launch
 * (kernels.rs:388-434); this is the building block of the pipelined sharded
 * GEMM. */
tg_status tg_gemm_accumulate(tg_semiring semiring, tg_layout layout,
                             int64_t m, int64_t n, int64_t k,
                             const float* a, int64_t lda,
                             const float* b, int64_t ldb,
                             float* c, int64_t ldc,
                             int32_t* argmax, int32_t k_offset,
                             void* stream);

/* Broadcast callback for tg_sharded_gemm: make the `bytes` bytes of device
 * memory at `buf` equal to rank `root`'s copy, enqueued on `stream` (for
 * example ncclBroadcast on the caller's communicator, so the library links no
 * collective library of its own).  Returns 0 on success. */
typedef int (*tg_broadcast_fn)(void* buf, size_t bytes, int root, void* stream, void* ctx);

/* One rank's part of a row-sharded GEMM across GPUs: B (k x n, row-major,
 * leading dimension ldb, one buffer per rank on its device) is made whole by
 * bcast(b, ..., root, stream, bcast_ctx), then this rank computes its own
 * m_local rows C_local = A_local (x) B (row-major, like tg_gemm with
 * TG_ROW_MAJOR).  C and argmax stay sharded: no reduction.  Every rank must
 * call it (m_local may be 0: the rank still takes part in the broadcast).
 * Column-major callers shard columns instead: pass the transposed problem
 * (B^T rows, A^T broadcast).  No reference counterpart: the reference has no
 * multi-GPU path; this is the sharded entry its CUDA crate would bind for one
 * process per GPU. */
tg_status tg_sharded_gemm(tg_semiring semiring, tg_dtype dtype,
                          int64_t m_local, int64_t n, int64_t k,
                          const void* a_local, int64_t lda,
                          void* b, int64_t ldb,
                          void* c_local, int64_t ldc,
                          int32_t* argmax_local,
                          int root, tg_broadcast_fn bcast, void* bcast_ctx,
                          void* stream);

/* Backward pass w.r.t. A:
 *   grad_a[i, argmax[i,j]] += grad_c[i,j] * w[i,j]
 * where w = 1 for MaxPlus/MinPlus and w = B[argmax[i,j], j] for MaxMul
 * (the multiplicative rule of pytorch.py:521-548; pass b for MaxMul, NULL
 * otherwise).  Indices outside [0, K) are skipped, as in the reference kernel.
 * accumulate == 0 overwrites grad_a (no pre-zeroing needed); != 0 adds into it.
 * Float types only.  Replaces tropical_backward_a_gpu_kernel
 * (crates/tropical-gemm-cuda/src/lib.rs:841-882) and the torch scatter_add_
 * backward (crates/tropical-gemm-python/python/tropical_gemm/pytorch.py:386-403). */
tg_status tg_backward_a(tg_semiring semiring, tg_dtype dtype, tg_layout layout,
                        int64_t batch, int64_t m, int64_t n, int64_t k,
                        const void* grad_c, int64_t ldc, int64_t stride_c,
                        const int32_t* argmax,
                        const void* b, int64_t ldb, int64_t stride_b,
                        void* grad_a, int64_t lda, int64_t stride_a,
                        int accumulate, void* stream);

/* Backward pass w.r.t. B:
 *   grad_b[argmax[i,j], j] += grad_c[i,j] * w[i,j]
 * with w = 1, or A[i, argmax[i,j]] for MaxMul (pass a).  Same conventions
 * as tg_backward_a.  Replaces tropical_backward_b_gpu_kernel
 * (crates/tropical-gemm-cuda/src/lib.rs:901-942). */
tg_status tg_backward_b(tg_semiring semiring, tg_dtype dtype, tg_layout layout,
                        int64_t batch, int64_t m, int64_t n, int64_t k,
                        const void* grad_c, int64_t ldc, int64_t stride_c,
                        const int32_t* argmax,
                        const void* a, int64_t lda, int64_t stride_a,
                        void* grad_b, int64_t ldb, int64_t stride_b,
                        int accumulate, void* stream);

/* Integer (i32) C = A (x) B, optionally with argmax, that allocates nothing.
 * No counterpart in the reference: it is an addition of this library.
 * For callers that cannot allocate device memory at call time -- e.g. a host
 * framework that has reserved the GPU's memory for its own pool, or a
 * serving / real-time loop that forbids cudaMalloc after start-up because an
 * allocation can block, fail or synchronise.  Same arguments and results as
 * tg_gemm with dtype TG_I32 (one matrix, no batch).  Its scratch (A and B as
 * f32, rows padded to 4 elements, plus a 256-byte header) lives in a fixed
 * 64 MiB device array that every GPU loading this library keeps until the
 * process exits; larger problems are rejected with TG_ERR_UNSUPPORTED and a
 * message (use tg_gemm for them).  The first call on a device looks up the
 * array's device address (cudaGetSymbolAddress); make that first call before
 * any stream capture.  All calls share the one array and it keeps the last
 * call's contents: calls that overlap on the GPU (different streams, or
 * different host threads on the same device) race and must be serialised by
 * the caller. */
tg_status tg_gemm_i32_noalloc(tg_semiring semiring, tg_layout layout,
                              int64_t m, int64_t n, int64_t k,
                              const void* a, int64_t lda,
                              const void* b, int64_t ldb,
                              void* c, int64_t ldc,
                              int32_t* argmax,
                              void* stream);

/* ------------------------------------------------------------------------
 * Rows held in 8 bits.
 *
 * A (rows x cols) matrix in 8-bit rows is q (int8, row-major, leading
 * dimension in elements) and scale (f32, one per row): element (r, c) stands
 * for q[r*ldq + c] * scale[r].  Every call below is row-major; dtype is
 * TG_F32, TG_F16 or TG_BF16; sizes of 0 are accepted.  Same conventions as
 * above otherwise (device pointers, stream order, status codes).  Some calls
 * take stream-ordered scratch from the library's own pool.
 * No reference counterpart: these are the ordinary (+, x) layers that stand
 * beside a tropical layer in a model.
 * ------------------------------------------------------------------------ */

/* q, scale = x in 8-bit rows: scale = max|x[r,:]| / 127, q = x / scale
 * rounded to nearest even, in [-127, 127] (ties of x * 127 / max exactly; a
 * quotient within 2^-15 of a tie that is none may take either neighbour, the
 * division being f32).  A row whose largest magnitude is
 * below 2^-120 becomes zeros with scale 0; a row that holds a NaN or an
 * infinity gets scale NaN, so that everything made of it is NaN. */
tg_status tg_rows8_quantize(tg_dtype dtype, int64_t rows, int64_t cols,
                            const void* x, int64_t ldx,
                            int8_t* q, int64_t ldq, float* scale, void* stream);

/* y = q * scale, the f32 product rounded to dtype. */
tg_status tg_rows8_dequantize(tg_dtype dtype, int64_t rows, int64_t cols,
                              const int8_t* q, int64_t ldq, const float* scale,
                              void* y, int64_t ldy, void* stream);

/* Root-mean-square norm with the residual's addition, out in 8-bit rows:
 *   h = x + residual;  u[r] = 1 / sqrt(mean(h[r,:]^2) + eps);  y = h * u * weight
 * q, scale = y in 8-bit rows (as tg_rows8_quantize).  All arithmetic and
 * the statistics are f32 on the unrounded sum; x, residual, weight and h are
 * of type dtype.  residual and h may be null (no addition; h not written).
 * Finite rows whose sum of squares passes f32's range (|h| from about 1e19 on)
 * have u = 0 and read as zeros.
 * For training, ckpt (ldk) and ckpt_scale receive h in 8-bit rows and rstd
 * receives u: what tg_rows8_rmsnorm_backward reads.  The three may be null. */
tg_status tg_rows8_rmsnorm(tg_dtype dtype, int64_t rows, int64_t cols,
                           const void* x, int64_t ldx, const void* residual, int64_t ldr,
                           const void* weight, float eps,
                           void* h, int64_t ldh,
                           int8_t* q, int64_t ldq, float* scale,
                           int8_t* ckpt, int64_t ldk, float* ckpt_scale, float* rstd,
                           void* stream);

/* Backward of the norm from its 8-bit checkpoint.  With v = ckpt * ckpt_scale
 * * rstd (the normalised row) and g = grad:
 *   grad_x = rstd * (g * weight - v * mean(g * weight * v)) + grad_h
 *   grad_weight = sum over rows of g * v
 * grad is of type grad_dtype (dtype, or TG_F32); grad_h (null for none),
 * weight, grad_x and grad_weight are of type dtype.  grad_x is the gradient
 * of x and of residual alike.  The rounding to 8 bits is passed straight
 * through.  The sum over rows has a fixed order: equal inputs give equal
 * bits.  grad_x or grad_weight may be null. */
tg_status tg_rows8_rmsnorm_backward(tg_dtype dtype, tg_dtype grad_dtype, int64_t rows, int64_t cols,
                                    const void* grad, int64_t ldg, const void* grad_h, int64_t ldgh,
                                    const void* weight, const int8_t* ckpt, int64_t ldk,
                                    const float* ckpt_scale, const float* rstd,
                                    void* grad_x, int64_t ldx, void* grad_weight, void* stream);

/* C[i,j] = a_scale[i] * b_scale[j] * sum_k A[i,k] * B[j,k] + bias[j]
 * A (m x k) and B (n x k) in 8-bit rows, C (m x n) of type dtype, bias (n) of
 * type dtype or null.  The integer sums are exact: k < 131072, beyond it
 * TG_ERR_UNSUPPORTED. */
tg_status tg_rows8_gemm(tg_dtype dtype, int64_t m, int64_t n, int64_t k,
                        const int8_t* a, int64_t lda, const float* a_scale,
                        const int8_t* b, int64_t ldb, const float* b_scale,
                        const void* bias, void* c, int64_t ldc, void* stream);

/* Gradient of tg_rows8_gemm with respect to one operand, from the other in
 * 8-bit rows (r x cols: the weights, or the activations' checkpoint):
 *   out[p, c] = sum_i g(p, i) * scale[i] * q[i, c]
 * transposed == 0: g is (p x r), g(p, i) = g[p*ldg + i]  (grad_A = grad B)
 * transposed != 0: g is (r x p), g(p, i) = g[i*ldg + p]  (grad_B = grad^T A)
 * g is of type grad_dtype, out (p x cols) of type out_dtype.  Sums are f32, the
 * tensor core's for some thousand terms and then added up, so that their error
 * does not grow with r.
 * Rounding of the factors: a TG_BF16 gradient meets the 8-bit operand's
 * values rounded once to bf16; TG_F16 and TG_F32 gradients are carried with
 * 16 and 24 significant bits. */
tg_status tg_rows8_gemm_backward(tg_dtype grad_dtype, tg_dtype out_dtype, int transposed,
                                 int64_t p, int64_t cols, int64_t r,
                                 const void* g, int64_t ldg,
                                 const int8_t* q, int64_t ldq, const float* scale,
                                 void* out, int64_t ldo, void* stream);

/* out[c] = sum over rows of x[r, c] (f32 sums, fixed order): the gradient of
 * tg_rows8_gemm's bias.  out is of type out_dtype. */
tg_status tg_rows8_column_sum(tg_dtype dtype, tg_dtype out_dtype, int64_t rows, int64_t cols,
                              const void* x, int64_t ldx, void* out, void* stream);

/* --------------------------------------------------------------------------
 * Layer norm.  Row-major; dtype is TG_F32, TG_F16 or TG_BF16; conventions as
 * for the 8-bit rows above (device pointers, stream order, status codes, sizes
 * of 0 rows accepted, scratch from the library's own pool).  No reference
 * counterpart.
 * ------------------------------------------------------------------------ */

/* h = x + residual;  u = (h - mean) * rstd;  y = u * weight + bias
 * with a row's mean and rstd = 1 / sqrt(variance + eps), the variance being the
 * mean square of h - mean.  All arithmetic is f32 on the unrounded sum; x,
 * residual, weight, bias, h and y are of type dtype.  residual, weight (ones),
 * bias (zeros), h, mean and rstd may be null, mean and rstd together.  Rows of
 * magnitudes up to 2^126 have finite statistics: where the squares of h - mean
 * add up to more than f32 holds (distances from about 1e19 / sqrt(cols) on),
 * rstd is 0, y is the bias, and grad_x is grad_h. */
tg_status tg_layernorm(tg_dtype dtype, int64_t rows, int64_t cols,
                       const void* x, int64_t ldx, const void* residual, int64_t ldr,
                       const void* weight, const void* bias, float eps,
                       void* h, int64_t ldh, void* y, int64_t ldy,
                       float* mean, float* rstd, void* stream);

/* Backward of the norm.  With u = (h - mean) * rstd and a = grad * weight:
 *   grad_x = rstd * (a - mean(a) - u * mean(a * u)) + grad_h
 *   grad_weight = sum over rows of grad * u;  grad_bias = sum over rows of grad
 * All of type dtype except mean and rstd (f32).  grad_h and weight may be
 * null, and each of the three results.  The sums over rows have a fixed order:
 * equal inputs give equal bits.
 * A 16-bit h that is the sum x + residual is that sum rounded: u is then off by
 * half a step of h times rstd, which a row far from zero shows in full.  The
 * call below takes the sum's parts. */
tg_status tg_layernorm_backward(tg_dtype dtype, int64_t rows, int64_t cols,
                                const void* grad, int64_t ldg, const void* grad_h, int64_t ldgh,
                                const void* weight, const void* h, int64_t ldh,
                                const float* mean, const float* rstd,
                                void* grad_x, int64_t ldx, void* grad_weight, void* grad_bias, void* stream);

/* The same with h = x + residual formed in f32 as tg_layernorm formed it, so
 * that u is that of y; residual may be null (h is x).  grad_x is the gradient
 * of x and of residual; its leading dimension is ldgx. */
tg_status tg_layernorm_residual_backward(tg_dtype dtype, int64_t rows, int64_t cols,
                                         const void* grad, int64_t ldg, const void* grad_h, int64_t ldgh,
                                         const void* weight, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                         const float* mean, const float* rstd,
                                         void* grad_x, int64_t ldgx, void* grad_weight, void* grad_bias, void* stream);

/* --------------------------------------------------------------------------
 * Matrices held in 8-bit floating point (e4m3, as bytes) with a scale for each
 * block of 128: element (r, c) stands for q[r*ldq + c] times the scale of
 *   its row's block of 128 columns   (tall == 1)
 *   its tile of 128 rows x columns   (tall == 128)
 * which is scale[(r / tall) * scale_row + (c / 128) * scale_block], f32.
 * A block at the matrix's edge is shorter.  Conventions as above; dtype is
 * TG_F32, TG_F16 or TG_BF16.
 *
 * The quantising calls take the least power of two, from 2^-126 on, that
 * brings a block's largest magnitude to 448 (the largest e4m3 value) or below,
 * and round to nearest even: a float code's precision does not depend on its
 * scale's mantissa, and with a power of two the rounding to 8 bits is the only
 * one.  A block that holds a NaN or an infinity gets scale NaN, so that
 * everything made of it is NaN.  The products take any f32 scales; two scales
 * that meet are multiplied first, so their product lies within f32's range.
 * Where all scales of a product are powers of two (or NaN) the tensor core
 * applies them itself; which way is taken is decided on the device.
 * ------------------------------------------------------------------------ */

/* q, scale = x with a scale per row and block of 128 columns.  qt (cols x
 * rows, or null): x transposed, with blocks of 128 along ITS rows; its element
 * (c, r) has the scale scale_t[c * scale_t_row + (r / 128) * scale_t_block].
 * column_sum (cols, or null): the sums of x's columns, f32 sums in a fixed
 * order, of type dtype.  One of q, qt and column_sum is there, all from one read. */
tg_status tg_blocks8_quantize(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                              void* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_block,
                              void* qt, int64_t ldqt, float* scale_t, int64_t scale_t_row, int64_t scale_t_block,
                              void* column_sum, void* stream);

/* q, scale = x with a scale per tile of 128 x 128.  qt (cols x rows, or null)
 * gets the same codes transposed, whose scales are scale transposed. */
tg_status tg_blocks8_quantize_tiles(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                                    void* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_block,
                                    void* qt, int64_t ldqt, void* stream);

/* Codes transposed: qt (cols x rows) = q (rows x cols).  A matrix in tiles of
 * 128 x 128 transposed has its scales transposed too. */
tg_status tg_blocks8_transpose(int64_t rows, int64_t cols, const void* q, int64_t ldq, void* qt, int64_t ldqt, void* stream);

/* y = q * scale, the f32 product rounded to dtype; tall is 1 or 128. */
tg_status tg_blocks8_dequantize(tg_dtype dtype, int64_t rows, int64_t cols, int tall,
                                const void* q, int64_t ldq, const float* scale, int64_t scale_row, int64_t scale_block,
                                void* y, int64_t ldy, void* stream);

/* tg_layernorm with its output in 8-bit blocks (tall == 1), quantised from the
 * unrounded f32 values. */
tg_status tg_blocks8_layernorm(tg_dtype dtype, int64_t rows, int64_t cols,
                               const void* x, int64_t ldx, const void* residual, int64_t ldr,
                               const void* weight, const void* bias, float eps, void* h, int64_t ldh,
                               void* q, int64_t ldq, float* scale, int64_t scale_row, int64_t scale_block,
                               float* mean, float* rstd, void* stream);

/* C[i,j] = sum over blocks b of a_scale(i, b) * b_scale(j, b) * sum over k in b
 * of A[i,k] * B[j,k], + bias[j]: A (m x k) with tall == 1, B (n x k) with
 * b_tall 1 or 128, C (m x n) and bias (n, or null) of type dtype.  Sums are
 * f32, in an order that depends on the sizes and not on the run: the tensor
 * core's over one block or over as many as keep its error below the output's
 * rounding, then added up. */
tg_status tg_blocks8_gemm(tg_dtype dtype, int64_t m, int64_t n, int64_t k,
                          const void* a, int64_t lda, const float* a_scale, int64_t a_scale_row, int64_t a_scale_block,
                          const void* b, int64_t ldb, int b_tall, const float* b_scale, int64_t b_scale_row, int64_t b_scale_block,
                          const void* bias, void* c, int64_t ldc, void* stream);

/* --------------------------------------------------------------------------
 * What a model answers with: log probabilities of tokens.  logits (rows x
 * vocab) of type dtype; conventions as above.
 *   p = softmax(row);  logprob = log p[token];  entropy = -sum p log p
 * Logits of -infinity have no part in it.  A row of nothing else has logprob
 * and alternatives -infinity, entropy 0 and no gradient; a row that holds a
 * NaN or +infinity gives NaN.  token == ignore_index gives logprob 0 and has
 * no part in the gradient; any other token outside 0 .. vocab - 1 gives NaN.
 * ------------------------------------------------------------------------ */

/* tokens and logprob may be null together; entropy and stats may be null.
 * stats (2 per row): the row's largest logit m, and log sum exp(logit - m).
 * top (0 .. 32, at most vocab): that many most likely tokens per row, and
 * their log probabilities, from the most likely on; of equal logits the lower
 * token comes first. */
tg_status tg_token_logprobs(tg_dtype dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                            const int64_t* tokens, int64_t ignore_index, float* logprob, float* entropy, float* stats,
                            int top, float* top_logprobs, int64_t* top_tokens, void* stream);

/* grad_logits[r, v] = grad_logprob[r] * ([v == token] - p_v)
 *                   - grad_entropy[r] * p_v * (log p_v + entropy[r])
 * from stats and entropy as tg_token_logprobs gave them.  grad_logprob or
 * grad_entropy may be null (zeros); tokens may be null with grad_logprob,
 * entropy with grad_entropy.  grad_logits, of type dtype, may be the logits
 * themselves (same address and ld). */
tg_status tg_token_logprobs_backward(tg_dtype dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                     const int64_t* tokens, int64_t ignore_index, const float* stats, const float* entropy,
                                     const float* grad_logprob, const float* grad_entropy,
                                     void* grad_logits, int64_t ldg, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TROPICAL_GEMM_B200_H */
