// Matrices in 8-bit floating point with a scale for each block of 128:
// quantisation along rows, along both directions at once, by tiles, and back.
// All are bound by memory: x is read once, codes are written once.
#include <algorithm>
#include "tg_blocks8.cuh"

namespace tgb {

struct QuantArgs {
  int64_t rows, cols, ldx, ldq, ldqt;
  const void* x;
  uint8_t *q, *qt;
  float *scale, *scale_t;
  int64_t scale_row, scale_block, scale_t_row, scale_t_block;
  int vec;   // x's rows start on 16-byte boundaries and cols is a multiple of 8
};

// Eight elements as f32, zeros behind the row.
template <typename T> __device__ __forceinline__ void load_values(const QuantArgs& p, int64_t row, int64_t c, float (&v)[8]) {
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  Vec8<T> a;
  if (p.vec) {
    if (c < p.cols) a.load(x + c); else a.zero();
    a.get(v);
  } else {
    load_any(a, x, c, p.cols);
    a.get(v);
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (c + e >= p.cols) v[e] = 0.f;
  }
}
__device__ __forceinline__ uint32_t top_of(const float (&v)[8]) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) top = mag_max(v[e], v[e + 1], top);
  return magnitude(top);
}

// Blocks along rows: 16 lanes per block, 8 elements each.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs p) {
  after_previous_kernel();
  const int64_t blocks = (p.cols + kBlock - 1) / kBlock, total = p.rows * blocks;
  const int lane = threadIdx.x & 15;
  const int64_t step = int64_t(gridDim.x) * 16;
  // whole half warps take part in the shuffles, past the end too
  for (int64_t first = int64_t(blockIdx.x) * 16; first < total; first += step) {
    const int64_t i = first + (threadIdx.x >> 4);
    const bool live = i < total;
    const int64_t row = live ? i / blocks : 0, b = live ? i - row * blocks : 0, c = b * kBlock + lane * 8;
    float v[8];
    load_values<T>(p, row, live ? c : p.cols, v);
    const Step s = step_of(half_warp_max(top_of(v)));
    if (!live || c >= p.cols) continue;
    store_codes(p.q + row * p.ldq, c, p.cols, codes8(v, s.inverse));
    if (lane == 0) p.scale[row * p.scale_row + b * p.scale_block] = s.scale;
  }
}

// A tile of 128 x 128 per thread block: codes along rows (q) and, transposed,
// along columns (qt), or with TILES both with the tile's own scale.  A thread
// holds 8 x 8 elements: rows 8 (t / 16) .., columns 8 (t % 16) ..
template <typename T, bool TILES>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const QuantArgs p) {
  __shared__ __align__(16) uint8_t turned[kBlock][kBlock];   // codes of column c at turned[c], 8-byte chunks swizzled
  __shared__ uint32_t tops[kBlock];
  after_previous_kernel();
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4;
  const int64_t c0 = int64_t(blockIdx.x) * kBlock, r0 = int64_t(blockIdx.y) * kBlock;
  const int64_t c = c0 + cx * 8;
  if (threadIdx.x < kBlock) tops[threadIdx.x] = 0;
  __syncthreads();
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int64_t row = r0 + ry * 8 + i;
    load_values<T>(p, row < p.rows ? row : 0, row < p.rows ? c : p.cols, v[i]);
  }
  // scales along columns, or the tile's
  float inv[8];
  if constexpr (TILES) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, top_of(v[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) atomicMax(&tops[0], top);
    __syncthreads();
    const Step s = step_of(tops[0]);
    if (threadIdx.x == 0) p.scale[blockIdx.y * p.scale_row + blockIdx.x * p.scale_block] = s.scale;
#pragma unroll
    for (int e = 0; e < 8; e++) inv[e] = s.inverse;
  } else {
    if (p.qt) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, magnitude(v[i][e]));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
        if ((threadIdx.x & 16) == 0) atomicMax(&tops[cx * 8 + e], top);
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; e++) inv[e] = step_of(tops[cx * 8 + e]).inverse;
      const int64_t col = c0 + threadIdx.x;
      if (threadIdx.x < kBlock && col < p.cols) p.scale_t[col * p.scale_t_row + blockIdx.y * p.scale_t_block] = step_of(tops[threadIdx.x]).scale;
    }
  }
  if (p.q) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t row = r0 + ry * 8 + i;
      float inverse = inv[0];
      if constexpr (!TILES) {
        const Step s = step_of(half_warp_max(top_of(v[i])));
        inverse = s.inverse;
        if (cx == 0 && row < p.rows) p.scale[row * p.scale_row + blockIdx.x * p.scale_block] = s.scale;
      }
      if (row < p.rows && c < p.cols) store_codes(p.q + row * p.ldq, c, p.cols, codes8(v[i], inverse));
    }
  }
  if (p.qt) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float column[8];
#pragma unroll
      for (int i = 0; i < 8; i++) column[i] = v[i][e];
      *reinterpret_cast<uint2*>(&turned[cx * 8 + e][(ry ^ cx) * 8]) = codes8(column, inv[e]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {   // 16 lanes along a column
      const int col = i * 16 + ry;
      if (c0 + col >= p.cols) continue;
      const uint2 w = *reinterpret_cast<const uint2*>(&turned[col][(cx ^ (col >> 3)) * 8]);
      if (r0 + cx * 8 < p.rows) store_codes(p.qt + (c0 + col) * p.ldqt, r0 + cx * 8, p.rows, w);
    }
  }
}

// Codes transposed, a tile of 128 x 128 per thread block.
__global__ void __launch_bounds__(256) turn_codes_kernel(int64_t rows, int64_t cols, const uint8_t* q, int64_t ldq, uint8_t* qt, int64_t ldqt) {
  __shared__ uint8_t tile[kBlock][kBlock + 4];
  after_previous_kernel();
  const int64_t c0 = int64_t(blockIdx.x) * kBlock;
  for (int64_t r0 = int64_t(blockIdx.y) * kBlock; r0 < rows; r0 += int64_t(gridDim.y) * kBlock) {
    for (int i = threadIdx.x; i < kBlock * kBlock; i += 256) {
      const int r = i >> 7, c = i & 127;
      if (r0 + r < rows && c0 + c < cols) tile[r][c] = q[(r0 + r) * ldq + c0 + c];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBlock * kBlock; i += 256) {
      const int c = i >> 7, r = i & 127;
      if (r0 + r < rows && c0 + c < cols) qt[(c0 + c) * ldqt + r0 + r] = tile[r][c];
    }
    __syncthreads();
  }
}

// Eight elements per thread.
template <typename T>
__global__ void __launch_bounds__(256) blocks_values_kernel(int64_t rows, int64_t cols, int tall, const uint8_t* q, int64_t ldq,
                                                            const float* scale, int64_t scale_row, int64_t scale_block, T* y, int64_t ldy) {
  after_previous_kernel();
  const int64_t per = (cols + 7) / 8, total = rows * per;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t row = i / per, c = (i - row * per) * 8;
    const uint8_t* from = q + row * ldq + c;
    uint2 w = make_uint2(0, 0);
    if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(from) & 7) == 0) {
      w = *reinterpret_cast<const uint2*>(from);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (c + e < cols) (e < 4 ? w.x : w.y) |= uint32_t(from[e]) << (8 * (e & 3));
    }
    const float s = scale[row / tall * scale_row + c / kBlock * scale_block];
    const float2 a = values2(w.x), b = values2(w.x >> 16), d = values2(w.y), f = values2(w.y >> 16);
    const float v[8] = {a.x * s, a.y * s, b.x * s, b.y * s, d.x * s, d.y * s, f.x * s, f.y * s};
    store_any(y + row * ldy, c, cols, v);
  }
}

}  // namespace tgb

namespace tgi {

using tgb::QuantArgs;

namespace {

tg_status check_blocks(tg_dtype dtype, int64_t rows, int64_t cols) {
  if (!elem8_size(dtype)) return fail(TG_ERR_INVALID_ARGUMENT, "8-bit blocks need f32, f16 or bf16, got dtype %d", int(dtype));
  if (rows < 0 || cols < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (rows=%lld cols=%lld)", (long long)rows, (long long)cols);
  if (rows > 0x7fffff00 || cols > 0x7fffff00) return fail(TG_ERR_UNSUPPORTED, "%lld x %lld elements", (long long)rows, (long long)cols);
  return TG_OK;
}
tg_status check_pitch(const char* name, int64_t ld, int64_t cols) {
  return ld < cols ? fail(TG_ERR_DIMENSION_MISMATCH, "%s=%lld < %lld", name, (long long)ld, (long long)cols) : TG_OK;
}
#define TG_CHECK(call)                  \
  do {                                  \
    const tg_status s_ = (call);        \
    if (s_ != TG_OK) return s_;         \
  } while (0)

template <bool TILES> tg_status launch_tiles(tg_dtype dtype, const QuantArgs& p, cudaStream_t st) {
  const int64_t tr = (p.rows + 127) / 128, tc = (p.cols + 127) / 128;
  return with_type8(dtype, [&](auto t) {
    // rows of tiles along grid.y, in as many launches as it takes
    for (int64_t at = 0; at < tr; at += 32768) {
      QuantArgs part = p;
      const int64_t first = at * 128;
      part.rows = std::min<int64_t>(p.rows - first, 32768 * 128);
      part.x = static_cast<const char*>(p.x) + first * p.ldx * int64_t(elem8_size(dtype));
      if (p.q) part.q += first * p.ldq;
      if (p.scale) part.scale += (TILES ? at : first) * p.scale_row;
      if (p.qt) part.qt += first;
      if (p.scale_t) part.scale_t += at * p.scale_t_block;
      launch_kernel(tgb::quantize_tile_kernel<decltype(t), TILES>, dim3(unsigned(tc), unsigned(std::min<int64_t>(tr - at, 32768))), 256, 0, 0, st, part);
    }
    return check_launch("blocks8 quantize");
  });
}

}  // namespace
}  // namespace tgi

using namespace tgi;

extern "C" {

tg_status tg_blocks8_quantize(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, void* q, int64_t ldq,
                              float* scale, int64_t scale_row, int64_t scale_block, void* qt, int64_t ldqt, float* scale_t,
                              int64_t scale_t_row, int64_t scale_t_block, void* stream) {
  clear_error();
  TG_CHECK(check_blocks(dtype, rows, cols));
  if (rows == 0 || cols == 0) return TG_OK;
  if (!x || (!q && !qt) || (q && !scale) || (qt && !scale_t)) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldx", ldx, cols));
  if (q) TG_CHECK(check_pitch("ldq", ldq, cols));
  if (qt) TG_CHECK(check_pitch("ldqt", ldqt, rows));
  QuantArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx;
  p.q = static_cast<uint8_t*>(q); p.ldq = ldq; p.scale = scale; p.scale_row = scale_row; p.scale_block = scale_block;
  p.qt = static_cast<uint8_t*>(qt); p.ldqt = ldqt; p.scale_t = scale_t; p.scale_t_row = scale_t_row; p.scale_t_block = scale_t_block;
  p.vec = aligned(x, 16) && (ldx * int64_t(elem8_size(dtype))) % 16 == 0 && cols % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (qt) return launch_tiles<false>(dtype, p, st);
  const int64_t blocks = rows * ((cols + 127) / 128);
  const unsigned grid = unsigned(std::min<int64_t>((blocks + 15) / 16, int64_t(sm_count()) * 64));
  return with_type8(dtype, [&](auto t) {
    launch_kernel(tgb::quantize_rows_kernel<decltype(t)>, grid, 256, 0, 0, st, p);
    return check_launch("blocks8 quantize");
  });
}

tg_status tg_blocks8_quantize_tiles(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, void* q, int64_t ldq,
                                    float* scale, int64_t scale_row, int64_t scale_block, void* qt, int64_t ldqt, void* stream) {
  clear_error();
  TG_CHECK(check_blocks(dtype, rows, cols));
  if (rows == 0 || cols == 0) return TG_OK;
  if (!x || !q || !scale) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldx", ldx, cols));
  TG_CHECK(check_pitch("ldq", ldq, cols));
  if (qt) TG_CHECK(check_pitch("ldqt", ldqt, rows));
  QuantArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx;
  p.q = static_cast<uint8_t*>(q); p.ldq = ldq; p.scale = scale; p.scale_row = scale_row; p.scale_block = scale_block;
  p.qt = static_cast<uint8_t*>(qt); p.ldqt = ldqt;
  p.vec = aligned(x, 16) && (ldx * int64_t(elem8_size(dtype))) % 16 == 0 && cols % 8 == 0;
  return launch_tiles<true>(dtype, p, static_cast<cudaStream_t>(stream));
}

tg_status tg_blocks8_transpose(int64_t rows, int64_t cols, const void* q, int64_t ldq, void* qt, int64_t ldqt, void* stream) {
  clear_error();
  TG_CHECK(check_blocks(TG_F32, rows, cols));
  if (rows == 0 || cols == 0) return TG_OK;
  if (!q || !qt) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldq", ldq, cols));
  TG_CHECK(check_pitch("ldqt", ldqt, rows));
  launch_kernel(tgb::turn_codes_kernel, dim3(unsigned((cols + 127) / 128), unsigned(std::min<int64_t>((rows + 127) / 128, 32768))), 256, 0, 0,
                static_cast<cudaStream_t>(stream), rows, cols, static_cast<const uint8_t*>(q), ldq, static_cast<uint8_t*>(qt), ldqt);
  return check_launch("blocks8 transpose");
}

tg_status tg_blocks8_dequantize(tg_dtype dtype, int64_t rows, int64_t cols, int tall, const void* q, int64_t ldq,
                                const float* scale, int64_t scale_row, int64_t scale_block, void* y, int64_t ldy, void* stream) {
  clear_error();
  TG_CHECK(check_blocks(dtype, rows, cols));
  if (tall != 1 && tall != 128) return fail(TG_ERR_INVALID_ARGUMENT, "blocks are 1 or 128 rows tall, got %d", tall);
  if (rows == 0 || cols == 0) return TG_OK;
  if (!q || !scale || !y) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldq", ldq, cols));
  TG_CHECK(check_pitch("ldy", ldy, cols));
  const int64_t threads = rows * ((cols + 7) / 8);
  const unsigned grid = unsigned(std::min<int64_t>((threads + 255) / 256, int64_t(sm_count()) * 64));
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    launch_kernel(tgb::blocks_values_kernel<T>, grid, 256, 0, 0, static_cast<cudaStream_t>(stream), rows, cols, tall,
                  static_cast<const uint8_t*>(q), ldq, scale, scale_row, scale_block, static_cast<T*>(y), ldy);
    return check_launch("blocks8 dequantize");
  });
}

}  // extern "C"
