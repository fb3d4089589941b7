// Matrices in 8-bit floating point with a scale for each block of 128:
// quantisation along rows, along both directions at once, by tiles, and back.
// All are bound by memory: x is read once, codes are written once.
#include <algorithm>
#include <type_traits>
#include "tg_blocks8.cuh"

namespace tgb {

struct QuantArgs {
  int64_t rows, cols, ldx, ldq, ldqt;
  const void* x;
  uint8_t *q, *qt;
  float *scale, *scale_t;
  int64_t scale_row, scale_block, scale_t_row, scale_t_block;
  float* sums;   // column sums of each row of tiles (tiles x cols), or null
  int vec;       // x's rows start on 16-byte boundaries and cols is a multiple of 8
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

// Few rows, blocks along them: 16 lanes per block, 8 elements each; blockIdx.x has
// 16 blocks of a row, blockIdx.y rows y, + gridDim.y, ..
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs p) {
  after_previous_kernel();
  const int64_t b = int64_t(blockIdx.x) * 16 + (threadIdx.x >> 4), c = b * kBlock + (threadIdx.x & 15) * 8;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    float v[8];
    load_values<T>(p, row, c, v);
    const Step s = step_of(half_warp_max(top_of(v)));   // whole half warps, past the row's end too
    if (c >= p.cols) continue;
    store_codes(p.q + row * p.ldq, c, p.cols, codes8(v, s.inverse));
    if ((threadIdx.x & 15) == 0) p.scale[row * p.scale_row + b * p.scale_block] = s.scale;
  }
}

// Largest magnitudes of eight columns, two 16-bit values per word where the
// elements are; a NaN stays.
template <typename T> struct Tops {
  uint32_t w[4];
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (std::is_same_v<T, bf16>) {
      const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&r);
    } else {
      const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&r);
    }
  }
  static __device__ __forceinline__ uint32_t bits(uint32_t half) {   // of the f32 value
    if constexpr (std::is_same_v<T, bf16>) return half << 16;
    else return __float_as_uint(__half2float(__ushort_as_half(uint16_t(half)))) & 0x7fffffffu;
  }
  __device__ __forceinline__ void start() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ void with(const Vec8<T>& a) {
    const uint32_t v[4] = {a.a.x, a.a.y, a.a.z, a.a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = larger(w[i], v[i] & 0x7fff7fffu);
  }
  __device__ __forceinline__ void with_lane(int d) {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = larger(w[i], __shfl_xor_sync(0xffffffffu, w[i], d));
  }
  __device__ __forceinline__ uint32_t column(int e) const { return bits(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu); }
  // rows' largest over 16 lanes, as f32 bits
  static __device__ __forceinline__ void rows(const Vec8<T> (&a)[8], uint32_t (&top)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {   // two rows to a word
      uint32_t r[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint4 v = a[i + j].a;
        r[j] = larger(larger(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), larger(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
      }
      uint32_t both = larger(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[0], r[1], 0x7632));
#pragma unroll
      for (int d = 8; d; d >>= 1) both = larger(both, __shfl_xor_sync(0xffffffffu, both, d));
      top[i] = bits(both & 0xffffu);
      top[i + 1] = bits(both >> 16);
    }
  }
};
template <> struct Tops<float> {
  float t[8];
  __device__ __forceinline__ void start() {
#pragma unroll
    for (int e = 0; e < 8; e++) t[e] = 0.f;
  }
  __device__ __forceinline__ void with(const Vec8<float>& a) {
    float v[8];
    a.get(v);
#pragma unroll
    for (int e = 0; e < 8; e++) t[e] = mag_max(v[e], v[e], t[e]);
  }
  __device__ __forceinline__ void with_lane(int d) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float o = __shfl_xor_sync(0xffffffffu, t[e], d);
      t[e] = mag_max(o, o, t[e]);
    }
  }
  __device__ __forceinline__ uint32_t column(int e) const { return magnitude(t[e]); }
  static __device__ __forceinline__ void rows(const Vec8<float> (&a)[8], uint32_t (&top)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float v[8];
      a[i].get(v);
      top[i] = half_warp_max(top_of(v));
    }
  }
};

// A tile of 128 x 128 per thread block: codes along rows (q) and, transposed,
// along columns (qt), or with TILES both with the tile's own scale.  A thread
// holds 8 x 8 elements: rows 8 (t / 16) .., columns 8 (t % 16) .., as they came,
// so that 16-bit ones leave room for four blocks on an SM (as f32 two fit:
// 8192 x 8192 bf16 both ways 139 us, tiles 95).
template <typename T, bool TILES>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) quantize_tile_kernel(const QuantArgs p) {
  __shared__ __align__(16) uint8_t turned[kBlock][kBlock];   // codes of column c at turned[c], 8-byte chunks swizzled
  __shared__ __align__(16) uint32_t tops[8][kBlock];         // per warp, or the tile's
  __shared__ __align__(16) float factor[kBlock];             // 1 / scale of the columns
  after_previous_kernel();
  const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = int64_t(blockIdx.x) * kBlock, r0 = int64_t(blockIdx.y) * kBlock;
  const int64_t c = c0 + cx * 8, left = p.cols - c;
  Vec8<T> a[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int64_t row = r0 + ry * 8 + i;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    a[i].zero();
    if (row >= p.rows || left <= 0) continue;
    if (p.vec) {
      a[i].load(x + c);
    } else {
      load_any(a[i], x, c, p.cols);
      if (left < 8) {
        union { Vec8<T> v; T e[8]; } u;
        u.v = a[i];
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (e >= left) u.e[e] = from_f32<T>(0.f);
        a[i] = u.v;
      }
    }
  }
  Tops<T> top;
  top.start();
  if (TILES || p.qt) {
#pragma unroll
    for (int i = 0; i < 8; i++) top.with(a[i]);
    top.with_lane(16);
  }
  float whole = 0.f;   // TILES: 1 / scale
  if constexpr (TILES) {
    uint32_t t = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) t = max(t, top.column(e));
    t = __reduce_max_sync(0xffffffffu, t);
    if (lane == 0) tops[0][warp] = t;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) t = max(t, tops[0][w]);
    const Step s = step_of(t);
    if (threadIdx.x == 0) p.scale[blockIdx.y * p.scale_row + blockIdx.x * p.scale_block] = s.scale;
    whole = s.inverse;
  } else if (p.qt) {
    if (lane < 16) {
      *reinterpret_cast<uint4*>(&tops[warp][cx * 8]) = make_uint4(top.column(0), top.column(1), top.column(2), top.column(3));
      *reinterpret_cast<uint4*>(&tops[warp][cx * 8 + 4]) = make_uint4(top.column(4), top.column(5), top.column(6), top.column(7));
    }
    __syncthreads();
    if (threadIdx.x < kBlock) {
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < 8; w++) t = max(t, tops[w][threadIdx.x]);
      const Step s = step_of(t);
      factor[threadIdx.x] = s.inverse;
      if (c0 + threadIdx.x < p.cols) p.scale_t[(c0 + threadIdx.x) * p.scale_t_row + blockIdx.y * p.scale_t_block] = s.scale;
    }
    __syncthreads();
  }
  if (!TILES && p.sums) {   // in a fixed order: 8 rows, two lanes, 8 warps
    uint64_t sum[4] = {};
#pragma unroll
    for (int i = 0; i < 8; i++) {
      uint64_t v[4];
      get_pairs(a[i], v);
#pragma unroll
      for (int j = 0; j < 4; j++) sum[j] = add_pair(sum[j], v[j]);
    }
    float f[8];
    from_pairs(sum, f);
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] += __shfl_xor_sync(0xffffffffu, f[e], 16);
    float(*parts)[kBlock] = reinterpret_cast<float(*)[kBlock]>(tops);   // the tops are read
    if (lane < 16) store8(&parts[warp][cx * 8], f);
    __syncthreads();
    if (threadIdx.x < kBlock && c0 + threadIdx.x < p.cols) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; w++) s += parts[w][threadIdx.x];
      p.sums[blockIdx.y * p.cols + c0 + threadIdx.x] = s;
    }
  }
  if (p.q) {
    uint32_t row_top[8];
    if constexpr (!TILES) Tops<T>::rows(a, row_top);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t row = r0 + ry * 8 + i;
      float inverse = whole;
      if constexpr (!TILES) {
        const Step s = step_of(row_top[i]);
        inverse = s.inverse;
        if (cx == 0 && row < p.rows) p.scale[row * p.scale_row + blockIdx.x * p.scale_block] = s.scale;
      }
      float v[8];
      a[i].get(v);
      if (row < p.rows && left > 0) store_codes(p.q + row * p.ldq, c, p.cols, codes8(v, inverse));
    }
  }
  if (p.qt) {
    // codes of each row with the columns' factors, then 8 x 8 bytes transposed
    uint64_t inv[4];
#pragma unroll
    for (int j = 0; j < 4; j++) inv[j] = TILES ? pair_of(whole) : pair_of(factor[cx * 8 + 2 * j], factor[cx * 8 + 2 * j + 1]);
    uint2 code[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      uint64_t v[4];
      get_pairs(a[i], v);
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 f = values_of(mul_pair(v[j], inv[j]));
        h[j] = code2(f.x, f.y);
      }
      code[i] = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {   // columns 4 half ..
      uint32_t lo[4], hi[4];   // rows 0-3 and 4-7 of a column
      auto turn = [&](uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t (&o)[4]) {
        const uint32_t a = __byte_perm(r0, r1, 0x5140), b = __byte_perm(r2, r3, 0x5140);   // columns 0, 1 of two rows each
        const uint32_t d = __byte_perm(r0, r1, 0x7362), e = __byte_perm(r2, r3, 0x7362);   // columns 2, 3
        o[0] = __byte_perm(a, b, 0x5410);
        o[1] = __byte_perm(a, b, 0x7632);
        o[2] = __byte_perm(d, e, 0x5410);
        o[3] = __byte_perm(d, e, 0x7632);
      };
      auto word = [&](int i) { return half ? code[i].y : code[i].x; };
      turn(word(0), word(1), word(2), word(3), lo);
      turn(word(4), word(5), word(6), word(7), hi);
#pragma unroll
      for (int e = 0; e < 4; e++) *reinterpret_cast<uint2*>(&turned[cx * 8 + half * 4 + e][(ry ^ cx) * 8]) = make_uint2(lo[e], hi[e]);
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
      if (p.sums) part.sums += at * p.cols;
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
                              int64_t scale_t_row, int64_t scale_t_block, void* column_sum, void* stream) {
  clear_error();
  TG_CHECK(check_blocks(dtype, rows, cols));
  if (cols && rows == 0 && column_sum) {   // a sum of nothing
    const cudaError_t e = cudaMemsetAsync(column_sum, 0, size_t(cols) * elem8_size(dtype), static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "memset: %s", cudaGetErrorString(e));
  }
  if (rows == 0 || cols == 0) return TG_OK;
  if (!x || (!q && !qt && !column_sum) || (q && !scale) || (qt && !scale_t)) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldx", ldx, cols));
  if (q) TG_CHECK(check_pitch("ldq", ldq, cols));
  if (qt) TG_CHECK(check_pitch("ldqt", ldqt, rows));
  QuantArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx;
  p.q = static_cast<uint8_t*>(q); p.ldq = ldq; p.scale = scale; p.scale_row = scale_row; p.scale_block = scale_block;
  p.qt = static_cast<uint8_t*>(qt); p.ldqt = ldqt; p.scale_t = scale_t; p.scale_t_row = scale_t_row; p.scale_t_block = scale_t_block;
  p.vec = aligned(x, 16) && (ldx * int64_t(elem8_size(dtype))) % 16 == 0 && cols % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (column_sum) {
    const int64_t tiles = (rows + 127) / 128;
    void* scratch = nullptr;
    const cudaError_t e = scratch_alloc(&scratch, size_t(tiles) * size_t(cols) * sizeof(float), st);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "blocks8 quantize scratch: %s", cudaGetErrorString(e));
    p.sums = static_cast<float*>(scratch);
    tg_status s = launch_tiles<false>(dtype, p, st);
    if (s == TG_OK)
      s = with_type8(dtype, [&](auto t) {
        using T = decltype(t);
        launch_kernel(tg8::column_join_kernel<T>, unsigned((cols + 31) / 32), 1024, 0, 0, st, tiles, cols, static_cast<const float*>(p.sums), static_cast<T*>(column_sum));
        return check_launch("blocks8 quantize");
      });
    scratch_free(scratch, st);
    return s;
  }
  // From 512 rows on the tile kernel is the faster one along rows alone, too (8192 x 8192 bf16 48 us row by row, 40).
  if (qt || rows >= 512) return launch_tiles<false>(dtype, p, st);
  const dim3 grid(unsigned((cols + 2047) / 2048), unsigned(rows));
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
