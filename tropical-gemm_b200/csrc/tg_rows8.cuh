// Shared by the 8-bit row kernels: element types, 8-element vector access,
// the quantisation rule and small host helpers.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include "tg_internal.h"

namespace tg8 {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(f16 v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ f16 from_f32<f16>(float v) { return __float2half_rn(v); }

// Eight consecutive elements as loaded (16-byte aligned), and as f32.
template <typename T> struct Vec8;
template <> struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
  __device__ __forceinline__ void zero() { a = b = make_float4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
};
template <> struct Vec8<bf16> {
  uint4 a;
  __device__ __forceinline__ void load(const bf16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};
template <> struct Vec8<f16> {
  uint4 a;
  __device__ __forceinline__ void load(const f16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(f16* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// How a row kernel reaches its rows.
//   kScalar  element by element, any alignment
//   kAligned groups of 8 elements that start on 16-byte boundaries
//   kShifted the same groups for rows that start anywhere: group k is elements
//            8 k - s .. 8 k - s + 7 with s the row start's distance from a boundary
//            of 8 elements, equal in all operands.  A group at an end of the row is
//            loaded whole where its 16 bytes hold an element of the row (they are
//            mapped then) and masked; it is stored element by element
enum Access { kScalar, kAligned, kShifted };

template <typename T> __device__ __forceinline__ int row_shift(const T* row) { return int((reinterpret_cast<uintptr_t>(row) / sizeof(T)) & 7); }

__device__ __forceinline__ void load_touching(Vec8<float>& v, const float* row, int c, int cols) {
  if (c + 4 > 0) v.a = *reinterpret_cast<const float4*>(row + c);
  if (c + 4 < cols) v.b = *reinterpret_cast<const float4*>(row + c + 4);
}
template <typename T> __device__ __forceinline__ void load_touching(Vec8<T>& v, const T* row, int c, int) { v.load(row + c); }

template <int ACCESS, typename T> __device__ __forceinline__ void load_group(Vec8<T>& v, const T* row, int c, int cols) {
  if constexpr (ACCESS == kAligned) {
    if (c < cols) v.load(row + c); else v.zero();
  } else {
    v.zero();
    if (c < cols) load_touching(v, row, c, cols);   // c > -8
  }
}
// Zeros for what a group at a row's end holds of its neighbours.
template <int ACCESS> __device__ __forceinline__ void mask_group(float (&v)[8], int c, int cols) {
  if (ACCESS == kShifted && (c < 0 || c + 8 > cols)) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (c + i < 0 || c + i >= cols) v[i] = 0.f;
  }
}
template <int ACCESS, typename T> __device__ __forceinline__ void store_group(T* row, int c, int cols, const float (&v)[8]) {
  if (ACCESS == kAligned ? c < cols : c >= 0 && c + 8 <= cols) {
    store8(row + c, v);
  } else if (ACCESS == kShifted) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (c + i >= 0 && c + i < cols) row[c + i] = from_f32<T>(v[i]);
  }
}
__device__ __forceinline__ uint2 load_bytes(const int8_t* row, int c, int cols) {
  return c < cols ? *reinterpret_cast<const uint2*>(row + c) : make_uint2(0, 0);
}
template <int ACCESS> __device__ __forceinline__ void store_bytes(int8_t* row, int c, int cols, uint2 w) {
  if (ACCESS == kAligned ? c < cols : c >= 0 && c + 8 <= cols) {
    *reinterpret_cast<uint2*>(row + c) = w;
  } else if (ACCESS == kShifted) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (c + i >= 0 && c + i < cols) row[c + i] = int8_t(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xff);
  }
}
// Place of column c in a row of f32 held in shared memory, c from -8: a word of
// padding after every eight, so that lanes eight columns apart meet all banks.
__device__ __forceinline__ int padded_at(int c) { return c + 8 + ((c + 8) >> 3); }
// padded_at(c + e) = padded_at(c) + padded_offset(shift, e) for the group that
// starts at c = 8 k - shift: an offset per element that a row's groups share.
__device__ __forceinline__ int padded_offset(int shift, int e) { return e + ((((8 - shift) & 7) + e) >> 3); }
__host__ __device__ __forceinline__ size_t padded_bytes(int64_t cols) { return size_t(cols + 16 + (cols + 16) / 8 + 1) * 4; }

// max(|a|, |b|, m) that keeps a NaN.
__device__ __forceinline__ float mag_max(float a, float b, float m) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(m));
  return r;
}

// One row's quantisation from its largest magnitude, given as the maximum of
// the values' bit patterns without the sign: unsigned order is magnitude
// order, with infinities and NaN on top, so a maximum never loses a NaN.
//
// A code is y * inv, rounded by adding `first` and then 1.5 * 2^23 - first, which
// leaves the integer in the low mantissa bits.  inv is 127 / top rounded up, off by
// less than 2^-23 of itself, and for most rows first = 1.5 * 2^23, one rounding:
// a quotient within 127 * 2^-23 of a tie may go to either side.  Ties themselves,
// 2 * 127 |y| = (2n + 1) top, go to the even code.  127 is a prime, so either
// 2n + 1 = 127 (y is half the largest value, 16-bit inputs hit it often): 63.5,
// made no less by inv, goes to 64.  Or 127 divides top's significand (by chance
// one row in 127): top / 127 is exact then, and first = 384.  384 + y * inv has
// units of 2^-15, so inv's error, below 126.5 * 2^-23 < 2^-16, is rounded away
// and the tie is met exactly by the second rounding.
struct Quant {
  float scale, inv, first;
};
constexpr float kWhole = 12582912.f;   // 1.5 * 2^23
__device__ __forceinline__ Quant quant_of(uint32_t top_bits) {
  Quant s;
  const float top = __uint_as_float(top_bits);
  s.first = kWhole;
  if (top_bits >= 0x7f800000u) {   // an infinity or a NaN: the row reads as NaN
    s.scale = __uint_as_float(0x7fffffffu);
    s.inv = 0.f;
  } else if (top < 7.52316385e-37f) {   // 2^-120: 127 / top would overflow not far below
    s.scale = s.inv = 0.f;
  } else {
    s.scale = top / 127.f;
    s.inv = __fdiv_ru(127.f, top);
    if (fmaf(s.scale, 127.f, -top) == 0.f) s.first = 384.f;
  }
  return s;
}
// The code as the low byte of the result (|y * inv| < 128).
__device__ __forceinline__ uint32_t quant8(float y, const Quant& s) {
  return __float_as_uint(fmaf(y, s.inv, s.first) + (kWhole - s.first));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
__device__ __forceinline__ uint2 quant_pack8(const float (&v)[8], const Quant& s) {
  uint32_t q[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2)   // two at a time
    asm("{\n.reg .b64 y, i, f, r;\nmov.b64 y, {%2, %3};\nmov.b64 i, {%4, %4};\nmov.b64 f, {%5, %5};\nmov.b64 r, {%6, %6};\n"
        "fma.rn.f32x2 y, y, i, f;\nadd.rn.f32x2 y, y, r;\nmov.b64 {%0, %1}, y;\n}\n"
        : "=r"(q[e]), "=r"(q[e + 1])
        : "f"(v[e]), "f"(v[e + 1]), "f"(s.inv), "f"(s.first), "f"(kWhole - s.first));
  return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}
// Byte i of w as a signed integer in f32, by way of 2^23 + (byte + 128).
template <int I> __device__ __forceinline__ float byte_f32(uint32_t w_biased) {
  return __uint_as_float(__byte_perm(w_biased, 0x4b000000u, 0x7650 | I)) - 8388736.f;
}
__device__ __forceinline__ void bytes_f32(uint2 w, float (&v)[8]) {
  const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
  v[0] = byte_f32<0>(a); v[1] = byte_f32<1>(a); v[2] = byte_f32<2>(a); v[3] = byte_f32<3>(a);
  v[4] = byte_f32<0>(b); v[5] = byte_f32<1>(b); v[6] = byte_f32<2>(b); v[7] = byte_f32<3>(b);
}

// Barrier `id` of the block's (1 to 15), for `threads` of them in whole warps whose
// lanes it wants together: a store by one lane before need not have left them so.
__device__ __forceinline__ void named_sync(int id, int threads) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Kernels of these calls are launched with programmatic stream serialisation:
// a kernel may be set up while the one before it ends, waits here before it
// touches global memory until that one is complete, and lets the next one be
// set up.  (norm, product: about 1 us less between two kernels.)
__device__ __forceinline__ void after_previous_kernel() {
  asm volatile("griddepcontrol.wait;\ngriddepcontrol.launch_dependents;" ::: "memory");
}

// out[c] = sum over slots of partial[slot, c]: 32 columns x 32 slot lanes per
// block, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) column_join_kernel(int64_t slots, int64_t cols, const float* partial, T* out) {
  __shared__ float part[32][33];
  after_previous_kernel();
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = int64_t(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = y; r < slots; r += 32) s += partial[r * cols + c];
  }
  part[y][lane] = s;
  __syncthreads();
  // warp y joins column y of the strip
  s = part[lane][y];
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  const int64_t column = int64_t(blockIdx.x) * 32 + y;
  if (lane == 0 && column < cols) out[column] = from_f32<T>(s);
}

}  // namespace tg8

namespace tgi {

// A launch of one of these kernels; clusters of `cluster` blocks along x.
// Errors are left to check_launch.
template <typename... P, typename... A>
void launch_kernel(void (*kern)(P...), dim3 grid, int block, size_t smem, int cluster, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(block));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {unsigned(cluster), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;   // 0: the kernel's own cluster size, if any
  (void)cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

inline size_t elem8_size(tg_dtype t) { return t == TG_F32 ? 4 : (t == TG_BF16 || t == TG_F16) ? 2 : 0; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// The access that a call's operands allow: kAligned when all rows start on a
// boundary of 8 elements, kShifted when all are the same distance from one.
class RowAccess {
 public:
  explicit RowAccess(int64_t cols) : cols_(cols) {}
  void add(const void* p, int64_t ld, size_t elem) {
    if (!p) return;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    const int phase = a % elem ? -1 : int(a / elem % 8), step = int(ld % 8);
    if (!any_) { phase_ = phase; step_ = step; }
    any_ = true;
    same_ = same_ && phase >= 0 && phase == phase_ && step == step_;
  }
  int get() const { return !same_ ? tg8::kScalar : phase_ == 0 && step_ == 0 && cols_ % 8 == 0 ? tg8::kAligned : tg8::kShifted; }

 private:
  int64_t cols_;
  int phase_ = 0, step_ = 0;
  bool any_ = false, same_ = true;
};

// f(T{}) for the element type of a tg_rows8 call; the caller has checked dtype.
template <typename F> tg_status with_type8(tg_dtype t, F&& f) {
  switch (t) {
    case TG_F32: return f(float{});
    case TG_F16: return f(tg8::f16{});
    case TG_BF16: return f(tg8::bf16{});
    default: return fail(TG_ERR_INVALID_ARGUMENT, "8-bit rows need f32, f16 or bf16, got dtype %d", int(t));
  }
}

}  // namespace tgi
