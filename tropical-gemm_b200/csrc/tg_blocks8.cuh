// Shared by the layer norm and the kernels of matrices held in 8-bit floating
// point: rows of any alignment, e4m3 codes and their scales.
#pragma once
#include <cuda_fp8.h>
#include "tg_rows8.cuh"

namespace tgb {

using namespace tg8;

constexpr int kBlock = 128;   // elements that share a scale

// Elements c .. c + 7 of a row of `cols` that may start at any element: the
// 16-byte words that hold at least one of them, shifted into place.  What lies
// behind the row is unspecified.
template <typename T> __device__ __forceinline__ void load_any(Vec8<T>& v, const T* row, int64_t c, int64_t cols) {
  static_assert(sizeof(T) == 2, "16-bit elements");
  v.zero();
  const int64_t left = (cols - c) * 2;   // bytes of the row from c on
  if (left <= 0) return;
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
  const uint32_t skew = uint32_t(at & 15);
  const uint4* words = reinterpret_cast<const uint4*>(at - skew);
  const uint4 lo = words[0];
  const uint4 hi = skew && int64_t(16 - skew) < left ? words[1] : make_uint4(0, 0, 0, 0);
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (skew & 8) {
#pragma unroll
    for (int k = 0; k < 6; k++) w[k] = w[k + 2];
  }
  if (skew & 4) {
#pragma unroll
    for (int k = 0; k < 5; k++) w[k] = w[k + 1];
  }
  const uint32_t bits = (skew & 2) * 8;
  v.a = make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                   __funnelshift_r(w[3], w[4], bits));
}
template <> __device__ __forceinline__ void load_any<float>(Vec8<float>& v, const float* row, int64_t c, int64_t cols) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = c + e < cols ? row[c + e] : 0.f;
  v.a = make_float4(f[0], f[1], f[2], f[3]);
  v.b = make_float4(f[4], f[5], f[6], f[7]);
}
// Eight elements to a row that may start at any element.
template <typename T> __device__ __forceinline__ void store_any(T* row, int64_t c, int64_t cols, const float (&v)[8]) {
  if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(row + c) & 15) == 0) {
    store8(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (c + e < cols) row[c + e] = from_f32<T>(v[e]);
  }
}
// The same of eight bytes.
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t c, int64_t cols, uint2 w) {
  if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(row + c) & 7) == 0) {
    *reinterpret_cast<uint2*>(row + c) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (c + e < cols) row[c + e] = uint8_t((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
  }
}

// Two f32 values side by side.
__device__ __forceinline__ uint64_t pair_of(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) { return pair_of(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ float2 values_of(uint64_t v) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ uint64_t pair_of(float a) { return pair_of(a, a); }
__device__ __forceinline__ void fma_pair(uint64_t& acc, uint64_t a, uint64_t b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b)); }
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair_of(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum_of(uint64_t v) {
  const float2 f = values_of(v);
  return f.x + f.y;
}
// Eight elements as four pairs: two f32 operations per instruction.
template <typename T> __device__ __forceinline__ void get_pairs(const Vec8<T>& a, uint64_t (&v)[4]) {
  float f[8];
  a.get(f);
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = pair_of(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void from_pairs(const uint64_t (&v)[4], float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 x = values_of(v[i]);
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block's scale and its inverse, from the bit pattern of its largest
// magnitude (as an unsigned number: infinities and NaN are on top).  448 =
// 1.75 * 2^8: the scale's exponent is the magnitude's less 8, or less 7 above
// a mantissa of 1.75.  Both are powers of two, so a code is one rounding of
// the value.
struct Step {
  float scale, inverse;
};
__device__ __forceinline__ Step step_of(uint32_t top) {
  if (top >= 0x7f800000u) return {__uint_as_float(0x7fffffffu), 0.f};
  const int e = max(int(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u), 1);   // biased; 1: 2^-126
  return {__uint_as_float(uint32_t(e) << 23), __uint_as_float(uint32_t(254 - e) << 23)};
}
// Codes of a and b, a in the low byte: round to nearest even.
__device__ __forceinline__ uint32_t code2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float inverse) {
  const uint32_t a = code2(v[0] * inverse, v[1] * inverse), b = code2(v[2] * inverse, v[3] * inverse);
  const uint32_t c = code2(v[4] * inverse, v[5] * inverse), d = code2(v[6] * inverse, v[7] * inverse);
  return make_uint2(a | b << 16, c | d << 16);
}
// The values of the two codes in the low half of w.
__device__ __forceinline__ float2 values2(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xffff), __NV_E4M3);   // exact
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Largest magnitude over the 16 lanes of a half warp.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t top) {
#pragma unroll
  for (int d = 8; d; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  return top;
}

}  // namespace tgb
