// Row kernels of the 8-bit row operators: quantisation, the root-mean-square
// norm with the residual's addition, its backward, and column sums.
//
// All are bound by memory.  A row of up to 16384 columns is read once, kept in
// registers between the statistics and the output, and written once; the norm
// reads its weights again for the output, from L1 (norm_stream_kernel keeps them).
// Longer rows are read two or three times, the later ones mostly from L2
// (2048 x 53248 bf16: quantise 186 us, 1.8 TB/s; norm with checkpoint 540).
#include <algorithm>
#include "tg_rows8.cuh"

namespace tg8 {

struct RowArgs {
  int64_t rows, cols;
  const void *x, *residual, *weight;
  void* h;
  int8_t *q, *ckpt;
  float *scale, *ckpt_scale, *rstd;
  int64_t ldx, ldr, ldh, ldq, ldk;
  float eps;
  int tpr;   // threads per row: 32 .. 1024
};

struct RowStats {
  float sum;        // of h^2
  uint32_t top_y;   // bit patterns of the largest |h * weight| ...
  uint32_t top_h;   // ... and |h|
};

__device__ __forceinline__ RowStats row_reduce(RowStats s, int tpr, RowStats* warp_stats) {
#pragma unroll
  for (int d = 16; d; d >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, d);
  s.top_y = __reduce_max_sync(0xffffffffu, s.top_y);
  s.top_h = __reduce_max_sync(0xffffffffu, s.top_h);
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, first = (threadIdx.x / tpr) * (tpr >> 5);
    __syncthreads();   // the last use of warp_stats is over
    if ((threadIdx.x & 31) == 0) warp_stats[warp] = s;
    __syncthreads();
    s = warp_stats[first];
    for (int w = 1; w < tpr >> 5; w++) {   // the same order in every thread
      const RowStats o = warp_stats[first + w];
      s.sum += o.sum;
      s.top_y = max(s.top_y, o.top_y);
      s.top_h = max(s.top_h, o.top_h);
    }
  }
  return s;
}

__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// One row per tpr threads, G groups of 8 elements per thread held in f32
// registers.  NORM: root-mean-square norm (and the checkpoint when asked for);
// otherwise the plain quantisation.
template <typename T, int G, int ACCESS, bool NORM>
__global__ void __launch_bounds__(G == 1 ? 1024 : 512) rows_kernel(RowArgs p) {
  __shared__ RowStats warp_stats[32];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int64_t row = int64_t(blockIdx.x) * per_block + sub;
  const bool live = row < p.rows;
  const T* x = static_cast<const T*>(p.x) + (live ? row : 0) * p.ldx;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + (live ? row : 0) * p.ldr : nullptr;
  const T* wgt = static_cast<const T*>(p.weight);
  const int cols = int(p.cols), shift = ACCESS == kShifted ? row_shift(x) : 0;
  auto at = [&](int g, int e) { return ACCESS == kScalar ? (g * 8 + e) * p.tpr + t : (g * p.tpr + t) * 8 + e - shift; };
  auto inside = [&](int g, int e) { return at(g, e) < cols && (ACCESS != kShifted || at(g, e) >= 0); };

  float v[G][8];
  if constexpr (ACCESS != kScalar) {
    Vec8<T> a[G], b[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
      a[g].zero();
      b[g].zero();
      if (live) load_group<ACCESS>(a[g], x, at(g, 0), cols);
      if (NORM && res && live) load_group<ACCESS>(b[g], res, at(g, 0), cols);
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      float r[8];
      a[g].get(v[g]);
      b[g].get(r);
      if (NORM && res) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[g][e] += r[e];
      }
      mask_group<ACCESS>(v[g], at(g, 0), cols);
    }
  } else {
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int c = at(g, e);
        const bool in = live && c < cols;
        v[g][e] = in ? to_f32(x[c]) : 0.f;
        if (NORM && res && in) v[g][e] += to_f32(res[c]);
      }
  }

  auto weight_of = [&](int g, float (&w)[8]) {
    if constexpr (ACCESS == kAligned) {
      Vec8<T> a;
      load_group<ACCESS>(a, wgt, at(g, 0), cols);
      a.get(w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = inside(g, e) ? to_f32(wgt[at(g, e)]) : 0.f;
    }
  };

  RowStats s{0.f, 0u, 0u};
  float top_h = 0.f, top_y = 0.f;
#pragma unroll
  for (int g = 0; g < G; g++) {
    float w[8];
    if (NORM) weight_of(g, w);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      top_h = mag_max(v[g][e], v[g][e + 1], top_h);
      if (NORM) {
        s.sum = fmaf(v[g][e], v[g][e], s.sum);
        s.sum = fmaf(v[g][e + 1], v[g][e + 1], s.sum);
        top_y = mag_max(v[g][e] * w[e], v[g][e + 1] * w[e + 1], top_y);
      }
    }
  }
  s.top_h = __float_as_uint(top_h);
  s.top_y = __float_as_uint(top_y);
  s = row_reduce(s, p.tpr, warp_stats);

  float u = 1.f;
  Quant qy;
  if (NORM) {
    u = 1.f / sqrtf(s.sum / float(cols) + p.eps);
    uint32_t top = mag_bits(__uint_as_float(s.top_y) * u);
    // max|h * w| * u stands for max|(h * u) * w| unless h * w left f32's range
    const bool redo = NORM && !(__uint_as_float(s.top_y) > 1e-25f && __uint_as_float(s.top_y) < 1e25f);
    if (__syncthreads_or(redo)) {   // rare: zero rows, tiny or huge values
      RowStats r{0.f, 0u, 0u};
#pragma unroll
      for (int g = 0; g < G; g++) {
        float w[8];
        weight_of(g, w);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if (inside(g, e)) r.top_y = max(r.top_y, mag_bits(v[g][e] * u * w[e]));
        }
      }
      r = row_reduce(r, p.tpr, warp_stats);
      if (redo) top = r.top_y;
    }
    qy = quant_of(top);
  } else {
    qy = quant_of(s.top_h);
  }
  if (!live) return;

  const Quant qh = quant_of(s.top_h);
  T* h = static_cast<T*>(p.h) + row * p.ldh;
  int8_t* q = p.q + row * p.ldq;
  int8_t* k = p.ckpt ? p.ckpt + row * p.ldk : nullptr;
  if (t == 0) {
    p.scale[row] = qy.scale;
    if (NORM && k) {
      p.ckpt_scale[row] = qh.scale;
      p.rstd[row] = u;
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++) {
    float w[8], y[8];
    if (NORM) weight_of(g, w);
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = NORM ? v[g][e] * u * w[e] : v[g][e];
    if constexpr (ACCESS != kScalar) {
      const int c = at(g, 0);
      store_bytes<ACCESS>(q, c, cols, quant_pack8(y, qy));
      if (NORM && k) store_bytes<ACCESS>(k, c, cols, quant_pack8(v[g], qh));
      if (NORM && p.h) store_group<ACCESS>(h, c, cols, v[g]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int c = at(g, e);
        if (c < cols) {
          q[c] = int8_t(quant8(y[e], qy));
          if (NORM && k) k[c] = int8_t(quant8(v[g][e], qh));
          if (NORM && p.h) h[c] = from_f32<T>(v[g][e]);
        }
      }
    }
  }
}

// Sums and maxima over the tpr threads of a row: one named barrier per row, two
// sets of partial results in turn.  The order is the same in every thread.
struct RowJoin {
  float4 (*stats)[16];   // [2][warps of the block]
  int tpr, sub, turn;
  __device__ __forceinline__ void barrier() const { asm volatile("bar.sync %0, %1;" ::"r"(sub + 1), "r"(tpr) : "memory"); }
  __device__ __forceinline__ RowStats operator()(RowStats s) {
#pragma unroll
    for (int d = 16; d; d >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, d);
    s.top_y = __reduce_max_sync(0xffffffffu, s.top_y);
    s.top_h = __reduce_max_sync(0xffffffffu, s.top_h);
    if (tpr > 32) {
      const int lane = threadIdx.x & 31, warps = tpr >> 5, first = sub * warps;
      if (lane == 0) stats[turn][threadIdx.x >> 5] = make_float4(s.sum, __uint_as_float(s.top_y), __uint_as_float(s.top_h), 0.f);
      barrier();
      const float4 o = stats[turn][first + (lane & (warps - 1))];
      turn ^= 1;
      s.sum = o.x;
      for (int d = warps >> 1; d; d >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, d);
      s.top_y = __reduce_max_sync(0xffffffffu, __float_as_uint(o.y));
      s.top_h = __reduce_max_sync(0xffffffffu, __float_as_uint(o.z));
    }
    return s;
  }
};

// The norm for many aligned rows: persistent, tpr threads per row with a fixed
// set of columns each, so the weights stay in registers as f32, and the next
// row is on its way while this one is worked on.  The kernel above is bound by
// instructions (78 % of the issue slots for 4096 x 8192 bf16, weights unpacked
// twice per row); this one needs about half of them.
// Rows that start anywhere would take their weights from shared memory and are
// slower so (16384 x 4001 bf16: 169 us, one row per block 137).
template <typename T, int G>
__global__ void __launch_bounds__(512) norm_stream_kernel(RowArgs p) {
  __shared__ float4 stats[2][16];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int cols = int(p.cols);
  auto at = [&](int g) { return (g * p.tpr + t) * 8; };
  RowJoin join{stats, p.tpr, sub, 0};
  float w[G][8];
  Vec8<T> nx[G], nr[G];
  const T *x = static_cast<const T*>(p.x), *res = static_cast<const T*>(p.residual);
#pragma unroll
  for (int g = 0; g < G; g++) {
    load_group<kAligned>(nx[g], static_cast<const T*>(p.weight), at(g), cols);
    nx[g].get(w[g]);
  }
  auto load = [&](int64_t row) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      load_group<kAligned>(nx[g], x + row * p.ldx, at(g), cols);
      if (res) load_group<kAligned>(nr[g], res + row * p.ldr, at(g), cols);
    }
  };
  const int64_t stride = int64_t(gridDim.x) * per_block;
  int64_t row = int64_t(blockIdx.x) * per_block + sub;
  if (row < p.rows) load(row);
  for (; row < p.rows; row += stride) {
    float v[G][8];
    RowStats s{0.f, 0u, 0u};
    float top_h = 0.f, top_y = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) {
      float r[8];
      nx[g].get(v[g]);
      if (res) {
        nr[g].get(r);
#pragma unroll
        for (int e = 0; e < 8; e++) v[g][e] += r[e];
      }
    }
    if (row + stride < p.rows) load(row + stride);
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        top_h = mag_max(v[g][e], v[g][e + 1], top_h);
        s.sum = fmaf(v[g][e], v[g][e], s.sum);
        s.sum = fmaf(v[g][e + 1], v[g][e + 1], s.sum);
        top_y = mag_max(v[g][e] * w[g][e], v[g][e + 1] * w[g][e + 1], top_y);
      }
    s.top_h = __float_as_uint(top_h);
    s.top_y = __float_as_uint(top_y);
    s = join(s);
    const float u = 1.f / sqrtf(s.sum / float(cols) + p.eps);
    const Quant qh = quant_of(s.top_h);
    // y = (h * weight) * u, so y / scale = (h * weight) * (127 / max|h * weight|),
    // unless the product left f32's comfortable range
    Quant qy;
    const bool redo = !(__uint_as_float(s.top_y) > 1e-25f && __uint_as_float(s.top_y) < 1e25f);
    if (redo) {   // uniform over the row's threads; zero rows, tiny or huge values
      RowStats r{0.f, 0u, 0u};
#pragma unroll
      for (int g = 0; g < G; g++)
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (at(g) < cols) r.top_y = max(r.top_y, mag_bits(v[g][e] * u * w[g][e]));
      qy = quant_of(join(r).top_y);
    } else {
      qy = quant_of(s.top_y);
      qy.scale = quant_of(mag_bits(__uint_as_float(s.top_y) * u)).scale;
    }
    if (t == 0) {
      p.scale[row] = qy.scale;
      if (p.ckpt) {
        p.ckpt_scale[row] = qh.scale;
        p.rstd[row] = u;
      }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int c = at(g);
      if (c >= cols) continue;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = redo ? v[g][e] * u * w[g][e] : v[g][e] * w[g][e];
      store_bytes<kAligned>(p.q + row * p.ldq, c, cols, quant_pack8(y, qy));
      if (p.ckpt) store_bytes<kAligned>(p.ckpt + row * p.ldk, c, cols, quant_pack8(v[g], qh));
      if (p.h) store_group<kAligned>(static_cast<T*>(p.h) + row * p.ldh, c, cols, v[g]);
    }
  }
}

// Rows too long for registers: one block per row, the row read three times
// (the second and third mostly from L2).
template <typename T, bool NORM>
__global__ void __launch_bounds__(1024) rows_long_kernel(RowArgs p) {
  __shared__ RowStats warp_stats[32];
  after_previous_kernel();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
  const T* wgt = static_cast<const T*>(p.weight);
  auto value = [&](int64_t c) { return to_f32(x[c]) + (NORM && res ? to_f32(res[c]) : 0.f); };
  RowStats s{0.f, 0u, 0u};
  for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float v = value(c);
    s.sum = fmaf(v, v, s.sum);
    s.top_h = max(s.top_h, mag_bits(v));
  }
  s = row_reduce(s, blockDim.x, warp_stats);
  float u = 1.f;
  Quant qy = quant_of(s.top_h);
  const Quant qh = qy;
  if (NORM) {
    u = 1.f / sqrtf(s.sum / float(p.cols) + p.eps);
    RowStats r{0.f, 0u, 0u};
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) r.top_y = max(r.top_y, mag_bits(value(c) * u * to_f32(wgt[c])));
    r = row_reduce(r, blockDim.x, warp_stats);
    qy = quant_of(r.top_y);
  }
  if (threadIdx.x == 0) {
    p.scale[row] = qy.scale;
    if (NORM && p.ckpt) {
      p.ckpt_scale[row] = qh.scale;
      p.rstd[row] = u;
    }
  }
  for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
    const float v = value(c);
    p.q[row * p.ldq + c] = int8_t(quant8(NORM ? v * u * to_f32(wgt[c]) : v, qy));
    if (NORM && p.ckpt) p.ckpt[row * p.ldk + c] = int8_t(quant8(v, qh));
    if (NORM && p.h) static_cast<T*>(p.h)[row * p.ldh + c] = from_f32<T>(v);
  }
}

// y = q * scale: 16 elements per thread, a shifted group of 8, or one.
template <typename T, int ACCESS>
__global__ void __launch_bounds__(256) dequantize_kernel(int64_t rows, int64_t cols, int64_t per, const int8_t* q, int64_t ldq,
                                                         const float* scale, T* y, int64_t ldy) {
  after_previous_kernel();
  const int64_t total = rows * per;
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t row = total <= 0xffffffffll ? int64_t(uint32_t(i) / uint32_t(per)) : i / per;
  const int64_t c = i - row * per;
  const float s = scale[row];
  float v[8];
  if constexpr (ACCESS == kAligned) {
    const uint4 w = *reinterpret_cast<const uint4*>(q + row * ldq + c * 16);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      bytes_f32(h ? make_uint2(w.z, w.w) : make_uint2(w.x, w.y), v);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= s;
      store8(y + row * ldy + c * 16 + h * 8, v);
    }
  } else if constexpr (ACCESS == kShifted) {
    const int first = int(c * 8) - row_shift(y + row * ldy);
    bytes_f32(load_bytes(q + row * ldq, first, int(cols)), v);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] *= s;
    store_group<ACCESS>(y + row * ldy, first, int(cols), v);
  } else {
    y[row * ldy + c] = from_f32<T>(float(q[row * ldq + c]) * s);
  }
}

// ------------------------------------------------------------------ backward
struct BackArgs {
  int64_t rows, cols;
  const void *grad, *grad_h, *weight;
  const int8_t* ckpt;
  const float *ckpt_scale, *rstd;
  void* grad_x;
  float* partial;   // (slots x cols) sums of grad * v over a slot's rows, or null
  int64_t ldg, ldgh, ldk, ldx;
  int tpr;
  int64_t slots;    // row groups running side by side; slot s takes rows s, s + slots, ...
};

__device__ __forceinline__ float row_sum(float s, int tpr, float* warp_sums) {
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (tpr > 32) {
    const int warp = threadIdx.x >> 5, first = (threadIdx.x / tpr) * (tpr >> 5);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warp_sums[warp] = s;
    __syncthreads();
    s = warp_sums[first];
    for (int w = 1; w < tpr >> 5; w++) s += warp_sums[first + w];
  }
  return s;
}

// What one thread reads of a row, as loaded; the columns are at(group, element).
template <typename T, typename GT, int G, int ACCESS> struct BackRow {
  Vec8<GT> grad[G];
  Vec8<T> gh[G];
  uint2 q[G];
  float u, s;
  int shift;
  __device__ __forceinline__ void load(const BackArgs& p, int64_t row, int t) {
    u = p.rstd[row];
    s = p.ckpt_scale[row];
    const GT* g = static_cast<const GT*>(p.grad) + row * p.ldg;
    const T* h = p.grad_h ? static_cast<const T*>(p.grad_h) + row * p.ldgh : nullptr;
    const int8_t* k = p.ckpt + row * p.ldk;
    const int cols = int(p.cols);
    shift = ACCESS == kShifted ? row_shift(g) : 0;
#pragma unroll
    for (int i = 0; i < G; i++) {
      const int c = (i * p.tpr + t) * 8 - shift;
      load_group<ACCESS>(grad[i], g, c, cols);
      q[i] = load_bytes(k, c, cols);
      if (h) load_group<ACCESS>(gh[i], h, c, cols); else gh[i].zero();
    }
  }
  __device__ __forceinline__ void get(int i, float (&g)[8], float (&v)[8]) const {
    grad[i].get(g);
    bytes_f32(q[i], v);
  }
  __device__ __forceinline__ void get_h(int i, float (&h)[8]) const { gh[i].get(h); }
};
template <typename T, typename GT, int G> struct BackRow<T, GT, G, kScalar> {
  GT grad[G][8];
  T gh[G][8];
  int8_t q[G][8];
  float u, s;
  static constexpr int shift = 0;
  __device__ __forceinline__ void load(const BackArgs& p, int64_t row, int t) {
    u = p.rstd[row];
    s = p.ckpt_scale[row];
#pragma unroll
    for (int i = 0; i < G; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int c = (i * 8 + e) * p.tpr + t;
        const bool in = c < p.cols;
        grad[i][e] = in ? static_cast<const GT*>(p.grad)[row * p.ldg + c] : from_f32<GT>(0.f);
        q[i][e] = in ? p.ckpt[row * p.ldk + c] : int8_t(0);
        gh[i][e] = in && p.grad_h ? static_cast<const T*>(p.grad_h)[row * p.ldgh + c] : from_f32<T>(0.f);
      }
  }
  __device__ __forceinline__ void get(int i, float (&g)[8], float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; e++) { g[e] = to_f32(grad[i][e]); v[e] = float(q[i][e]); }
  }
  __device__ __forceinline__ void get_h(int i, float (&h)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; e++) h[e] = to_f32(gh[i][e]);
  }
};

// Each slot (tpr threads) walks its rows; the sums over its rows stay with it
// and are joined by column_join_kernel in a fixed order.  A thread has a fixed
// set of columns and keeps their sums in registers, except where rows start
// anywhere: there sums and weights are in shared memory (a column has one
// thread per row, and a barrier lies between rows).  The next row is loaded
// before this one's sum is joined, so a row is always on its way.
template <typename T, typename GT, int G, int ACCESS>
__global__ void __launch_bounds__(512) norm_backward_kernel(BackArgs p) {
  constexpr bool kShift = ACCESS == kShifted;
  extern __shared__ float shared_cols[];   // kShifted: the weights, then a slot's sums each
  __shared__ float4 stats[2][16];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int cols = int(p.cols);
  const T* wgt = static_cast<const T*>(p.weight);
  auto at = [&](int g, int e, int shift) { return ACCESS == kScalar ? (g * 8 + e) * p.tpr + t : (g * p.tpr + t) * 8 + e - shift; };
  RowJoin join{stats, p.tpr, sub, 0};
  float* sums = shared_cols + (1 + sub) * (padded_bytes(cols) / 4);
  if constexpr (kShift) {
    for (int c = int(threadIdx.x) - 8; c < cols + 8; c += blockDim.x) shared_cols[padded_at(c)] = c >= 0 && c < cols ? to_f32(wgt[c]) : 0.f;
    for (int c = t; c < cols; c += p.tpr) sums[padded_at(c)] = 0.f;
    __syncthreads();
  }
  // what fits the registers: the next row (up to 16 elements per thread), and
  // the weights as f32 beside 16-bit rows; else the weights come from L1
  constexpr bool kAhead = G <= 2 && ACCESS != kScalar, kHold = G <= 2 && sizeof(T) == 2 && ACCESS == kAligned;
  float dw[kShift ? 1 : G][8] = {}, held[kHold ? G : 1][8];
  auto weight_of = [&](int i, int shift, float (&w)[8]) {
    if constexpr (ACCESS == kAligned) {
      Vec8<T> a;
      load_group<ACCESS>(a, wgt, at(i, 0, 0), cols);
      a.get(w);
    } else if constexpr (kShift) {
      const float* from = shared_cols + padded_at(at(i, 0, shift));
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = at(i, 0, shift) < cols ? from[padded_offset(shift, e)] : 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) w[e] = at(i, e, 0) < cols ? to_f32(wgt[at(i, e, 0)]) : 0.f;
    }
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < G; i++) weight_of(i, 0, held[i]);
  }
  const float inv_cols = 1.f / float(cols);
  const int64_t slot = int64_t(blockIdx.x) * per_block + sub;
  BackRow<T, GT, G, ACCESS> next;
  int64_t row = slot;
  if (kAhead && row < p.rows) next.load(p, row, t);
  for (; row < p.rows; row += p.slots) {
    if (!kAhead) next.load(p, row, t);
    float gw[G][8], v[G][8];
    const BackRow<T, GT, G, ACCESS> cur = next;   // of which grad_h is needed below
    const float u = cur.u, s = cur.s * u;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < G; i++) {
      float g[8], w[8];
      cur.get(i, g, v[i]);
      if constexpr (!kHold) weight_of(i, cur.shift, w);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int c = at(i, ACCESS == kAligned ? 0 : e, cur.shift);
        gw[i][e] = 0.f;
        if (c < cols && (!kShift || c >= 0)) {   // a NaN scale must not reach columns that are not there
          v[i][e] *= s;
          if (kShift) sums[padded_at(at(i, 0, cur.shift)) + padded_offset(cur.shift, e)] += g[e] * v[i][e];
          else dw[kShift ? 0 : i][e] = fmaf(g[e], v[i][e], dw[kShift ? 0 : i][e]);
          gw[i][e] = g[e] * (kHold ? held[kHold ? i : 0][e] : w[e]);
          dot = fmaf(gw[i][e], v[i][e], dot);
        }
      }
    }
    if (kAhead && row + p.slots < p.rows) next.load(p, row + p.slots, t);
    if (!p.grad_x && !kShift) continue;   // uniform over the grid
    const float mean = join(RowStats{dot, 0u, 0u}).sum * inv_cols;   // kShifted: also the barrier between rows' sums
    if (kShift) __syncwarp();
    if (!p.grad_x) continue;
    T* out = static_cast<T*>(p.grad_x) + row * p.ldx;
#pragma unroll
    for (int i = 0; i < G; i++) {
      float o[8], h[8];
      cur.get_h(i, h);
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = fmaf(u, fmaf(-mean, v[i][e], gw[i][e]), h[e]);
      if constexpr (ACCESS != kScalar) {
        store_group<ACCESS>(out, at(i, 0, cur.shift), cols, o);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (at(i, e, 0) < cols) out[at(i, e, 0)] = from_f32<T>(o[e]);
      }
    }
  }
  if (p.partial && slot < p.slots) {
    float* o = p.partial + slot * p.cols;
    if constexpr (kShift) {
      join(RowStats{0.f, 0u, 0u});   // the last row's sums are complete
      __syncwarp();
      for (int c = t; c < cols; c += p.tpr) o[c] = sums[padded_at(c)];
    } else {
#pragma unroll
      for (int i = 0; i < G; i++) {
        if constexpr (ACCESS == kAligned) {
          if (at(i, 0, 0) < cols) store8(o + at(i, 0, 0), dw[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (at(i, e, 0) < cols) o[at(i, e, 0)] = dw[i][e];
        }
      }
    }
  }
}

// Rows too long for registers, grad_x: one block per row.
template <typename T, typename GT>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(BackArgs p) {
  __shared__ float warp_sums[32];
  after_previous_kernel();
  const int64_t row = blockIdx.x;
  const float u = p.rstd[row], s = p.ckpt_scale[row] * u;
  const GT* grad = static_cast<const GT*>(p.grad) + row * p.ldg;
  const int8_t* k = p.ckpt + row * p.ldk;
  const T* wgt = static_cast<const T*>(p.weight);
  float dot = 0.f;
  for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) dot = fmaf(to_f32(grad[c]) * to_f32(wgt[c]), float(k[c]) * s, dot);
  const float c_mean = row_sum(dot, blockDim.x, warp_sums) / float(p.cols);
  for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
    float o = u * (to_f32(grad[c]) * to_f32(wgt[c]) - float(k[c]) * s * c_mean);
    if (p.grad_h) o += to_f32(static_cast<const T*>(p.grad_h)[row * p.ldgh + c]);
    static_cast<T*>(p.grad_x)[row * p.ldx + c] = from_f32<T>(o);
  }
}

// Partial column sums, one thread per column, slot blockIdx.y takes rows
// y, y + slots, ...: sum of x (ckpt null) or of x * v (the norm's weight).
template <typename GT>
__global__ void __launch_bounds__(256) column_partial_kernel(int64_t rows, int64_t cols, const GT* x, int64_t ldx,
                                                             const int8_t* ckpt, int64_t ldk, const float* ckpt_scale,
                                                             const float* rstd, float* partial) {
  after_previous_kernel();
  const int64_t c = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = to_f32(x[r * ldx + c]);
    s = ckpt ? fmaf(g, float(ckpt[r * ldk + c]) * (ckpt_scale[r] * rstd[r]), s) : s + g;
  }
  partial[int64_t(blockIdx.y) * cols + c] = s;
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

using tg8::BackArgs;
using tg8::RowArgs;

constexpr int64_t kRowLimit = 16384;   // longest row kept in registers
constexpr int64_t kGridLimit = 0x7fffffff;

// Threads per row and groups of 8 elements per thread (1, 2 or 4), for rows of
// at most kRowLimit: as few threads as max_groups allows (more loads in
// flight per thread, cheaper sums) when there are rows enough to fill the GPU;
// one group per thread when there are not, and latency counts.  Threads are a
// power of two (RowJoin), or a multiple of `step`.
struct RowShape {
  int tpr, groups, block;
};
RowShape row_shape(int64_t rows, int64_t cols, int max_groups, int max_threads, int step = 0) {
  const int64_t groups = (cols + 7) / 8;
  int g = rows >= 2 * sm_count() ? max_groups : 1;
  while (groups > int64_t(g) * (g == 1 ? max_threads : 512)) g *= 2;
  int tpr = 32;
  while (int64_t(tpr) * g < groups) tpr *= 2;
  while (g > 1 && int64_t(tpr) * (g / 2) >= groups) g /= 2;
  if (step) tpr = std::max(step, int(((groups + g - 1) / g + step - 1) / step * step));
  return {tpr, g, tpr >= 128 ? tpr : 128 / tpr * tpr};
}

template <typename F> void with_access(int access, F&& f) {
  if (access == tg8::kAligned) f(std::integral_constant<int, tg8::kAligned>{});
  else if (access == tg8::kShifted) f(std::integral_constant<int, tg8::kShifted>{});
  else f(std::integral_constant<int, tg8::kScalar>{});
}

template <typename T, bool NORM>
tg_status launch_rows(RowArgs p, int access, cudaStream_t st) {
  if (p.cols > kRowLimit) {
    if (p.rows > kGridLimit) return fail(TG_ERR_UNSUPPORTED, "%lld rows", (long long)p.rows);
    launch_kernel(tg8::rows_long_kernel<T, NORM>, unsigned(p.rows), 1024, 0, 0, st, p);
    return check_launch("rows8");
  }
  if constexpr (NORM) {
    // many aligned rows: persistent, 32 elements per thread (f32: 16, which
    // holds 8192 columns).  8192 x 8192 bf16 with the checkpoint: 99 us, one
    // row per block 124.  The plain quantisation has no weights to keep and
    // gains nothing (46 us either way).
    constexpr int kGroups = sizeof(T) == 4 ? 2 : 4;
    if (access == tg8::kAligned && p.rows >= 4 * int64_t(sm_count()) && p.cols <= 512 * 8 * kGroups) {
      const RowShape s = row_shape(p.rows, p.cols, kGroups, 512);
      p.tpr = s.tpr;
      const int per = s.block / s.tpr;
      const int64_t blocks = std::min<int64_t>((p.rows + per - 1) / per, int64_t(sm_count()) * (512 / s.block));
      if (s.groups == 1) launch_kernel(tg8::norm_stream_kernel<T, 1>, unsigned(blocks), s.block, 0, 0, st, p);
      else if (s.groups == 2) launch_kernel(tg8::norm_stream_kernel<T, 2>, unsigned(blocks), s.block, 0, 0, st, p);
      else launch_kernel(tg8::norm_stream_kernel<T, kGroups>, unsigned(blocks), s.block, 0, 0, st, p);
      return check_launch("rows8");
    }
  }
  if (access == tg8::kShifted && p.cols + 7 > kRowLimit) access = tg8::kScalar;
  // a shifted row may need a group more
  const RowShape s = row_shape(p.rows, p.cols + (access == tg8::kShifted ? 7 : 0), 4, 1024, 32);
  p.tpr = s.tpr;
  const int per = s.block / s.tpr;
  const int64_t grid = (p.rows + per - 1) / per;
  if (grid > kGridLimit) return fail(TG_ERR_UNSUPPORTED, "%lld rows", (long long)p.rows);
  auto go = [&](auto access_c) {
    constexpr int V = decltype(access_c)::value;
    if (s.groups == 1) launch_kernel(tg8::rows_kernel<T, 1, V, NORM>, unsigned(grid), s.block, 0, 0, st, p);
    else if (s.groups == 2) launch_kernel(tg8::rows_kernel<T, 2, V, NORM>, unsigned(grid), s.block, 0, 0, st, p);
    else launch_kernel(tg8::rows_kernel<T, 4, V, NORM>, unsigned(grid), s.block, 0, 0, st, p);
  };
  with_access(access, go);
  return check_launch("rows8");
}

template <typename T, typename GT>
tg_status launch_norm_backward(BackArgs p, T* grad_w, int access, cudaStream_t st) {
  const bool lng = p.cols > kRowLimit;
  if (access == tg8::kShifted && p.cols + 7 > kRowLimit) access = tg8::kScalar;
  RowShape s = lng ? RowShape{1024, 4, 1024} : row_shape(p.rows, p.cols + (access == tg8::kShifted ? 7 : 0), 2, 512);
  const int per = s.block / s.tpr;
  p.tpr = s.tpr;
  // at most four slots per SM: each leaves a row of sums to be joined
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((p.rows + per - 1) / per, sm_count() * int64_t(std::max(1, std::min(4 / per, 1024 / s.block)))));
  p.slots = lng ? std::max<int64_t>(1, std::min<int64_t>(p.rows, 64)) : blocks * per;
  if (lng && p.rows > kGridLimit) return fail(TG_ERR_UNSUPPORTED, "%lld rows", (long long)p.rows);
  void* scratch = nullptr;
  if (grad_w) {
    const cudaError_t e = scratch_alloc(&scratch, size_t(p.slots) * size_t(p.cols) * sizeof(float), st);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "norm backward scratch: %s", cudaGetErrorString(e));
    p.partial = static_cast<float*>(scratch);
  }
  if (lng) {
    if (p.grad_x) launch_kernel(tg8::norm_backward_long_kernel<T, GT>, unsigned(p.rows), 1024, 0, 0, st, p);
    if (grad_w)
      launch_kernel(tg8::column_partial_kernel<GT>, dim3(unsigned((p.cols + 255) / 256), unsigned(p.slots)), 256, 0, 0, st, p.rows, p.cols, static_cast<const GT*>(p.grad), p.ldg, p.ckpt, p.ldk, p.ckpt_scale, p.rstd, p.partial);
  } else {
    tg_status sized = TG_OK;
    with_access(access, [&](auto access_c) {
      constexpr int A = decltype(access_c)::value;
      const size_t smem = A == tg8::kShifted ? size_t(1 + per) * tg8::padded_bytes(p.cols) : 0;
      auto run = [&](auto kern) {
        if (smem) sized = ensure_smem(reinterpret_cast<const void*>(kern), 2 * tg8::padded_bytes(kRowLimit));
        if (sized == TG_OK) launch_kernel(kern, unsigned(blocks), s.block, smem, 0, st, p);
      };
      if (s.groups == 1) run(tg8::norm_backward_kernel<T, GT, 1, A>);
      else if (s.groups == 2) run(tg8::norm_backward_kernel<T, GT, 2, A>);
      else run(tg8::norm_backward_kernel<T, GT, 4, A>);
    });
    if (sized != TG_OK) {
      if (scratch) scratch_free(scratch, st);
      return sized;
    }
  }
  tg_status r = check_launch("rows8 norm backward");
  if (grad_w) {
    if (r == TG_OK) {
      launch_kernel(tg8::column_join_kernel<T>, unsigned((p.cols + 31) / 32), 1024, 0, 0, st, p.slots, p.cols, p.partial, grad_w);
      r = check_launch("rows8 norm backward");
    }
    scratch_free(scratch, st);
  }
  return r;
}

tg_status check_rows(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (rows=%lld cols=%lld)", (long long)rows, (long long)cols);
  if (cols > kGridLimit) return fail(TG_ERR_UNSUPPORTED, "cols=%lld", (long long)cols);
  return TG_OK;
}
tg_status check_ld(const char* name, int64_t ld, int64_t cols) {
  if (ld < cols) return fail(TG_ERR_DIMENSION_MISMATCH, "%s=%lld < %lld", name, (long long)ld, (long long)cols);
  return TG_OK;
}
tg_status check_type8(tg_dtype t) {
  if (!elem8_size(t)) return fail(TG_ERR_INVALID_ARGUMENT, "8-bit rows need f32, f16 or bf16, got dtype %d", int(t));
  return TG_OK;
}

}  // namespace tgi

using namespace tgi;

#define TG8_CHECK(call)                 \
  do {                                  \
    const tg_status s_ = (call);        \
    if (s_ != TG_OK) return s_;         \
  } while (0)

extern "C" {

tg_status tg_rows8_quantize(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, int8_t* q,
                            int64_t ldq, float* scale, void* stream) {
  clear_error();
  TG8_CHECK(check_type8(dtype));
  TG8_CHECK(check_rows(rows, cols));
  if (rows == 0) return TG_OK;
  if (!scale || (cols && (!x || !q))) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG8_CHECK(check_ld("ldx", ldx, cols));
  TG8_CHECK(check_ld("ldq", ldq, cols));
  RowArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx; p.q = q; p.ldq = ldq; p.scale = scale;
  RowAccess access(cols);
  access.add(x, ldx, elem8_size(dtype));
  access.add(q, ldq, 1);
  return with_type8(dtype, [&](auto t) { return launch_rows<decltype(t), false>(p, access.get(), static_cast<cudaStream_t>(stream)); });
}

tg_status tg_rows8_dequantize(tg_dtype dtype, int64_t rows, int64_t cols, const int8_t* q, int64_t ldq,
                              const float* scale, void* y, int64_t ldy, void* stream) {
  clear_error();
  TG8_CHECK(check_type8(dtype));
  TG8_CHECK(check_rows(rows, cols));
  if (rows == 0 || cols == 0) return TG_OK;
  if (!q || !scale || !y) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG8_CHECK(check_ld("ldq", ldq, cols));
  TG8_CHECK(check_ld("ldy", ldy, cols));
  RowAccess access(cols);
  access.add(y, ldy, elem8_size(dtype));
  access.add(q, ldq, 1);
  int how = access.get();
  if (how == tg8::kAligned && (cols % 16 || ldq % 16 || !aligned(q, 16))) how = tg8::kShifted;   // by 8 elements, without edges
  if (how == tg8::kShifted && cols > kGridLimit - 32) how = tg8::kScalar;   // a shifted group counts its columns in 32 bits, to 22 past the row
  const int64_t per = how == tg8::kAligned ? cols / 16 : how == tg8::kShifted ? (cols + 7 + 7) / 8 : cols;
  if (rows > (kGridLimit * 256) / per) return fail(TG_ERR_UNSUPPORTED, "%lld x %lld elements", (long long)rows, (long long)cols);
  const unsigned grid = unsigned((rows * per + 255) / 256);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    with_access(how, [&](auto access_c) {
      launch_kernel(tg8::dequantize_kernel<T, decltype(access_c)::value>, grid, 256, 0, 0, st, rows, cols, per, q, ldq, scale, static_cast<T*>(y), ldy);
    });
    return check_launch("rows8 dequantize");
  });
}

tg_status tg_rows8_rmsnorm(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                           const void* residual, int64_t ldr, const void* weight, float eps, void* h, int64_t ldh,
                           int8_t* q, int64_t ldq, float* scale, int8_t* ckpt, int64_t ldk, float* ckpt_scale,
                           float* rstd, void* stream) {
  clear_error();
  TG8_CHECK(check_type8(dtype));
  TG8_CHECK(check_rows(rows, cols));
  if (!(eps >= 0.f)) return fail(TG_ERR_INVALID_ARGUMENT, "eps=%g is negative", double(eps));
  if ((ckpt != nullptr) != (ckpt_scale != nullptr) || (ckpt != nullptr) != (rstd != nullptr))
    return fail(TG_ERR_INVALID_ARGUMENT, "ckpt, ckpt_scale and rstd are given together or not at all");
  if (rows == 0 || cols == 0) {
    if (rows && (!scale || ckpt)) return fail(TG_ERR_INVALID_ARGUMENT, "a row of no columns has no norm");
    if (rows) {
      const cudaError_t e = cudaMemsetAsync(scale, 0, size_t(rows) * sizeof(float), static_cast<cudaStream_t>(stream));
      if (e != cudaSuccess) return fail(TG_ERR_CUDA, "memset: %s", cudaGetErrorString(e));
    }
    return TG_OK;
  }
  if (!x || !weight || !q || !scale) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG8_CHECK(check_ld("ldx", ldx, cols));
  if (residual) TG8_CHECK(check_ld("ldr", ldr, cols));
  if (h) TG8_CHECK(check_ld("ldh", ldh, cols));
  TG8_CHECK(check_ld("ldq", ldq, cols));
  if (ckpt) TG8_CHECK(check_ld("ldk", ldk, cols));
  RowArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx; p.residual = residual; p.ldr = ldr; p.weight = weight;
  p.eps = eps; p.h = h; p.ldh = ldh; p.q = q; p.ldq = ldq; p.scale = scale;
  p.ckpt = ckpt; p.ldk = ldk; p.ckpt_scale = ckpt_scale; p.rstd = rstd;
  const size_t e = elem8_size(dtype);
  RowAccess access(cols);
  access.add(x, ldx, e);
  access.add(residual, ldr, e);
  access.add(h, ldh, e);
  access.add(q, ldq, 1);
  access.add(ckpt, ldk, 1);
  const int how = access.get() == tg8::kAligned && !aligned(weight, 16) ? tg8::kScalar : access.get();
  return with_type8(dtype, [&](auto t) { return launch_rows<decltype(t), true>(p, how, static_cast<cudaStream_t>(stream)); });
}

tg_status tg_rows8_rmsnorm_backward(tg_dtype dtype, tg_dtype grad_dtype, int64_t rows, int64_t cols, const void* grad,
                                    int64_t ldg, const void* grad_h, int64_t ldgh, const void* weight,
                                    const int8_t* ckpt, int64_t ldk, const float* ckpt_scale, const float* rstd,
                                    void* grad_x, int64_t ldx, void* grad_weight, void* stream) {
  clear_error();
  TG8_CHECK(check_type8(dtype));
  if (grad_dtype != dtype && grad_dtype != TG_F32) return fail(TG_ERR_INVALID_ARGUMENT, "grad is of type dtype or f32, got dtype %d", int(grad_dtype));
  TG8_CHECK(check_rows(rows, cols));
  if (cols == 0 || (!grad_x && !grad_weight)) return TG_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {   // a sum of nothing; the operands, the weight among them, may be null
    const cudaError_t e = grad_weight ? cudaMemsetAsync(grad_weight, 0, size_t(cols) * elem8_size(dtype), st) : cudaSuccess;
    return e == cudaSuccess ? TG_OK : fail(TG_ERR_CUDA, "memset: %s", cudaGetErrorString(e));
  }
  if (!grad || !weight || !ckpt || !ckpt_scale || !rstd) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG8_CHECK(check_ld("ldg", ldg, cols));
  if (grad_h) TG8_CHECK(check_ld("ldgh", ldgh, cols));
  TG8_CHECK(check_ld("ldk", ldk, cols));
  if (grad_x) TG8_CHECK(check_ld("ldx", ldx, cols));
  BackArgs p{};
  p.rows = rows; p.cols = cols; p.grad = grad; p.ldg = ldg; p.grad_h = grad_h; p.ldgh = ldgh; p.weight = weight;
  p.ckpt = ckpt; p.ldk = ldk; p.ckpt_scale = ckpt_scale; p.rstd = rstd; p.grad_x = grad_x; p.ldx = ldx;
  const size_t e = elem8_size(dtype);
  RowAccess access(cols);
  access.add(grad, ldg, elem8_size(grad_dtype));
  access.add(grad_h, ldgh, e);
  access.add(ckpt, ldk, 1);
  access.add(grad_x, ldx, e);
  const int how = access.get() == tg8::kAligned && !aligned(weight, 16) ? tg8::kScalar : access.get();
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    if (grad_dtype == dtype) return launch_norm_backward<T, T>(p, static_cast<T*>(grad_weight), how, st);
    return launch_norm_backward<T, float>(p, static_cast<T*>(grad_weight), how, st);
  });
}

tg_status tg_rows8_column_sum(tg_dtype dtype, tg_dtype out_dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                              void* out, void* stream) {
  clear_error();
  TG8_CHECK(check_type8(dtype));
  TG8_CHECK(check_type8(out_dtype));
  TG8_CHECK(check_rows(rows, cols));
  if (cols == 0) return TG_OK;
  if (!out || (rows && !x)) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (rows) TG8_CHECK(check_ld("ldx", ldx, cols));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // enough slots to fill the GPU, no more than there are rows
  const int64_t strips = (cols + 255) / 256;
  const int64_t slots = std::max<int64_t>(1, std::min<int64_t>({rows, 1024, (8 * int64_t(sm_count()) + strips - 1) / strips}));
  void* scratch = nullptr;
  const cudaError_t e = scratch_alloc(&scratch, size_t(slots) * size_t(cols) * sizeof(float), st);
  if (e != cudaSuccess) return fail(TG_ERR_CUDA, "column sum scratch: %s", cudaGetErrorString(e));
  float* partial = static_cast<float*>(scratch);
  tg_status r = with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    launch_kernel(tg8::column_partial_kernel<T>, dim3(unsigned(strips), unsigned(slots)), 256, 0, 0, st, rows, cols, static_cast<const T*>(x), ldx, nullptr, 0, nullptr, nullptr, partial);
    return check_launch("rows8 column sum");
  });
  if (r == TG_OK)
    r = with_type8(out_dtype, [&](auto t) {
      using T = decltype(t);
      launch_kernel(tg8::column_join_kernel<T>, unsigned((cols + 31) / 32), 1024, 0, 0, st, slots, cols, partial, static_cast<T*>(out));
      return check_launch("rows8 column sum");
    });
  scratch_free(scratch, st);
  return r;
}

}  // extern "C"
