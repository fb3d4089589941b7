// Layer norm: forward (rows or 8-bit blocks out), backward with the gradients
// of weight and bias.
//
//   h = x + residual, u = (h - mean) rstd, y = u weight + bias
//   grad_x = rstd (a - mean(a) - u mean(a u)) + grad_h,  a = grad weight
//
// All are bound by memory: a row is read once, kept in registers between its
// sums and its output, and written once.
#include <algorithm>
#include "tg_blocks8.cuh"

namespace tgb {

struct NormArgs {
  int64_t rows, cols, slots;
  const void *x, *residual, *weight, *bias;
  void *h, *y;
  uint8_t* q;                 // the output in 8-bit blocks, in place of y
  float *scale, *mean, *rstd;
  int64_t ldx, ldr, ldh, ldy, ldq, scale_row, scale_block;
  float eps;
  int tpr;                    // threads per row: 32 .. 512, a power of two
};

// Two sums over the tpr threads of a row: one named barrier per row, two sets
// of partial results in turn.  The order is the same in every thread.
struct PairJoin {
  float2 (*sums)[16];   // [2][warps of the block]
  int tpr, sub, turn;
  __device__ __forceinline__ float2 operator()(float2 s) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, d);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, d);
    }
    if (tpr > 32) {
      const int lane = threadIdx.x & 31, warps = tpr >> 5, first = sub * warps;
      if (lane == 0) sums[turn][threadIdx.x >> 5] = s;
      asm volatile("bar.sync %0, %1;" ::"r"(sub + 1), "r"(tpr) : "memory");
      s = sums[turn][first + (lane & (warps - 1))];
      turn ^= 1;
      for (int d = warps >> 1; d; d >>= 1) {
        s.x += __shfl_xor_sync(0xffffffffu, s.x, d);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, d);
      }
    }
    return s;
  }
};

template <int ACCESS, typename T> __device__ __forceinline__ void load_at(Vec8<T>& v, const T* row, int c, int cols) {
  if constexpr (ACCESS == kScalar) load_any(v, row, c, cols);
  else load_group<ACCESS>(v, row, c, cols);
}
template <int ACCESS> __device__ __forceinline__ bool inside(int c, int e, int cols) {
  return ACCESS == kAligned ? c < cols : c + e < cols && (ACCESS == kScalar || c + e >= 0);
}
// Zeros for what a group holds of other rows.
template <int ACCESS> __device__ __forceinline__ void mask_at(float (&v)[8], int c, int cols) {
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (ACCESS != kAligned && !inside<ACCESS>(c, e, cols)) v[e] = 0.f;
}
template <int ACCESS, typename T> __device__ __forceinline__ void store_at(T* row, int c, int cols, const float (&v)[8]) {
  if constexpr (ACCESS == kScalar) store_any(row, c, cols, v);
  else store_group<ACCESS>(row, c, cols, v);
}
// A group of a vector over the columns (weight, bias), as it lies in memory.
template <int ACCESS, typename T> __device__ __forceinline__ void load_columns(Vec8<T>& v, const T* from, int c, int cols) {
  if constexpr (ACCESS == kAligned) {
    load_group<kAligned>(v, from, c, cols);
  } else {
    union { Vec8<T> v; T e[8]; } u;
#pragma unroll
    for (int e = 0; e < 8; e++) u.e[e] = inside<ACCESS>(c, e, cols) ? from[c + e] : from_f32<T>(0.f);
    v = u.v;
  }
}

// Mean and rstd from the row's mean (the sum's, rounded), the sum of h - mean and
// of its square: what the rounding of the first mean left is taken out again.
__device__ __forceinline__ float2 finish_stats(float mean, float2 off, float cols, float eps) {
  const float d = off.x / cols;
  float var = off.y / cols - d * d;
  if (var < 0.f) var = 0.f;   // a NaN stays
  return make_float2(mean + d, 1.f / sqrtf(var + eps));
}

// Codes and scale of eight outputs per lane, 16 lanes per block; c < 0 or past
// the row: no part in it.
__device__ __forceinline__ void store_block(const NormArgs& p, int64_t row, int64_t c, const float (&y)[8]) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 2)
    top = mag_max(c + e < p.cols ? y[e] : 0.f, c + e + 1 < p.cols ? y[e + 1] : 0.f, top);
  const Step s = step_of(half_warp_max(magnitude(top)));
  if (c >= p.cols) return;
  store_codes(p.q + row * p.ldq, c, p.cols, codes8(y, s.inverse));
  if ((c & (kBlock - 1)) == 0) p.scale[row * p.scale_row + c / kBlock * p.scale_block] = s.scale;
}

// tpr threads per row, G groups of 8 elements per thread.  A slot (tpr threads)
// walks rows slot, slot + slots, ..; its threads have fixed columns, so weight
// and bias stay in registers (rows that start anywhere: slots is a multiple of
// 8, so all rows of a slot start at the same distance from a boundary).  The
// next row is on its way while this one is worked on.
template <typename T, int G, int ACCESS, bool BLOCKS>
__global__ void __launch_bounds__(512) layernorm_kernel(const NormArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int cols = int(p.cols);
  int64_t row = int64_t(blockIdx.x) * per_block + sub;
  if (row >= p.rows || row >= p.slots) return;
  const T *x = static_cast<const T*>(p.x), *res = static_cast<const T*>(p.residual);
  const int shift = ACCESS == kShifted ? row_shift(x + row * p.ldx) : 0;
  auto at = [&](int g) { return (g * p.tpr + t) * 8 - shift; };
  PairJoin join{sums, p.tpr, sub, 0};
  Vec8<T> nx[G], nr[G], w[G], b[G];
  auto load = [&](int64_t r) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      load_at<ACCESS>(nx[g], x + r * p.ldx, at(g), cols);
      if (res) load_at<ACCESS>(nr[g], res + r * p.ldr, at(g), cols);
    }
  };
  load(row);
#pragma unroll
  for (int g = 0; g < G; g++) {
    if (p.weight) load_columns<ACCESS>(w[g], static_cast<const T*>(p.weight), at(g), cols);
    if (p.bias) load_columns<ACCESS>(b[g], static_cast<const T*>(p.bias), at(g), cols);
  }
  const float n = float(cols);
  for (; row < p.rows; row += p.slots) {
    float v[G][8], sum = 0.f;
#pragma unroll
    for (int g = 0; g < G; g++) {
      nx[g].get(v[g]);
      if (res) {
        float r[8];
        nr[g].get(r);
#pragma unroll
        for (int e = 0; e < 8; e++) v[g][e] += r[e];
      }
      mask_at<ACCESS>(v[g], at(g), cols);
    }
    if (row + p.slots < p.rows) load(row + p.slots);
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int e = 0; e < 8; e++) sum += v[g][e];
    const float rough = join(make_float2(sum, 0.f)).x / n;
    float2 off = make_float2(0.f, 0.f);
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = inside<ACCESS>(at(g), e, cols) ? v[g][e] - rough : 0.f;
        off.x += d;
        off.y = fmaf(d, d, off.y);
      }
    const float2 st = finish_stats(rough, join(off), n, p.eps);
    if (t == 0 && p.mean) {
      p.mean[row] = st.x;
      p.rstd[row] = st.y;
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int c = at(g);
      float y[8], k[8];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = (v[g][e] - st.x) * st.y;
      if (p.weight) {
        w[g].get(k);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] *= k[e];
      }
      if (p.bias) {
        b[g].get(k);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] += k[e];
      }
      if (p.h) store_at<ACCESS>(static_cast<T*>(p.h) + row * p.ldh, c, cols, v[g]);
      if constexpr (BLOCKS) store_block(p, row, c, y);
      else store_at<ACCESS>(static_cast<T*>(p.y) + row * p.ldy, c, cols, y);
    }
  }
}

// Rows too long for registers: one block per row, which reads it three times
// (the second and third from L2).
template <typename T, bool BLOCKS>
__global__ void __launch_bounds__(512) layernorm_long_kernel(const NormArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  PairJoin join{sums, 512, 0, 0};
  const float n = float(p.cols);
  const int64_t last = (p.cols + 511 * 8 + 7) / (512 * 8);   // turns of the block
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    auto load = [&](int64_t c, float (&v)[8]) {
      Vec8<T> a;
      load_any(a, x, c, p.cols);
      a.get(v);
      if (res) {
        float r[8];
        load_any(a, res, c, p.cols);
        a.get(r);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += r[e];
      }
    };
    float sum = 0.f;
    for (int64_t i = 0; i < last; i++) {
      const int64_t c = (i * 512 + threadIdx.x) * 8;
      float v[8];
      load(c, v);
#pragma unroll
      for (int e = 0; e < 8; e++) sum += c + e < p.cols ? v[e] : 0.f;
    }
    const float rough = join(make_float2(sum, 0.f)).x / n;
    float2 off = make_float2(0.f, 0.f);
    for (int64_t i = 0; i < last; i++) {
      const int64_t c = (i * 512 + threadIdx.x) * 8;
      float v[8];
      load(c, v);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = c + e < p.cols ? v[e] - rough : 0.f;
        off.x += d;
        off.y = fmaf(d, d, off.y);
      }
    }
    const float2 st = finish_stats(rough, join(off), n, p.eps);
    if (threadIdx.x == 0 && p.mean) {
      p.mean[row] = st.x;
      p.rstd[row] = st.y;
    }
    for (int64_t i = 0; i < last; i++) {
      const int64_t c = (i * 512 + threadIdx.x) * 8;
      float v[8], y[8];
      load(c, v);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool in = c + e < p.cols;
        y[e] = (v[e] - st.x) * st.y;
        if (p.weight) y[e] *= in ? to_f32(static_cast<const T*>(p.weight)[c + e]) : 0.f;
        if (p.bias) y[e] += in ? to_f32(static_cast<const T*>(p.bias)[c + e]) : 0.f;
      }
      if (p.h) store_any(static_cast<T*>(p.h) + row * p.ldh, c, p.cols, v);
      if constexpr (BLOCKS) store_block(p, row, c, y);
      else store_any(static_cast<T*>(p.y) + row * p.ldy, c, p.cols, y);
    }
  }
}

struct NormBackArgs {
  int64_t rows, cols, slots;
  const void *grad, *grad_h, *weight, *h;
  const float *mean, *rstd;
  void* grad_x;
  float *partial_w, *partial_b;   // (slots x cols), or null
  int64_t ldg, ldgh, ldh, ldx;
  int tpr;
};

// As layernorm_kernel; a thread also keeps its columns' sums of grad * u and of
// grad over the slot's rows, joined by column_join_kernel in a fixed order.
template <typename T, int G, int ACCESS>
__global__ void __launch_bounds__(512) layernorm_backward_kernel(const NormBackArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int cols = int(p.cols);
  const int64_t slot = int64_t(blockIdx.x) * per_block + sub;
  if (slot >= p.slots) return;
  const T *grad = static_cast<const T*>(p.grad), *h = static_cast<const T*>(p.h), *gh = static_cast<const T*>(p.grad_h);
  const int shift = ACCESS == kShifted ? row_shift(grad + slot * p.ldg) : 0;
  auto at = [&](int g) { return (g * p.tpr + t) * 8 - shift; };
  PairJoin join{sums, p.tpr, sub, 0};
  constexpr bool kAhead = G * sizeof(T) <= 4;   // the next row fits the registers
  Vec8<T> ng[G], nh[G], w[G];
  float2 ns;
  float dw[G][8] = {}, db[G][8] = {};
  auto load = [&](int64_t r) {
    ns = make_float2(p.mean[r], p.rstd[r]);
#pragma unroll
    for (int g = 0; g < G; g++) {
      load_at<ACCESS>(ng[g], grad + r * p.ldg, at(g), cols);
      load_at<ACCESS>(nh[g], h + r * p.ldh, at(g), cols);
    }
  };
  int64_t row = slot;
  if (kAhead && row < p.rows) load(row);
#pragma unroll
  for (int g = 0; g < G; g++)
    if (p.weight) load_columns<ACCESS>(w[g], static_cast<const T*>(p.weight), at(g), cols);
  const float n = float(cols);
  for (; row < p.rows; row += p.slots) {
    if (!kAhead) load(row);
    Vec8<T> ch[G];
    if (gh && p.grad_x) {
#pragma unroll
      for (int g = 0; g < G; g++) load_at<ACCESS>(ch[g], gh + row * p.ldgh, at(g), cols);
    }
    float a[G][8], u[G][8];
    const float2 st = ns;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int g = 0; g < G; g++) {
      ng[g].get(a[g]);
      nh[g].get(u[g]);
      float k[8];
      if (p.weight) w[g].get(k);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool in = inside<ACCESS>(at(g), e, cols);
        u[g][e] = in ? (u[g][e] - st.x) * st.y : 0.f;
        a[g][e] = in ? a[g][e] : 0.f;
        dw[g][e] = fmaf(a[g][e], u[g][e], dw[g][e]);
        db[g][e] += a[g][e];
        if (p.weight) a[g][e] *= k[e];
        if (ACCESS != kAligned && !in) a[g][e] = 0.f;
        s.x += a[g][e];
        s.y = fmaf(a[g][e], u[g][e], s.y);
      }
    }
    if (kAhead && row + p.slots < p.rows) load(row + p.slots);
    if (!p.grad_x) continue;
    s = join(s);
    s.x /= n;
    s.y /= n;
    T* out = static_cast<T*>(p.grad_x) + row * p.ldx;
#pragma unroll
    for (int g = 0; g < G; g++) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = st.y * (a[g][e] - s.x - u[g][e] * s.y);
      if (gh) {
        float k[8];
        ch[g].get(k);
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] += k[e];
      }
      store_at<ACCESS>(out, at(g), cols, o);
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int c = at(g);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (c + e < 0 || c + e >= cols) continue;
      if (p.partial_w) p.partial_w[slot * p.cols + c + e] = dw[g][e];
      if (p.partial_b) p.partial_b[slot * p.cols + c + e] = db[g][e];
    }
  }
}

// Rows too long for registers, grad_x: one block per row, read twice.
template <typename T>
__global__ void __launch_bounds__(512) layernorm_backward_long_kernel(const NormBackArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  PairJoin join{sums, 512, 0, 0};
  const float n = float(p.cols);
  const T* wgt = static_cast<const T*>(p.weight);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    const T *grad = static_cast<const T*>(p.grad) + row * p.ldg, *h = static_cast<const T*>(p.h) + row * p.ldh;
    const T* gh = p.grad_h ? static_cast<const T*>(p.grad_h) + row * p.ldgh : nullptr;
    auto load = [&](int64_t c, float (&a)[8], float (&u)[8]) {
      Vec8<T> v;
      load_any(v, grad, c, p.cols);
      v.get(a);
      load_any(v, h, c, p.cols);
      v.get(u);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool in = c + e < p.cols;
        u[e] = in ? (u[e] - mean) * rstd : 0.f;
        a[e] = !in ? 0.f : wgt ? a[e] * to_f32(wgt[c + e]) : a[e];
      }
    };
    float2 s = make_float2(0.f, 0.f);
    for (int64_t c = threadIdx.x * 8; c < p.cols; c += 512 * 8) {
      float a[8], u[8];
      load(c, a, u);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        s.x += a[e];
        s.y = fmaf(a[e], u[e], s.y);
      }
    }
    s = join(s);
    s.x /= n;
    s.y /= n;
    for (int64_t c = threadIdx.x * 8; c < p.cols; c += 512 * 8) {
      float a[8], u[8];
      load(c, a, u);
#pragma unroll
      for (int e = 0; e < 8; e++) a[e] = rstd * (a[e] - s.x - u[e] * s.y);
      if (gh) {
        Vec8<T> v;
        load_any(v, gh, c, p.cols);
        v.get(u);
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] += u[e];
      }
      store_any(static_cast<T*>(p.grad_x) + row * p.ldx, c, p.cols, a);
    }
  }
}

// The same rows' column sums: eight columns per thread, slot blockIdx.y takes
// rows y, y + slots, ..
template <typename T>
__global__ void __launch_bounds__(128) layernorm_columns_kernel(const NormBackArgs p) {
  after_previous_kernel();
  const int64_t c = (int64_t(blockIdx.x) * 128 + threadIdx.x) * 8;
  if (c >= p.cols) return;
  float dw[8] = {}, db[8] = {};
  for (int64_t row = blockIdx.y; row < p.rows; row += p.slots) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    Vec8<T> v;
    float a[8], u[8];
    load_any(v, static_cast<const T*>(p.grad) + row * p.ldg, c, p.cols);
    v.get(a);
    load_any(v, static_cast<const T*>(p.h) + row * p.ldh, c, p.cols);
    v.get(u);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      dw[e] = fmaf(a[e], (u[e] - mean) * rstd, dw[e]);
      db[e] += a[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; e++) {
    if (c + e >= p.cols) break;
    if (p.partial_w) p.partial_w[int64_t(blockIdx.y) * p.cols + c + e] = dw[e];
    if (p.partial_b) p.partial_b[int64_t(blockIdx.y) * p.cols + c + e] = db[e];
  }
}

}  // namespace tgb

namespace tgi {

using tgb::NormArgs;
using tgb::NormBackArgs;

namespace {

constexpr int64_t kColumnLimit = 0x7fffff00;

// Threads per row (a power of two) and groups of 8 per thread, at most
// `most`; `extra` elements may lie before a row's first group.
struct RowPlan {
  int tpr, groups, block;
  int64_t blocks, slots;
};
RowPlan row_plan(int64_t rows, int64_t cols, int access, int most, int per_sm) {
  const int64_t groups = (cols + (access == tg8::kShifted ? 7 : 0) + 7) / 8;
  RowPlan r;
  r.groups = rows >= 2 * int64_t(sm_count()) ? most : 1;
  while (groups > int64_t(r.groups) * 512) r.groups *= 2;
  r.tpr = 32;
  while (int64_t(r.tpr) * r.groups < groups) r.tpr *= 2;
  while (r.groups > 1 && int64_t(r.tpr) * (r.groups / 2) >= groups) r.groups /= 2;
  r.block = std::max(r.tpr, 128);
  const int per = r.block / r.tpr;
  r.blocks = std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, int64_t(sm_count()) * per_sm * std::max(1, 512 / r.block)));
  r.slots = r.blocks * per;
  if (access == tg8::kShifted && r.slots < rows) {   // a slot's rows start alike
    r.slots = std::max<int64_t>(8, r.slots / 8 * 8);
    r.blocks = (r.slots + per - 1) / per;
  }
  return r;
}
template <typename F> void with_groups(int groups, F&& f) {
  if (groups == 1) f(std::integral_constant<int, 1>{});
  else if (groups == 2) f(std::integral_constant<int, 2>{});
  else f(std::integral_constant<int, 4>{});
}
template <typename F> void with_mode(int access, F&& f) {
  if (access == tg8::kAligned) f(std::integral_constant<int, tg8::kAligned>{});
  else if (access == tg8::kShifted) f(std::integral_constant<int, tg8::kShifted>{});
  else f(std::integral_constant<int, tg8::kScalar>{});
}

template <typename T, bool BLOCKS> tg_status launch_norm(NormArgs p, int access, cudaStream_t st) {
  constexpr int kMost = sizeof(T) == 4 ? 2 : 4;
  if (p.cols + 7 > 512 * 8 * kMost) {
    launch_kernel(tgb::layernorm_long_kernel<T, BLOCKS>, unsigned(std::min<int64_t>(p.rows, 0x7fffffff)), 512, 0, 0, st, p);
    return check_launch("layernorm");
  }
  const RowPlan r = row_plan(p.rows, p.cols, access, kMost, 1);
  p.tpr = r.tpr;
  p.slots = r.slots;
  with_mode(access, [&](auto mode) {
    constexpr int A = decltype(mode)::value;
    if constexpr (!(BLOCKS && A == tg8::kShifted)) {
      with_groups(r.groups, [&](auto g) {
        constexpr int G = decltype(g)::value;
        if constexpr (G <= kMost) launch_kernel(tgb::layernorm_kernel<T, G, A, BLOCKS>, unsigned(r.blocks), r.block, 0, 0, st, p);
      });
    }
  });
  return check_launch("layernorm");
}

tg_status check_shape(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (rows=%lld cols=%lld)", (long long)rows, (long long)cols);
  if (cols > kColumnLimit) return fail(TG_ERR_UNSUPPORTED, "cols=%lld", (long long)cols);
  if (rows && cols == 0) return fail(TG_ERR_INVALID_ARGUMENT, "a row of no columns has no norm");
  return TG_OK;
}
tg_status check_pitch(const char* name, const void* p, int64_t ld, int64_t cols) {
  return p && ld < cols ? fail(TG_ERR_DIMENSION_MISMATCH, "%s=%lld < %lld", name, (long long)ld, (long long)cols) : TG_OK;
}
tg_status check_type(tg_dtype t) {
  return elem8_size(t) ? TG_OK : fail(TG_ERR_INVALID_ARGUMENT, "layer norm needs f32, f16 or bf16, got dtype %d", int(t));
}

#define TG_CHECK(call)                  \
  do {                                  \
    const tg_status s_ = (call);        \
    if (s_ != TG_OK) return s_;         \
  } while (0)

tg_status norm_forward(tg_dtype dtype, NormArgs p, cudaStream_t st) {
  TG_CHECK(check_type(dtype));
  TG_CHECK(check_shape(p.rows, p.cols));
  if (!(p.eps >= 0.f)) return fail(TG_ERR_INVALID_ARGUMENT, "eps=%g is negative", double(p.eps));
  if ((p.mean != nullptr) != (p.rstd != nullptr)) return fail(TG_ERR_INVALID_ARGUMENT, "mean and rstd are given together or not at all");
  if (p.rows == 0) return TG_OK;
  if (!p.x || (!p.y && !p.q) || (p.q && !p.scale)) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldx", p.x, p.ldx, p.cols));
  TG_CHECK(check_pitch("ldr", p.residual, p.ldr, p.cols));
  TG_CHECK(check_pitch("ldh", p.h, p.ldh, p.cols));
  TG_CHECK(check_pitch("ldy", p.y, p.ldy, p.cols));
  TG_CHECK(check_pitch("ldq", p.q, p.ldq, p.cols));
  const size_t e = elem8_size(dtype);
  RowAccess access(p.cols);
  access.add(p.x, p.ldx, e);
  access.add(p.residual, p.ldr, e);
  access.add(p.h, p.ldh, e);
  access.add(p.y, p.ldy, e);
  int how = access.get();
  if (how == tg8::kAligned && !(aligned(p.weight, 16) && aligned(p.bias, 16))) how = tg8::kScalar;
  if (p.q && how == tg8::kShifted) how = tg8::kScalar;   // a block's 16 lanes start at its first element
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    return p.q ? launch_norm<T, true>(p, how, st) : launch_norm<T, false>(p, how, st);
  });
}

template <typename T> tg_status launch_backward(NormBackArgs p, T* grad_w, T* grad_b, int access, cudaStream_t st) {
  constexpr int kMost = 2;
  const bool lng = p.cols + 7 > 512 * 8 * kMost;
  RowPlan r = row_plan(p.rows, std::min<int64_t>(p.cols, 512 * 8), access, kMost, 1);
  if (!lng) r = row_plan(p.rows, p.cols, access, kMost, 1);
  p.tpr = r.tpr;
  p.slots = lng ? std::max<int64_t>(1, std::min<int64_t>(p.rows, 64)) : r.slots;
  void* scratch = nullptr;
  const size_t part = size_t(p.slots) * size_t(p.cols);
  if (grad_w || grad_b) {
    const cudaError_t e = scratch_alloc(&scratch, part * sizeof(float) * ((grad_w ? 1 : 0) + (grad_b ? 1 : 0)), st);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "layernorm backward scratch: %s", cudaGetErrorString(e));
    float* at = static_cast<float*>(scratch);
    if (grad_w) { p.partial_w = at; at += part; }
    if (grad_b) p.partial_b = at;
  }
  if (lng) {
    if (p.grad_x) launch_kernel(tgb::layernorm_backward_long_kernel<T>, unsigned(std::min<int64_t>(p.rows, 0x7fffffff)), 512, 0, 0, st, p);
    if (scratch) launch_kernel(tgb::layernorm_columns_kernel<T>, dim3(unsigned((p.cols + 1023) / 1024), unsigned(p.slots)), 128, 0, 0, st, p);
  } else {
    with_mode(access, [&](auto mode) {
      constexpr int A = decltype(mode)::value;
      if (r.groups == 1) launch_kernel(tgb::layernorm_backward_kernel<T, 1, A>, unsigned(r.blocks), r.block, 0, 0, st, p);
      else launch_kernel(tgb::layernorm_backward_kernel<T, 2, A>, unsigned(r.blocks), r.block, 0, 0, st, p);
    });
  }
  const unsigned strips = unsigned((p.cols + 31) / 32);
  if (grad_w) launch_kernel(tg8::column_join_kernel<T>, strips, 1024, 0, 0, st, p.slots, p.cols, p.partial_w, grad_w);
  if (grad_b) launch_kernel(tg8::column_join_kernel<T>, strips, 1024, 0, 0, st, p.slots, p.cols, p.partial_b, grad_b);
  const tg_status s = check_launch("layernorm backward");
  if (scratch) scratch_free(scratch, st);
  return s;
}

}  // namespace
}  // namespace tgi

using namespace tgi;

extern "C" {

tg_status tg_layernorm(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual,
                       int64_t ldr, const void* weight, const void* bias, float eps, void* h, int64_t ldh, void* y,
                       int64_t ldy, float* mean, float* rstd, void* stream) {
  clear_error();
  NormArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx; p.residual = residual; p.ldr = ldr; p.weight = weight; p.bias = bias;
  p.eps = eps; p.h = h; p.ldh = ldh; p.y = y; p.ldy = ldy; p.mean = mean; p.rstd = rstd;
  return norm_forward(dtype, p, static_cast<cudaStream_t>(stream));
}

tg_status tg_blocks8_layernorm(tg_dtype dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual,
                               int64_t ldr, const void* weight, const void* bias, float eps, void* h, int64_t ldh, void* q,
                               int64_t ldq, float* scale, int64_t scale_row, int64_t scale_block, float* mean, float* rstd,
                               void* stream) {
  clear_error();
  NormArgs p{};
  p.rows = rows; p.cols = cols; p.x = x; p.ldx = ldx; p.residual = residual; p.ldr = ldr; p.weight = weight; p.bias = bias;
  p.eps = eps; p.h = h; p.ldh = ldh; p.mean = mean; p.rstd = rstd;
  p.q = static_cast<uint8_t*>(q); p.ldq = ldq; p.scale = scale; p.scale_row = scale_row; p.scale_block = scale_block;
  return norm_forward(dtype, p, static_cast<cudaStream_t>(stream));
}

tg_status tg_layernorm_backward(tg_dtype dtype, int64_t rows, int64_t cols, const void* grad, int64_t ldg, const void* grad_h,
                                int64_t ldgh, const void* weight, const void* h, int64_t ldh, const float* mean,
                                const float* rstd, void* grad_x, int64_t ldx, void* grad_weight, void* grad_bias, void* stream) {
  clear_error();
  TG_CHECK(check_type(dtype));
  TG_CHECK(check_shape(rows, cols));
  if (cols == 0 || (!grad_x && !grad_weight && !grad_bias)) return TG_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {   // sums of nothing
    for (void* out : {grad_weight, grad_bias}) {
      const cudaError_t e = out ? cudaMemsetAsync(out, 0, size_t(cols) * elem8_size(dtype), st) : cudaSuccess;
      if (e != cudaSuccess) return fail(TG_ERR_CUDA, "memset: %s", cudaGetErrorString(e));
    }
    return TG_OK;
  }
  if (!grad || !h || !mean || !rstd) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldg", grad, ldg, cols));
  TG_CHECK(check_pitch("ldgh", grad_h, ldgh, cols));
  TG_CHECK(check_pitch("ldh", h, ldh, cols));
  TG_CHECK(check_pitch("ldx", grad_x, ldx, cols));
  NormBackArgs p{};
  p.rows = rows; p.cols = cols; p.grad = grad; p.ldg = ldg; p.grad_h = grad_h; p.ldgh = ldgh; p.weight = weight;
  p.h = h; p.ldh = ldh; p.mean = mean; p.rstd = rstd; p.grad_x = grad_x; p.ldx = ldx;
  const size_t e = elem8_size(dtype);
  RowAccess access(cols);
  access.add(grad, ldg, e);
  access.add(grad_h, ldgh, e);
  access.add(h, ldh, e);
  access.add(grad_x, ldx, e);
  int how = access.get();
  if (how == tg8::kAligned && !aligned(weight, 16)) how = tg8::kScalar;
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    return launch_backward<T>(p, static_cast<T*>(grad_weight), static_cast<T*>(grad_bias), how, st);
  });
}

}  // extern "C"
