// Layer norm: forward (rows or 8-bit blocks out), backward with the gradients
// of weight and bias.
//
//   h = x + residual, u = (h - mean) rstd, y = u weight + bias
//   grad_x = rstd (a - mean(a) - u mean(a u)) + grad_h,  a = grad weight
//
// All are bound by memory.  A row that fits registers is read once, kept there
// between its sums and its output, and written once; a longer one (forward: f32
// above 8192 columns, 16-bit above 16384; backward: above 8192) is read three times.
// The backward's rows, of two to four operands beside the columns' sums, come by
// bulk copies into a ring in shared memory where there are many, which keeps more
// of them on the way than registers could (8192 x 8192 bf16, us: grad, h and grad_h
// 106; with h's parts in its place, four operands, 117; three loaded directly 389
// with f32 arithmetic one by one).
#include <algorithm>
#include "tg_blocks8.cuh"
#include "tg_umma.cuh"

namespace tgb {

struct NormArgs {
  int64_t rows, cols, slots;
  const void *x, *residual, *weight, *bias;
  void *h, *y;
  uint8_t* q;                 // the output in 8-bit blocks, in place of y
  float *scale, *mean, *rstd;
  int64_t ldx, ldr, ldh, ldy, ldq, scale_row, scale_block;
  float eps;
  int tpr;                    // threads per row: 32 .. 512, a multiple of 32
};

// Sums over the tpr threads of a row (a multiple of 32), one or two at a time:
// one named barrier per row, two sets of partial results in turn.  The order is
// the same in every thread.
struct RowSums {
  float2 (*sums)[16];   // [2][warps of the block]
  int tpr, sub, turn;
  __device__ __forceinline__ float2 across(float2 s) {
    if (tpr > 32) {
      const int warps = tpr >> 5, first = sub * warps;
      if ((threadIdx.x & 31) == 0) sums[turn][threadIdx.x >> 5] = s;
      named_sync(sub + 1, tpr);
      const float2* from = &sums[turn][first];
      turn ^= 1;
      uint64_t all = pair_of(from[0].x, from[0].y);
      if (warps == 16) {
#pragma unroll
        for (int w = 1; w < 16; w++) all = add_pair(all, pair_of(from[w].x, from[w].y));
      } else {
#pragma unroll 4
        for (int w = 1; w < warps; w++) all = add_pair(all, pair_of(from[w].x, from[w].y));
      }
      s = values_of(all);
    }
    return s;
  }
  __device__ __forceinline__ float one(float s) {
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    return across(make_float2(s, 0.f)).x;
  }
  __device__ __forceinline__ float2 two(float2 s) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, d);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, d);
    }
    return across(s);
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
template <int ACCESS> __device__ __forceinline__ void mask_pairs(uint64_t (&v)[4], int c, int cols) {
  if (ACCESS != kAligned && (c < 0 || c + 8 > cols)) {   // a row's ends
    float f[8];
    from_pairs(v, f);
    mask_at<ACCESS>(f, c, cols);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = pair_of(f[2 * i], f[2 * i + 1]);
  }
}
template <int ACCESS, typename T> __device__ __forceinline__ void store_at(T* row, int c, int cols, const float (&v)[8]) {
  if constexpr (ACCESS == kScalar) store_any(row, c, cols, v);
  else store_group<ACCESS>(row, c, cols, v);
}
// A group of a vector over the columns (weight, bias), as it lies in memory;
// `otherwise` in all places where there is none.
template <int ACCESS, typename T> __device__ __forceinline__ void load_columns(Vec8<T>& v, const void* columns, float otherwise, int c, int cols) {
  const T* from = static_cast<const T*>(columns);
  if (ACCESS == kAligned && from) {
    load_group<kAligned>(v, from, c, cols);
  } else if (from && c >= 0 && c + 8 <= cols) {
    load_any(v, from, c, cols);
  } else {
    union { Vec8<T> v; T e[8]; } u;
#pragma unroll
    for (int e = 0; e < 8; e++) u.e[e] = from && inside<ACCESS>(c, e, cols) ? from[c + e] : from_f32<T>(otherwise);
    v = u.v;
  }
}

// Mean and rstd from the row's mean (the sum's, rounded), the sum of h - mean and
// of its square: what the rounding of the first mean left is taken out again.
// Squares that pass f32's range say that rstd is 0; the sum beside them may have
// passed it too, in both directions, and is left out.
__device__ __forceinline__ float2 finish_stats(float mean, float2 off, float inv_cols, float eps) {
  const float d = off.y == __int_as_float(0x7f800000) ? 0.f : off.x * inv_cols;
  float var = fmaf(off.y, inv_cols, -d * d);
  if (var < 0.f) var = 0.f;   // a NaN stays
  return make_float2(mean + d, rsqrtf(var + eps));   // within two units of the last place
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

// The two passes over a row that its threads hold: its statistics, and its
// outputs.  Groups past the row take no part.
template <int G, int ACCESS>
__device__ __forceinline__ float2 row_stats(const uint64_t (&v)[G][4], int tpr, int t, int shift, int cols, float inv_cols, float eps, RowSums& join) {
  auto at = [&](int g) { return (g * tpr + t) * 8 - shift; };
  uint64_t sum = 0;   // of h / cols, which stays within f32's range where h does
  const uint64_t share = pair_of(inv_cols);
#pragma unroll
  for (int g = 0; g < G; g++) {
    if (at(g) >= cols) continue;
#pragma unroll
    for (int i = 0; i < 4; i++) fma_pair(sum, v[g][i], share);
  }
  const float rough = join.one(sum_of(sum));
  const uint64_t minus = pair_of(-rough);
  uint64_t off = 0, square = 0;
#pragma unroll
  for (int g = 0; g < G; g++) {
    if (at(g) >= cols) continue;
    uint64_t d[4];
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = add_pair(v[g][i], minus);
    mask_pairs<ACCESS>(d, at(g), cols);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      off = add_pair(off, d[i]);
      fma_pair(square, d[i], d[i]);
    }
  }
  return finish_stats(rough, join.two(make_float2(sum_of(off), sum_of(square))), inv_cols, eps);
}
template <typename T, int G, int ACCESS, bool BLOCKS>
__device__ __forceinline__ void finish_row(const NormArgs& p, int64_t row, int t, int shift, const uint64_t (&v)[G][4], const Vec8<T> (&w)[G],
                                           const Vec8<T> (&b)[G], float2 st) {
  if (t == 0 && p.mean) {
    p.mean[row] = st.x;
    p.rstd[row] = st.y;
  }
  const int cols = int(p.cols);
  const uint64_t minus = pair_of(-st.x), scale = pair_of(st.y);
  T* h = static_cast<T*>(p.h) + row * p.ldh;
  T* out = static_cast<T*>(p.y) + row * p.ldy;
  if (p.h) {
#pragma unroll
    for (int g = 0; g < G; g++) {
      const int c = (g * p.tpr + t) * 8 - shift;
      float f[8];
      from_pairs(v[g], f);
      store_at<ACCESS>(h, c, cols, f);
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int c = (g * p.tpr + t) * 8 - shift;
    if (!BLOCKS && c >= cols) continue;
    uint64_t y[4], kw[4], kb[4];
    get_pairs(w[g], kw);
    get_pairs(b[g], kb);
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = fma_pair_of(mul_pair(add_pair(v[g][i], minus), scale), kw[i], kb[i]);
    float f[8];
    from_pairs(y, f);
    if constexpr (BLOCKS) store_block(p, row, c, f);
    else store_at<ACCESS>(out, c, cols, f);
  }
}

// tpr threads per row, G groups of 8 elements per thread.  A slot (tpr threads)
// walks rows slot, slot + slots, ..; its threads have fixed columns, so weight
// and bias stay in registers (rows that start anywhere: slots is a multiple of
// 8, so all rows of a slot start at the same distance from a boundary).  The
// next row is on its way while this one is worked on.
//
// MOST threads per block: 512, of which an SM has one, or 320, of which it has two.
template <typename T, int G, int ACCESS, bool BLOCKS, int MOST>
__global__ void __launch_bounds__(MOST, MOST == 320 ? 2 : 1) layernorm_kernel(const NormArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int cols = int(p.cols);
  int64_t row = int64_t(blockIdx.x) * per_block + sub;
  if (row >= p.rows || row >= p.slots) return;
  const T *x = static_cast<const T*>(p.x), *res = static_cast<const T*>(p.residual);
  const int shift = ACCESS == kShifted ? row_shift(x + row * p.ldx) : 0;
  auto at = [&](int g) { return (g * p.tpr + t) * 8 - shift; };
  RowSums join{sums, p.tpr, sub, 0};
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
    load_columns<ACCESS>(w[g], p.weight, 1.f, at(g), cols);
    load_columns<ACCESS>(b[g], p.bias, 0.f, at(g), cols);
  }
  const float inv_cols = 1.f / float(cols);
  for (; row < p.rows; row += p.slots) {
    uint64_t v[G][4];
#pragma unroll
    for (int g = 0; g < G; g++) {
      get_pairs(nx[g], v[g]);
      if (res) {
        uint64_t r[4];
        get_pairs(nr[g], r);
#pragma unroll
        for (int i = 0; i < 4; i++) v[g][i] = add_pair(v[g][i], r[i]);
      }
      mask_pairs<ACCESS>(v[g], at(g), cols);
    }
    if (row + p.slots < p.rows) load(row + p.slots);
    const float2 st = row_stats<G, ACCESS>(v, p.tpr, t, shift, cols, inv_cols, p.eps, join);
    finish_row<T, G, ACCESS, BLOCKS>(p, row, t, shift, v, w, b, st);
  }
}

// Rows too long for registers: one block per row, which reads it three times
// (the second and third from L2).
template <typename T, bool BLOCKS>
__global__ void __launch_bounds__(512) layernorm_long_kernel(const NormArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  RowSums join{sums, 512, 0, 0};
  const float inv_cols = 1.f / float(p.cols);
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
      for (int e = 0; e < 8; e++) sum = fmaf(c + e < p.cols ? v[e] : 0.f, inv_cols, sum);
    }
    const float rough = join.one(sum);
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
    const float2 st = finish_stats(rough, join.two(off), inv_cols, p.eps);
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

// u is that of the output only where h is the sum that the forward took its
// statistics of: a 16-bit h is that sum rounded, which u would show in full
// (errors of the gradients against 64 bits 1.5 times those of their own rounding,
// more where a row is far from zero).  With a residual, h is x and the sum is
// formed again, as the forward did.
struct NormBackArgs {
  int64_t rows, cols, slots;
  const void *grad, *grad_h, *weight, *h, *residual;   // grad_h, weight, residual: or null
  const float *mean, *rstd;
  void* grad_x;
  float *partial_w, *partial_b;   // (slots x cols), or null
  int64_t ldg, ldgh, ldh, ldr, ldx;
  int tpr;
};

// The backward's two passes over a group: a = grad * weight and u, and their part
// in the sums; then grad_x from the row's means.  SUM: h is x + res.
template <int ACCESS, bool SUM, typename T>
__device__ __forceinline__ void back_group(const Vec8<T>& grad, const Vec8<T>& h, const Vec8<T>& res, const Vec8<T>& w, int c, int cols,
                                           uint64_t minus, uint64_t rstd, uint64_t (&a)[4], uint64_t (&u)[4], uint64_t (&dw)[4], uint64_t (&db)[4],
                                           uint64_t& s, uint64_t& su) {
  uint64_t k[4];
  get_pairs(grad, a);
  get_pairs(h, u);
  if (SUM) {
    get_pairs(res, k);
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = add_pair(u[i], k[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) u[i] = mul_pair(add_pair(u[i], minus), rstd);
  mask_pairs<ACCESS>(a, c, cols);
  mask_pairs<ACCESS>(u, c, cols);
  get_pairs(w, k);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    fma_pair(dw[i], a[i], u[i]);
    db[i] = add_pair(db[i], a[i]);
    a[i] = mul_pair(a[i], k[i]);
    s = add_pair(s, a[i]);
    fma_pair(su, a[i], u[i]);
  }
}
// rstd * (a - mean - u * mean_u) + more
template <bool MORE, typename T>
__device__ __forceinline__ void back_out(const uint64_t (&a)[4], const uint64_t (&u)[4], uint64_t minus_mean, uint64_t minus_mean_u, uint64_t rstd,
                                         const Vec8<T>& more, float (&o)[8]) {
  uint64_t r[4], k[4];
  if (MORE) get_pairs(more, k);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    r[i] = add_pair(fma_pair_of(u[i], minus_mean_u, a[i]), minus_mean);
    r[i] = MORE ? fma_pair_of(r[i], rstd, k[i]) : mul_pair(r[i], rstd);
  }
  from_pairs(r, o);
}

// As layernorm_kernel; a thread also keeps its columns' sums of grad * u and of
// grad over the slot's rows, joined by layernorm_join_kernel in a fixed order.
// SUM, the sum formed again, is a variant of its own: as a branch it took 14 us of
// 109 from the rows without (8192 x 8192 bf16, by copies).
template <typename T, int G, int ACCESS, bool SUM>
__global__ void __launch_bounds__(512) layernorm_backward_kernel(const NormBackArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, per_block = blockDim.x / p.tpr;
  const int cols = int(p.cols);
  const int64_t slot = int64_t(blockIdx.x) * per_block + sub;
  if (slot >= p.slots) return;
  const T *grad = static_cast<const T*>(p.grad), *h = static_cast<const T*>(p.h), *gh = static_cast<const T*>(p.grad_h);
  const T* res = SUM ? static_cast<const T*>(p.residual) : nullptr;
  const int shift = ACCESS == kShifted ? row_shift(grad + slot * p.ldg) : 0;
  auto at = [&](int g) { return (g * p.tpr + t) * 8 - shift; };
  RowSums join{sums, p.tpr, sub, 0};
  constexpr bool kAhead = G * sizeof(T) <= 4;   // the next row fits the registers
  Vec8<T> ng[G], nh[G], w[G];
  float2 ns;
  uint64_t dw[G][4] = {}, db[G][4] = {};
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
    load_columns<ACCESS>(w[g], p.weight, 1.f, at(g), cols);
  const float inv_cols = 1.f / float(cols);
  for (; row < p.rows; row += p.slots) {
    if (!kAhead) load(row);
    Vec8<T> ch[G], cr[G];
    if (SUM) {
#pragma unroll
      for (int g = 0; g < G; g++) load_at<ACCESS>(cr[g], res + row * p.ldr, at(g), cols);
    }
    if (gh && p.grad_x) {
#pragma unroll
      for (int g = 0; g < G; g++) load_at<ACCESS>(ch[g], gh + row * p.ldgh, at(g), cols);
    }
    uint64_t a[G][4], u[G][4], s = 0, su = 0;
    const uint64_t rstd = pair_of(ns.y), minus = pair_of(-ns.x);
#pragma unroll
    for (int g = 0; g < G; g++)
      if (at(g) < cols) back_group<ACCESS, SUM>(ng[g], nh[g], cr[g], w[g], at(g), cols, minus, rstd, a[g], u[g], dw[g], db[g], s, su);
    if (kAhead && row + p.slots < p.rows) load(row + p.slots);
    if (!p.grad_x) continue;
    const float2 sums2 = join.two(make_float2(sum_of(s), sum_of(su)));
    const uint64_t mean = pair_of(-sums2.x * inv_cols), mean_u = pair_of(-sums2.y * inv_cols);
    T* out = static_cast<T*>(p.grad_x) + row * p.ldx;
#pragma unroll
    for (int g = 0; g < G; g++) {
      if (at(g) >= cols) continue;
      float o[8];
      if (gh) back_out<true>(a[g], u[g], mean, mean_u, rstd, ch[g], o);
      else back_out<false>(a[g], u[g], mean, mean_u, rstd, ch[g], o);
      store_at<ACCESS>(out, at(g), cols, o);
    }
  }
#pragma unroll
  for (int g = 0; g < G; g++) {
    const int c = at(g);
    float fw[8], fb[8];
    from_pairs(dw[g], fw);
    from_pairs(db[g], fb);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      if (c + e < 0 || c + e >= cols) continue;
      if (p.partial_w) p.partial_w[slot * p.cols + c + e] = fw[e];
      if (p.partial_b) p.partial_b[slot * p.cols + c + e] = fb[e];
    }
  }
}

// ------------------------------------------------------------------------------- rows by bulk copies
// A stage holds one row of each of up to four operands for each of the `per`
// rows that a block works on at once; a row is copied from the 16-byte boundary
// before its first element, 16 bytes into its place.
constexpr int kMostStages = 8;
struct RowRing {
  uint32_t base, full, empty;   // shared memory; barriers
  int stages, per, ops, pitch;
  __device__ __forceinline__ uint32_t at(int stage, int op, int sub) const { return base + uint32_t(((stage * ops + op) * per + sub) * pitch); }
};
// One warp starts the copies of a batch's rows into a stage: a lane has one row
// of one operand (ops * per is at most 32).
template <int ACCESS, typename T> struct RowCopies {
  const char* x;   // this lane's operand at row `sub` of batch 0
  int64_t step;    // bytes from one batch to the next
  int sub;
  uint32_t to, bytes;
  __device__ __forceinline__ RowCopies(const RowRing& r, int64_t cols, const void* const (&rows)[4], const int64_t (&ld)[4]) {
    const int lane = threadIdx.x & 31, op = lane / r.per;
    sub = lane - op * r.per;
    if (op >= r.ops) sub = 1 << 30;
    const void* from = op == 0 ? rows[0] : op == 1 ? rows[1] : op == 2 ? rows[2] : rows[3];
    const int64_t pitch = (op == 0 ? ld[0] : op == 1 ? ld[1] : op == 2 ? ld[2] : ld[3]) * int64_t(sizeof(T));
    x = static_cast<const char*>(from) + (op < r.ops ? sub * pitch : 0);
    step = pitch * r.per;
    bytes = uint32_t(cols * sizeof(T));
    to = r.at(0, op < r.ops ? op : 0, op < r.ops ? sub : 0) + 16;
  }
  __device__ __forceinline__ void operator()(const RowRing& r, int64_t rows, int64_t batch, int stage) const {
    const int here = int(min(int64_t(r.per), rows - batch * r.per));
    const uintptr_t from = reinterpret_cast<uintptr_t>(x) + uintptr_t(batch * step), a = from & ~uintptr_t(15);
    const uint32_t size = ACCESS == kAligned ? bytes : uint32_t(((from + bytes + 15) & ~uintptr_t(15)) - a);
    const bool mine = sub < here;
    uint32_t total = uint32_t(r.ops * here) * bytes;
    if (ACCESS != kAligned) total = __reduce_add_sync(0xffffffffu, mine ? size : 0u);
    if ((threadIdx.x & 31) == 0) umma::bar_expect(r.full + 8 * stage, total);
    __syncwarp();
    if (mine) umma::bulk_load(to + uint32_t(stage * r.ops * r.per * r.pitch), reinterpret_cast<const void*>(a), size, r.full + 8 * stage);
  }
};
__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
// Eight elements from shared memory; kScalar: from any element on.
template <int ACCESS, typename T> __device__ __forceinline__ void take8(Vec8<T>& v, uint32_t at) {
  if constexpr (sizeof(T) == 4) {
    if constexpr (ACCESS != kScalar) {
      const uint4 a = load_shared16(at), b = load_shared16(at + 16);
      v.a = make_float4(__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w));
      v.b = make_float4(__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w));
    } else {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; e++) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[e]) : "r"(at + 4 * e));
      v.a = make_float4(f[0], f[1], f[2], f[3]);
      v.b = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else if constexpr (ACCESS != kScalar) {
    v.a = load_shared16(at);
  } else {
    const uint32_t skew = at & 15;
    const uint4 lo = load_shared16(at - skew), hi = load_shared16(at - skew + 16);
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
}
template <typename T> __device__ __forceinline__ uint32_t skew_of(const T* row) { return uint32_t(reinterpret_cast<uintptr_t>(row) & 15); }

// Many rows: as layernorm_backward_kernel, rows by bulk copies.  The block's
// sums over its rows are joined across its `per` threads of a column at the end.
template <typename T, int G, int ACCESS, bool SUM>
__global__ void __launch_bounds__(512) layernorm_backward_ring_kernel(const NormBackArgs p, int per, int stages, int pitch) {
  extern __shared__ __align__(16) uint8_t ring_store[];
  __shared__ __align__(8) uint64_t bars[2 * kMostStages];
  __shared__ float2 sums[2][16];
  const int workers = per * p.tpr, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *grad = static_cast<const T*>(p.grad), *h = static_cast<const T*>(p.h), *gh = p.grad_x ? static_cast<const T*>(p.grad_h) : nullptr;
  const T* res = SUM ? static_cast<const T*>(p.residual) : nullptr;
  const int op_res = gh ? 3 : 2;   // its place in a stage
  RowRing ring{umma::smem_u32(ring_store), umma::smem_u32(bars), umma::smem_u32(bars + kMostStages), stages, per, op_res + (SUM ? 1 : 0), pitch};
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) {
      umma::bar_init(ring.full + 8 * s, 1);
      umma::bar_init(ring.empty + 8 * s, workers >> 5);
    }
    umma::bar_init_fence();
  }
  after_previous_kernel();
  __syncthreads();
  const RowCopies<ACCESS, T> copies(ring, p.cols, {grad, h, gh || !SUM ? gh : res, res}, {p.ldg, p.ldh, gh || !SUM ? p.ldgh : p.ldr, p.ldr});
  auto bring = [&](int64_t batch, int stage) { copies(ring, p.rows, batch, stage); };
  if (warp == 0)
    for (int s = 0; s < stages && (blockIdx.x + int64_t(s) * gridDim.x) * per < p.rows; s++) bring(blockIdx.x + int64_t(s) * gridDim.x, s);
  const int sub = threadIdx.x / p.tpr, t = threadIdx.x % p.tpr, cols = int(p.cols);
  const int shift = ACCESS == kShifted ? row_shift(grad + (int64_t(blockIdx.x) * per + sub) * p.ldg) : 0;
  auto at = [&](int g) { return (g * p.tpr + t) * 8 - shift; };
  RowSums join{sums, p.tpr, sub, 0};
  Vec8<T> w[G];
#pragma unroll
  for (int g = 0; g < G; g++)
    load_columns<ACCESS>(w[g], p.weight, 1.f, at(g), cols);
  uint64_t dw[G][4] = {}, db[G][4] = {};
  const float inv_cols = 1.f / float(cols);
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  float2 next = make_float2(0.f, 0.f);
  if (int64_t(blockIdx.x) * per + sub < p.rows) next = make_float2(p.mean[int64_t(blockIdx.x) * per + sub], p.rstd[int64_t(blockIdx.x) * per + sub]);
  for (int64_t batch = blockIdx.x; batch * per < p.rows; batch += gridDim.x) {
    const int64_t row = batch * per + sub, after = row + int64_t(gridDim.x) * per;
    const uint64_t rstd = pair_of(next.y), minus = pair_of(-next.x);
    if (after < p.rows) next = make_float2(p.mean[after], p.rstd[after]);
    if (ok) ok = umma::bar_wait(ring.full + 8 * stage, parity);
    if (row < p.rows) {   // the same in all threads of a row
      uint64_t a[G][4], u[G][4], s = 0, su = 0;
      const uint32_t from = ring.at(stage, 0, sub) + 16 + (ACCESS == kAligned ? 0 : skew_of(grad + row * p.ldg));
      const uint32_t from_h = ring.at(stage, 1, sub) + 16 + (ACCESS == kAligned ? 0 : skew_of(h + row * p.ldh));
      const uint32_t from_r = SUM ? ring.at(stage, op_res, sub) + 16 + (ACCESS == kAligned ? 0 : skew_of(res + row * p.ldr)) : 0;
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int c = at(g);
        if (c >= cols) continue;
        Vec8<T> vg, vh, vr;
        take8<ACCESS>(vg, from + c * int(sizeof(T)));
        take8<ACCESS>(vh, from_h + c * int(sizeof(T)));
        if (SUM) take8<ACCESS>(vr, from_r + c * int(sizeof(T)));
        back_group<ACCESS, SUM>(vg, vh, vr, w[g], c, cols, minus, rstd, a[g], u[g], dw[g], db[g], s, su);
      }
      if (p.grad_x) {
        float2 sums2 = join.two(make_float2(sum_of(s), sum_of(su)));
        if (!ok) sums2.x = __uint_as_float(0x7fffffffu);   // a wait ran out: the outputs say so
        const uint64_t mean = pair_of(-sums2.x * inv_cols), mean_u = pair_of(-sums2.y * inv_cols);
        const uint32_t more = gh ? ring.at(stage, 2, sub) + 16 + (ACCESS == kAligned ? 0 : skew_of(gh + row * p.ldgh)) : 0;
        T* out = static_cast<T*>(p.grad_x) + row * p.ldx;
#pragma unroll
        for (int g = 0; g < G; g++) {
          const int c = at(g);
          if (c >= cols) continue;
          float o[8];
          Vec8<T> vh;
          if (gh) {
            take8<ACCESS>(vh, more + c * int(sizeof(T)));
            back_out<true>(a[g], u[g], mean, mean_u, rstd, vh, o);
          } else {
            back_out<false>(a[g], u[g], mean, mean_u, rstd, vh, o);
          }
          store_at<ACCESS>(out, c, cols, o);
        }
      }
    }
    __syncwarp();
    if (lane == 0) umma::bar_arrive(ring.empty + 8 * stage);
    const int64_t ahead = batch + int64_t(stages) * gridDim.x;
    if (warp == 0 && ahead * per < p.rows) {
      // Waits may run out in some lanes alone.  Rows off the boundaries add up their
      // bytes across the warp, so its lanes go on by vote; whole ones have a
      // __syncwarp there, which lanes that gave up meet in the next turn (a vote here
      // would take 5 us of 106, 8192 x 8192 bf16).
      if (ok) ok = umma::bar_wait(ring.empty + 8 * stage, parity);
      if (ACCESS != kAligned) ok = __all_sync(0xffffffffu, ok);
      if (ok) bring(ahead, stage);
    }
    if (++stage == stages) { stage = 0; parity ^= 1; }
  }
  if (!ok) umma::drain_copies();
  // all rows have been used: the ring holds the sums of the block's threads of a column
  float* store = reinterpret_cast<float*>(ring_store);
  auto join_columns = [&](const uint64_t (&d)[G][4], float* partial) {
    if (!partial) return;
#pragma unroll
    for (int g = 0; g < G; g++) {
      float f[8];
      from_pairs(d[g], f);
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (inside<kShifted>(at(g), e, cols)) store[sub * cols + at(g) + e] = ok ? f[e] : __uint_as_float(0x7fffffffu);
    }
    named_sync(15, workers);
    for (int c = threadIdx.x; c < cols; c += workers) {
      float sum = 0.f;
      for (int i = 0; i < per; i++) sum += store[i * cols + c];
      partial[int64_t(blockIdx.x) * p.cols + c] = sum;
    }
    named_sync(15, workers);
  };
  if (p.partial_w || p.partial_b) named_sync(15, workers);
  join_columns(dw, p.partial_w);
  join_columns(db, p.partial_b);
}

// Rows too long for registers, grad_x: one block per row, read twice.
template <typename T>
__global__ void __launch_bounds__(512) layernorm_backward_long_kernel(const NormBackArgs p) {
  __shared__ float2 sums[2][16];
  after_previous_kernel();
  RowSums join{sums, 512, 0, 0};
  const float inv_cols = 1.f / float(p.cols);
  const T* wgt = static_cast<const T*>(p.weight);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    const T *grad = static_cast<const T*>(p.grad) + row * p.ldg, *h = static_cast<const T*>(p.h) + row * p.ldh;
    const T* gh = p.grad_h ? static_cast<const T*>(p.grad_h) + row * p.ldgh : nullptr;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    auto load = [&](int64_t c, float (&a)[8], float (&u)[8]) {
      Vec8<T> v;
      load_any(v, h, c, p.cols);
      v.get(u);
      if (res) {
        load_any(v, res, c, p.cols);
        v.get(a);
#pragma unroll
        for (int e = 0; e < 8; e++) u[e] += a[e];
      }
      load_any(v, grad, c, p.cols);
      v.get(a);
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
    s = join.two(s);
    s.x *= inv_cols;
    s.y *= inv_cols;
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
    load_any(v, static_cast<const T*>(p.h) + row * p.ldh, c, p.cols);
    v.get(u);
    if (p.residual) {
      load_any(v, static_cast<const T*>(p.residual) + row * p.ldr, c, p.cols);
      v.get(a);
#pragma unroll
      for (int e = 0; e < 8; e++) u[e] += a[e];
    }
    load_any(v, static_cast<const T*>(p.grad) + row * p.ldg, c, p.cols);
    v.get(a);
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

// out[c] = sum over slots of partial[slot, c], for the weight (blockIdx.y 0) and
// the bias: 32 columns x 32 slot lanes per block, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_join_kernel(int64_t slots, int64_t cols, const float* partial_w, const float* partial_b, T* grad_w, T* grad_b) {
  __shared__ float part[32][33];
  after_previous_kernel();
  const float* partial = blockIdx.y || !grad_w ? partial_b : partial_w;
  T* out = blockIdx.y || !grad_w ? grad_b : grad_w;
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = int64_t(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = y; r < slots; r += 32) s += partial[r * cols + c];
  }
  part[y][lane] = s;
  __syncthreads();
  s = part[lane][y];   // warp y joins column y of the strip
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  const int64_t column = int64_t(blockIdx.x) * 32 + y;
  if (lane == 0 && column < cols) out[column] = from_f32<T>(s);
}

}  // namespace tgb

namespace tgi {

using tgb::NormArgs;
using tgb::NormBackArgs;

namespace {

constexpr int64_t kColumnLimit = 0x7fffff00;

// Groups of 8 elements of a row; one more where it may start behind a boundary.
int64_t groups_of(int64_t cols, int access) { return (cols + (access == tg8::kShifted ? 7 : 0) + 7) / 8; }
bool in_registers(int64_t cols, int access, int most) { return groups_of(cols, access) <= int64_t(most) * 512; }
int64_t round32(int64_t v) { return (v + 31) / 32 * 32; }

// Threads per row (a multiple of 32) and groups of 8 elements per thread, for
// rows loaded directly, 512 threads per SM.  Few rows: one group, for the latency,
// where 512 threads hold the row.  Many: two, which needs half as many sums
// across warps (8192 rows, us, one group / two: 1024 f32 28 / 24, 2048 bf16
// 36 / 26, 4096 bf16 70 / 50, four 57; 300 rows of 2048 f32 4.4 / 4.9).
//
// Rows of 257 to 320 threads leave many idle at one block per SM; with `narrow`
// there are two, in 96 registers (8192 rows bf16, us, one block / two: 4608 67 / 45,
// 5120 70 / 47, 777 f16 rows of 5001 13.1 / 9.4; f32, whose registers spill, 5120 88 / 105;
// 384 threads in 80 registers 6144 74 / 69, with residual 87 / 88).
struct RowPlan {
  int tpr, groups, block;
  int64_t blocks, slots;
  bool two;   // blocks per SM
};
RowPlan row_plan(int64_t rows, int64_t cols, int access, bool narrow) {
  const int64_t groups = groups_of(cols, access);
  RowPlan r;
  r.groups = rows >= 2 * int64_t(sm_count()) && groups > 32 ? 2 : 1;
  while (groups > int64_t(r.groups) * 512) r.groups *= 2;
  r.tpr = int(round32((groups + r.groups - 1) / r.groups));
  const int per = std::max(1, 128 / r.tpr);
  r.block = per * r.tpr;
  r.two = narrow && r.groups == 2 && r.tpr > 256 && r.tpr <= 320;
  r.blocks = std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, int64_t(sm_count()) * (r.two ? 2 : std::max(1, 512 / r.block))));
  r.slots = r.blocks * per;
  if (access == tg8::kShifted && r.slots < rows) {   // a slot's rows start alike
    r.slots = std::max<int64_t>(8, r.slots / 8 * 8);
    r.blocks = (r.slots + per - 1) / per;
  }
  return r;
}

// The same for rows by bulk copies: one block per SM, up to `most` groups per
// thread, as many stages as shared memory holds.
struct RingPlan {
  int tpr, groups, per, block, stages, pitch;
  size_t smem;
  int64_t blocks;
  bool fits;
};
RingPlan ring_plan(int64_t rows, int64_t cols, size_t elem, int ops, int access, int most) {
  constexpr int workers = 512;
  RingPlan r{};
  const int64_t groups = groups_of(cols, access);
  if (groups > int64_t(most) * 512) return r;
  r.groups = 1;
  while (r.groups < most && groups > int64_t(r.groups) * 128) r.groups *= 2;   // up to 128 threads with one group each
  r.tpr = int(round32((groups + r.groups - 1) / r.groups));
  r.per = std::min(std::max(1, workers / r.tpr), 32 / ops);   // a lane of the copying warp for each row
  r.block = r.per * r.tpr;
  r.pitch = int((cols * int64_t(elem) + 15) / 16 * 16 + 64);
  const size_t stage = size_t(ops) * r.per * r.pitch, share = size_t(216 * 1024);
  r.stages = int(std::min<size_t>(tgb::kMostStages, share / stage));
  if (r.stages < 2) return r;
  r.smem = r.stages * stage;
  r.blocks = std::min<int64_t>((rows + r.per - 1) / r.per, int64_t(sm_count()));
  if (access == tg8::kShifted && r.blocks * r.per < rows) {   // a thread's rows start alike
    const int64_t unit = 8 / (r.per % 8 == 0 ? 8 : r.per % 4 == 0 ? 4 : r.per % 2 == 0 ? 2 : 1);
    r.blocks = std::max(unit, r.blocks / unit * unit);
  }
  r.fits = true;
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
  if (access == tg8::kShifted && !in_registers(p.cols, access, kMost)) access = tg8::kScalar;
  if (!in_registers(p.cols, access, kMost)) {
    launch_kernel(tgb::layernorm_long_kernel<T, BLOCKS>, unsigned(std::min<int64_t>(p.rows, 0x7fffffff)), 512, 0, 0, st, p);
    return check_launch("layernorm");
  }
  const RowPlan r = row_plan(p.rows, p.cols, access, sizeof(T) == 2);
  p.tpr = r.tpr;
  p.slots = r.slots;
  with_mode(access, [&](auto mode) {
    constexpr int A = decltype(mode)::value;
    if constexpr (!(BLOCKS && A == tg8::kShifted)) {
      with_groups(r.groups, [&](auto g) {
        constexpr int G = decltype(g)::value;
        auto go = [&](auto kern) { launch_kernel(kern, unsigned(r.blocks), r.block, 0, 0, st, p); };
        if constexpr (G == 2 && sizeof(T) == 2) {
          if (r.two) return go(tgb::layernorm_kernel<T, G, A, BLOCKS, 320>);
        }
        if constexpr (G <= kMost) go(tgb::layernorm_kernel<T, G, A, BLOCKS, 512>);
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
  if (access == tg8::kShifted && !in_registers(p.cols, access, kMost)) access = tg8::kScalar;
  const bool lng = !in_registers(p.cols, access, kMost);
  RingPlan ring{};
  // by copies from a row per SM on (us, by copies / directly, bf16: 74 x 4096 11.2 / 9.6, 148 x 4096 11.2 / 11.8, 148 x 8192 16 / 21, 2400 x 8192 44 / 61)
  if (p.rows >= sm_count()) ring = ring_plan(p.rows, p.cols, sizeof(T), 2 + (p.grad_h && p.grad_x ? 1 : 0) + (p.residual ? 1 : 0), access, kMost);
  RowPlan r{};
  if (lng) p.slots = std::max<int64_t>(1, std::min<int64_t>(p.rows, 64));
  else if (ring.fits) { p.slots = ring.blocks; p.tpr = ring.tpr; }
  else { r = row_plan(p.rows, p.cols, access, false); p.slots = r.slots; p.tpr = r.tpr; }
  void* scratch = nullptr;
  const size_t part = size_t(p.slots) * size_t(p.cols);
  if (grad_w || grad_b) {
    const cudaError_t e = scratch_alloc(&scratch, part * sizeof(float) * ((grad_w ? 1 : 0) + (grad_b ? 1 : 0)), st);
    if (e != cudaSuccess) return fail(TG_ERR_CUDA, "layernorm backward scratch: %s", cudaGetErrorString(e));
    float* at = static_cast<float*>(scratch);
    if (grad_w) { p.partial_w = at; at += part; }
    if (grad_b) p.partial_b = at;
  }
  tg_status s = TG_OK;
  if (lng) {
    if (p.grad_x) launch_kernel(tgb::layernorm_backward_long_kernel<T>, unsigned(std::min<int64_t>(p.rows, 0x7fffffff)), 512, 0, 0, st, p);
    if (scratch) launch_kernel(tgb::layernorm_columns_kernel<T>, dim3(unsigned((p.cols + 1023) / 1024), unsigned(p.slots)), 128, 0, 0, st, p);
  } else {
    with_mode(access, [&](auto mode) {
      constexpr int A = decltype(mode)::value;
      auto go = [&](auto direct, auto by_copies) {
        if (!ring.fits) {
          launch_kernel(direct, unsigned(r.blocks), r.block, 0, 0, st, p);
        } else {
          s = ensure_smem(reinterpret_cast<const void*>(by_copies), 216 * 1024);
          if (s == TG_OK) launch_kernel(by_copies, unsigned(ring.blocks), ring.block, ring.smem, 0, st, p, ring.per, ring.stages, ring.pitch);
        }
      };
      auto with = [&](auto g, auto sum) {
        constexpr int G = decltype(g)::value;
        constexpr bool SUM = decltype(sum)::value;
        go(tgb::layernorm_backward_kernel<T, G, A, SUM>, tgb::layernorm_backward_ring_kernel<T, G, A, SUM>);
      };
      const bool one = (ring.fits ? ring.groups : r.groups) == 1;
      using One = std::integral_constant<int, 1>;
      using Two = std::integral_constant<int, 2>;
      if (p.residual && one) with(One{}, std::true_type{});
      else if (p.residual) with(Two{}, std::true_type{});
      else if (one) with(One{}, std::false_type{});
      else with(Two{}, std::false_type{});
    });
  }
  if (scratch && s == TG_OK)
    launch_kernel(tgb::layernorm_join_kernel<T>, dim3(unsigned((p.cols + 31) / 32), grad_w && grad_b ? 2 : 1), 1024, 0, 0, st, p.slots, p.cols, p.partial_w, p.partial_b, grad_w, grad_b);
  if (s == TG_OK) s = check_launch("layernorm backward");
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

tg_status tg_layernorm_residual_backward(tg_dtype dtype, int64_t rows, int64_t cols, const void* grad, int64_t ldg, const void* grad_h,
                                         int64_t ldgh, const void* weight, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                         const float* mean, const float* rstd, void* grad_x, int64_t ldgx, void* grad_weight, void* grad_bias,
                                         void* stream) {
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
  if (!grad || !x || !mean || !rstd) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TG_CHECK(check_pitch("ldg", grad, ldg, cols));
  TG_CHECK(check_pitch("ldgh", grad_h, ldgh, cols));
  TG_CHECK(check_pitch(residual ? "ldx" : "ldh", x, ldx, cols));
  TG_CHECK(check_pitch("ldr", residual, ldr, cols));
  TG_CHECK(check_pitch(residual ? "ldgx" : "ldx", grad_x, ldgx, cols));
  NormBackArgs p{};
  p.rows = rows; p.cols = cols; p.grad = grad; p.ldg = ldg; p.grad_h = grad_h; p.ldgh = ldgh; p.weight = weight;
  p.h = x; p.ldh = ldx; p.residual = residual; p.ldr = ldr; p.mean = mean; p.rstd = rstd; p.grad_x = grad_x; p.ldx = ldgx;
  const size_t e = elem8_size(dtype);
  RowAccess access(cols);
  access.add(grad, ldg, e);
  access.add(grad_h, ldgh, e);
  access.add(x, ldx, e);
  access.add(residual, ldr, e);
  access.add(grad_x, ldgx, e);
  int how = access.get();
  if (how == tg8::kAligned && !aligned(weight, 16)) how = tg8::kScalar;
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    return launch_backward<T>(p, static_cast<T*>(grad_weight), static_cast<T*>(grad_bias), how, st);
  });
}

tg_status tg_layernorm_backward(tg_dtype dtype, int64_t rows, int64_t cols, const void* grad, int64_t ldg, const void* grad_h,
                                int64_t ldgh, const void* weight, const void* h, int64_t ldh, const float* mean,
                                const float* rstd, void* grad_x, int64_t ldx, void* grad_weight, void* grad_bias, void* stream) {
  return tg_layernorm_residual_backward(dtype, rows, cols, grad, ldg, grad_h, ldgh, weight, h, ldh, nullptr, 0, mean, rstd, grad_x, ldx, grad_weight,
                                        grad_bias, stream);
}

}  // extern "C"
