// The tensor-core kernel of the 8-bit row products.
//
//   forward    C[i,j]   = a_scale[i] b_scale[j] sum_k A[i,k] B[j,k] + bias[j]
//              8-bit integer products, 32-bit integer sums: exact.
//   backward   out[p,c] = sum_i g(p,i) scale[i] q[i,c]
//              bf16 products, f32 sums; the 8-bit operand is expanded to bf16
//              on its way to the tensor core, so it is read as bytes.
//
// Both: a pair of CTAs on two SMs computes 256 x 256 outputs (one tcgen05.mma
// covers both), CTA r holding rows 128 r .. 128 r + 127 of the left operand
// and half of the right one.  The sum advances by 128 bytes of each left row
// per stage of a TMA ring; two 256-column accumulators in tensor memory let
// the epilogue of one tile run under the products of the next.  Persistent:
// a pair walks tiles in groups of row panels, so what it reads stays in L2.
#pragma once
#include "tg_rows8.cuh"
#include "tg_umma.cuh"

namespace tg8 {

enum ProductMode { kForward = 0, kBackRows = 1, kBackCols = 2 };   // Back: g's sum index contiguous, or g's outer one

struct ProductArgs {
  int64_t m, n, ldc;          // outputs
  void* c;
  const float *row_scale, *col_scale;   // forward
  const void* bias;                     // forward, or null
  const float* sum_scale;     // backward: one factor per index of the sum, or null (taken into g)
  int sum;                    // length of the sum (of one plane)
  int blocks, planes;         // stages per plane, planes of g
  int tiles_m, tiles_n;
  int vec;                    // 16-byte stores of C's rows
};

constexpr int kTile = 256, kHalf = 128;
constexpr int kStageA = 16384, kStageB = 16384, kStageRaw = 8192;
constexpr int kEpiWarps = 4, kConvWarps = 4;
constexpr int kEpiPitch = 33;

template <int MODE> struct ProductShape {
  static constexpr bool kBack = MODE != kForward;
  static constexpr int kStages = kBack ? 5 : 6;
  static constexpr int kStage = kStageA + kStageB + (kBack ? kStageRaw : 0);
  static constexpr int kThreads = 32 * (4 + kEpiWarps + (kBack ? kConvWarps : 0));
  static constexpr int kOffStaging = kStages * kStage;
  static constexpr int kOffCols = kOffStaging + kEpiWarps * 32 * kEpiPitch * 4;   // b_scale, bias of the tile
  static constexpr int kOffBars = kOffCols + (kBack ? 0 : 2 * kTile * 4);
  static constexpr int kBars = 4 * kStages + 4;
  static constexpr int kOffSlot = kOffBars + kBars * 8;
  static constexpr int kSmem = kOffSlot + 16 + 1024;   // the ring starts on a 1024-byte boundary
};

// Tile t of the walk: groups of 8 row panels, columns outside rows in a group.
__device__ __forceinline__ void tile_at(const ProductArgs& p, int t, int64_t& m0, int64_t& n0) {
  constexpr int kGroup = 8;
  const int per = kGroup * p.tiles_n, g = t / per, first = g * kGroup, rows = min(kGroup, p.tiles_m - first);
  const int in = t - g * per;
  m0 = int64_t(first + in % rows) * kTile;
  n0 = int64_t(in / rows) * kTile;
}

// One row of 32 outputs in the row's own thread, or through shared memory by
// rows when C's rows are not 16-byte aligned or end inside.
template <typename T>
__device__ __forceinline__ void store_rows32(const ProductArgs& p, const float (&z)[32], float* staging, int lane,
                                             int64_t row0, int64_t col) {
  if (p.vec && col + 32 <= p.n) {
    const int64_t row = row0 + lane;
    if (row < p.m) {
      T* c = static_cast<T*>(p.c) + row * p.ldc + col;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = z[8 * i + e];
        store8(c + 8 * i, v);
      }
    }
    return;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; i++) staging[lane * kEpiPitch + i] = z[i];
  __syncwarp();
  if (col + lane < p.n) {
    const int rows = int(min(int64_t(32), p.m - row0));
    T* c = static_cast<T*>(p.c) + row0 * p.ldc + col + lane;
    for (int r = 0; r < rows; r++) c[r * p.ldc] = from_f32<T>(staging[r * kEpiPitch + lane]);
  }
}

template <int MODE, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(ProductShape<MODE>::kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const ProductArgs p) {
  using S = ProductShape<MODE>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (umma::smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - umma::smem_u32(smem_raw));
  const uint32_t bars = base + S::kOffBars;
  auto full = [&](int s) { return bars + 8 * s; };                       // A and B landed (leader)
  auto empty = [&](int s) { return bars + 8 * (S::kStages + s); };       // products that read the stage are done
  auto raw = [&](int s) { return bars + 8 * (2 * S::kStages + s); };     // 8-bit tile landed (each CTA)
  auto conv = [&](int s) { return bars + 8 * (3 * S::kStages + s); };    // expanded in both CTAs (leader)
  auto acc_full = [&](int b) { return bars + 8 * (4 * S::kStages + b); };
  auto acc_empty = [&](int b) { return bars + 8 * (4 * S::kStages + 2 + b); };   // (leader)
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + S::kOffSlot);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = umma::cta_rank();
  const int tiles = p.tiles_m * p.tiles_n, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int steps = p.blocks * p.planes;

  if (warp == 0 && lane == 0) {
    umma::tma_prefetch(&map_a);
    umma::tma_prefetch(&map_b);
    for (int s = 0; s < S::kStages; s++) {
      umma::bar_init(full(s), 1);
      umma::bar_init(empty(s), 1);
      umma::bar_init(raw(s), 1);
      umma::bar_init(conv(s), 2 * kConvWarps);
    }
    for (int b = 0; b < 2; b++) {
      umma::bar_init(acc_full(b), 1);
      umma::bar_init(acc_empty(b), 2 * kEpiWarps);
    }
    umma::bar_init_fence();
  }
  if (warp == 2) umma::tmem_alloc<2>(base + S::kOffSlot, 512);
  umma::fence_before();
  umma::cluster_sync();
  umma::fence_after();
  const uint32_t tmem = *slot;
  bool ok = true;   // false once a wait of this role ran out

  if (warp == 0) {
    // ---- producer: this CTA's half of each operand
    if (lane == 0) {
      int it = 0;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int64_t m0, n0;
        tile_at(p, t, m0, n0);
        const int row = int(m0) + int(rank) * kHalf, col = int(n0) + int(rank) * kHalf;
        for (int step = 0; step < steps; step++, it++) {
          const int s = it % S::kStages;
          if (!umma::bar_wait(empty(s), ((it / S::kStages) & 1) ^ 1)) { ok = false; break; }
          const uint32_t a = base + s * S::kStage, b = a + kStageA;
          const uint32_t bar = umma::map_rank(full(s), 0);
          if (rank == 0) umma::bar_expect(full(s), S::kBack ? 2 * kStageA : 2 * (kStageA + kStageB));
          if (MODE == kForward) {
            umma::tma_load_3d_pair(a, &map_a, step * 128, row, 0, bar);
            umma::tma_load_3d_pair(b, &map_b, step * 128, col, 0, bar);
          } else {
            const int plane = step / p.blocks, r0 = (step - plane * p.blocks) * 64;
            if (MODE == kBackRows) {
              umma::tma_load_3d_pair(a, &map_a, r0, row, plane, bar);
            } else {
              umma::tma_load_3d_pair(a, &map_a, row, r0, plane, bar);
              umma::tma_load_3d_pair(a + kStageA / 2, &map_a, row + 64, r0, plane, bar);
            }
            umma::bar_expect(raw(s), kStageRaw);
            umma::tma_load_3d_pair(b + kStageB, &map_b, col, r0, 0, umma::map_rank(raw(s), rank));
          }
        }
      }
      if (!ok) umma::drain_copies();
    }
  } else if (warp == 1) {
    // ---- products, issued by one thread of the leader for both SMs
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = MODE == kForward ? umma::instr_desc(2, 1, false, false, kTile, kTile)
                                                  : umma::instr_desc(1, 1, MODE == kBackCols, true, kTile, kTile);
      // bytes from one instruction's slice of the sum to the next: 32 along a
      // 128-byte row, or 16 rows
      constexpr uint32_t step_a = MODE == kBackCols ? 2048 : 32, step_b = MODE == kForward ? 32 : 2048;
      int it = 0, n = 0;
      for (int t = pair; t < tiles && ok; t += pairs, n++) {
        const int buf = n & 1;
        if (!umma::bar_wait(acc_empty(buf), ((n >> 1) & 1) ^ 1)) { ok = false; break; }
        umma::fence_after();
        for (int step = 0; step < steps; step++, it++) {
          const int s = it % S::kStages;
          const uint32_t parity = (it / S::kStages) & 1;
          if (!umma::bar_wait(full(s), parity) || (S::kBack && !umma::bar_wait(conv(s), parity))) { ok = false; break; }
          umma::fence_after();
          const uint32_t a = base + s * S::kStage, b = a + kStageA;
          // contiguous along the sum: 8-row groups 1024 bytes apart; else
          // 64-wide columns of 64 rows 8192 bytes apart
          const uint64_t da = umma::smem_desc(a, MODE == kBackCols ? 8192 : 16, 1024);
          const uint64_t db = umma::smem_desc(b, S::kBack ? 8192 : 16, 1024);
#pragma unroll
          for (int i = 0; i < 4; i++)
            umma::mma<2, MODE == kForward>(tmem + buf * kTile, da + (i * step_a >> 4), db + (i * step_b >> 4), idesc, step | i);
          umma::mma_commit<2>(empty(s));
        }
        if (ok) umma::mma_commit<2>(acc_full(buf));
      }
      if (!ok) umma::drain_copies();
    }
  } else if (warp >= 4 && warp < 4 + kEpiWarps) {
    // ---- epilogue: warp w reads lanes 32 w .. 32 w + 31 of tensor memory
    const int w = warp - 4, tid = threadIdx.x - 128;
    float* staging = reinterpret_cast<float*>(smem + S::kOffStaging) + w * 32 * kEpiPitch;
    float* cols = reinterpret_cast<float*>(smem + S::kOffCols);
    int n = 0;
    for (int t = pair; t < tiles; t += pairs, n++) {
      int64_t m0, n0;
      tile_at(p, t, m0, n0);
      const int buf = n & 1;
      const int64_t row0 = m0 + rank * kHalf + w * 32, row = row0 + lane;
      float rs = 0.f;
      if (MODE == kForward) {
        asm volatile("bar.sync 1, 128;" ::: "memory");   // the last tile's columns are no longer read
        for (int i = tid; i < kTile; i += 128) {
          const bool in = n0 + i < p.n;
          cols[i] = in ? p.col_scale[n0 + i] : 0.f;
          cols[kTile + i] = in && p.bias ? to_f32(static_cast<const T*>(p.bias)[n0 + i]) : 0.f;
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (row < p.m) rs = p.row_scale[row];
      }
      if (ok && !umma::bar_wait(acc_full(buf), (n >> 1) & 1)) ok = false;
      umma::fence_after();
      for (int c = 0; c < kTile; c += 32) {
        uint32_t acc[32];
        float z[32];
        umma::tmem_load32(tmem + buf * kTile + c + (uint32_t(w * 32) << 16), acc);
        umma::tmem_load_wait();
        if (c + 32 == kTile) {   // read out: the next tile's products may have the accumulator
          umma::fence_before();
          __syncwarp();
          if (lane == 0) umma::bar_arrive_cluster(umma::map_rank(acc_empty(buf), 0));
        }
        if (n0 + c >= p.n) continue;
#pragma unroll
        for (int i = 0; i < 32; i++) {
          if (MODE == kForward) {
            z[i] = float(int(acc[i])) * rs * cols[c + i] + (p.bias ? cols[kTile + c + i] : 0.f);
          } else {
            z[i] = __uint_as_float(acc[i]);
          }
          if (!ok) z[i] = __uint_as_float(0x7fffffffu);   // a wait ran out: the outputs say so
        }
        store_rows32<T>(p, z, staging, lane, row0, n0 + c);
      }
    }
    if (!ok) umma::drain_copies();
  } else if (S::kBack && warp >= 4 + kEpiWarps) {
    // ---- 8-bit tile (64 of the sum x 128 columns) to bf16, 128-byte swizzled
    // columns of 64.  Lanes 0-7 take eight rows of one 16-byte chunk: the
    // swizzle spreads them over all banks on both sides.
    const int w = warp - 4 - kEpiWarps, r8 = lane & 7, c4 = lane >> 3;
    const uint32_t out0 = base + kStageA, in0 = out0 + kStageB;
    int it = 0;
    for (int t = pair; t < tiles && ok; t += pairs) {
      for (int step = 0; step < steps; step++, it++) {
        const int s = it % S::kStages;
        const int r0 = (step % p.blocks) * 64 + w * 16 + r8;
        float sc[2];
#pragma unroll
        for (int i = 0; i < 2; i++) sc[i] = p.sum_scale ? (r0 + 8 * i < p.sum ? p.sum_scale[r0 + 8 * i] : 0.f) : 1.f;
        if (!umma::bar_wait(raw(s), (it / S::kStages) & 1)) { ok = false; break; }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int r = w * 16 + i * 8 + r8;
#pragma unroll
          for (int j = 0; j < 2; j++) {
            uint32_t q[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3])
                         : "r"(in0 + s * S::kStage + r * 128 + (((j * 4 + c4) ^ r8) << 4)));
            uint32_t o[8];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const uint32_t x = q[k] ^ 0x80808080u;
              const __nv_bfloat162 lo = __floats2bfloat162_rn(byte_f32<0>(x) * sc[i], byte_f32<1>(x) * sc[i]);
              const __nv_bfloat162 hi = __floats2bfloat162_rn(byte_f32<2>(x) * sc[i], byte_f32<3>(x) * sc[i]);
              o[2 * k] = *reinterpret_cast<const uint32_t*>(&lo);
              o[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&hi);
            }
#pragma unroll
            for (int k = 0; k < 2; k++)
              asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(out0 + s * S::kStage + j * 8192 + r * 128 + (((2 * c4 + k) ^ r8) << 4)),
                           "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]), "r"(o[4 * k + 3]) : "memory");
          }
        }
        umma::fence_async_smem();
        __syncwarp();
        if (lane == 0) umma::bar_arrive_cluster(umma::map_rank(conv(s), 0));
      }
    }
  }

  __syncwarp();
  umma::fence_before();
  umma::cluster_sync();
  if (warp == 2) {
    umma::fence_after();
    umma::tmem_free<2>(tmem, 512);
  }
}

// g * scale (scale null: g) in `planes` bf16 parts, each padded to rows of
// ldo: parts 0 .. planes - 1 from the smallest to the largest, so that the
// sums take the small ones first.  The upper parts are truncations, which
// leaves an exact rest: three parts hold all 24 bits, two hold 16 rounded.
template <typename GT>
__global__ void __launch_bounds__(256) split_kernel(int64_t rows, int64_t cols, const GT* g, int64_t ldg, const float* scale,
                                                    int scale_rows, bf16* out, int64_t ldo, int planes) {
  const int64_t c = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (c >= ldo) return;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    float v = 0.f;
    if (c < cols) {
      v = to_f32(g[r * ldg + c]);
      if (scale) v *= scale[scale_rows ? r : c];
    }
    const bool finite = fabsf(v) < __uint_as_float(0x7f800000u);
    for (int i = planes - 1; i >= 0; i--) {
      const uint32_t bits = __float_as_uint(v) & 0xffff0000u;
      bf16 part = i && finite ? __ushort_as_bfloat16(uint16_t(bits >> 16)) : __float2bfloat16_rn(v);
      out[(int64_t(i) * rows + r) * ldo + c] = part;
      v = finite ? v - __bfloat162float(part) : 0.f;
    }
  }
}

// 8-bit rows copied to rows of ldo, a multiple of 16, zeros behind.
__global__ void __launch_bounds__(256) pad8_kernel(int64_t rows, int64_t cols, const int8_t* q, int64_t ldq, int8_t* out, int64_t ldo) {
  const int64_t c = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (c >= ldo) return;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (c + e < cols) v |= uint32_t(uint8_t(q[r * ldq + c + e])) << (8 * e);
    *reinterpret_cast<uint32_t*>(out + r * ldo + c) = v;
  }
}

}  // namespace tg8
