// The tensor-core kernels of products in 8-bit floating point with a scale for
// each block of 128 along the sum:
//
//   C[i,j] = sum_b a_scale(i,b) b_scale(j,b) sum_{k in b} A[i,k] B[j,k] + bias[j]
//
// A block is one step of 128 bytes per row: four products of 32 into an
// accumulator in tensor memory.  Where all scales are powers of two the tensor
// core applies them on the way in (pairs of CTAs) and the sum stays there;
// otherwise the epilogue warps take each block's sums out, scale them and add them
// to f32 sums in registers while the next block goes into another accumulator.
#pragma once
#include "tg_blocks8.cuh"
#include "tg_rows8_umma.cuh"
#include "tg_umma.cuh"

namespace tgb {

struct ProductArgs8 {
  int64_t m, n, ldc;          // outputs
  void* c;
  const void* bias;           // or null
  const float *a_scale, *b_scale;
  int64_t a_row, a_block, b_row, b_block;   // strides of the scales
  int blocks;                 // of the sum
  int tiles_m, tiles_n;       // tiles of 256 x 2 half_n
  int half_n;                 // columns of a tile per CTA: 128, or 64 for outputs of at most 128 columns
  int splits, split_blocks;   // the sum in parts, one pair each (1: whole); blocks per part
  float* part;                // sums of the parts, (splits x m x ldp)
  int64_t ldp;
  int vec;                    // 16-byte stores of C's rows
  // scales that are powers of two, packed for the tensor core (pack_scales_kernel)
  uint32_t *words_a, *words_b;   // (groups of 4 blocks) x (rows of A, of B, to whole tiles)
  int64_t pitch_a, pitch_b;
  int* other;                 // kPackBlocks flags: some scale is not a power of two
  int chunk;                  // blocks that the tensor core may sum (scaled kernel)
};

// Two pairs from shared memory.
__device__ __forceinline__ void load_pairs(uint32_t from, uint64_t& a, uint64_t& b) {
  asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(from));
}

// ------------------------------------------------------------------------------- scales that are powers of two
// Exponents of four blocks' scales per word, and whether all scales are powers of
// two (from 2^-126 on) or NaN.  Rows past the last get zeros.
constexpr int kPackBlocks = 256;
static __global__ void __launch_bounds__(256) pack_scales_kernel(const ProductArgs8 p, int b_tall) {
  after_previous_kernel();
  const int64_t groups = (p.blocks + 3) / 4, total_a = groups * p.pitch_a, total = total_a + groups * p.pitch_b;
  bool bad = false;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const bool is_a = i < total_a;
    const int64_t at = is_a ? i : i - total_a, pitch = is_a ? p.pitch_a : p.pitch_b, g = at / pitch, r = at - g * pitch;
    uint32_t w = 0;
    if (r < (is_a ? p.m : p.n)) {
      const float* s = is_a ? p.a_scale + r * p.a_row : p.b_scale + r / b_tall * p.b_row;
      const int64_t step = is_a ? p.a_block : p.b_block;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (g * 4 + j >= p.blocks) break;
        const uint32_t bits = __float_as_uint(s[(g * 4 + j) * step]);
        uint32_t e = bits >> 23;   // 255: NaN
        if ((bits & 0x7fffffffu) > 0x7f800000u) e = 255;
        else if (bits & 0x007fffffu || e == 0 || e >= 255) bad = true;
        w |= (e & 255) << (8 * j);
      }
    }
    (is_a ? p.words_a : p.words_b)[at] = w;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) p.other[blockIdx.x] = bad;
}
// Whether some scale is not a power of two: the same in all threads.
__device__ __forceinline__ bool other_scales(const int* other) { return __syncthreads_or(threadIdx.x < kPackBlocks && other[threadIdx.x]); }

// ------------------------------------------------------------------------------- pairs of CTAs, tiles of 256 x 256
// Persistent; CTA r of a pair holds rows 128 r .. of A's tile and half of B's.
//
// Scales that are powers of two the tensor core applies itself, from tensor
// memory, and the sum stays there.  Warps 4-7 bring them: four blocks' exponents
// are one word per row, of which a CTA takes its 128 rows of A and all 256 of B
// to each quarter of the lanes of its own tensor memory, in four slots in turn.
// One accumulator of 256 columns fits beside them: a tile's sum is taken to
// registers before the next one begins (about 1000 cycles; a tile of 8192 takes
// 33000).  The tensor core's f32 sums lose in proportion to their length, so they
// are taken out and added up in f32 every `chunk` blocks.
//
// With other scales each block goes into an accumulator of its own, of two in
// turn, which the epilogue scales and adds up: a hand-over of 800 cycles and 500
// of reads and arithmetic per block of 512, so this takes about twice as long
// (8192^3 bf16: 0.39 and 0.76 ms), and with a scale for each of B's rows, which is
// read from shared memory and multiplied for each output and block, 1.76 ms.
//
// What bounds it: power (8192^3 2.8 PFLOP/s, operands of zeros 3.8); 4096^3, 56 us, is
// 256 tiles on 74 pairs, four rounds for 3.46.
struct PairShape {
  static constexpr int kStages = 6, kStage = 2 * tg8::kOperand, kEpi = 8, kSlots = 4, kThreads = 512;
  static constexpr int kLow = 48, kHigh = 208;   // registers per thread of the first two warpgroups, and of the epilogue's two
  static constexpr int kOffStaging = kStages * kStage;
  static constexpr int kOffBias = kOffStaging + kEpi * tg8::kStagingBytes;
  static constexpr int kOffScales = kOffBias + 256 * 4;      // other scales, ROWS: per epilogue warp 128 column scales
  static constexpr int kOffBars = kOffScales + kEpi * 512;
  static constexpr int kBars = 2 * (kStages + kSlots + 2);
  static constexpr int kOffSlot = kOffBars + kBars * 8;
  static constexpr int kSmem = kOffSlot + 16 + 1024;
};
static_assert(PairShape::kSmem <= 227 * 1024, "shared memory");

struct PairItem {
  int64_t m0, n0;
  int b0, b1;
};
// Tile (or part of one) i of a pair's walk: groups of 8 row panels, columns outside rows.
__device__ __forceinline__ bool pair_item(const ProductArgs8& p, int pair, int pairs, int i, PairItem& it) {
  if (p.splits > 1) {
    const int tile = pair / p.splits, part = pair - tile * p.splits;
    it.m0 = int64_t(tile % p.tiles_m) * 256;
    it.n0 = int64_t(tile / p.tiles_m) * 2 * p.half_n;
    it.b0 = part * p.split_blocks;
    it.b1 = min(p.blocks, it.b0 + p.split_blocks);
    return i == 0;
  }
  it.b0 = 0;
  it.b1 = p.blocks;
  const int64_t t = pair + int64_t(i) * pairs;
  if (t >= int64_t(p.tiles_m) * p.tiles_n) return false;
  constexpr int kGroup = 8;
  const int64_t per = int64_t(kGroup) * p.tiles_n, g = t / per;
  const int first = int(g) * kGroup, rows = min(kGroup, p.tiles_m - first), in = int(t - g * per);
  it.m0 = int64_t(first + in % rows) * 256;
  it.n0 = int64_t(in / rows) * 2 * p.half_n;
  return true;
}

// ROWS: B has a scale per row and block; else per tile of 128 rows.
template <typename T, bool ROWS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairShape::kThreads, 1)
blocks_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const ProductArgs8 p) {
  using S = PairShape;
  using tg8::kOperand;
  after_previous_kernel();
  const bool other = other_scales(p.other);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (umma::smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - umma::smem_u32(smem_raw));
  const uint32_t bars = base + S::kOffBars;
  auto full = [&](int s) { return bars + 8 * s; };                              // operands in place in both CTAs (leader)
  auto empty = [&](int s) { return bars + 8 * (S::kStages + s); };              // products that read them are done (each CTA)
  auto scales_full = [&](int s) { return bars + 8 * (2 * S::kStages + s); };    // scales in both CTAs' tensor memory (leader)
  auto scales_empty = [&](int s) { return bars + 8 * (2 * S::kStages + S::kSlots + s); };   // and used (each CTA)
  auto acc_full = [&](int b) { return bars + 8 * (2 * S::kStages + 2 * S::kSlots + b); };       // sum done (each CTA)
  auto acc_empty = [&](int b) { return bars + 8 * (2 * S::kStages + 2 * S::kSlots + 2 + b); };   // and taken out in both CTAs (leader)
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + S::kOffSlot);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = umma::cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 0 && lane == 0) {
    umma::tma_prefetch(&map_a);
    umma::tma_prefetch(&map_b);
    for (int s = 0; s < S::kStages; s++) {
      umma::bar_init(full(s), 1);
      umma::bar_init(empty(s), 1);
    }
    for (int s = 0; s < S::kSlots; s++) {
      umma::bar_init(scales_full(s), 8);
      umma::bar_init(scales_empty(s), 1);
    }
    for (int b = 0; b < 2; b++) {
      umma::bar_init(acc_full(b), 1);
      umma::bar_init(acc_empty(b), 2 * S::kEpi);
    }
    umma::bar_init_fence();
  }
  if (warp == 2) umma::tmem_alloc<2>(base + S::kOffSlot, 512);
  umma::fence_before();
  umma::cluster_sync();
  umma::fence_after();
  const uint32_t tmem = *slot, scales = tmem + 256;   // slot s: A's 4 columns at scales + 16 s, B's 8 behind them
  bool ok = true;   // false once a wait of this role ran out

  if (warp < 4) {
    umma::registers_down<S::kLow>();
    const bool issue = umma::elect_one();
    tg8::RingAt<S::kStages> at;
    PairItem item;
    if (warp == 0) {
      // ---- producer: this CTA's half of each operand
      for (int i = 0; ok && pair_item(p, pair, pairs, i, item); i++) {
        const int row = int(item.m0) + int(rank) * 128, col = int(item.n0) + int(rank) * p.half_n;
        for (int b = item.b0; b < item.b1; b++, at.next()) {
          if (!umma::bar_wait(empty(at.slot), at.parity ^ 1)) { ok = false; break; }
          const uint32_t to = base + at.slot * S::kStage, bar = umma::map_rank(full(at.slot), 0);
          if (issue) {
            if (rank == 0) umma::bar_expect(full(at.slot), 4 * kOperand);
            umma::tma_load_3d_pair(to, &map_b, b * 128, col, 0, bar);
            umma::tma_load_3d_pair(to + kOperand, &map_a, b * 128, row, 0, bar);
          }
        }
      }
      if (!ok) umma::drain_copies();
    } else if (warp == 1 && rank == 0) {
      // ---- products, issued by one thread of the leader for both SMs
      const uint64_t db0 = umma::smem_desc(base, 16, 1024), da0 = umma::smem_desc(base + kOperand, 16, 1024);
      uint32_t n = 0;   // sums so far
      if (other) {      // sum n, one block, goes into accumulator n % 2
        const uint32_t idesc = umma::instr_desc(1, 0, false, false, 256, 2 * p.half_n);
        for (int i = 0; ok && pair_item(p, pair, pairs, i, item); i++) {
          for (int b = item.b0; b < item.b1; b++, at.next(), n++) {
            const uint32_t buf = n & 1;
            if (!umma::bar_wait(full(at.slot), at.parity) || !umma::bar_wait<true>(acc_empty(buf), ((n >> 1) & 1) ^ 1)) { ok = false; break; }
            umma::fence_after();
            const uint32_t off = at.slot * (S::kStage >> 4);
            if (issue) {
#pragma unroll
              for (int j = 0; j < 4; j++) umma::mma_f8<2>(tmem + buf * 256, da0 + (off + j * 2), db0 + (off + j * 2), idesc, j > 0);
              umma::mma_commit<2>(empty(at.slot));
              umma::mma_commit<2>(acc_full(buf));
            }
          }
          __syncwarp();
        }
      } else {
        const uint32_t idesc = umma::instr_desc_scaled(256, 2 * p.half_n);
        tg8::RingAt<S::kSlots> sc;
        for (int i = 0; ok && pair_item(p, pair, pairs, i, item); i++) {
          int left = 0;   // of the chunk
          for (int b = item.b0; ok && b < item.b1; b += 4) {   // four blocks with one slot of scales
            if (!umma::bar_wait<true>(scales_full(sc.slot), sc.parity)) { ok = false; break; }
            const uint32_t sa = scales + 16 * sc.slot;
            const int blocks = min(4, item.b1 - b);
#pragma unroll
            for (int j = 0; j < 4; j++) {
              if (j >= blocks) break;
              const bool first = left == 0;
              if (first) {
                left = min(p.chunk, item.b1 - (b + j));
                if (!umma::bar_wait<true>(acc_empty(0), (n & 1) ^ 1)) { ok = false; break; }
              }
              if (!umma::bar_wait(full(at.slot), at.parity)) { ok = false; break; }
              umma::fence_after();
              left--;
              const uint32_t off = at.slot * (S::kStage >> 4), id = idesc | umma::scale_byte(j);
              if (issue) {
#pragma unroll
                for (int q = 0; q < 4; q++) umma::mma_f8_scaled(tmem, da0 + (off + q * 2), db0 + (off + q * 2), id, sa, sa + 4, !first || q);
                umma::mma_commit<2>(empty(at.slot));
                if (j + 1 == blocks) umma::mma_commit<2>(scales_empty(sc.slot));
                if (left == 0) umma::mma_commit<2>(acc_full(0));
              }
              if (left == 0) n++;
              at.next();
            }
            sc.next();
          }
          __syncwarp();
        }
      }
      if (!ok) umma::drain_copies();
    }
  } else if (warp < 8) {
    umma::registers_down<S::kLow>();
    // ---- scales: each warp writes all of this CTA's to its quarter of the lanes
    const uint32_t quarter = scales + (uint32_t((warp & 3) * 32) << 16);
    tg8::RingAt<S::kSlots> sc;
    PairItem item;
    for (int i = 0; ok && !other && pair_item(p, pair, pairs, i, item); i++) {
      const int g1 = (item.b1 - 1) / 4;   // item.b0 is a multiple of 4
      const uint32_t *wa = p.words_a + item.m0 + rank * 128 + lane, *wb = p.words_b + item.n0 + lane;
      uint32_t a[4], b[8];
      auto load = [&](int64_t g) {
#pragma unroll
        for (int j = 0; j < 4; j++) a[j] = wa[g * p.pitch_a + 32 * j];
#pragma unroll
        for (int j = 0; j < 8; j++) b[j] = j < 4 || p.half_n == 128 ? wb[g * p.pitch_b + 32 * j] : 0u;
      };
      load(item.b0 / 4);
      for (int g = item.b0 / 4; g <= g1; g++, sc.next()) {
        if (!umma::bar_wait(scales_empty(sc.slot), sc.parity ^ 1)) { ok = false; break; }
        umma::fence_after();
        umma::tmem_store4(quarter + 16 * sc.slot, a);
        umma::tmem_store8(quarter + 16 * sc.slot + 4, b);
        if (g < g1) load(g + 1);
        umma::tmem_store_wait();
        umma::fence_before();
        __syncwarp();
        if (lane == 0) umma::bar_arrive_cluster(umma::map_rank(scales_full(sc.slot), 0));
      }
    }
    if (!ok) umma::drain_copies();
  } else {
    umma::registers_up<S::kHigh>();
    // ---- epilogue: warp w has lanes 32 (w % 4) .. of tensor memory and one half of the columns
    const int w = warp & 3, half = (warp - 8) >> 2, tid = threadIdx.x - 256;
    const uint32_t staging = base + S::kOffStaging + (warp - 8) * tg8::kStagingBytes;
    float* bias = reinterpret_cast<float*>(smem + S::kOffBias);
    const int columns = min(128, 2 * p.half_n - half * 128);   // of this warp's half: none in narrow tiles' second
    const uint32_t from = tmem + half * 128 + (uint32_t(w * 32) << 16);
    PairItem item;
    uint32_t n = 0;
    for (int i = 0; pair_item(p, pair, pairs, i, item); i++) {
      const int64_t row0 = item.m0 + rank * 128 + w * 32, col0 = item.n0 + half * 128;
      const bool parts = p.splits > 1;
      if (!parts) {
        named_sync(1, 256);   // the last tile's bias is no longer read
        bias[tid] = p.bias && item.n0 + tid < p.n ? to_f32(static_cast<const T*>(p.bias)[item.n0 + tid]) : 0.f;
        named_sync(1, 256);
      }
      float acc[128];
      auto taken = [&](int buf) {   // the next sum may have the accumulator
        umma::fence_before();
        __syncwarp();
        if (lane == 0) umma::bar_arrive_cluster(umma::map_rank(acc_empty(buf), 0));
      };
      if (!other) {
        for (int b = item.b0; b < item.b1; b += p.chunk, n++) {
          for (int k = 0; ok; k++) {   // a whole sum: the limit grows with its length
            if (umma::bar_wait(acc_full(0), n & 1)) break;
            if (k >= min(p.chunk, item.b1 - b) >> 10) ok = false;
          }
          umma::fence_after();
          if (columns > 0 && b == item.b0) {
#pragma unroll
            for (int c = 0; c < 128; c += 32) umma::tmem_load32(from + c, reinterpret_cast<uint32_t(&)[32]>(acc[c]));
            umma::tmem_load_wait();
          } else if (columns > 0) {
#pragma unroll
            for (int c = 0; c < 128; c += 16) {
              uint32_t t[16];
              umma::tmem_load16(from + c, t);
              umma::tmem_load_wait();
#pragma unroll
              for (int e = 0; e < 16; e++) acc[c + e] += __uint_as_float(t[e]);
            }
          }
          taken(0);
        }
      } else {
        const int64_t row = row0 + lane;
        const bool live = row < p.m && col0 < p.n && columns > 0;
        const float* sa = p.a_scale + (live ? row : 0) * p.a_row;
        const float* sb = p.b_scale + (col0 < p.n ? (ROWS ? col0 : col0 / kBlock) : 0) * p.b_row;
        const uint32_t mine = base + S::kOffScales + (warp - 8) * 512;
#pragma unroll
        for (int c = 0; c < 128; c++) acc[c] = 0.f;
#pragma unroll 1
        for (int b = item.b0; b < item.b1; b++, n++) {
          const uint32_t buf = n & 1;
          float s = live ? sa[b * p.a_block] : 0.f;
          if (ROWS) {
            __syncwarp();   // the last block's are read
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int64_t col = lane + 32 * j;
              const float v = col < columns && col0 + col < p.n ? sb[col * p.b_row + b * p.b_block] : 0.f;
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + uint32_t(col) * 4), "f"(v) : "memory");
            }
            __syncwarp();
          } else if (live) {
            s *= sb[b * p.b_block];
          }
          if (ok) ok = umma::bar_wait(acc_full(buf), (n >> 1) & 1);
          umma::fence_after();
          if (columns > 0) {
#pragma unroll
            for (int c = 0; c < 128; c += 16) {
              uint32_t t[16];
              umma::tmem_load16(from + buf * 256 + c, t);
              umma::tmem_load_wait();
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                float k[4] = {1.f, 1.f, 1.f, 1.f};
                if (ROWS) asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(k[0]), "=f"(k[1]), "=f"(k[2]), "=f"(k[3]) : "r"(mine + (c + e) * 4));
#pragma unroll
                for (int q = 0; q < 4; q++) acc[c + e + q] = fmaf(__uint_as_float(t[e + q]), ROWS ? s * k[q] : s, acc[c + e + q]);   // the scales first: a sum of 2^24 and one scale may pass f32's range
              }
            }
          }
          taken(buf);
        }
      }
      if (columns <= 0) continue;
      const int rows = int(max(int64_t(0), min(int64_t(32), p.m - row0)));
#pragma unroll
      for (int c = 0; c < 128; c += 16) {
        if (c >= columns || col0 + c >= p.n) break;
        uint32_t z[16];
        if (parts || sizeof(T) == 4) {   // 16 columns
#pragma unroll
          for (int e = 0; e < 16; e++) z[e] = ok ? __float_as_uint(parts ? acc[c + e] : acc[c + e] + bias[half * 128 + c + e]) : 0x7fffffffu;   // a wait ran out: the outputs say so
          if (parts) tg8::store_rows64(p.part + (int64_t(pair % p.splits) * p.m + row0) * p.ldp + col0 + c, p.ldp, rows, p.ldp - col0 - c, true, z, staging, lane);
          else if constexpr (sizeof(T) == 4) tg8::store_rows64(static_cast<T*>(p.c) + row0 * p.ldc + col0 + c, p.ldc, rows, p.n - col0 - c, p.vec, z, staging, lane);
        } else if constexpr (sizeof(T) == 2) {   // 32 columns
          if (c % 32) continue;
#pragma unroll
          for (int e = 0; e < 16; e++) {
            float x = acc[c + 2 * e] + bias[half * 128 + c + 2 * e], y = acc[c + 2 * e + 1] + bias[half * 128 + c + 2 * e + 1];
            if (!ok) x = y = __uint_as_float(0x7fffffffu);
            z[e] = tg8::pack_pair<T>(x, y);
          }
          tg8::store_rows64(static_cast<T*>(p.c) + row0 * p.ldc + col0 + c, p.ldc, rows, p.n - col0 - c, p.vec, z, staging, lane);
        }
      }
    }
    if (!ok) umma::drain_copies();
  }

  __syncwarp();
  umma::fence_before();
  umma::cluster_sync();
  if (warp == 2) {
    umma::fence_after();
    umma::tmem_free<2>(tmem, 512);
  }
}

// Adds up the parts of a sum, in order, and the bias.  Four columns per thread.
template <typename T>
__global__ void __launch_bounds__(256) blocks_join_kernel(const ProductArgs8 p) {
  after_previous_kernel();
  const int64_t c0 = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (c0 >= p.n) return;
  for (int64_t row = blockIdx.y; row < p.m; row += gridDim.y) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < p.splits; i++) {
      const float4 v = *reinterpret_cast<const float4*>(p.part + (int64_t(i) * p.m + row) * p.ldp + c0);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float z[4] = {s.x, s.y, s.z, s.w};
    T* c = static_cast<T*>(p.c) + row * p.ldc + c0;
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (c0 + e < p.n) c[e] = from_f32<T>(z[e] + (p.bias ? to_f32(static_cast<const T*>(p.bias)[c0 + e]) : 0.f));
  }
}

// A sum of nothing: the bias, or zeros.
template <typename T>
__global__ void __launch_bounds__(256) blocks_bias_kernel(const ProductArgs8 p) {
  after_previous_kernel();
  const int64_t col = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (col >= p.n) return;
  const T v = p.bias ? static_cast<const T*>(p.bias)[col] : from_f32<T>(0.f);
  for (int64_t row = blockIdx.y; row < p.m; row += gridDim.y) static_cast<T*>(p.c)[row * p.ldc + col] = v;
}

// ------------------------------------------------------------------------------- few tokens
// What few tokens have to do is read the weights once, so the roles are
// swapped: 128 rows of B are the tensor core's rows and NT tokens its columns;
// the sum is split over the S CTAs of a cluster (1 to 8), so that all SMs read.
// Each CTA finishes a share of the tokens: the others write their parts into its
// shared memory.  Four epilogue warps, one row of B per thread.
//
// What bounds it: launch and set-up where the weights are few (1 x 4096 x 4096
// 5.1 us, their read 2.6), then what an SM takes from memory: one step of 16 KB of
// weights per 0.22 us and CTA (16 x 8192 x 4096 8.1 us, floor 5.2).
//
// A CTA that waits for its cluster must not wait for tensor memory held by one
// that waits for another cluster: with split > 1 a CTA asks for more than half
// of an SM's shared memory, so no two of these share an SM; it takes at most 256
// of the 512 columns.  Nor must one that waits for the kernel before it hold what
// that one's CTAs still ask for: tensor memory is taken behind that wait.
template <int NT> struct FewShape {
  static constexpr int kStage = tg8::kOperand + NT * 128, kThreads = 192;
  static constexpr int kExchange = (NT < 32 ? 32 : NT) * 512;       // parts of this CTA's tokens (shares of 4) from the whole cluster
  static constexpr int kMost = (200 * 1024 - kExchange) / kStage;   // stages
  static constexpr int kBufs = NT <= 32 ? 8 : 256 / NT;             // accumulators
  static constexpr int kColumns = NT * kBufs;
  static constexpr int kBars = 2 * (kMost + kBufs);
  static constexpr int kAlone = 118 * 1024;                         // shared memory of which an SM has no two
};

template <int NT, typename T, bool ROWS>
__global__ void __launch_bounds__(192) blocks_few_kernel(const __grid_constant__ CUtensorMap map_tokens, const __grid_constant__ CUtensorMap map_weights,
                                                         const ProductArgs8 p, int split, int stages) {
  using S = FewShape<NT>;
  __shared__ __align__(8) uint64_t bar_store[S::kBars];
  __shared__ uint32_t slot;
  __shared__ __align__(16) float token_scales[4][2][NT];
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (umma::smem_u32(smem_raw) + 1023) & ~1023u, bars = umma::smem_u32(bar_store);
  const uint32_t exchange = base + stages * S::kStage;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (S::kMost + s); };
  auto acc_full = [&](int b) { return bars + 8 * (2 * S::kMost + b); };
  auto acc_empty = [&](int b) { return bars + 8 * (2 * S::kMost + S::kBufs + b); };
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % split;
  const int64_t n0 = int64_t(blockIdx.x / split) * 128;
  const int t0 = int(blockIdx.y) * NT, tokens = int(min(int64_t(NT), p.m - t0));
  const int first = rank * p.split_blocks, steps = max(0, min(p.split_blocks, p.blocks - first));   // the last CTAs may have no share

  if (warp == 0 && lane == 0) {
    umma::tma_prefetch(&map_weights);
    umma::tma_prefetch(&map_tokens);
    for (int s = 0; s < stages; s++) {
      umma::bar_init(full(s), 1);
      umma::bar_init(empty(s), 1);
    }
    for (int b = 0; b < S::kBufs; b++) {
      umma::bar_init(acc_full(b), 1);
      umma::bar_init(acc_empty(b), 4);
    }
    umma::bar_init_fence();
  }
  after_previous_kernel();
  if (warp == 1) umma::tmem_alloc<1>(umma::smem_u32(&slot), S::kColumns);
  umma::fence_before();
  __syncthreads();
  umma::fence_after();
  if (split > 1) umma::cluster_arrive();   // all of the cluster has started: waited for before the first store
  const uint32_t tmem = slot;
  bool ok = true;

  if (warp == 0) {
    const bool issue = umma::elect_one();
    int s = 0;
    uint32_t parity = 0;
    for (int i = 0; i < steps; i++) {
      if (!umma::bar_wait(empty(s), parity ^ 1)) { ok = false; break; }
      const uint32_t a = base + s * S::kStage;
      if (issue) {
        umma::bar_expect(full(s), S::kStage);
        umma::tma_load_3d(a, &map_weights, (first + i) * 128, int(n0), 0, full(s));
        umma::tma_load_3d(a + tg8::kOperand, &map_tokens, (first + i) * 128, t0, 0, full(s));
      }
      if (++s == stages) { s = 0; parity ^= 1; }
    }
    if (!ok) umma::drain_copies();
    __syncwarp();
    if (split > 1) {
      umma::cluster_wait();
      umma::cluster_sync();
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma::instr_desc(1, 0, false, false, 128, NT);
    const uint64_t da0 = umma::smem_desc(base, 16, 1024), db0 = umma::smem_desc(base + tg8::kOperand, 16, 1024);
    const bool issue = umma::elect_one();
    int s = 0, buf = 0;
    uint32_t parity = 0, turn = 0;
    for (int i = 0; i < steps; i++) {
      if (!umma::bar_wait(full(s), parity) || !umma::bar_wait(acc_empty(buf), turn ^ 1)) { ok = false; break; }
      umma::fence_after();
      const uint32_t off = s * (S::kStage >> 4);
      if (issue) {
#pragma unroll
        for (int j = 0; j < 4; j++) umma::mma_f8<1>(tmem + buf * NT, da0 + (off + j * 2), db0 + (off + j * 2), idesc, j > 0);
        umma::mma_commit<1>(empty(s));
        umma::mma_commit<1>(acc_full(buf));
      }
      if (++s == stages) { s = 0; parity ^= 1; }
      if (++buf == S::kBufs) { buf = 0; turn ^= 1; }
    }
    if (!ok) umma::drain_copies();
    __syncwarp();
    if (split > 1) {
      umma::cluster_wait();
      umma::cluster_sync();
    }
  } else {
    const int quarter = warp & 3, tid = quarter * 32 + lane;   // tensor memory's lanes go by the warp's number
    const int64_t col = n0 + tid;
    const bool live = col < p.n;
    const float* sa = p.a_scale + int64_t(t0) * p.a_row;
    const float* sb = p.b_scale + (ROWS ? (live ? col : 0) : n0 / kBlock) * p.b_row;
    auto weight_scale = [&](int i) { return i < steps ? sb[(first + i) * p.b_block] : 0.f; };
    constexpr int kPer = (NT + 31) / 32;
    float next[kPer];
    auto scales_of = [&](int i) {
#pragma unroll
      for (int j = 0; j < kPer; j++) next[j] = i < steps && lane + 32 * j < tokens ? sa[(lane + 32 * j) * p.a_row + (first + i) * p.a_block] : 0.f;
    };
    scales_of(0);
    float w0 = weight_scale(0), w1 = weight_scale(1);
    uint64_t acc[NT / 2];
#pragma unroll
    for (int j = 0; j < NT / 2; j++) acc[j] = 0;
    int buf = 0;
    uint32_t turn = 0;
    const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
#pragma unroll 1
    for (int i = 0; i < steps; i++) {
      const uint32_t mine = umma::smem_u32(&token_scales[quarter][i & 1][0]);
#pragma unroll
      for (int j = 0; j < kPer; j++)
        if (NT >= 32 || lane < NT) asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + (lane + 32 * j) * 4), "f"(next[j]) : "memory");
      __syncwarp();
      scales_of(i + 1);
      const uint64_t w2 = pair_of(w0, w0);
      w0 = w1;
      w1 = weight_scale(i + 2);
      if (ok) ok = umma::bar_wait(acc_full(buf), turn);
      umma::fence_after();
      constexpr int kChunk = NT < 32 ? 16 : 32;
#pragma unroll
      for (int c = 0; c < NT; c += kChunk) {
        uint32_t t[kChunk];
        if constexpr (kChunk == 16) umma::tmem_load16(lanes + buf * NT + c, t);
        else umma::tmem_load32(lanes + buf * NT + c, t);
        umma::tmem_load_wait();
        if (c + kChunk == NT) {
          umma::fence_before();
          __syncwarp();
          if (lane == 0) umma::bar_arrive(acc_empty(buf));
        }
#pragma unroll
        for (int j = 0; j < kChunk / 4; j++) {
          uint64_t c0, c1;
          load_pairs(mine + (c + 4 * j) * 4, c0, c1);
          // the scales first: a sum of 2^24 and one scale may pass f32's range
          fma_pair(acc[c / 2 + 2 * j], pair_of(t[4 * j], t[4 * j + 1]), mul_pair(c0, w2));
          fma_pair(acc[c / 2 + 2 * j + 1], pair_of(t[4 * j + 2], t[4 * j + 3]), mul_pair(c1, w2));
        }
      }
      if (++buf == S::kBufs) { buf = 0; turn ^= 1; }
    }
    if (!ok) {
      umma::drain_copies();
#pragma unroll
      for (int j = 0; j < NT / 2; j++) acc[j] = pair_of(0x7fffffffu, 0x7fffffffu);   // a wait ran out: the outputs say so
    }
    const float bias = p.bias && live ? to_f32(static_cast<const T*>(p.bias)[col]) : 0.f;
    T* c = static_cast<T*>(p.c) + int64_t(t0) * p.ldc + col;
    if (split == 1) {
#pragma unroll
      for (int t = 0; t < NT; t += 2) {
        const float2 v = values_of(acc[t / 2]);
        if (live && t < tokens) c[int64_t(t) * p.ldc] = from_f32<T>(v.x + bias);
        if (live && t + 1 < tokens) c[int64_t(t + 1) * p.ldc] = from_f32<T>(v.y + bias);
      }
    } else {
      __syncwarp();
      umma::cluster_wait();
      const int share = ((tokens + split - 1) / split + 3) & ~3;   // tokens a CTA of the cluster finishes, by fours
      const uint32_t at = exchange + tid * 16, row4 = 128 * 16;    // (source x share / 4 x 128 rows of B x 4 tokens)
#pragma unroll
      for (int t = 0; t < NT; t += 4) {
        if (t >= tokens) break;
        const int owner = t / share, local = t - owner * share;
        const float2 lo = values_of(acc[t / 2]), hi = values_of(acc[t / 2 + 1]);
        umma::store_cluster(umma::map_rank(at + uint32_t(rank * share + local) / 4 * row4, owner), __float_as_uint(lo.x), __float_as_uint(lo.y),
                            __float_as_uint(hi.x), __float_as_uint(hi.y));
      }
      __syncwarp();
      umma::cluster_sync();
      const int last = min(tokens - rank * share, share);
#pragma unroll 2
      for (int t = 0; t < last; t += 4) {
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < 8; r++) {
          if (r >= split) break;
          float4 v;
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at + uint32_t(r * share + t) / 4 * row4));
          sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        const float z[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int token = rank * share + t + e;
          if (live && token < tokens) c[int64_t(token) * p.ldc] = from_f32<T>(z[e] + bias);
        }
      }
    }
  }
  umma::fence_before();
  __syncthreads();
  if (warp == 1) {
    umma::fence_after();
    umma::tmem_free<1>(tmem, S::kColumns);
  }
}

}  // namespace tgb
