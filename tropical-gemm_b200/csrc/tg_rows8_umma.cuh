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
// and half of the right one, or two such tiles one below the other that share
// the right operand.  The sum advances by 128 bytes of each left row per stage
// of a TMA ring; the two accumulators in tensor memory are 256 columns each.
// Persistent: a pair walks tiles in groups of row panels, so what it reads
// stays in L2.
//
// What bounds it: power for long sums (8192^3 forward: one call 0.33 ms, called on
// end 0.38, with zero operands 0.25), and shared memory.  Per 256 x 256 x (128 bytes) step an SM's tensor core
// needs 512 cycles and reads 32 KB (256 cycles at 128 bytes per cycle); TMA writes
// 32 KB more (forward: 512 in all).  Backward a step writes 16 + 8 KB, and the
// expansion reads 8 and writes 16: 640 cycles.  Two tiles that share the right
// operand bring that to 1024 per 1024 of tensor work (8192 x 8192 x 4096: 0.44 ms
// one tile at a time, 0.36 two, called on end 0.43); forward they gain nothing (0.176, 0.196 ms).
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
  int tiles_m, tiles_n;       // tiles of 256 x 2 half_n
  int half_n;                 // columns of a tile per CTA: 128, or 64 for outputs of at most 128 columns
  int splits, split_blocks;   // the sum in parts, one pair each (1: whole); blocks per part
  int chunk;                  // blocks after which the accumulator is added up in f32 (see Walk)
  float4* work;               // those sums of the pairs' current tiles, or null; L2 keeps them
  uint32_t* part;             // raw sums of the parts, (splits x m x ldp), joined by join_kernel
  int64_t ldp;
  int doubles;                // two-tile items, taken first (a multiple of the pairs)
  int singles;                // one-tile items
  int vec;                    // 16-byte stores of C's rows
};

constexpr int kTile = 256, kHalf = 128;
constexpr int kOperand = 16384;                 // bytes of one operand's stage: 128 rows x 128 bytes
constexpr int kRawBytes = 8192;                 // the 8-bit tile that is expanded to one stage
constexpr int kEpiWarps = 8, kConvWarps = 4, kConvGroups = 2;   // a group of conv warps per 8-bit tile, in turn
constexpr int kStagingBytes = 2048;             // per epilogue warp: 64 bytes of 32 rows

// Shared memory and barriers: a ring of both operands.  Backward the right
// operand's stages are written by the conv warps from a ring of 8-bit tiles
// of its own, which run ahead; a stage is full when the left operand has
// landed and both CTAs' conv warps have arrived, so the products wait and
// commit once per stage, as in the forward kernel (a barrier and a commit of
// its own for the expanded operand: 0.36 -> 0.40 ms without any expansion).
template <int MODE> struct ProductShape {
  static constexpr bool kBack = MODE != kForward;
  static constexpr int kHalves = kBack ? 2 : 1;                  // tiles of an item that share the right operand
  static constexpr int kStages = kBack ? 4 : 6;
  static constexpr int kStage = (1 + kHalves) * kOperand;        // right operand, left operands
  // 8-bit tiles on their way: two of their own, and while no item has two
  // tiles, two in each stage's unused half of the left operands: a short
  // product is bound by the way from memory (1000 cycles a stage with two)
  static constexpr int kOwnRaws = kBack ? 2 : 0, kRaws = kBack ? 2 + 2 * kStages : 0;
  // a slot belongs to one conv group for good: a group that met a slot every
  // other turn could take the parity of a turn it did not see for its own
  static_assert(kConvGroups == 2 && kOwnRaws % kConvGroups == 0 && kRaws % kConvGroups == 0 && kStages % kConvGroups == 0, "rings and groups");
  static constexpr int kThreads = 32 * (4 + kEpiWarps + (kBack ? kConvWarps * kConvGroups : 0));
  static constexpr int kOffRaw = kStages * kStage;
  static constexpr int kOffStaging = kOffRaw + kOwnRaws * kRawBytes;
  static constexpr int kOffCols = kOffStaging + kEpiWarps * kStagingBytes;   // b_scale, bias of the tile
  static constexpr int kOffBars = kOffCols + (kBack ? 0 : 2 * kTile * 4);
  static constexpr int kBars = 2 * (kStages + kRaws + 2);
  static constexpr int kOffSlot = kOffBars + kBars * 8;
  static constexpr int kSmem = kOffSlot + 16 + 1024;   // the rings start on a 1024-byte boundary
};

// A place in a ring: its slot and the parity of its turn.
template <int N> struct RingAt {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == N) { slot = 0; parity ^= 1; }
  }
};

// Bytes I and I + 1 of w_biased (offset by 128) times f as a pair of bf16,
// each rounded once: two values per f32 add and multiply.
template <int I> __device__ __forceinline__ uint32_t bytes_scaled(uint32_t w_biased, float f) {
  uint32_t r;
  asm("{\n.reg .b64 v, m, s;\n.reg .f32 x, y;\n"
      "mov.b64 v, {%1, %2};\nmov.b64 m, {%3, %3};\nmov.b64 s, {%4, %4};\n"
      "add.rn.f32x2 v, v, m;\nmul.rn.f32x2 v, v, s;\nmov.b64 {x, y}, v;\ncvt.rn.bf16x2.f32 %0, y, x;\n}\n"
      : "=r"(r)
      : "r"(__byte_perm(w_biased, 0x4b000000u, 0x7650 | I)), "r"(__byte_perm(w_biased, 0x4b000000u, 0x7650 | (I + 1))),
        "f"(-8388736.f), "f"(f));
  return r;
}

// The same for a ring whose size is known when the kernel runs.
struct RingOf {
  int n, slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == n) { slot = 0; parity ^= 1; }
  }
};

// Item i of a pair's walk: the tile at (m0, n0) and, if halves is 2, the one
// below it.  Double items first, in whole rounds of all pairs; then the rest
// one tile at a time, so the last round is as even as single tiles make it.
// Doubles go in groups of 4 (8 panels of 256 rows), columns outside rows.
// b0 .. b1: the item's blocks of the sum.
struct Item {
  int64_t m0, n0;
  int halves, b0, b1;
};
__device__ __forceinline__ bool item_at(const ProductArgs& p, int pair, int pairs, int i, Item& it) {
  if (p.splits > 1) {   // one part of one tile per pair
    const int tile = pair / p.splits, part = pair - tile * p.splits;
    it.m0 = int64_t(tile % p.tiles_m) * kTile;
    it.n0 = int64_t(tile / p.tiles_m) * 2 * p.half_n;
    it.halves = 1;
    it.b0 = part * p.split_blocks;
    it.b1 = min(p.blocks, it.b0 + p.split_blocks);
    return i == 0;
  }
  it.b0 = 0;
  it.b1 = p.blocks;
  constexpr int kGroup = 4;
  const int panels = p.tiles_m >> 1;
  int d, half = 0;
  if (i < p.doubles / pairs) {
    d = pair + i * pairs;
    it.halves = 2;
  } else {
    const int64_t s = pair + int64_t(i - p.doubles / pairs) * pairs;
    if (s >= p.singles) return false;
    it.halves = 1;
    d = p.doubles + int(s >> 1);
    half = int(s & 1);
    if (d >= panels * p.tiles_n) {   // the last panel, when their number is odd
      it.m0 = int64_t(p.tiles_m - 1) * kTile;
      it.n0 = (s - 2 * int64_t(panels * p.tiles_n - p.doubles)) * 2 * p.half_n;
      return true;
    }
  }
  const int per = kGroup * p.tiles_n, g = d / per, first = g * kGroup, rows = min(kGroup, panels - first);
  const int in = d - g * per;
  it.m0 = int64_t(2 * (first + in % rows) + half) * kTile;
  it.n0 = int64_t(in / rows) * 2 * p.half_n;
  return true;
}

// The order of an item's stages: chunks of blocks, in each the planes of g from
// the smallest parts to the largest, in each the chunk's blocks.  The tensor
// core's f32 sums lose in proportion to the additions (norm of the error over
// that of the result: 3.1e-7 after 512 terms, 6.6e-7 after 1024, 1.3e-6 after 2048,
// 7e-5 after 65536, 3e-4 after 262144; the plain f32 product of 8192 terms 1.6e-6),
// so after a chunk the epilogue adds the accumulator to a running f32 sum.  A
// chunk's loss stays below what g's own parts carry: with three planes (f32) 16
// blocks, 1024 terms; with two (f16, 16 bits) 128 blocks, 8e-6; with one (bf16)
// 256 blocks, 1.5e-5, beside factors of 8 bits.  From then on it does not grow:
// 262144 terms of f16 8.1e-6, of bf16 1.5e-5, f32 5.7e-7.  Cost of the chunks at
// 8192 x 8192 x 32768: bf16 2.89 -> 2.97 ms, f16 none to measure.
struct Walk {
  int block, plane, c0, c1, chunk, b1, planes;
  __device__ __forceinline__ Walk(const ProductArgs& p, const Item& it)
      : block(it.b0), plane(0), c0(it.b0), c1(min(it.b0 + p.chunk, it.b1)), chunk(p.chunk), b1(it.b1), planes(p.planes) {}
  __device__ __forceinline__ bool first() const { return block == c0 && plane == 0; }   // of a chunk
  __device__ __forceinline__ bool last() const { return block + 1 == c1 && plane + 1 == planes; }
  __device__ __forceinline__ bool more() const { return c0 < b1; }
  __device__ __forceinline__ void next() {
    if (++block < c1) return;
    block = c0;
    if (++plane < planes) return;
    plane = 0;
    block = c0 = c1;
    c1 = min(c1 + chunk, b1);
  }
};

// 64 bytes of each of 32 rows, one row per lane, to global memory through
// shared memory, so that a warp's store covers 8 rows' 64 bytes (a store of 32
// lanes' own rows touches 32 lines: 900 cycles for 32 columns instead of 250).  c: the
// first row's first element; rows, cols: how many exist; vec: 16-byte aligned
// rows.  Two rows share 128 bytes of shared memory; the chunks are swizzled so
// that eight lanes meet all banks either way.
template <typename T>
__device__ __forceinline__ void store_rows64(T* c, int64_t ld, int rows, int64_t cols, bool vec, const uint32_t (&w)[16],
                                             uint32_t staging, int lane) {
  constexpr int kPer = 16 / int(sizeof(T));   // elements of a 16-byte chunk
  __syncwarp();                               // the last chunk is read
#pragma unroll
  for (int j = 0; j < 4; j++)
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(staging + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)),
                 "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3]) : "memory");
  __syncwarp();
  const int j = lane & 3, r0 = lane >> 2;   // rows r0, r0 + 8, ..: the same place in the swizzle
  uint32_t v[4][4];
#pragma unroll
  for (int k = 0; k < 4; k++)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[k][0]), "=r"(v[k][1]), "=r"(v[k][2]), "=r"(v[k][3])
                 : "r"(staging + r0 * 64 + k * 512 + ((j ^ ((r0 >> 1) & 3)) << 4)));
  T* to = c + r0 * ld + j * kPer;
  if (vec && rows == 32 && cols >= 4 * kPer) {   // uniform
#pragma unroll
    for (int k = 0; k < 4; k++) *reinterpret_cast<uint4*>(to + k * 8 * ld) = make_uint4(v[k][0], v[k][1], v[k][2], v[k][3]);
    return;
  }
  if (vec && cols % kPer == 0) {   // whole chunks only
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (r0 + 8 * k < rows && (j + 1) * kPer <= cols) *reinterpret_cast<uint4*>(to + k * 8 * ld) = make_uint4(v[k][0], v[k][1], v[k][2], v[k][3]);
    return;
  }
  // any alignment: lanes along the row, one element each
  constexpr int kWide = 64 / int(sizeof(T));   // 16 or 32 elements: two rows or one at a time
  const int e = lane % kWide;
  if (e < cols) {
    T* at = c + e;
#pragma unroll 8
    for (int r = lane / kWide; r < rows; r += 32 / kWide) {
      const uint32_t from = staging + r * 64 + (((e / kPer) ^ ((r >> 1) & 3)) << 4) + (e % kPer) * int(sizeof(T));
      if constexpr (sizeof(T) == 4) {
        uint32_t x;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(from));
        reinterpret_cast<uint32_t*>(at)[r * ld] = x;
      } else {
        uint16_t x;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(from));
        reinterpret_cast<uint16_t*>(at)[r * ld] = x;
      }
    }
  }
}

template <typename T> __device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_pair<bf16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack_pair<f16>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// SUMS: a sum has several chunks (kept out of the other instances: a short
// product is on the GPU for 5 us and pays for every instruction it fetches).
template <int MODE, typename T, bool SUMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(ProductShape<MODE>::kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const ProductArgs p) {
  using S = ProductShape<MODE>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (umma::smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - umma::smem_u32(smem_raw));
  // barriers of the leader unless noted: a pair's products are issued there
  const uint32_t bars = base + S::kOffBars;
  auto full = [&](int s) { return bars + 8 * s; };                         // operands in place in both CTAs
  auto empty = [&](int s) { return bars + 8 * (S::kStages + s); };         // products that read them are done (each CTA)
  constexpr int kR = 2 * S::kStages, kAcc = kR + 2 * S::kRaws;
  auto raw_full = [&](int s) { return bars + 8 * (kR + s); };              // 8-bit tile landed (each CTA)
  auto raw_empty = [&](int s) { return bars + 8 * (kR + S::kRaws + s); };  // and is read (each CTA)
  auto acc_full = [&](int b) { return bars + 8 * (kAcc + b); };            // tile summed (each CTA)
  auto acc_empty = [&](int b) { return bars + 8 * (kAcc + 2 + b); };       // and read out in both CTAs
  const int raws = p.doubles ? S::kOwnRaws : S::kRaws;
  auto raw_tile = [&](int s) {
    return s < S::kOwnRaws ? base + S::kOffRaw + s * kRawBytes
                           : base + ((s - S::kOwnRaws) >> 1) * S::kStage + 2 * kOperand + ((s - S::kOwnRaws) & 1) * kRawBytes;
  };
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + S::kOffSlot);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp: uniform
  const uint32_t rank = umma::cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 0 && lane == 0) {
    umma::tma_prefetch(&map_a);
    umma::tma_prefetch(&map_b);
    for (int s = 0; s < S::kStages; s++) {
      umma::bar_init(full(s), 1 + (S::kBack ? 2 * kConvWarps : 0));
      umma::bar_init(empty(s), 1);
    }
    for (int s = 0; s < S::kRaws; s++) {
      umma::bar_init(raw_full(s), 1);
      umma::bar_init(raw_empty(s), kConvWarps);
    }
    for (int b = 0; b < 2; b++) {
      umma::bar_init(acc_full(b), 1);
      umma::bar_init(acc_empty(b), 2 * kEpiWarps);
    }
    umma::bar_init_fence();
  }
  if (warp == 2) umma::tmem_alloc<2>(base + S::kOffSlot, 512);
  after_previous_kernel();
  umma::fence_before();
  umma::cluster_sync();
  umma::fence_after();
  const uint32_t tmem = *slot;
  bool ok = true;   // false once a wait of this role ran out

  if (warp == 0) {
    // ---- producer: this CTA's half of each operand (backward: of the left one)
    const bool issue = umma::elect_one();
    RingAt<S::kStages> at;
    Item item;
    for (int i = 0; ok && item_at(p, pair, pairs, i, item); i++) {
      const int row = int(item.m0) + int(rank) * kHalf, col = int(item.n0) + int(rank) * p.half_n;
      for (Walk at_sum(p, item); at_sum.more(); at_sum.next(), at.next()) {
        if (!umma::bar_wait(empty(at.slot), at.parity ^ 1)) { ok = false; break; }
        const uint32_t b = base + at.slot * S::kStage, bar = umma::map_rank(full(at.slot), 0);
        const int block = at_sum.block, plane = at_sum.plane;
        if (issue) {
          if (rank == 0) umma::bar_expect(full(at.slot), 2 * kOperand * (item.halves + (S::kBack ? 0 : 1)));
          if (MODE == kForward) umma::tma_load_3d_pair(b, &map_b, block * 128, col, 0, bar);
#pragma unroll
          for (int h = 0; h < S::kHalves; h++) {
            if (h == item.halves) break;
            const uint32_t a = b + kOperand * (1 + h);
            const int r = row + h * kTile;
            if (MODE == kForward) {
              umma::tma_load_3d_pair(a, &map_a, block * 128, r, 0, bar);
            } else if (MODE == kBackRows) {
              umma::tma_load_3d_pair(a, &map_a, block * 64, r, plane, bar);
            } else {
              umma::tma_load_3d_pair(a, &map_a, r, block * 64, plane, bar);
              umma::tma_load_3d_pair(a + kOperand / 2, &map_a, r + 64, block * 64, plane, bar);
            }
          }
        }
      }
    }
    if (!ok) umma::drain_copies();
  } else if (S::kBack && warp == 3) {
    // ---- producer of the 8-bit tiles
    const bool issue = umma::elect_one();
    RingOf at{raws};
    Item item;
    for (int i = 0; ok && item_at(p, pair, pairs, i, item); i++) {
      const int col = int(item.n0) + int(rank) * p.half_n;
      for (Walk at_sum(p, item); at_sum.more(); at_sum.next(), at.next()) {
        if (!umma::bar_wait(raw_empty(at.slot), at.parity ^ 1)) { ok = false; break; }
        if (issue) {
          umma::bar_expect(raw_full(at.slot), kRawBytes);
          umma::tma_load_3d_pair(raw_tile(at.slot), &map_b, col, at_sum.block * 64, 0, umma::map_rank(raw_full(at.slot), rank));
        }
      }
    }
    if (!ok) umma::drain_copies();
  } else if (warp == 1 && rank == 0) {
    // ---- products, issued by one thread of the leader for both SMs
    const uint32_t idesc = MODE == kForward ? umma::instr_desc(2, 1, false, false, kTile, 2 * p.half_n)
                                            : umma::instr_desc(1, 1, MODE == kBackCols, true, kTile, 2 * p.half_n);
    // bytes from one instruction's slice of the sum to the next: 32 along a
    // 128-byte row, or 16 rows
    constexpr uint32_t step_a = MODE == kBackCols ? 2048 : 32, step_b = MODE == kForward ? 32 : 2048;
    // contiguous along the sum: 8-row groups 1024 bytes apart; else 64-wide
    // columns of 64 rows 8192 bytes apart
    const uint64_t db0 = umma::smem_desc(base, S::kBack ? 8192 : 16, 1024);
    const uint64_t da0 = umma::smem_desc(base + kOperand, MODE == kBackCols ? 8192 : 16, 1024);
    const bool issue = umma::elect_one();
    RingAt<S::kStages> at;
    Item item;
    int n = 0;   // sums so far: sum n goes into accumulator n % 2
    for (int i = 0; ok && item_at(p, pair, pairs, i, item); i++) {
      for (Walk at_sum(p, item); at_sum.more(); at_sum.next(), at.next()) {
        if (!umma::bar_wait<S::kBack>(full(at.slot), at.parity)) { ok = false; break; }
        const uint32_t off = at.slot * (S::kStage >> 4);
        const bool first = at_sum.first();
#pragma unroll
        for (int h = 0; h < S::kHalves; h++) {
          if (h == item.halves) break;
          const int buf = (n + h) & 1;
          if (first && !umma::bar_wait<true>(acc_empty(buf), (((n + h) >> 1) & 1) ^ 1)) { ok = false; break; }
          umma::fence_after();
          const uint32_t offa = off + h * (kOperand >> 4);
          if (issue) {
#pragma unroll
            for (int j = 0; j < 4; j++)
              umma::mma<2, MODE == kForward>(tmem + buf * kTile, da0 + (offa + (j * step_a >> 4)), db0 + (off + (j * step_b >> 4)), idesc, !first || j);
          }
        }
        if (!ok) break;
        if (issue) umma::mma_commit<2>(empty(at.slot));
        if (at_sum.last()) {
          if (issue)
            for (int h = 0; h < item.halves; h++) umma::mma_commit<2>(acc_full((n + h) & 1));
          n += item.halves;
        }
      }
      __syncwarp();
    }
    if (!ok) umma::drain_copies();
  } else if (warp >= 4 && warp < 4 + kEpiWarps) {
    // ---- epilogue: warp w reads lanes 32 (w % 4) .. of tensor memory and one
    // half of the columns, 64 bytes of output at a time
    const int w = (warp - 4) & 3, half = (warp - 4) >> 2, tid = threadIdx.x - 128;
    const uint32_t staging = base + S::kOffStaging + (warp - 4) * kStagingBytes;
    float* cols = reinterpret_cast<float*>(smem + S::kOffCols);
    Item item;
    int n = 0;
    for (int i = 0; item_at(p, pair, pairs, i, item); i++) {
      const int chunks = SUMS ? (item.b1 - item.b0 + p.chunk - 1) / p.chunk : 1;
      for (int ch = 0, h = 0; ch < chunks; n++) {   // h: the tile within the item
        const int tile = h, buf = n & 1;
        const bool first = !SUMS || ch == 0, last = !SUMS || ch + 1 == chunks;
        const int64_t n0 = item.n0, row0 = item.m0 + tile * kTile + rank * kHalf + w * 32, row = row0 + lane;
        const int rows = int(max(int64_t(0), min(int64_t(32), p.m - row0)));
        const int columns = min(128, 2 * p.half_n - half * 128);   // of this warp's half: none in narrow tiles' second
        if (++h == item.halves) { h = 0; ch++; }
        float rs = 0.f;
        if (MODE == kForward && p.splits == 1) {
          named_sync(1, 256);   // the last tile's columns are no longer read
          const bool in = n0 + tid < p.n;
          cols[tid] = in ? p.col_scale[n0 + tid] : 0.f;
          cols[kTile + tid] = in && p.bias ? to_f32(static_cast<const T*>(p.bias)[n0 + tid]) : 0.f;
          named_sync(1, 256);
          if (row < p.m) rs = p.row_scale[row];
        }
        if (ok) {   // a whole sum: the limit grows with its length
          bool done = false;
          for (int k = 0; k <= (item.b1 - item.b0) * p.planes >> 10 && !done; k++) done = umma::bar_wait(acc_full(buf), (n >> 1) & 1);
          ok = done;
        }
        umma::fence_after();
        const uint32_t from = tmem + buf * kTile + half * 128 + (uint32_t(w * 32) << 16);
        const int64_t col0 = n0 + half * 128;
        auto read_out = [&] {   // the next sum may have the accumulator
          umma::fence_before();
          __syncwarp();
          if (lane == 0) umma::bar_arrive_cluster(umma::map_rank(acc_empty(buf), 0));
        };
        auto value = [&](uint32_t acc, int c) {
          float z = __uint_as_float(acc);
          if (MODE == kForward) z = float(int(acc)) * rs * cols[half * 128 + c] + cols[kTile + half * 128 + c];
          return ok ? z : __uint_as_float(0x7fffffffu);   // a wait ran out: the outputs say so
        };
        // 16 columns' sums so far, kept where the same thread finds them again
        auto add_up = [&](uint32_t* acc, int c) {
          if (!SUMS || (first && last)) return;
          float4* kept = p.work + (((int64_t(pair) * 2 + rank) * 2 + tile) * kEpiWarps + (warp - 4)) * 1024 + c / 4 * 32 + lane;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float4 o = first ? make_float4(0.f, 0.f, 0.f, 0.f) : kept[j * 32];
            o.x += __uint_as_float(acc[4 * j]);
            o.y += __uint_as_float(acc[4 * j + 1]);
            o.z += __uint_as_float(acc[4 * j + 2]);
            o.w += __uint_as_float(acc[4 * j + 3]);
            if (!last) kept[j * 32] = o;
            acc[4 * j] = __float_as_uint(o.x);
            acc[4 * j + 1] = __float_as_uint(o.y);
            acc[4 * j + 2] = __float_as_uint(o.z);
            acc[4 * j + 3] = __float_as_uint(o.w);
          }
        };
        if (columns <= 0) {
          read_out();
        } else if (p.splits > 1 || sizeof(T) == 4) {
#pragma unroll 1
          for (int c = 0; c < columns; c += 16) {
            uint32_t acc[16];
            umma::tmem_load16(from + c, acc);
            umma::tmem_load_wait();
            if (c + 16 == columns) read_out();
            if (col0 + c >= p.n) continue;
            add_up(acc, c);
            if (!last) continue;
            if (p.splits > 1) {
              if (!ok) {   // NaN, or a value no integer sum takes
#pragma unroll
                for (int e = 0; e < 16; e++) acc[e] = MODE == kForward ? 0x80000000u : 0x7fffffffu;
              }
              store_rows64(p.part + (int64_t(pair % p.splits) * p.m + row0) * p.ldp + col0 + c, p.ldp, rows, p.ldp - col0 - c, true, acc, staging, lane);
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
              for (int e = 0; e < 16; e++) acc[e] = __float_as_uint(value(acc[e], c + e));
              store_rows64(static_cast<T*>(p.c) + row0 * p.ldc + col0 + c, p.ldc, rows, p.n - col0 - c, p.vec, acc, staging, lane);
            }
          }
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll 1
          for (int c = 0; c < columns; c += 32) {
            uint32_t acc[32], z[16];
            umma::tmem_load32(from + c, acc);
            umma::tmem_load_wait();
            if (c + 32 == columns) read_out();
            if (col0 + c >= p.n) continue;
            add_up(acc, c);
            add_up(acc + 16, c + 16);
            if (!last) continue;
#pragma unroll
            for (int e = 0; e < 16; e++) z[e] = pack_pair<T>(value(acc[2 * e], c + 2 * e), value(acc[2 * e + 1], c + 2 * e + 1));
            store_rows64(static_cast<T*>(p.c) + row0 * p.ldc + col0 + c, p.ldc, rows, p.n - col0 - c, p.vec, z, staging, lane);
          }
        }
      }
    }
    if (!ok) umma::drain_copies();
  } else if (S::kBack && warp >= 4 + kEpiWarps) {
    // ---- 8-bit tile (64 of the sum x 128 columns) to bf16, 128-byte swizzled
    // columns of 64.  Lanes 0-7 take eight rows of one 16-byte chunk: the
    // swizzle spreads them over all banks on both sides.
    const int w = (warp - 4 - kEpiWarps) % kConvWarps, group = (warp - 4 - kEpiWarps) / kConvWarps;
    const int r8 = lane & 7, c4 = lane >> 3;
    RingOf rw{raws};
    RingAt<S::kStages> cv;
    float sc[2], next[2];
    auto factors = [&](int block, float (&f)[2]) {
      const int r0 = block * 64 + w * 16 + r8;
#pragma unroll
      for (int i = 0; i < 2; i++) f[i] = p.sum_scale ? (r0 + 8 * i < p.sum ? p.sum_scale[r0 + 8 * i] : 0.f) : 1.f;
    };
    for (int i = 0; i < group; i++) { rw.next(); cv.next(); }
    Item item;
    bool started = false;
    int turn = 0;   // stages go to the groups in turn
    for (int it = 0; ok && item_at(p, pair, pairs, it, item); it++)
    for (Walk at_sum(p, item); at_sum.more(); at_sum.next(), turn ^= 1) {   // one nest: every stage of every item
      if (turn != group) continue;
      if (!started) factors(at_sum.block, next);
      started = true;
      sc[0] = next[0];
      sc[1] = next[1];
      // a turn ahead, so that the load's latency stays out of the wait (factors
      // are there only with one plane, whose walk is straight, and all items of a
      // pair have the same blocks)
      int ahead = at_sum.block + kConvGroups;
      while (ahead >= item.b1) ahead -= item.b1 - item.b0;
      factors(ahead, next);
      if (!umma::bar_wait(raw_full(rw.slot), rw.parity)) { ok = false; break; }
      const uint32_t in = raw_tile(rw.slot) + (w * 16 + r8) * 128;
      const bool wide = p.half_n == 128;   // else the first 64 columns only
      uint32_t q[4][4];
#pragma unroll
      for (int i = 0; i < 4; i++)   // rows + 8 (i / 2), 64 columns (i % 2)
        if (wide || !(i & 1)) asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q[i][0]), "=r"(q[i][1]), "=r"(q[i][2]), "=r"(q[i][3])
                     : "r"(in + (i >> 1) * 1024 + ((((i & 1) * 4 + c4) ^ r8) << 4)));
      if (!umma::bar_wait(empty(cv.slot), cv.parity ^ 1)) { ok = false; break; }
      const uint32_t out = base + cv.slot * S::kStage + (w * 16 + r8) * 128;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (!wide && (i & 1)) continue;
        uint32_t o[8];
        const float f = sc[i >> 1];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t x = q[i][k] ^ 0x80808080u;
          o[2 * k] = bytes_scaled<0>(x, f);
          o[2 * k + 1] = bytes_scaled<2>(x, f);
        }
#pragma unroll
        for (int k = 0; k < 2; k++)
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(out + (i >> 1) * 1024 + (i & 1) * 8192 + (((2 * c4 + k) ^ r8) << 4)),
                       "r"(o[4 * k]), "r"(o[4 * k + 1]), "r"(o[4 * k + 2]), "r"(o[4 * k + 3]) : "memory");
      }
      // The 8-bit tile is given back only now that its values have been used: an
      // arrival right after the loads overtook them under load, and the next
      // tile was read in their place.
      __syncwarp();
      if (lane == 0) umma::bar_arrive(raw_empty(rw.slot));
      umma::fence_async_smem();
      __syncwarp();
      if (lane == 0) umma::bar_arrive_cluster(umma::map_rank(full(cv.slot), 0));
      for (int i = 0; i < kConvGroups; i++) { rw.next(); cv.next(); }
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

// The forward product for few tokens (decoding): what it has to do is read the
// weights once, so the roles are swapped.  128 weight rows are the tensor
// core's rows and up to NT tokens its columns; the sum is split over the S
// CTAs of a cluster (S from 1 to 8, so that all SMs read).  Each CTA finishes a
// share of the tokens: the others write their integer parts into its shared
// memory (stores need no answer; fetching the parts took 860 cycles a round).
// A CTA's whole share of the weights is in flight at once where it fits its
// shared memory.
//
// A CTA that waits for its cluster must not wait for tensor memory held by
// one that waits for another cluster: with split > 1 a CTA has at least 37 KB
// of shared memory (NT = 128: 65 KB), so the CTAs that fit an SM together ask
// for at most 416 of its 512 columns, and none fits beside a paired CTA.
template <int NT> struct TokensShape {
  static constexpr int kStage = kOperand + NT * 128;
  static constexpr int kExchange = (NT < 32 ? 32 : NT) * 512;   // parts of this CTA's tokens (shares of 4) from the whole cluster
  static constexpr int kMost = (200 * 1024 - kExchange) / kStage;   // stages
  static constexpr int kBars = 2 * kMost + 1;
  static constexpr int kColumns = NT < 32 ? 32 : NT;
};

template <int NT, typename T>
__global__ void __launch_bounds__(128) tokens_kernel(const __grid_constant__ CUtensorMap map_tokens,
                                                     const __grid_constant__ CUtensorMap map_weights, const ProductArgs p,
                                                     int split, int stages) {
  using S = TokensShape<NT>;
  __shared__ __align__(8) uint64_t bar_store[S::kBars];
  __shared__ uint32_t slot;
  __shared__ float scales[NT];
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (umma::smem_u32(smem_raw) + 1023) & ~1023u, bars = umma::smem_u32(bar_store);
  const uint32_t exchange = base + stages * S::kStage;
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (S::kMost + s); };
  const uint32_t done = bars + 8 * (2 * S::kMost);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % split;
  const int n0 = int(blockIdx.x / split) * 128, t0 = int(blockIdx.y) * NT, tokens = min(NT, int(p.m) - t0);
  const int first = rank * p.split_blocks, steps = max(0, min(p.split_blocks, p.blocks - first));   // the last CTAs may have no share

  if (warp == 0 && lane == 0) {
    umma::tma_prefetch(&map_weights);
    umma::tma_prefetch(&map_tokens);
    for (int s = 0; s < stages; s++) {
      umma::bar_init(full(s), 1);
      umma::bar_init(empty(s), 1);
    }
    umma::bar_init(done, 1);
    umma::bar_init_fence();
  }
  after_previous_kernel();   // before tensor memory is taken, which that kernel's CTAs may still ask for
  if (warp == 2) umma::tmem_alloc<1>(umma::smem_u32(&slot), S::kColumns);
  umma::fence_before();
  __syncthreads();
  umma::fence_after();
  if (split > 1) umma::cluster_arrive();   // all of the cluster has started: waited for before the first store
  const uint32_t tmem = slot;
  bool ok = true;
  const int64_t col = int64_t(n0) + threadIdx.x;
  float cs = 0.f, bias = 0.f;
  if (col < p.n) {
    cs = p.col_scale[col];
    if (p.bias) bias = to_f32(static_cast<const T*>(p.bias)[col]);
  }
  if (warp >= 2)
    for (int t = threadIdx.x - 64; t < tokens; t += 64) scales[t] = p.row_scale[t0 + t];

  if (warp == 0) {
    const bool issue = umma::elect_one();
    int s = 0;
    uint32_t parity = 0;
    for (int i = 0; i < steps; i++) {
      if (!umma::bar_wait(empty(s), parity ^ 1)) { ok = false; break; }
      const uint32_t a = base + s * S::kStage;
      if (issue) {
        umma::bar_expect(full(s), S::kStage);
        umma::tma_load_3d(a, &map_weights, (first + i) * 128, n0, 0, full(s));
        umma::tma_load_3d(a + kOperand, &map_tokens, (first + i) * 128, t0, 0, full(s));
      }
      if (++s == stages) { s = 0; parity ^= 1; }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma::instr_desc(2, 1, false, false, 128, NT);
    const uint64_t da0 = umma::smem_desc(base, 16, 1024), db0 = umma::smem_desc(base + kOperand, 16, 1024);
    const bool issue = umma::elect_one();
    int s = 0;
    uint32_t parity = 0;
    for (int i = 0; i < steps; i++) {
      if (!umma::bar_wait(full(s), parity)) { ok = false; break; }
      umma::fence_after();
      const uint32_t off = s * (S::kStage >> 4);
      if (issue) {
#pragma unroll
        for (int j = 0; j < 4; j++) umma::mma<1, true>(tmem, da0 + (off + j * 2), db0 + (off + j * 2), idesc, i | j);
        umma::mma_commit<1>(empty(s));
      }
      if (++s == stages) { s = 0; parity ^= 1; }
    }
    if (issue && ok) umma::mma_commit<1>(done);
  }
  __syncwarp();
  if (!umma::bar_wait(done, 0)) ok = false;
  umma::fence_after();
  if (!ok) umma::drain_copies();
  __syncthreads();   // the tokens' scales

  // four tokens of this thread's weight row
  T* c = static_cast<T*>(p.c) + int64_t(t0) * p.ldc + col;
  auto emit4 = [&](int t, const int (&sum)[4], bool bad) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float z = float(sum[i]) * scales[t + i] * cs + bias;   // scales: NT of them, a multiple of 4
      if (bad) z = __uint_as_float(0x7fffffffu);
      if (t + i < tokens && col < p.n) c[int64_t(t + i) * p.ldc] = from_f32<T>(z);
    }
  };
  if (split > 1) umma::cluster_wait();
  const int share = ((tokens + split - 1) / split + 3) & ~3;   // tokens a CTA of the cluster finishes, by fours
  const uint32_t mine = exchange + threadIdx.x * 16, row4 = 128 * 16;   // (source x share / 4 x 128 weight rows x 4 tokens)
#pragma unroll 1
  for (int t = 0; t < tokens; t += 16) {
    uint32_t acc[16];
    umma::tmem_load16(tmem + t + (uint32_t(warp * 32) << 16), acc);
    umma::tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      if (split == 1) {
        emit4(t + i, {int(acc[i]), int(acc[i + 1]), int(acc[i + 2]), int(acc[i + 3])}, !ok);
      } else if (t + i < tokens) {
        if (!ok || !steps) acc[i] = acc[i + 1] = acc[i + 2] = acc[i + 3] = ok ? 0u : 0x80000000u;
        const int owner = (t + i) / share, local = t + i - owner * share;
        umma::store_cluster(umma::map_rank(mine + uint32_t(rank * share + local) / 4 * row4, owner), acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
      }
    }
  }
  if (split > 1) {
    umma::cluster_sync();
    const int last = min(tokens - rank * share, share);
#pragma unroll 2
    for (int t = 0; t < last; t += 4) {
      int sum[4] = {};
      bool bad = false;
#pragma unroll
      for (int r = 0; r < 8; r++) {
        if (r >= split) break;
        uint32_t v[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                     : "r"(mine + uint32_t(r * share + t) / 4 * row4));
#pragma unroll
        for (int i = 0; i < 4; i++) {
          sum[i] += int(v[i]);
          bad |= v[i] == 0x80000000u;   // no sum takes this value
        }
      }
      emit4(rank * share + t, sum, bad);
    }
  }
  umma::fence_before();
  __syncthreads();
  if (warp == 2) {
    umma::fence_after();
    umma::tmem_free<1>(tmem, S::kColumns);
  }
}

// Joins the parts of a sum, in order: forward integer sums with their scales
// and bias, backward f32 sums.  Four columns per thread.
template <bool FORWARD, typename T>
__global__ void __launch_bounds__(256) join_kernel(const ProductArgs p) {
  after_previous_kernel();
  const int64_t c0 = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (c0 >= p.n) return;
  for (int64_t row = blockIdx.y; row < p.m; row += gridDim.y) {
    int si[4] = {};
    float sf[4] = {};
    bool bad = false;
    for (int s = 0; s < p.splits; s++) {
      const uint4 v = *reinterpret_cast<const uint4*>(p.part + (int64_t(s) * p.m + row) * p.ldp + c0);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (FORWARD) { si[e] += int(w[e]); bad |= w[e] == 0x80000000u; } else sf[e] += __uint_as_float(w[e]);
      }
    }
    T* c = static_cast<T*>(p.c) + row * p.ldc + c0;
    const float rs = FORWARD ? p.row_scale[row] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (c0 + e >= p.n) break;
      float z = sf[e];
      if (FORWARD) {
        z = float(si[e]) * rs * p.col_scale[c0 + e] + (p.bias ? to_f32(static_cast<const T*>(p.bias)[c0 + e]) : 0.f);
        if (bad) z = __uint_as_float(0x7fffffffu);
      }
      c[e] = from_f32<T>(z);
    }
  }
}

// g * scale (scale null: g) in `planes` bf16 parts, each padded to rows of
// ldo: parts 0 .. planes - 1 from the smallest to the largest, so that the
// sums take the small ones first.  The upper parts are truncations, which
// leaves an exact rest: three parts hold all 24 bits, two hold 16 rounded.
// Eight columns per thread; vec: g's rows are 16-byte aligned.
template <typename GT>
__global__ void __launch_bounds__(256) split_kernel(int64_t rows, int64_t cols, const GT* g, int64_t ldg, const float* scale,
                                                    int scale_rows, bf16* out, int64_t ldo, int planes, int vec) {
  after_previous_kernel();
  const int64_t c = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (c >= ldo) return;
  float by_col[8];
#pragma unroll
  for (int e = 0; e < 8; e++) by_col[e] = scale && !scale_rows && c + e < cols ? scale[c + e] : 1.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    float v[8];
    if (vec && c + 8 <= cols) {
      Vec8<GT> a;
      a.load(g + r * ldg + c);
      a.get(v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = c + e < cols ? to_f32(g[r * ldg + c + e]) : 0.f;
    }
    const float by_row = scale && scale_rows ? scale[r] : 1.f;
    bool finite[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      v[e] *= scale_rows ? by_row : by_col[e];
      finite[e] = fabsf(v[e]) < __uint_as_float(0x7f800000u);
    }
    for (int i = planes - 1; i >= 0; i--) {
      float part[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        part[e] = i && finite[e] ? __uint_as_float(__float_as_uint(v[e]) & 0xffff0000u) : __bfloat162float(__float2bfloat16_rn(v[e]));
        v[e] = finite[e] ? v[e] - part[e] : 0.f;
      }
      store8(out + (int64_t(i) * rows + r) * ldo + c, part);
    }
  }
}

}  // namespace tg8
