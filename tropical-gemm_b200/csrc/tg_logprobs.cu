// Log probabilities of given tokens, entropies and the most likely tokens from
// rows of logits, and the gradient of the logits.
//
//   m = max x, S = sum exp(x - m), E = sum exp(x - m) (x - m)
//   logprob = (x_token - m) - log S,  entropy = log S - E / S
//   grad_v = g_lp ([v == token] - p_v) - g_H p_v (log p_v + entropy)
//
// One pass, in powers of two: with t = (x - m) log2 e, S = sum 2^t, E = sum 2^t t:
//   logprob = (x_token - m) - log S,  entropy = (log2 S - E / S) log 2
// Each thread keeps m, S and E of what it has seen and rescales them when a
// larger logit comes; each warp keeps its most likely tokens sorted across its
// lanes.
//
// 4096 x 65536 bf16 takes 131 us.  Neither its read (82) nor the exponentials (60, at
// 16 per clock and SM) nor issue slots (62 %) fill that time: a batch is loaded and
// then worked on, and 28 of an SM's 64 warps do not cover the one with the other.
#include <algorithm>
#include "tg_blocks8.cuh"
#include "tg_umma.cuh"

namespace tgb {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kMostTop = 32;   // alternatives: one per lane
constexpr int kManyRows = 128, kFewRows = 512;   // threads per row and CTA
constexpr int kSorted = 6;     // of a warp's 32 logits: more than these are cheaper to sort than to insert one by one
constexpr int kGroups = 4;     // of 8 logits per thread on their way at once

__device__ __forceinline__ float neg_inf() { return __int_as_float(int(0xff800000)); }
__device__ __forceinline__ float exp2_fast(float x) {   // within 2^-22 of itself; 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Where 2^t is zero its product with t is too (t may be -infinity).
__device__ __forceinline__ float least_power(float t) { return fmaxf(t, -200.f); }

struct Sums {
  float m, s, e;   // largest logit, S, E
};
__device__ __forceinline__ Sums nothing() { return {neg_inf(), 0.f, 0.f}; }
// What is measured from while there is nothing but -infinity: any finite value does.
__device__ __forceinline__ float base_of(float m) { return m == neg_inf() ? 0.f : m; }
// The same sums from m on, which is at least a.m.
__device__ __forceinline__ Sums rebase(const Sums& a, float m) {
  if (a.m == m || a.s == 0.f) return {m, a.s, a.e};
  const float d = (base_of(a.m) - m) * kLog2e, f = exp2_fast(d);
  return {m, a.s * f, fmaf(a.s, least_power(d), a.e) * f};
}
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  const Sums x = rebase(a, m), y = rebase(b, m);
  return {m, x.s + y.s, x.e + y.e};
}
__device__ __forceinline__ Sums from_lane(const Sums& a, int lane) {
  return {__shfl_xor_sync(0xffffffffu, a.m, lane), __shfl_xor_sync(0xffffffffu, a.s, lane), __shfl_xor_sync(0xffffffffu, a.e, lane)};
}

// Order of the alternatives as one whole number: larger logits first (one zero,
// NaN on top), of equal ones the lower token.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) b = 0x7fffffffu;
  b ^= b >> 31 ? 0xffffffffu : 0x80000000u;
  return uint64_t(b) << 32 | uint32_t(~token);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t b = uint32_t(key >> 32);
  return __uint_as_float(b >> 31 ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ uint32_t token_of(uint64_t key) { return ~uint32_t(key); }

// Descending over the lanes.
template <typename K> __device__ __forceinline__ K sort_lanes(K v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int d = size / 2; d; d >>= 1) {
      const K o = __shfl_xor_sync(0xffffffffu, v, d);
      const bool descending = (lane & size) == 0 || size == 32, low = (lane & d) == 0;
      v = (descending == low) == (v > o) ? v : o;
    }
  return v;
}

// A warp's best keys so far, sorted, one per lane; 0 is below every key.
struct Best {
  uint64_t key;
  __device__ __forceinline__ void insert(uint64_t k, int lane) {   // k: the same in all lanes
    const bool after = key < k;
    const uint64_t up = __shfl_up_sync(0xffffffffu, key, 1);
    const bool first = after && (lane == 0 || up >= k);
    if (after) key = first ? k : up;
  }
  // the best 32 of two sorted lists: the larger of each lane and its mirror
  // image form a bitonic sequence
  __device__ __forceinline__ void merge(uint64_t other, int lane) {
    const uint64_t mirror = __shfl_sync(0xffffffffu, other, 31 - lane);
    key = key > mirror ? key : mirror;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const uint64_t o = __shfl_xor_sync(0xffffffffu, key, d);
      const bool low = (lane & d) == 0;
      key = low == (key > o) ? key : o;
    }
  }
};

// The best 32 of a sorted list and of 32 more keys.  A call, for the sake of the
// loop that it stands in four times (4096 x 65536 with 20 alternatives, inline 267 us).
__device__ __noinline__ uint64_t merge_keys(uint64_t best, uint64_t keys) {
  const int lane = threadIdx.x & 31;
  Best b{best};
  b.merge(sort_lanes(keys, lane), lane);
  return b.key;
}

// A value's place in the order alone: larger for larger values, one zero, NaN on top.
__device__ __forceinline__ uint32_t rank_of(float x) { return uint32_t(key_of(x, 0) >> 32); }
__device__ __forceinline__ float value_of_rank(uint32_t r) { return __uint_as_float(r >> 31 ? r ^ 0x80000000u : ~r); }
// The largest, or a NaN.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The ranks of the lanes' largest logits in descending order; a group that holds a NaN counts for nothing.
__device__ __forceinline__ uint32_t lane_ranks(const float (&tops)[kGroups], int lane) {
  float top = neg_inf();
#pragma unroll
  for (int u = 0; u < kGroups; u++) top = fmaxf(top, tops[u]);
  return sort_lanes(top == neg_inf() ? 0u : rank_of(top), lane);
}

struct TokenArgs {
  int64_t rows, vocab, ld;
  const void* logits;
  const int64_t* tokens;
  int64_t ignore;
  float *logprob, *entropy, *stats, *top_logprobs;
  int64_t* top_tokens;
  int top;
  int split;        // CTAs (of a cluster) per row
  int64_t share;    // groups of 8 logits of each
};

// The lists of `count` warps (or CTAs) to one: four warps take a quarter each, then warp 0 theirs.
__device__ __forceinline__ void merge_lists(uint64_t (*lists)[kMostTop], int count, Best& best, int warp, int lane) {
  if (count > 4) {
    if (warp < 4) {
      best.key = warp < count ? lists[warp][lane] : 0;
      for (int i = warp + 4; i < count; i += 4) best.merge(lists[i][lane], lane);
      lists[warp][lane] = best.key;   // only this warp reads or writes it
    }
    __syncthreads();
  }
  if (warp == 0) {
    best.key = lists[0][lane];
    for (int i = 1; i < min(count, 4); i++) best.merge(lists[i][lane], lane);
  }
}

// One row per cluster of `split` CTAs, rows in turn.
//
// The alternatives: logits below a bound that k of them are known to reach are
// passed over.  It comes from the largest logits of the first batch's lanes, and
// from the lists after one, two, four .. batches (of 8 warps' 1024 normal logits
// each about three reach it in the second batch, for k = 20), and from the
// warp's own k-th best.
//
// Many rows take 128 threads each (4096 x 65536 bf16, us without / with 20
// alternatives: 512 threads 179 / 446, 256 144 / 266, 128 131 / 235, 64 125 / 236; now
// 252, and 1060 where every logit is larger than the one before it, which took 12400
// before many at once were sorted into the list): fewer lists to fill, more rows on an SM.  Few rows take 512, and several CTAs each (one
// of 131072, 20 alternatives: 512 threads 11.5, 128 17.5).
template <typename T, int ACCESS, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, (TOP ? 768 : 1024) / THREADS) token_logprobs_kernel(const TokenArgs p) {
  constexpr int kWarps = THREADS / 32;
  __shared__ Sums warp_sums[kWarps];
  __shared__ __align__(16) float4 cta_sums[8];   // m, S, E
  __shared__ uint64_t lists[kWarps][kMostTop];
  __shared__ uint64_t cta_lists[8][kMostTop];
  __shared__ uint32_t bounds[2][32];
  after_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = p.split > 1 ? int(umma::cta_rank()) : 0;
  const int64_t clusters = gridDim.x / p.split;
  if (p.split > 1) umma::cluster_arrive();   // all of the cluster has started: waited for before the first store to another CTA
  bool started = false;
  const uint64_t log2e = pair_of(kLog2e);
  for (int64_t row = blockIdx.x / p.split; row < p.rows; row += clusters) {
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    const int shift = ACCESS == kShifted ? row_shift(x) : 0;
    const int vocab = int(p.vocab), begin = int(rank * p.share), end = min((vocab - 1 + shift) / 8 + 1, begin + int(p.share));
    Sums own = nothing();
    uint64_t s = 0, e2 = 0, minus = 0;   // own.s, own.e and -own.m for pairs
    Best best{0};
    uint64_t least = 0;          // the top-th best key so far
    float bound = neg_inf();     // what is less is passed over
    bool rising = false;         // many of this warp's last batch came into its list
    auto logits_of = [&](const Vec8<T>& a, int g, float (&v)[8]) {
      a.get(v);
      if (ACCESS != kAligned) {
        const int c = g * 8 - shift;
        if (c < 0 || c > vocab - 8) {   // a row's ends
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (c + e < 0 || c + e >= vocab) v[e] = neg_inf();
        }
      }
    };
    auto take = [&](const Vec8<T>& a, int g) {   // a group's alternatives; whole warps
      const int c = g * 8 - shift;
      float v[8];
      uint32_t mine = 0;   // of this lane's eight
      if (g < end) {
        logits_of(a, g, v);
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (!(v[e] < bound) && (ACCESS == kAligned || (c + e >= 0 && c + e < vocab))) mine |= 1u << e;
      }
      // each lane offers the first of its eight that would enter the list; a few are taken one
      // at a time, more are sorted and merged
      while (__any_sync(0xffffffffu, mine != 0)) {
        const int e = __ffs(mine) - 1;
        float x1 = v[0];
#pragma unroll
        for (int i = 1; i < 8; i++)
          if (e == i) x1 = v[i];
        const uint64_t key = mine ? key_of(x1, uint32_t(c + e)) : 0;
        const uint32_t lanes = __ballot_sync(0xffffffffu, key > least);
        const int from = __ffs(lanes) - 1;
        const bool many = __popc(lanes) > kSorted;
        if (key <= least || lane == from || many) mine &= mine - 1;
        if (!lanes) continue;
        rising |= many;
        if (many) best.key = merge_keys(best.key, key);
        else best.insert(__shfl_sync(0xffffffffu, key, from), lane);
        least = __shfl_sync(0xffffffffu, best.key, p.top - 1);
        if (least) bound = fmaxf(bound, value_of_rank(uint32_t(least >> 32)));   // a NaN is passed over by its key
      }
    };
    // A bound from what the block has seen: each warp gives its 32 / W best, `mine`
    // being ranks in descending order over the lanes; k of them reach the k-th.
    int bounded = 0;
    auto tighten = [&](uint32_t mine) {
      const int per = 32 / warps, set = bounded & 1;
      if (lane < per) bounds[set][warp * per + lane] = mine;
      __syncthreads();
      const uint32_t sorted = sort_lanes(lane < per * warps ? bounds[set][lane] : 0u, lane);
      const uint32_t kth = __shfl_sync(0xffffffffu, sorted, p.top - 1);
      if (kth) bound = fmaxf(bound, value_of_rank(kth));
      bounded++;
    };
    int batch = 0;
    // whole warps (TOP: the block) go round together
    for (int g0 = begin; g0 < end || (TOP && batch == 0); g0 += int(blockDim.x) * kGroups, batch++) {
      Vec8<T> a[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; u++) {
        const int g = g0 + u * int(blockDim.x) + int(threadIdx.x), c = g * 8 - shift;
        if (g < end) {
          if constexpr (ACCESS == kScalar) load_any(a[u], x, c, vocab);
          else load_group<ACCESS>(a[u], x, c, vocab);
        }
      }
      float tops[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; u++) {
        const int g = g0 + u * int(blockDim.x) + int(threadIdx.x);
        tops[u] = neg_inf();
        if (g >= end) continue;
        float v[8];
        logits_of(a[u], g, v);
        // NaN stays out of m: it is in the sums
        const float top = TOP ? max_nan(max_nan(v[0], v[1], v[2]), max_nan(v[3], v[4], v[5]), max_nan(v[6], v[7], v[7]))
                              : fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
        tops[u] = top;
        if (top > own.m) {
          own.s = sum_of(s);
          own.e = sum_of(e2);
          own = rebase(own, top);
          s = pair_of(own.s, 0.f);
          e2 = pair_of(own.e, 0.f);
          minus = pair_of(-own.m);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 t = values_of(mul_pair(add_pair(pair_of(v[2 * i], v[2 * i + 1]), minus), log2e));
          const uint64_t f = pair_of(exp2_fast(t.x), exp2_fast(t.y));
          s = add_pair(s, f);
          fma_pair(e2, f, pair_of(least_power(t.x), least_power(t.y)));
        }
      }
      if constexpr (TOP) {
        if (batch == 0) {   // no lists yet: the lanes' largest logits
          tighten(lane_ranks(tops, lane));
        } else if ((batch & (batch - 1)) == 0) {
          tighten(uint32_t(best.key >> 32));
        }
        if (rising) {   // the warp's own bound, as in the first batch
          rising = false;
          const uint32_t kth = __shfl_sync(0xffffffffu, lane_ranks(tops, lane), p.top - 1);
          if (kth) bound = fmaxf(bound, value_of_rank(kth));
        }
#pragma unroll
        for (int u = 0; u < kGroups; u++)
          if (__any_sync(0xffffffffu, g0 + u * int(blockDim.x) + int(threadIdx.x) < end && !(tops[u] < bound)))
            take(a[u], g0 + u * int(blockDim.x) + int(threadIdx.x));
      }
    }
    own.s = sum_of(s);
    own.e = sum_of(e2);
    // the CTA's sums and list
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const Sums o = from_lane(own, d);
      own = lane & d ? join(o, own) : join(own, o);
    }
    if (lane == 0) warp_sums[warp] = own;
    if (TOP) lists[warp][lane] = best.key;
    __syncthreads();
    if (p.split > 1 && !started) umma::cluster_wait();
    started = true;
    if (TOP) merge_lists(lists, warps, best, warp, lane);
    if (warp == 0) {
      own = lane < warps ? warp_sums[lane] : nothing();
#pragma unroll
      for (int d = 8; d; d >>= 1) {
        const Sums o = from_lane(own, d);
        own = lane & d ? join(o, own) : join(own, o);
      }
      if (p.split > 1) {
        const uint32_t to = umma::map_rank(umma::smem_u32(&cta_sums[rank]), 0);
        if (lane == 0) umma::store_cluster(to, __float_as_uint(own.m), __float_as_uint(own.s), __float_as_uint(own.e), 0u);
        if (TOP)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(umma::map_rank(umma::smem_u32(&cta_lists[rank][lane]), 0)), "l"(best.key) : "memory");
      }
    }
    if (p.split > 1) umma::cluster_sync();
    if (p.split > 1 && rank == 0 && TOP) merge_lists(cta_lists, p.split, best, warp, lane);
    if (warp == 0 && rank == 0) {
      if (p.split > 1) {
        own = lane < p.split ? Sums{cta_sums[lane].x, cta_sums[lane].y, cta_sums[lane].z} : nothing();
#pragma unroll
        for (int d = 4; d; d >>= 1) {
          const Sums o = from_lane(own, d);
          own = lane & d ? join(o, own) : join(own, o);
        }
      }
      own = {__shfl_sync(0xffffffffu, own.m, 0), __shfl_sync(0xffffffffu, own.s, 0), __shfl_sync(0xffffffffu, own.e, 0)};
      const bool empty = own.m == neg_inf() && own.s == 0.f;
      const float logs = logf(own.s);
      auto logp = [&](float v) { return empty ? neg_inf() : (v - own.m) - logs; };
      if (lane == 0) {
        if (p.logprob) {
          const int64_t token = p.tokens[row];
          float lp = __int_as_float(0x7fffffff);
          if (token == p.ignore) lp = 0.f;
          else if (token >= 0 && token < p.vocab) lp = logp(to_f32(x[token]));
          p.logprob[row] = lp;
        }
        if (p.entropy) p.entropy[row] = empty ? 0.f : logs - own.e / own.s * kLn2;
        if (p.stats) {
          p.stats[2 * row] = own.m;
          p.stats[2 * row + 1] = logs;   // -infinity of an empty row
        }
      }
      if (TOP && lane < p.top) {
        p.top_logprobs[row * p.top + lane] = logp(logit_of(best.key));
        p.top_tokens[row * p.top + lane] = token_of(best.key);
      }
    }
    if (p.split > 1) umma::cluster_sync();   // the lists are read
    else __syncthreads();
  }
}

struct TokenBackArgs {
  int64_t rows, vocab, ld, ldg;
  const void* logits;
  const int64_t* tokens;
  int64_t ignore;
  const float *stats, *entropy, *grad_logprob, *grad_entropy;
  void* grad;
};

// Parts of kPart groups of a row, kGroups of 8 logits per thread at a time.
constexpr int64_t kPart = 256 * kGroups * 2;
template <typename T, int ACCESS>
__global__ void __launch_bounds__(256) token_logprobs_backward_kernel(const TokenBackArgs p, int64_t parts) {
  after_previous_kernel();
  const uint64_t log2e = pair_of(kLog2e);
  for (int64_t item = blockIdx.x; item < p.rows * parts; item += gridDim.x) {
    const int64_t row = item / parts, from = (item - row * parts) * kPart;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    T* out = static_cast<T*>(p.grad) + row * p.ldg;
    const int shift = ACCESS == kShifted ? row_shift(x) : 0;
    const int64_t end = min((p.vocab + shift + 7) / 8, from + kPart);
    const float m = p.stats[2 * row], logs = p.stats[2 * row + 1];
    const bool empty = m == neg_inf() && logs == m;
    const int64_t token = p.grad_logprob ? p.tokens[row] : p.ignore;
    float g = token != p.ignore ? p.grad_logprob[row] : 0.f;
    if (token != p.ignore && (token < 0 || token >= p.vocab)) g = __int_as_float(0x7fffffff);
    const float gh = p.grad_entropy ? p.grad_entropy[row] : 0.f, h = p.grad_entropy ? p.entropy[row] : 0.f;
    const uint64_t minus_m = pair_of(-m), minus_s = pair_of(-logs);
    const uint64_t slope = pair_of(-gh * kLn2), offset = pair_of(-fmaf(gh, h, g));
    for (int64_t i = from + threadIdx.x; i < end; i += 256 * kGroups) {
      Vec8<T> a[kGroups];
#pragma unroll
      for (int u = 0; u < kGroups; u++) {
        const int64_t c = (i + u * 256) * 8 - shift;
        if (i + u * 256 < end) {
          if constexpr (ACCESS == kScalar) load_any(a[u], x, c, p.vocab);
          else load_group<ACCESS>(a[u], x, int(c), int(p.vocab));
        }
      }
#pragma unroll
      for (int u = 0; u < kGroups; u++) {
        const int64_t c = (i + u * 256) * 8 - shift;
        if (i + u * 256 >= end) continue;
        uint64_t v[4];
        float o[8];
        get_pairs(a[u], v);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float2 t = values_of(mul_pair(add_pair(add_pair(v[j], minus_m), minus_s), log2e));   // log2 p
          v[j] = mul_pair(pair_of(exp2_fast(t.x), exp2_fast(t.y)), fma_pair_of(pair_of(least_power(t.x), least_power(t.y)), slope, offset));
        }
        from_pairs(v, o);
        if (token >= c && token < c + 8) {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (c + e == token) o[e] += g;
        }
        if (empty) {
#pragma unroll
          for (int e = 0; e < 8; e++) o[e] = 0.f;
        }
        if constexpr (ACCESS == kScalar) store_any(out, c, p.vocab, o);
        else store_group<ACCESS>(out, int(c), int(p.vocab), o);
      }
    }
  }
}

}  // namespace tgb

namespace tgi {

using tgb::kGroups;
using tgb::kFewRows;
using tgb::kManyRows;
using tgb::TokenArgs;
using tgb::TokenBackArgs;

namespace {

tg_status check_logits(tg_dtype dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld) {
  if (!elem8_size(dtype)) return fail(TG_ERR_INVALID_ARGUMENT, "logits must be f32, f16 or bf16, got dtype %d", int(dtype));
  if (rows < 0 || vocab < 0) return fail(TG_ERR_INVALID_ARGUMENT, "negative size (rows=%lld vocab=%lld)", (long long)rows, (long long)vocab);
  if (vocab > 0x7fffff00) return fail(TG_ERR_UNSUPPORTED, "vocab=%lld", (long long)vocab);
  if (rows == 0) return TG_OK;
  if (vocab == 0) return fail(TG_ERR_INVALID_ARGUMENT, "a row of no logits has no distribution");
  if (!logits) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (ld < vocab) return fail(TG_ERR_DIMENSION_MISMATCH, "ld=%lld < %lld", (long long)ld, (long long)vocab);
  return TG_OK;
}
template <typename F> void with_mode(int access, F&& f) {
  if (access == tg8::kAligned) f(std::integral_constant<int, tg8::kAligned>{});
  else if (access == tg8::kShifted) f(std::integral_constant<int, tg8::kShifted>{});
  else f(std::integral_constant<int, tg8::kScalar>{});
}
#define TG_CHECK(call)                  \
  do {                                  \
    const tg_status s_ = (call);        \
    if (s_ != TG_OK) return s_;         \
  } while (0)

}  // namespace
}  // namespace tgi

using namespace tgi;

extern "C" {

tg_status tg_token_logprobs(tg_dtype dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld, const int64_t* tokens,
                            int64_t ignore_index, float* logprob, float* entropy, float* stats, int top, float* top_logprobs,
                            int64_t* top_tokens, void* stream) {
  clear_error();
  TG_CHECK(check_logits(dtype, rows, vocab, logits, ld));
  if (top < 0 || top > tgb::kMostTop) return fail(TG_ERR_INVALID_ARGUMENT, "top must be 0 to %d, got %d", tgb::kMostTop, top);
  if (rows == 0) return TG_OK;
  if (top > vocab) return fail(TG_ERR_INVALID_ARGUMENT, "top=%d of %lld tokens", top, (long long)vocab);
  if ((tokens != nullptr) != (logprob != nullptr)) return fail(TG_ERR_INVALID_ARGUMENT, "tokens and logprob are given together or not at all");
  if (top && (!top_logprobs || !top_tokens)) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  TokenArgs p{};
  p.rows = rows; p.vocab = vocab; p.ld = ld; p.logits = logits; p.tokens = tokens; p.ignore = ignore_index;
  p.logprob = logprob; p.entropy = entropy; p.stats = stats; p.top = top; p.top_logprobs = top_logprobs; p.top_tokens = top_tokens;
  RowAccess access(vocab);
  access.add(logits, ld, elem8_size(dtype));
  const int64_t groups = (vocab + 7 + 7) / 8;
  // Few rows: several CTAs share one, each with at least one round of its threads.
  p.split = 1;
  while (p.split < 8 && rows * p.split * 2 <= sm_count() && groups >= kFewRows * kGroups * p.split) p.split *= 2;
  p.share = (groups + p.split - 1) / p.split;
  // (us, 128 / 512 threads: 600 x 131072 bf16 71 / 57, 900 x 131072 73 / 77; with 20 alternatives 296 x 50000 30 / 29, 444 x 50000 34 / 43)
  const bool many = rows * p.split >= (top ? 3 : 5) * int64_t(sm_count());
  // threads for one round of kGroups groups each
  const int threads = int(std::max<int64_t>(32, std::min<int64_t>(many ? kManyRows : kFewRows, (p.share + 32 * kGroups - 1) / (32 * kGroups) * 32)));
  const int64_t clusters = std::min<int64_t>(rows, int64_t(1) << 16);   // rows beyond that in turn
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    with_mode(access.get(), [&](auto mode) {
      constexpr int A = decltype(mode)::value;
      const dim3 grid(unsigned(clusters * p.split));
      const int cluster = p.split > 1 ? p.split : 0;
      auto go = [&](auto kern) { launch_kernel(kern, grid, threads, 0, cluster, static_cast<cudaStream_t>(stream), p); };
      if (many && top) go(tgb::token_logprobs_kernel<T, A, true, kManyRows>);
      else if (many) go(tgb::token_logprobs_kernel<T, A, false, kManyRows>);
      else if (top) go(tgb::token_logprobs_kernel<T, A, true, kFewRows>);
      else go(tgb::token_logprobs_kernel<T, A, false, kFewRows>);
    });
    return check_launch("token logprobs");
  });
}

tg_status tg_token_logprobs_backward(tg_dtype dtype, int64_t rows, int64_t vocab, const void* logits, int64_t ld,
                                     const int64_t* tokens, int64_t ignore_index, const float* stats, const float* entropy,
                                     const float* grad_logprob, const float* grad_entropy, void* grad_logits, int64_t ldg,
                                     void* stream) {
  clear_error();
  TG_CHECK(check_logits(dtype, rows, vocab, logits, ld));
  if (rows == 0) return TG_OK;
  if (!stats || !grad_logits || (grad_logprob && !tokens) || (grad_entropy && !entropy)) return fail(TG_ERR_INVALID_ARGUMENT, "null operand");
  if (ldg < vocab) return fail(TG_ERR_DIMENSION_MISMATCH, "ldg=%lld < %lld", (long long)ldg, (long long)vocab);
  TokenBackArgs p{};
  p.rows = rows; p.vocab = vocab; p.ld = ld; p.ldg = ldg; p.logits = logits; p.tokens = tokens; p.ignore = ignore_index;
  p.stats = stats; p.entropy = entropy; p.grad_logprob = grad_logprob; p.grad_entropy = grad_entropy; p.grad = grad_logits;
  const size_t e = elem8_size(dtype);
  RowAccess access(vocab);
  access.add(logits, ld, e);
  access.add(grad_logits, ldg, e);
  const int64_t parts = (vocab + 7 + 7) / 8 / tgb::kPart + 1;
  const unsigned grid = unsigned(std::min<int64_t>(rows * parts, int64_t(sm_count()) * 8));
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    with_mode(access.get(), [&](auto mode) {
      launch_kernel(tgb::token_logprobs_backward_kernel<T, decltype(mode)::value>, grid, 256, 0, 0, static_cast<cudaStream_t>(stream), p, parts);
    });
    return check_launch("token logprobs backward");
  });
}

}  // extern "C"
