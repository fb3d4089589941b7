// Log probabilities of given tokens, entropies and the most likely tokens from
// rows of logits, and the gradient of the logits.
//
//   m = max x, S = sum exp(x - m), E = sum exp(x - m) (x - m)
//   logprob = (x_token - m) - log S,  entropy = log S - E / S
//   grad_v = g_lp ([v == token] - p_v) - g_H p_v (log p_v + entropy)
//
// One pass: each thread keeps m, S and E of what it has seen and rescales them
// when a larger logit comes; each warp keeps its most likely tokens sorted
// across its lanes.  Bound by memory, one exponential per logit beside it.
#include <algorithm>
#include "tg_blocks8.cuh"
#include "tg_umma.cuh"

namespace tgb {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMostTop = 32;   // alternatives: one per lane
constexpr int kWarps = 16;

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// x - m for the sums: below -1000 the exponential is zero either way, and a
// product with it must not be 0 * infinity.  Keeps a NaN.
__device__ __forceinline__ float below(float x, float m) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x - m), "f"(-1000.f));
  return r;
}

struct Sums {
  float m, s, e;   // largest logit, sum of exp(x - m), sum of exp(x - m) (x - m)
};
// What a thread with nothing but -infinity so far measures from: any finite value does.
__device__ __forceinline__ float base_of(float m) { return m == -__int_as_float(0x7f800000) ? 0.f : m; }
__device__ __forceinline__ Sums rebase(const Sums& a, float m) {
  if (a.m == m || a.s == 0.f) return {m, a.s, a.e};
  const float d = below(a.m, m), f = exp2_fast(d * kLog2e);
  return {m, a.s * f, (a.e + a.s * d) * f};
}
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  const Sums x = rebase(a, m), y = rebase(b, m);
  return {m, x.s + y.s, x.e + y.e};
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

// One row per cluster of `split` CTAs, rows in turn.
template <typename T, int ACCESS, bool TOP>
__global__ void __launch_bounds__(512) token_logprobs_kernel(const TokenArgs p) {
  __shared__ Sums warp_sums[kWarps];
  __shared__ Sums cta_sums[8];
  __shared__ uint64_t lists[kWarps][kMostTop];
  __shared__ uint64_t cta_lists[8][kMostTop];
  after_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = p.split > 1 ? int(umma::cta_rank()) : 0;
  const int64_t clusters = gridDim.x / p.split;
  if (p.split > 1) umma::cluster_arrive();   // all of the cluster has started: waited for before the first store to another CTA
  bool started = false;
  for (int64_t row = blockIdx.x / p.split; row < p.rows; row += clusters) {
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    const int shift = ACCESS == kShifted ? row_shift(x) : 0;
    const int64_t end = min((p.vocab + shift + 7) / 8, (rank + 1) * p.share);
    Sums own{-__int_as_float(0x7f800000), 0.f, 0.f};
    Best best{0};
    uint64_t least = 0;   // the top-th best key so far
    // whole warps go round together
    for (int64_t g0 = rank * p.share + warp * 32; g0 < end; g0 += warps * 32) {
      const int64_t g = g0 + lane, c = g * 8 - shift;
      float v[8];
      Vec8<T> a;
      if (g < end) {
        if constexpr (ACCESS == kScalar) load_any(a, x, c, p.vocab);
        else load_group<ACCESS>(a, x, int(c), int(p.vocab));
      } else {
        a.zero();
      }
      a.get(v);
      float top = -__int_as_float(0x7f800000);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        if (g >= end || c + e < 0 || c + e >= p.vocab) v[e] = -__int_as_float(0x7f800000);
        top = fmaxf(top, v[e]);
      }
      if (top > own.m) own = rebase(own, top);
      const float base = base_of(own.m);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = below(v[e], base), f = exp2_fast(d * kLog2e);
        own.s += f;
        own.e = fmaf(f, d, own.e);
      }
      if constexpr (TOP) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const bool in = g < end && c + e >= 0 && c + e < p.vocab;
          const uint64_t k = in ? key_of(v[e], uint32_t(c + e)) : 0;
          uint32_t more = __ballot_sync(0xffffffffu, k > least);
          while (more) {
            const uint64_t next = __shfl_sync(0xffffffffu, k, __ffs(more) - 1);
            more &= more - 1;
            if (next <= least) continue;
            best.insert(next, lane);
            least = __shfl_sync(0xffffffffu, best.key, p.top - 1);
          }
        }
      }
    }
    // the CTA's sums and list
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const Sums o{__shfl_xor_sync(0xffffffffu, own.m, d), __shfl_xor_sync(0xffffffffu, own.s, d), __shfl_xor_sync(0xffffffffu, own.e, d)};
      own = lane & d ? join(o, own) : join(own, o);
    }
    if (lane == 0) warp_sums[warp] = own;
    if (TOP) lists[warp][lane] = best.key;
    __syncthreads();
    if (p.split > 1 && !started) umma::cluster_wait();
    started = true;
    if (warp == 0) {
      own = warp_sums[0];
      for (int w = 1; w < warps; w++) own = join(own, warp_sums[w]);
      if (TOP)
        for (int w = 1; w < warps; w++) best.merge(lists[w][lane], lane);
      if (p.split > 1) {
        const uint32_t to = umma::map_rank(umma::smem_u32(&cta_sums[rank]), 0);
        if (lane == 0) {
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(own.m) : "memory");
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(own.s) : "memory");
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(own.e) : "memory");
        }
        if (TOP)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(umma::map_rank(umma::smem_u32(&cta_lists[rank][lane]), 0)), "l"(best.key) : "memory");
      }
    }
    if (p.split > 1) umma::cluster_sync();
    if (warp == 0 && rank == 0) {
      if (p.split > 1) {
        own = cta_sums[0];
        for (int r = 1; r < p.split; r++) own = join(own, cta_sums[r]);
        if (TOP)
          for (int r = 1; r < p.split; r++) best.merge(cta_lists[r][lane], lane);
      }
      const bool empty = own.m == -__int_as_float(0x7f800000) && own.s == 0.f;
      const float logs = logf(own.s);
      if (lane == 0) {
        if (p.logprob) {
          const int64_t token = p.tokens[row];
          float lp = __int_as_float(0x7fffffff);
          if (token == p.ignore) lp = 0.f;
          else if (token >= 0 && token < p.vocab) lp = empty ? -__int_as_float(0x7f800000) : (to_f32(x[token]) - own.m) - logs;
          p.logprob[row] = lp;
        }
        if (p.entropy) p.entropy[row] = empty ? 0.f : logs - own.e / own.s;
        if (p.stats) {
          p.stats[2 * row] = own.m;
          p.stats[2 * row + 1] = logs;
        }
      }
      if (TOP && lane < p.top) {
        p.top_logprobs[row * p.top + lane] = empty ? -__int_as_float(0x7f800000) : (logit_of(best.key) - own.m) - logs;
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

template <typename T, int ACCESS>
__global__ void __launch_bounds__(256) token_logprobs_backward_kernel(const TokenBackArgs p) {
  after_previous_kernel();
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    T* out = static_cast<T*>(p.grad) + row * p.ldg;
    const int shift = ACCESS == kShifted ? row_shift(x) : 0;
    const float m = p.stats[2 * row], logs = p.stats[2 * row + 1];
    const bool empty = m == -__int_as_float(0x7f800000) && logs == m;
    const int64_t token = p.grad_logprob ? p.tokens[row] : p.ignore;
    float g = token != p.ignore ? p.grad_logprob[row] : 0.f;
    if (token != p.ignore && (token < 0 || token >= p.vocab)) g = __int_as_float(0x7fffffff);
    const float gh = p.grad_entropy ? p.grad_entropy[row] : 0.f, h = p.grad_entropy ? p.entropy[row] : 0.f;
    const int64_t groups = (p.vocab + shift + 7) / 8;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < groups; i += int64_t(gridDim.x) * 256) {
      const int64_t c = i * 8 - shift;
      Vec8<T> a;
      float v[8];
      if constexpr (ACCESS == kScalar) load_any(a, x, c, p.vocab);
      else load_group<ACCESS>(a, x, int(c), int(p.vocab));
      a.get(v);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float logp = below(v[e], m) - logs, prob = exp2_fast(logp * kLog2e);
        float d = -prob * fmaf(gh, logp + h, g);
        if (c + e == token) d += g;
        v[e] = empty ? 0.f : d;
      }
      if constexpr (ACCESS == kScalar) store_any(out, c, p.vocab, v);
      else store_group<ACCESS>(out, int(c), int(p.vocab), v);
    }
  }
}

}  // namespace tgb

namespace tgi {

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
  p.split = 1;
  while (p.split < 8 && rows * p.split * 2 <= 2 * int64_t(sm_count()) && groups >= 512 * 2 * p.split) p.split *= 2;
  p.share = (groups + p.split - 1) / p.split;
  const int64_t clusters = std::min<int64_t>(rows, std::max<int64_t>(1, 4 * int64_t(sm_count()) / p.split));
  const int threads = int(std::max<int64_t>(32, std::min<int64_t>(512, (p.share + 31) / 32 * 32)));
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    with_mode(access.get(), [&](auto mode) {
      constexpr int A = decltype(mode)::value;
      const dim3 grid(unsigned(clusters * p.split));
      const int cluster = p.split > 1 ? p.split : 0;
      if (top) launch_kernel(tgb::token_logprobs_kernel<T, A, true>, grid, threads, 0, cluster, static_cast<cudaStream_t>(stream), p);
      else launch_kernel(tgb::token_logprobs_kernel<T, A, false>, grid, threads, 0, cluster, static_cast<cudaStream_t>(stream), p);
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
  const unsigned across = unsigned(std::min<int64_t>((vocab + 7 + 2047) / 2048, 64));
  return with_type8(dtype, [&](auto t) {
    using T = decltype(t);
    with_mode(access.get(), [&](auto mode) {
      launch_kernel(tgb::token_logprobs_backward_kernel<T, decltype(mode)::value>, dim3(across, unsigned(std::min<int64_t>(rows, 65535))), 256, 0, 0,
                    static_cast<cudaStream_t>(stream), p);
    });
    return check_launch("token logprobs backward");
  });
}

}  // extern "C"
