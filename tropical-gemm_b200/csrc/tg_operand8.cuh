// Host side of the products of 8-bit matrices: scratch of one call, and copies
// of operands whose rows a TMA load cannot take.
#pragma once
#include <algorithm>
#include "tg_rows8.cuh"

namespace tg8 {

// 8-bit rows copied to rows of ldo, a multiple of 16, zeros behind; up to two
// matrices in one launch (blockIdx.z).  16 bytes per thread: the one or two
// aligned 16-byte words that hold them (each with at least one byte of the
// row), shifted into place.
struct PadArgs {
  const int8_t* q[2];
  int8_t* out[2];
  int64_t rows[2], cols[2], ldq[2], ldo[2];
};
static __global__ void __launch_bounds__(256) pad8_kernel(const __grid_constant__ PadArgs p) {   // indexed in place: a copy per thread took 17 of 31 us at 4096 x 4095
  after_previous_kernel();
  const int z = blockIdx.z;
  const int64_t per = p.ldo[z] / 16, total = p.rows[z] * per;
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t r = total <= 0xffffffffll ? int64_t(uint32_t(i) / uint32_t(per)) : i / per, c = (i - r * per) * 16;
    const int64_t left = p.cols[z] - c;   // bytes of the row from c on
    uint32_t o[4] = {0, 0, 0, 0};
    if (left > 0) {
      const int8_t* from = p.q[z] + r * p.ldq[z] + c;
      const uint32_t skew = uint32_t(reinterpret_cast<uintptr_t>(from) & 15);
      const uint4* words = reinterpret_cast<const uint4*>(from - skew);
      const uint4 lo = words[0], hi = skew && 16 < left + skew ? words[1] : make_uint4(0, 0, 0, 0);
      uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      if (skew & 8) {
#pragma unroll
        for (int k = 0; k < 6; k++) w[k] = w[k + 2];
      }
      if (skew & 4) {
#pragma unroll
        for (int k = 0; k < 5; k++) w[k] = w[k + 1];
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        o[k] = __funnelshift_r(w[k], w[k + 1], (skew & 3) * 8);
        const int64_t valid = left - 4 * k;
        if (valid < 4) o[k] = valid <= 0 ? 0u : o[k] & ((1u << (8 * valid)) - 1);
      }
    }
    *reinterpret_cast<uint4*>(p.out[z] + r * p.ldo[z] + c) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

}  // namespace tg8

namespace tgi {

// Scratch of one call, freed in stream order when the call returns.
class Scratch {
 public:
  explicit Scratch(cudaStream_t st) : st_(st) {}
  Scratch(const Scratch&) = delete;
  ~Scratch() {
    if (p_) scratch_free(p_, st_);
  }
  cudaError_t reserve(size_t bytes) { return scratch_alloc(&p_, bytes, st_); }
  template <typename T> T* take(size_t count) {
    T* r = reinterpret_cast<T*>(static_cast<char*>(p_) + used_);
    used_ += size_of<T>(count);
    return r;
  }
  template <typename T> static size_t size_of(size_t count) { return (count * sizeof(T) + 255) & ~size_t(255); }

 private:
  void* p_ = nullptr;
  size_t used_ = 0;
  cudaStream_t st_;
};

// Rows and columns of C: the kernels count them, and the edges of the last tiles,
// in 32 bits (TMA's coordinates are 32-bit too).
constexpr int64_t kMostOutputs = 0x7ffffc00;

inline int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// 8-bit rows a TMA load can take: 16-byte aligned rows of at least one byte.
inline bool tma_rows8(const int8_t* q, int64_t ld, int64_t rows, int64_t cols) {
  return cols > 0 && aligned(q, 16) && (ld % 16 == 0 || rows == 1);
}
struct Operand8 {
  const int8_t* q;
  int64_t ld, rows, cols;
  bool pad;
  Operand8(const int8_t* q_, int64_t ld_, int64_t rows_, int64_t cols_)
      : q(q_), ld(ld_), rows(rows_), cols(cols_), pad(!tma_rows8(q_, ld_, rows_, cols_)) {}
  int64_t padded() const { return std::max<int64_t>(16, round_up(cols, 16)); }
  size_t scratch() const { return pad ? Scratch::size_of<int8_t>(size_t(rows) * size_t(padded())) : 0; }
  // Takes the place of a padded copy where the rows are not aligned, to be
  // filled by pad_operands; a sum of nothing becomes a sum over one zero.
  void place(Scratch& s, tg8::PadArgs& p, int& count) {
    if (pad) {
      int8_t* out = s.take<int8_t>(size_t(rows) * size_t(padded()));
      p.q[count] = q;
      p.out[count] = out;
      p.rows[count] = rows;
      p.cols[count] = cols;
      p.ldq[count] = ld;
      p.ldo[count] = padded();
      count++;
      q = out;
      ld = padded();
      cols = std::max<int64_t>(cols, 1);
    } else if (rows == 1) {
      ld = padded();
    }
  }
  bool map(uint32_t box_cols, uint32_t box_rows, CUtensorMap* m) const {
    return encode_tma(CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q, cols, rows, ld, 1, 0, box_cols, box_rows, m);
  }
};

inline void pad_operands(const tg8::PadArgs& p, int count, cudaStream_t st) {
  int64_t most = 0;
  for (int i = 0; i < count; i++) most = std::max(most, (p.rows[i] * (p.ldo[i] / 16) + 255) / 256);
  if (most) launch_kernel(tg8::pad8_kernel, dim3(unsigned(std::min<int64_t>(most, 8192)), 1, unsigned(count)), 256, 0, 0, st, p);
}

}  // namespace tgi
