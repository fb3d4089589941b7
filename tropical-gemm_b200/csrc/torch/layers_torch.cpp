// torch binding of layer norm, of linear layers in 8-bit floating point and of
// token log probabilities: argument checks, outputs from torch's allocator,
// torch's current stream, autograd.  The work is the C ABI's
// (include/tropical_gemm_b200.h).
#include "binding.h"
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/variable.h>

namespace {

int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

void check_columns(const Tensor& t, const Tensor& like, int64_t k, const char* what) {
  if (t.defined() && (t.scalar_type() != like.scalar_type() || t.dim() != 1 || t.size(0) != k))
    refuse(what, " must be ", name(like.scalar_type()), " of shape (", k, ",), got ", name(t.scalar_type()), " ", shape(t.sizes()));
}
void check_like(const Tensor& t, const Tensor& like, const char* what, const char* whose) {
  if (t.defined() && (t.scalar_type() != like.scalar_type() || t.sizes() != like.sizes()))
    refuse(what, " must be like ", whose, " (", name(like.scalar_type()), " ", shape(like.sizes()), "), got ", name(t.scalar_type()), " ", shape(t.sizes()));
}
void check_row_values(const Tensor& t, const Tensor& rows, const char* what) {   // one f32 per row
  if (t.defined() && (t.scalar_type() != at::kFloat || t.sizes() != rows.sizes().slice(0, rows.dim() - 1)))
    refuse(what, " must be float32 of shape ", shape(rows.sizes().slice(0, rows.dim() - 1)), ", got ", name(t.scalar_type()), " ", shape(t.sizes()));
}

// ------------------------------------------------------------------------------------------------ 8-bit blocks
struct Blocks {   // codes and scales as tensors
  Tensor q, scale;
};
// Codes with rows of a multiple of 16 bytes (what the tensor core's loads take).
Tensor make_codes(at::IntArrayRef sizes, const Tensor& like) {
  at::DimVector padded(sizes.begin(), sizes.end());
  const int64_t k = padded.back();
  padded.back() = (k + 15) / 16 * 16;
  Tensor t = make(padded, like, at::kFloat8_e4m3fn);
  return padded.back() == k ? t : t.narrow(-1, 0, k);
}
// One scale per row and block, rows next to one another.
Tensor make_scales(at::IntArrayRef sizes, const Tensor& like) {
  at::DimVector size(sizes.begin(), sizes.end()), stride(sizes.size());
  size.back() = blocks_of(sizes.back());
  int64_t rows = 1;
  for (int64_t i = int64_t(sizes.size()) - 2; i >= 0; i--) {
    stride[i] = std::max<int64_t>(rows, 1);
    rows *= sizes[i];
  }
  stride.back() = std::max<int64_t>(rows, 1);
  if (watched()) return at::empty_strided(size, stride, like.options().dtype(at::kFloat).requires_grad(false));
  return Tensor(at::detail::empty_strided_cuda(size, stride, at::kFloat, like.device()));
}
int64_t pitch(const Tensor& q) { return q.size(-1) == 0 ? 0 : (q.size(-1) + 15) / 16 * 16; }   // of make_codes

// Scales as (rows, blocks) with strides.
struct FlatScale {
  Tensor t;
  explicit FlatScale(const Tensor& s) {
    t = s.detach();
    if (t.dim() != 2) t = t.reshape({rows_of(s), s.size(-1)});
  }
  float* ptr() const { return f32(t); }
  int64_t row() const { return t.size(0) > 1 ? t.stride(0) : 0; }
  int64_t block() const { return t.size(1) > 1 ? t.stride(1) : 0; }
};

// 1 or 128, the rows that share a scale.
int check_blocks8(const Tensor& q, const Tensor& s, const char* what) {
  if (q.scalar_type() != at::kFloat8_e4m3fn || s.scalar_type() != at::kFloat)
    refuse(what, " must be float8_e4m3fn codes with float32 scales, got ", name(q.scalar_type()), " and ", name(s.scalar_type()));
  if (q.dim() > 0 && s.dim() == q.dim() && s.size(-1) == blocks_of(q.size(-1))) {
    if (s.sizes().slice(0, s.dim() - 1) == q.sizes().slice(0, q.dim() - 1)) return 1;
    if (q.dim() == 2 && s.size(0) == blocks_of(q.size(0))) return 128;
  }
  refuse(what, " needs one scale per row and block of 128 columns, or (two-dimensional) per tile of 128 x 128: q is ", shape(q.sizes()), ", scale is ", shape(s.sizes()));
}

// x along its rows, with `turned` along its columns (as rows of x^T; leading dimensions make one), and its columns' sums.
void quantize_into(const Tensor& x, Blocks* rows, Blocks* turned, Tensor* sum = nullptr) {
  const tg_dtype code = type(x.scalar_type(), "x");
  on(x.device());
  if (x.dim() == 0) refuse("expected a tensor with at least one dimension");
  c10::cuda::CUDAGuard guard(x.device());
  const Flat f(x);
  const int64_t m = rows_of(x), k = x.size(-1);
  void *q = nullptr, *qt = nullptr;
  float *s = nullptr, *st = nullptr;
  int64_t ldq = 0, ldqt = 0;
  if (rows) {
    rows->q = make_codes(x.sizes(), x);
    rows->scale = make_scales(x.sizes(), x);
    q = ptr(rows->q); s = f32(rows->scale); ldq = pitch(rows->q);
  }
  if (turned) {
    turned->q = make_codes({k, m}, x);
    turned->scale = make_scales({k, m}, x);
    qt = ptr(turned->q); st = f32(turned->scale); ldqt = pitch(turned->q);
  }
  if (sum) *sum = make({k}, x, x.scalar_type());
  check(tg_blocks8_quantize(code, m, k, f.ptr(), f.ld, q, ldq, s, 1, m, qt, ldqt, st, 1, k, sum ? ptr(*sum) : nullptr, stream(x.device())));
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x) {
  Blocks r;
  quantize_into(x, &r, nullptr);
  return {r.q, r.scale};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> quantize_both(const Tensor& x) {
  Blocks r, t;
  quantize_into(x, &r, &t);
  return {r.q, r.scale, t.q, t.scale};
}

void quantize_tiles_into(const Tensor& w, Blocks* tiles, Tensor* turned) {
  const tg_dtype code = type(w.scalar_type(), "w");
  on(w.device());
  if (w.dim() != 2) refuse("w must be two-dimensional, got ", shape(w.sizes()));
  c10::cuda::CUDAGuard guard(w.device());
  const Flat f(w);
  const int64_t n = w.size(0), k = w.size(1);
  tiles->q = make_codes(w.sizes(), w);
  tiles->scale = make({blocks_of(n), blocks_of(k)}, w, at::kFloat);
  if (turned) *turned = make_codes({k, n}, w);
  check(tg_blocks8_quantize_tiles(code, n, k, f.ptr(), f.ld, ptr(tiles->q), pitch(tiles->q), f32(tiles->scale), blocks_of(k), 1,
                                  turned ? ptr(*turned) : nullptr, turned ? pitch(*turned) : 0, stream(w.device())));
}
std::tuple<Tensor, Tensor, Tensor> quantize_tiles(const Tensor& w, bool turn) {
  Blocks r;
  Tensor t;
  quantize_tiles_into(w, &r, turn ? &t : nullptr);
  return {r.q, r.scale, t};
}

Tensor dequantize(const Tensor& q, const Tensor& scale, const py::object& dtype) {
  const int tall = check_blocks8(q, scale, "blocks");
  on(q.device(), {&scale});
  const at::ScalarType t = dtype_arg(dtype, at::kBFloat16, "dtype");
  c10::cuda::CUDAGuard guard(q.device());
  const Flat f(q);
  const FlatScale s(scale);
  const int64_t k = q.size(-1);
  Tensor y = make(q.sizes(), q, t);
  check(tg_blocks8_dequantize(type(t, "dtype"), rows_of(q), k, tall, f.ptr(), f.ld, s.ptr(), s.row(), s.block(), ptr(y), k, stream(q.device())));
  return y;
}

Tensor transpose(const Tensor& q) {
  if (q.scalar_type() != at::kFloat8_e4m3fn || q.dim() != 2) refuse("expected two-dimensional float8_e4m3fn codes, got ", name(q.scalar_type()), " ", shape(q.sizes()));
  on(q.device());
  c10::cuda::CUDAGuard guard(q.device());
  const Flat f(q);
  Tensor t = make_codes({q.size(1), q.size(0)}, q);
  check(tg_blocks8_transpose(q.size(0), q.size(1), f.ptr(), f.ld, ptr(t), pitch(t), stream(q.device())));
  return t;
}

Tensor matmul(const Tensor& aq, const Tensor& a_scale, const Tensor& bq, const Tensor& b_scale, const OptTensor& bias_arg, at::ScalarType t) {
  const Tensor& bias = or_none(bias_arg);
  if (check_blocks8(aq, a_scale, "a") != 1) refuse("a must have one scale per row and block of 128 columns: q is ", shape(aq.sizes()), ", scale is ", shape(a_scale.sizes()));
  const int tall = check_blocks8(bq, b_scale, "b");
  const at::Device dev = aq.device();
  on(dev, {&a_scale, &bq, &b_scale, &bias});
  if (bq.dim() != 2) refuse("b must be two-dimensional (channels, K), got ", shape(bq.sizes()));
  const int64_t n = bq.size(0), k = bq.size(1);
  if (aq.size(-1) != k) refuse("Dimension mismatch: a has ", aq.size(-1), " columns, b has ", k);
  if (bias.defined() && (bias.scalar_type() != t || bias.dim() != 1 || bias.size(0) != n))
    refuse("bias must be ", name(t), " of shape (", n, ",), got ", name(bias.scalar_type()), " ", shape(bias.sizes()));
  c10::cuda::CUDAGuard guard(dev);
  const Flat a(aq), b(bq);
  const FlatScale as(a_scale), bs(b_scale);
  const Tensor bi = dense(bias);
  Tensor c = make(with_last(aq, n), aq, t);
  check(tg_blocks8_gemm(type(t, "dtype"), rows_of(aq), n, k, a.ptr(), a.ld, as.ptr(), as.row(), as.block(), b.ptr(), b.ld, tall,
                        bs.ptr(), bs.row(), bs.block(), ptr(bi), ptr(c), n, stream(dev)));
  return c;
}

// ------------------------------------------------------------------------------------------------ layer norm
struct Norm {
  Tensor y, h, mean, rstd;
  Blocks blocks;
};
Norm norm(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps, bool stats, bool in_blocks) {
  const tg_dtype code = type(x.scalar_type(), "x");
  const at::Device dev = x.device();
  on(dev, {&weight, &bias, &residual});
  const int64_t k = x.dim() ? x.size(-1) : 0;
  if (k == 0) refuse("x needs at least one column");
  check_columns(weight, x, k, "weight");
  check_columns(bias, x, k, "bias");
  check_like(residual, x, "residual", "x");
  if (!(eps >= 0)) refuse("eps must not be negative, got ", eps);
  c10::cuda::CUDAGuard guard(dev);
  const Flat xf(x), rf(residual);
  const Tensor w = dense(weight), b = dense(bias);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  const int64_t rows = rows_of(x);
  Norm r;
  if (residual.defined()) r.h = make(x.sizes(), x, x.scalar_type());
  if (stats) {
    r.mean = make(lead, x, at::kFloat);
    r.rstd = make(lead, x, at::kFloat);
  }
  if (in_blocks) {
    r.blocks = {make_codes(x.sizes(), x), make_scales(x.sizes(), x)};
    check(tg_blocks8_layernorm(code, rows, k, xf.ptr(), xf.ld, rf.ptr(), rf.ld, ptr(w), ptr(b), float(eps), ptr(r.h), k, ptr(r.blocks.q),
                               pitch(r.blocks.q), f32(r.blocks.scale), 1, rows, f32(r.mean), f32(r.rstd), stream(dev)));
  } else {
    r.y = make(x.sizes(), x, x.scalar_type());
    check(tg_layernorm(code, rows, k, xf.ptr(), xf.ld, rf.ptr(), rf.ld, ptr(w), ptr(b), float(eps), ptr(r.h), k, ptr(r.y), k, f32(r.mean),
                       f32(r.rstd), stream(dev)));
  }
  return r;
}
std::tuple<Tensor, Tensor, Tensor, Tensor> layernorm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& residual,
                                                     double eps, bool stats) {
  const Norm r = norm(x, or_none(weight), or_none(bias), or_none(residual), eps, stats, false);
  return {r.y, residual ? r.h : x, r.mean, r.rstd};
}
std::tuple<Tensor, Tensor, Tensor> layernorm_blocks8(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& residual, double eps) {
  const Norm r = norm(x, or_none(weight), or_none(bias), or_none(residual), eps, false, true);
  return {r.blocks.q, r.blocks.scale, residual ? r.h : x};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& grad, const Tensor& h, const Tensor& mean, const Tensor& rstd, const Tensor& weight,
                                                 const Tensor& grad_h, const Tensor& residual, bool want_x, bool want_weight, bool want_bias) {
  const tg_dtype code = type(h.scalar_type(), "h");
  const at::Device dev = grad.device();
  on(dev, {&h, &mean, &rstd, &weight, &grad_h, &residual});
  const int64_t k = h.dim() ? h.size(-1) : 0;
  if (k == 0) refuse("h needs at least one column");
  check_like(grad, h, "grad", "h");
  check_like(grad_h, h, "grad_h", "h");
  check_like(residual, h, "residual", "h");
  check_columns(weight, h, k, "weight");
  check_row_values(mean, h, "mean");
  check_row_values(rstd, h, "rstd");
  c10::cuda::CUDAGuard guard(dev);
  const Flat gf(grad), hf(h), ghf(grad_h), rf(residual);
  const Tensor w = dense(weight), mu = dense(mean), r = dense(rstd);
  Tensor grad_x, grad_w, grad_b;
  if (want_x) grad_x = make(h.sizes(), h, h.scalar_type());
  if (want_weight) grad_w = make({k}, h, h.scalar_type());
  if (want_bias) grad_b = make({k}, h, h.scalar_type());
  check(tg_layernorm_residual_backward(code, rows_of(h), k, gf.ptr(), gf.ld, ghf.ptr(), ghf.ld, ptr(w), hf.ptr(), hf.ld, rf.ptr(), rf.ld, f32(mu), f32(r),
                                       ptr(grad_x), k, ptr(grad_w), ptr(grad_b), stream(dev)));
  return {grad_x, grad_w, grad_b};
}

void once(const char* what) {
  if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(what) + " cannot be differentiated twice");
}
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool any_wants(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (wants(*t)) return true;
  return false;
}

// A backward that is captured into a graph adds to its leaves on the stream of
// the autograd graph that met them first.  Where an eager one is still alive
// that is a stream outside of the capture, which breaks it off: said here,
// while the forward is captured and nothing has gone wrong yet.
void check_capture(std::initializer_list<const Tensor*> inputs) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const Tensor* t : inputs) {
    if (!wants(*t) || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    if (!node || !node->stream()) continue;
    if (*node->stream() != at::cuda::getCurrentCUDAStream(t->device().index()).unwrap())
      throw std::runtime_error("a leaf of this captured call belongs to an autograd graph that is alive on another stream: "
                               "release what holds that graph (losses, outputs) before the capture");
  }
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                                const OptTensor& residual, double eps, bool train) {
    const Norm r = norm(x, or_none(weight), or_none(bias), or_none(residual), eps, train, false);
    if (train) {
      // h in 16 bits is the sum rounded: the backward takes its parts
      const bool parts = residual && x.scalar_type() != at::kFloat;
      ctx->save_for_backward({residual && !parts ? r.h : x, r.mean, r.rstd, or_none(weight), parts ? *residual : Tensor()});
      ctx->saved_data["needs"] = std::vector<int64_t>{wants(x), wants(or_none(weight)), wants(or_none(bias)), wants(or_none(residual))};
      ctx->set_materialize_grads(false);
    }
    return {r.y, residual ? r.h : x.view_as(x)};   // an output must not be the input itself
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    once("layernorm");
    const auto saved = ctx->get_saved_variables();
    const auto needs = ctx->saved_data["needs"].toIntVector();
    const Tensor &grad_y = grads[0], &grad_h = grads[1];
    Tensor grad_x, grad_w, grad_b;
    if (grad_y.defined())
      std::tie(grad_x, grad_w, grad_b) = norm_backward(grad_y, saved[0], saved[1], saved[2], saved[3], grad_h, saved[4], needs[0] || needs[3], needs[1], needs[2]);
    else
      grad_x = grad_h;
    const Tensor none;
    return {needs[0] ? grad_x : none, grad_w, grad_b, needs[3] ? grad_x : none, none, none};
  }
};
std::tuple<Tensor, Tensor> layernorm_grad(const Tensor& x, const OptTensor& weight, const OptTensor& bias, const OptTensor& residual, double eps) {
  const bool train = any_wants({&x, &or_none(weight), &or_none(bias), &or_none(residual)});
  if (train) check_capture({&x, &or_none(weight), &or_none(bias), &or_none(residual)});
  auto out = LayerNorm::apply(x, weight, bias, residual, eps, train);
  return {out[0], out[1]};
}

// ------------------------------------------------------------------------------------------------ linear
// Kept for the backward, in 8 bits: x along the tokens (the weight's gradient
// sums over them) and the weight transposed.
struct Linear : torch::autograd::Function<Linear> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& weight_scale,
                                                const OptTensor& bias, bool train) {
    const bool need_x = train && wants(x), need_w = train && !weight_scale && wants(weight);
    Blocks a, a_turned, w;
    Tensor w_turned;
    quantize_into(x, &a, need_w ? &a_turned : nullptr);
    if (weight_scale) {
      w = {weight, *weight_scale};
      if (need_x) w_turned = transpose(weight);
    } else {
      quantize_tiles_into(weight, &w, need_x ? &w_turned : nullptr);
    }
    Tensor z = matmul(a.q, a.scale, w.q, w.scale, bias, x.scalar_type());
    if (train) {
      ctx->save_for_backward({a_turned.q, a_turned.scale, w_turned, need_x ? w.scale : Tensor()});
      ctx->saved_data["needs"] = std::vector<int64_t>{need_x, need_w, wants(or_none(bias))};
      ctx->set_materialize_grads(false);
    }
    return {z};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    once("linear_blocks8");
    const auto saved = ctx->get_saved_variables();
    const auto needs = ctx->saved_data["needs"].toIntVector();
    const Tensor& g = grads[0];
    Tensor grad_x, grad_w, grad_b;
    if (g.defined()) {
      Blocks rows, turned;
      quantize_into(g, needs[0] ? &rows : nullptr, needs[1] ? &turned : nullptr, needs[2] ? &grad_b : nullptr);
      if (needs[0]) grad_x = matmul(rows.q, rows.scale, saved[2], saved[3].t(), std::nullopt, g.scalar_type());
      if (needs[1]) grad_w = matmul(turned.q, turned.scale, saved[0], saved[1], std::nullopt, g.scalar_type());
    }
    const Tensor none;
    return {grad_x, grad_w, none, grad_b, none};
  }
};
Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& weight_scale, const OptTensor& bias) {
  type(x.scalar_type(), "x");
  if (!weight_scale && (weight.scalar_type() != x.scalar_type() || weight.dim() != 2))
    refuse("weight must be a two-dimensional ", name(x.scalar_type()), " tensor or Blocks8, got ", name(weight.scalar_type()), " ", shape(weight.sizes()));
  if (x.dim() == 0) refuse("expected a tensor with at least one dimension");
  if (weight.dim() != 2 || x.size(-1) != weight.size(1)) refuse("Dimension mismatch: x is ", shape(x.sizes()), ", weight is ", shape(weight.sizes()));
  const bool train = any_wants({&x, &or_none(bias)}) || (!weight_scale && any_wants({&weight}));
  if (weight_scale && check_blocks8(weight, *weight_scale, "weight") != 128 && train && wants(x) && weight.size(0) > 1)
    refuse("a weight whose scales are per row has no gradient for x in 8-bit blocks: use tiles of 128 x 128");
  on(x.device(), {&weight, &or_none(weight_scale), &or_none(bias)});
  if (train) check_capture({&x, &weight, &or_none(bias)});
  // frozen blocks are constants, their scales included
  const OptTensor frozen = weight_scale && weight_scale->requires_grad() ? OptTensor(weight_scale->detach()) : weight_scale;
  return Linear::apply(x, weight, frozen, bias, train)[0];
}

// ------------------------------------------------------------------------------------------------ token log probabilities
struct Tokens {
  Tensor logprob, entropy, stats, top_logprobs, top_tokens;
};
Tokens tokens_of(const Tensor& logits, const Tensor& tokens, int64_t top, int64_t ignore) {
  const tg_dtype code = type(logits.scalar_type(), "logits");
  const at::Device dev = logits.device();
  on(dev, {&tokens});
  const int64_t v = logits.dim() ? logits.size(-1) : 0;
  if (v == 0) refuse("logits need at least one column");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  if (tokens.defined() && (tokens.scalar_type() != at::kLong || tokens.sizes() != lead))
    refuse("tokens must be int64 of shape ", shape(lead), ", got ", name(tokens.scalar_type()), " ", shape(tokens.sizes()));
  if (top < 0 || top > 32 || top > v) refuse("top must be 0 to ", std::min<int64_t>(32, v), ", got ", top);
  c10::cuda::CUDAGuard guard(dev);
  const Flat f(logits);
  const Tensor t = dense(tokens);
  Tokens r;
  if (tokens.defined()) r.logprob = make(lead, logits, at::kFloat);
  r.entropy = make(lead, logits, at::kFloat);
  at::DimVector pair(lead.begin(), lead.end());
  pair.push_back(2);
  r.stats = make(pair, logits, at::kFloat);
  if (top) {
    r.top_logprobs = make(with_last(logits, top), logits, at::kFloat);
    r.top_tokens = make(with_last(logits, top), logits, at::kLong);
  }
  check(tg_token_logprobs(code, rows_of(logits), v, f.ptr(), f.ld, static_cast<const int64_t*>(ptr(t)), ignore, f32(r.logprob), f32(r.entropy),
                          f32(r.stats), int(top), f32(r.top_logprobs), static_cast<int64_t*>(ptr(r.top_tokens)), stream(dev)));
  return r;
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const OptTensor& tokens, int64_t top, int64_t ignore) {
  const Tokens r = tokens_of(logits, or_none(tokens), top, ignore);
  return {r.logprob, r.entropy, r.top_logprobs, r.top_tokens, r.stats};
}
Tensor tokens_backward(const Tensor& logits, const Tensor& tokens, const Tensor& stats, const Tensor& entropy, const Tensor& grad_logprob,
                       const Tensor& grad_entropy, int64_t ignore) {
  const tg_dtype code = type(logits.scalar_type(), "logits");
  const at::Device dev = logits.device();
  on(dev, {&tokens, &stats, &entropy, &grad_logprob, &grad_entropy});
  const int64_t v = logits.dim() ? logits.size(-1) : 0;
  if (v == 0) refuse("logits need at least one column");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  if (tokens.defined() && (tokens.scalar_type() != at::kLong || tokens.sizes() != lead))
    refuse("tokens must be int64 of shape ", shape(lead), ", got ", name(tokens.scalar_type()), " ", shape(tokens.sizes()));
  at::DimVector pair(lead.begin(), lead.end());
  pair.push_back(2);
  if (stats.scalar_type() != at::kFloat || stats.sizes() != at::IntArrayRef(pair)) refuse("stats must be float32 of shape ", shape(pair), ", got ", name(stats.scalar_type()), " ", shape(stats.sizes()));
  check_row_values(entropy, logits, "entropy");
  check_row_values(grad_logprob, logits, "grad_logprob");
  check_row_values(grad_entropy, logits, "grad_entropy");
  if (grad_logprob.defined() && !tokens.defined()) refuse("grad_logprob needs tokens");
  if (grad_entropy.defined() && !entropy.defined()) refuse("grad_entropy needs entropy");
  c10::cuda::CUDAGuard guard(dev);
  const Flat f(logits);
  const Tensor t = dense(tokens), s = dense(stats), h = dense(entropy), gl = dense(grad_logprob), ge = dense(grad_entropy);
  Tensor out = make(logits.sizes(), logits, logits.scalar_type());
  check(tg_token_logprobs_backward(code, rows_of(logits), v, f.ptr(), f.ld, static_cast<const int64_t*>(ptr(t)), ignore, f32(s), f32(h), f32(gl), f32(ge),
                                   ptr(out), v, stream(dev)));
  return out;
}
struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t ignore, bool train) {
    const Tokens r = tokens_of(logits, tokens, 0, ignore);
    if (train) {
      ctx->save_for_backward({logits, tokens, r.stats, r.entropy});
      ctx->saved_data["ignore"] = ignore;
      ctx->set_materialize_grads(false);
    }
    return {r.logprob, r.entropy};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    once("token_logprobs");
    const auto saved = ctx->get_saved_variables();
    Tensor grad;
    if (grads[0].defined() || grads[1].defined())
      grad = tokens_backward(saved[0], saved[1], saved[2], saved[3], grads[0], grads[1], ctx->saved_data["ignore"].toInt());
    const Tensor none;
    return {grad, none, none, none};
  }
};
std::tuple<Tensor, Tensor> token_logprobs_grad(const Tensor& logits, const Tensor& tokens, int64_t ignore) {
  const bool train = any_wants({&logits});
  if (train) check_capture({&logits});
  auto out = TokenLogprobs::apply(logits, tokens, ignore, train);
  return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(_layers_torch, m) {
  m.def("layernorm", &layernorm);
  m.def("layernorm_blocks8", &layernorm_blocks8);
  m.def("layernorm_backward", [](const Tensor& grad, const Tensor& h, const Tensor& mean, const Tensor& rstd, const OptTensor& weight, const OptTensor& grad_h,
                                  const OptTensor& residual) {
    return norm_backward(grad, h, mean, rstd, or_none(weight), or_none(grad_h), or_none(residual), true, true, true);
  });
  m.def("layernorm_grad", &layernorm_grad);
  m.def("quantize", &quantize);
  m.def("quantize_both", &quantize_both);
  m.def("quantize_tiles", &quantize_tiles);
  m.def("dequantize", &dequantize);
  m.def("transpose", &transpose);
  m.def("matmul", [](const Tensor& aq, const Tensor& as, const Tensor& bq, const Tensor& bs, const OptTensor& bias, const py::object& dtype) {
    return matmul(aq, as, bq, bs, bias, dtype_arg(dtype, at::kBFloat16, "dtype"));
  });
  m.def("linear", &linear);
  m.def("token_logprobs", &token_logprobs);
  m.def("token_logprobs_backward", [](const Tensor& logits, const OptTensor& tokens, const Tensor& stats, const OptTensor& entropy, const OptTensor& gl,
                                      const OptTensor& ge, int64_t ignore) {
    return tokens_backward(logits, or_none(tokens), stats, or_none(entropy), or_none(gl), or_none(ge), ignore);
  });
  m.def("token_logprobs_grad", &token_logprobs_grad);
}
