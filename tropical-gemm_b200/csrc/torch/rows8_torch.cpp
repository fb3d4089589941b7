// torch binding of the 8-bit row calls: argument checks, outputs from torch's
// allocator, torch's current stream.  In C++ because these calls are small:
// a norm of one token is 3 us on the GPU and was 18 us of Python around it.
// The work is the C ABI's (include/tropical_gemm_b200.h).
#include "binding.h"

namespace {

void check_rows8(const Tensor& q, const Tensor& s, const char* what) {
  if (q.scalar_type() != at::kChar || s.scalar_type() != at::kFloat)
    refuse(what, " must be int8 rows with float32 scales, got ", name(q.scalar_type()), " and ", name(s.scalar_type()));
  if (q.dim() == 0 || s.sizes() != q.sizes().slice(0, q.dim() - 1))
    refuse(what, " needs one scale per row: q is ", shape(q.sizes()), ", scale is ", shape(s.sizes()));
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x) {
  const tg_dtype code = type(x.scalar_type(), "x");
  on(x.device());
  if (x.dim() == 0) refuse("expected a tensor with at least one dimension");
  c10::cuda::CUDAGuard guard(x.device());
  const Flat f(x);
  const int64_t k = x.size(-1);
  Tensor q = make(x.sizes(), x, at::kChar), scale = make(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  check(tg_rows8_quantize(code, rows_of(x), k, f.ptr(), f.ld, q.data_ptr<int8_t>(), k, f32(scale), stream(x.device())));
  return {q, scale};
}

Tensor dequantize(const Tensor& q, const Tensor& scale, const py::object& dtype) {
  check_rows8(q, scale, "rows");
  on(q.device(), {&scale});
  const at::ScalarType t = dtype_arg(dtype, at::kBFloat16, "dtype");
  c10::cuda::CUDAGuard guard(q.device());
  const Flat f(q);
  const Tensor s = dense(scale);
  const int64_t k = q.size(-1);
  Tensor y = make(q.sizes(), q, t);
  check(tg_rows8_dequantize(type(t, "dtype"), rows_of(q), k, f.q(), f.ld, f32(s), y.data_ptr(), k, stream(q.device())));
  return y;
}

// q, scale, h, and with the checkpoint q and scale of h, 1 / root mean square
using Norm = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
Norm rmsnorm(const Tensor& x, const Tensor& weight, const OptTensor& residual_arg, double eps, bool checkpoint) {
  const Tensor& residual = or_none(residual_arg);
  const tg_dtype code = type(x.scalar_type(), "x");
  const at::Device dev = x.device();
  on(dev, {&weight, &residual});
  const int64_t k = x.dim() ? x.size(-1) : 0;
  if (k == 0) refuse("x needs at least one column");
  if (weight.scalar_type() != x.scalar_type() || weight.dim() != 1 || weight.size(0) != k)
    refuse("weight must be ", name(x.scalar_type()), " of shape (", k, ",), got ", name(weight.scalar_type()), " ", shape(weight.sizes()));
  if (residual.defined() && (residual.scalar_type() != x.scalar_type() || residual.sizes() != x.sizes()))
    refuse("residual must be like x (", name(x.scalar_type()), " ", shape(x.sizes()), "), got ", name(residual.scalar_type()), " ", shape(residual.sizes()));
  if (!(eps >= 0)) refuse("eps must not be negative, got ", eps);
  c10::cuda::CUDAGuard guard(dev);
  const Flat xf(x), rf(residual);
  const Tensor w = dense(weight);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  Tensor q = make(x.sizes(), x, at::kChar), scale = make(lead, x, at::kFloat), h, ck, cs, rstd;
  if (residual.defined()) h = make(x.sizes(), x, x.scalar_type());
  if (checkpoint) {
    ck = make(x.sizes(), x, at::kChar);
    cs = make(lead, x, at::kFloat);
    rstd = make(lead, x, at::kFloat);
  }
  check(tg_rows8_rmsnorm(code, rows_of(x), k, xf.ptr(), xf.ld, rf.ptr(), rf.ld, w.data_ptr(), float(eps), ptr(h), k,
                         q.data_ptr<int8_t>(), k, f32(scale), static_cast<int8_t*>(ptr(ck)), k, f32(cs), f32(rstd), stream(dev)));
  return {q, scale, residual.defined() ? h : x, ck, cs, rstd};
}

std::tuple<Tensor, Tensor> rmsnorm_backward(const Tensor& grad, const Tensor& ck, const Tensor& ck_scale, const Tensor& rstd,
                           const Tensor& weight, const OptTensor& grad_h_arg) {
  const Tensor& grad_h = or_none(grad_h_arg);
  check_rows8(ck, ck_scale, "checkpoint");
  const tg_dtype code = type(weight.scalar_type(), "weight"), gcode = type(grad.scalar_type(), "grad");
  const at::Device dev = grad.device();
  on(dev, {&ck, &ck_scale, &rstd, &weight, &grad_h});
  const int64_t k = ck.size(-1);
  if (k == 0) refuse("the checkpoint needs at least one column");
  if (grad.sizes() != ck.sizes()) refuse("grad must have the checkpoint's shape ", shape(ck.sizes()), ", got ", shape(grad.sizes()));
  if (gcode != code && gcode != TG_F32) refuse("grad must be float32 or weight's ", name(weight.scalar_type()), ", got ", name(grad.scalar_type()));
  if (weight.dim() != 1 || weight.size(0) != k) refuse("weight must have shape (", k, ",), got ", shape(weight.sizes()));
  if (rstd.scalar_type() != at::kFloat || rstd.sizes() != ck_scale.sizes())
    refuse("rstd must be float32 of shape ", shape(ck_scale.sizes()), ", got ", name(rstd.scalar_type()), " ", shape(rstd.sizes()));
  if (grad_h.defined() && (grad_h.scalar_type() != weight.scalar_type() || grad_h.sizes() != grad.sizes()))
    refuse("grad_h must be ", name(weight.scalar_type()), " of shape ", shape(grad.sizes()), ", got ", name(grad_h.scalar_type()), " ", shape(grad_h.sizes()));
  c10::cuda::CUDAGuard guard(dev);
  const Flat gf(grad), kf(ck), hf(grad_h);
  const Tensor w = dense(weight), s = dense(ck_scale), r = dense(rstd);
  Tensor grad_x = make(grad.sizes(), grad, weight.scalar_type()), grad_w = make({k}, grad, weight.scalar_type());
  check(tg_rows8_rmsnorm_backward(code, gcode, rows_of(ck), k, gf.ptr(), gf.ld, hf.ptr(), hf.ld, w.data_ptr(), kf.q(), kf.ld,
                                  f32(s), f32(r), grad_x.data_ptr(), k, grad_w.data_ptr(), stream(dev)));
  return {grad_x, grad_w};
}

Tensor matmul(const Tensor& aq, const Tensor& a_scale, const Tensor& bq, const Tensor& b_scale, const OptTensor& bias_arg,
              at::ScalarType t) {
  const Tensor& bias = or_none(bias_arg);
  check_rows8(aq, a_scale, "a");
  check_rows8(bq, b_scale, "b");
  const at::Device dev = aq.device();
  on(dev, {&a_scale, &bq, &b_scale, &bias});
  if (bq.dim() != 2) refuse("b must be two-dimensional (channels, K), got ", shape(bq.sizes()));
  const int64_t n = bq.size(0), k = bq.size(1);
  if (aq.size(-1) != k) refuse("Dimension mismatch: a has ", aq.size(-1), " columns, b has ", k);
  if (bias.defined() && (bias.scalar_type() != t || bias.dim() != 1 || bias.size(0) != n))
    refuse("bias must be ", name(t), " of shape (", n, ",), got ", name(bias.scalar_type()), " ", shape(bias.sizes()));
  c10::cuda::CUDAGuard guard(dev);
  const Flat a(aq), b(bq);
  const Tensor as = dense(a_scale), bs = dense(b_scale), bi = dense(bias);
  Tensor c = make(with_last(aq, n), aq, t);
  check(tg_rows8_gemm(type(t, "dtype"), rows_of(aq), n, k, a.q(), a.ld, f32(as), b.q(), b.ld, f32(bs), ptr(bi), c.data_ptr(), n, stream(dev)));
  return c;
}

std::tuple<Tensor, Tensor> matmul_backward(const Tensor& grad, const OptTensor& aq, const OptTensor& a_scale, const OptTensor& bq,
                                           const OptTensor& b_scale, at::ScalarType ta, at::ScalarType tb) {
  const tg_dtype code = type(grad.scalar_type(), "grad");
  const at::Device dev = grad.device();
  on(dev);
  if (grad.dim() == 0) refuse("expected a gradient with at least one dimension");
  if (aq) check_rows8(*aq, *a_scale, "a");
  if (bq) check_rows8(*bq, *b_scale, "b");
  on(dev, {&or_none(aq), &or_none(a_scale), &or_none(bq), &or_none(b_scale)});
  const int64_t n = grad.size(-1), rows = rows_of(grad);
  if (bq && (bq->dim() != 2 || bq->size(0) != n)) refuse("Dimension mismatch: grad is ", shape(grad.sizes()), ", b is ", shape(bq->sizes()));
  if (aq && aq->sizes().slice(0, aq->dim() - 1) != grad.sizes().slice(0, grad.dim() - 1))
    refuse("Dimension mismatch: grad is ", shape(grad.sizes()), ", a is ", shape(aq->sizes()));
  c10::cuda::CUDAGuard guard(dev);
  const Flat g(grad);
  Tensor ga, gb;
  if (bq) {
    const Flat b(*bq);
    const Tensor s = dense(*b_scale);
    const int64_t k = bq->size(1);
    ga = make(with_last(grad, k), grad, ta);
    check(tg_rows8_gemm_backward(code, type(ta, "dtype_a"), 0, rows, k, n, g.ptr(), g.ld, b.q(), b.ld, f32(s), ga.data_ptr(), k, stream(dev)));
  }
  if (aq) {
    const Flat a(*aq);
    const Tensor s = dense(*a_scale);
    const int64_t k = aq->size(-1);
    gb = make({n, k}, grad, tb);
    check(tg_rows8_gemm_backward(code, type(tb, "dtype_b"), 1, n, k, rows, g.ptr(), g.ld, a.q(), a.ld, f32(s), gb.data_ptr(), k, stream(dev)));
  }
  return {ga, gb};
}

Tensor column_sum(const Tensor& x, at::ScalarType t) {
  const tg_dtype code = type(x.scalar_type(), "x");
  on(x.device());
  if (x.dim() == 0) refuse("expected a tensor with at least one dimension");
  c10::cuda::CUDAGuard guard(x.device());
  const Flat f(x);
  Tensor out = make({x.size(-1)}, x, t);
  check(tg_rows8_column_sum(code, type(t, "dtype"), rows_of(x), x.size(-1), f.ptr(), f.ld, out.data_ptr(), stream(x.device())));
  return out;
}

// norm of x + residual -> linear, both in 8-bit rows, with gradients.  Kept for
// the backward, in 8 bits: the normalised activations (the product's own
// operand), h, and the weight's rows.
struct NormLinear : torch::autograd::Function<NormLinear> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& norm_weight,
                                                const Tensor& weight, const OptTensor& weight_scale, const OptTensor& residual,
                                                const OptTensor& bias, double eps, bool train) {
    auto [q, scale, h, ck, ck_scale, rstd] = rmsnorm(x, norm_weight, residual, eps, train);
    const auto [bq, b_scale] = weight_scale ? std::make_tuple(weight, *weight_scale) : quantize(weight);
    Tensor z = matmul(q, scale, bq, b_scale, bias, x.scalar_type());
    if (train) {
      ctx->save_for_backward({q, scale, ck, ck_scale, rstd, bq, b_scale, norm_weight});
      ctx->saved_data["needs"] = std::vector<int64_t>{x.requires_grad(), norm_weight.requires_grad(),
                                                      !weight_scale && weight.requires_grad(), residual && residual->requires_grad(),
                                                      bias && bias->requires_grad()};
      ctx->set_materialize_grads(false);
    }
    return {z, residual ? h : x.view_as(x)};   // an output must not be the input itself
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled()) throw std::runtime_error("rmsnorm_linear_rows8 cannot be differentiated twice");
    const auto saved = ctx->get_saved_variables();
    const auto needs = ctx->saved_data["needs"].toIntVector();
    const Tensor &grad_z = grads[0], &grad_h = grads[1];
    Tensor grad_x, grad_norm, grad_w, grad_bias;
    if (grad_z.defined()) {
      const bool norm = needs[0] || needs[1] || needs[3];
      // the norm's incoming gradient stays float32: one rounding less, at its output
      Tensor grad_y;
      std::tie(grad_y, grad_w) = matmul_backward(
          grad_z, needs[2] ? OptTensor(saved[0]) : OptTensor(), needs[2] ? OptTensor(saved[1]) : OptTensor(),
          norm ? OptTensor(saved[5]) : OptTensor(), norm ? OptTensor(saved[6]) : OptTensor(), at::kFloat, grad_z.scalar_type());
      if (norm)
        std::tie(grad_x, grad_norm) = rmsnorm_backward(grad_y, saved[2], saved[3], saved[4], saved[7],
                                                       grad_h.defined() ? OptTensor(grad_h) : OptTensor());
      if (needs[4]) grad_bias = column_sum(grad_z, grad_z.scalar_type());
    } else {
      grad_x = grad_h;
    }
    const Tensor none;
    return {needs[0] ? grad_x : none, needs[1] ? grad_norm : none, grad_w, none, needs[3] ? grad_x : none, grad_bias, none, none};
  }
};

std::tuple<Tensor, Tensor> rmsnorm_linear(const Tensor& x, const Tensor& norm_weight, const Tensor& weight, const OptTensor& weight_scale,
                                          const OptTensor& residual, const OptTensor& bias, double eps) {
  if (!weight_scale && (weight.scalar_type() != x.scalar_type() || weight.dim() != 2))
    refuse("weight must be a two-dimensional ", name(x.scalar_type()), " tensor or Rows8, got ", name(weight.scalar_type()), " ", shape(weight.sizes()));
  const bool train = at::GradMode::is_enabled() &&
                     (x.requires_grad() || norm_weight.requires_grad() || (!weight_scale && weight.requires_grad()) ||
                      (residual && residual->requires_grad()) || (bias && bias->requires_grad()));
  // frozen rows are constants, their scales included: else a scale that requires a
  // gradient would make a node of a call that kept nothing for its backward
  const OptTensor frozen = weight_scale && weight_scale->requires_grad() ? OptTensor(weight_scale->detach()) : weight_scale;
  auto out = NormLinear::apply(x, norm_weight, weight, frozen, residual, bias, eps, train);
  return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(_rows8_torch, m) {
  m.def("quantize", &quantize);
  m.def("dequantize", &dequantize);
  m.def("rmsnorm", &rmsnorm);
  m.def("rmsnorm_backward", &rmsnorm_backward);
  m.def("matmul", [](const Tensor& aq, const Tensor& as, const Tensor& bq, const Tensor& bs, const OptTensor& bias, const py::object& dtype) {
    return matmul(aq, as, bq, bs, bias, dtype_arg(dtype, at::kBFloat16, "dtype"));
  });
  m.def("matmul_backward", [](const Tensor& grad, const OptTensor& aq, const OptTensor& as, const OptTensor& bq, const OptTensor& bs,
                              const py::object& dtype_a, const py::object& dtype_b) {
    return matmul_backward(grad, aq, as, bq, bs, dtype_arg(dtype_a, grad.scalar_type(), "dtype_a"), dtype_arg(dtype_b, grad.scalar_type(), "dtype_b"));
  });
  m.def("column_sum", [](const Tensor& x, const py::object& dtype) { return column_sum(x, dtype_arg(dtype, x.scalar_type(), "dtype")); });
  m.def("rmsnorm_linear", &rmsnorm_linear);
}
