// Shared by the torch bindings: argument checks, rows and columns of a tensor,
// torch's current stream, and the engine's status codes as exceptions.
#pragma once
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <optional>
#include <sstream>
#include "../../../include/tropical_gemm_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

template <typename... A> [[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw py::value_error(s.str());
}

std::string name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    default: return c10::toString(t);
  }
}
std::string shape(at::IntArrayRef s) {
  std::ostringstream o;
  o << '(';
  for (size_t i = 0; i < s.size(); i++) o << (i ? ", " : "") << s[i];
  o << (s.size() == 1 ? ",)" : ")");
  return o.str();
}

bool type_of(at::ScalarType t, tg_dtype* out) {
  switch (t) {
    case at::kFloat: *out = TG_F32; return true;
    case at::kHalf: *out = TG_F16; return true;
    case at::kBFloat16: *out = TG_BF16; return true;
    default: return false;
  }
}
tg_dtype type(at::ScalarType t, const char* what) {
  tg_dtype r;
  if (!type_of(t, &r)) refuse(what, " must be float32, float16 or bfloat16, got ", name(t));
  return r;
}
at::ScalarType dtype_arg(const py::object& o, at::ScalarType otherwise, const char* what) {
  if (o.is_none()) return otherwise;
  if (!THPDtype_Check(o.ptr())) throw py::type_error(std::string(what) + " must be a torch.dtype");
  const at::ScalarType t = reinterpret_cast<THPDtype*>(o.ptr())->scalar_type;
  type(t, what);
  return t;
}

void on(const at::Device& dev, std::initializer_list<const Tensor*> others = {}) {
  if (!dev.is_cuda()) throw std::runtime_error("the tropical-gemm engine needs CUDA tensors");
  for (const Tensor* t : others)
    if (t->defined() && t->device() != dev) refuse("Tensors must be on the same device: got ", dev.str(), " and ", t->device().str());
}
const Tensor& or_none(const OptTensor& t) {
  static const Tensor none;
  return t ? *t : none;
}

int64_t rows_of(const Tensor& t) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); i++) n *= t.size(i);
  return n;
}

// t as rows and columns with a row stride; a copy only where a row is not
// contiguous or the rows do not form one dimension.
struct Flat {
  Tensor t;
  int64_t ld = 0;
  Flat() = default;
  explicit Flat(const Tensor& x) {
    if (!x.defined()) return;
    if (x.is_contiguous()) {
      t = x;
      ld = x.size(-1);
      return;
    }
    t = x.detach();
    if (t.dim() != 2) t = t.reshape({rows_of(t), t.size(-1)});
    if (!(t.stride(1) == 1 && t.stride(0) >= std::max<int64_t>(1, t.size(1)))) t = t.contiguous();
    ld = t.size(0) > 1 ? std::max<int64_t>(1, t.stride(0)) : std::max<int64_t>(1, t.size(1));
  }
  void* ptr() const { return t.defined() ? t.data_ptr() : nullptr; }
  const int8_t* q() const { return static_cast<const int8_t*>(ptr()); }
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* f32(const Tensor& t) { return static_cast<float*>(ptr(t)); }
Tensor dense(const Tensor& t) { return !t.defined() || t.is_contiguous() ? t : t.detach().contiguous(); }
void* stream(const at::Device& d) { return at::cuda::getCurrentCUDAStream(d.index()).stream(); }

void check(tg_status s) {
  if (s == TG_OK) return;
  py::gil_scoped_acquire gil;   // autograd's threads come without it
  py::module_::import("tropical_gemm._native").attr("check")(int(s));
}

// Whether somebody is to see a new tensor: a dispatch mode that watches calls, or
// the deterministic mode's filling of what is not written.
bool watched() { return c10::impl::dispatch_mode_enabled() || at::globalContext().deterministicAlgorithms(); }
// Outputs, on like's device: CUDA tensors only, so torch's choice of a backend
// (0.4 us each) is left out where nobody watches it.
Tensor make(at::IntArrayRef sizes, const Tensor& like, at::ScalarType t) {
  if (watched()) return at::empty(sizes, like.options().dtype(t).requires_grad(false));
  return Tensor(at::detail::empty_cuda(sizes, t, like.device(), std::nullopt));
}

at::DimVector with_last(const Tensor& t, int64_t last) {
  at::DimVector v(t.sizes().begin(), t.sizes().end());
  v.back() = last;
  return v;
}

}  // namespace
