// torch glue of the token-path ops (layer norm, rotary positions): checks the
// tensors and calls one extern "C" entry point of libpkv.so on the current
// CUDA stream.  A fragment of the `adahead` library registered in
// adahead_bind.cpp.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../include/pkv.h"

namespace pkv_torch {
namespace {

using at::Tensor;

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == PKV_OK, what, ": ", pkv_error_string(rc), " (code ", rc, ")");
}

void* stream_of(const Tensor& t) {
  return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

int type_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PKV_BF16;
    case at::kHalf: return PKV_FP16;
    case at::kFloat: return PKV_FP32;
    default: TORCH_CHECK(false, what, " must be bf16, fp16 or fp32");
  }
}

// ---- layer norm -------------------------------------------------------------
struct NormParams {
  Tensor w, b;  // undefined when absent
  int64_t groups = 1;
  int wtype = PKV_FP32;
};

void check_norm_x(const Tensor& x, const char* op, const char* name) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, op, ": ", name, " must be a [rows, cols] CUDA tensor");
  TORCH_CHECK(x.size(1) > 0, op, ": ", name, " has no channels");
}

NormParams norm_params(const char* op, const Tensor& x, const std::optional<Tensor>& weight,
                       const std::optional<Tensor>& bias) {
  NormParams p;
  p.wtype = type_code(x, op);
  bool first = true;
  for (const auto* t : {&weight, &bias}) {
    if (!t->has_value() || !(*t)->defined()) continue;
    const Tensor& v = **t;
    TORCH_CHECK(v.device() == x.device(), op, ": weight / bias must be on x's device");
    TORCH_CHECK((v.dim() == 1 || v.dim() == 2) && v.size(-1) == x.size(1), op,
                ": weight / bias must be [cols] or [groups, cols] of x's ", x.size(1),
                " channels");
    const int64_t g = v.dim() == 2 ? v.size(0) : 1;
    TORCH_CHECK(g > 0 && x.size(0) % g == 0, op, ": ", g, " groups do not divide ", x.size(0),
                " rows");
    const int code = type_code(v, op);
    TORCH_CHECK(code == type_code(x, op) || code == PKV_FP32, op,
                ": weight / bias must have x's type or be fp32");
    TORCH_CHECK(first || (g == p.groups && code == p.wtype), op,
                ": weight and bias must have one shape and type");
    p.groups = g;
    p.wtype = code;
    first = false;
    (t == &weight ? p.w : p.b) = v.contiguous();
  }
  return p;
}

const void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

Tensor dense_rows(const Tensor& x) { return x.stride(1) == 1 || x.size(1) == 1 ? x : x.contiguous(); }

std::tuple<Tensor, Tensor, Tensor> op_layer_norm(Tensor x, std::optional<Tensor> weight,
                                                 std::optional<Tensor> bias, double eps,
                                                 bool one_plus, bool stats) {
  const char* op = "pkv_layer_norm";
  check_norm_x(x, op, "x");
  TORCH_CHECK(eps >= 0.0, op, ": eps must not be negative");
  const int dt = type_code(x, op);
  const c10::cuda::CUDAGuard g(x.device());
  const NormParams p = norm_params(op, x, weight, bias);
  const Tensor xx = dense_rows(x);
  const Tensor y = at::empty(x.sizes(), x.options());
  const auto f32 = x.options().dtype(at::kFloat);
  const Tensor mean = at::empty({stats ? x.size(0) : 0}, f32);
  const Tensor rstd = at::empty({stats ? x.size(0) : 0}, f32);
  check_rc(pkv_layer_norm(ptr(xx), xx.stride(0), ptr(p.w), ptr(p.b), dt, p.wtype, x.size(0),
                          x.size(1), p.groups, float(eps), one_plus, mut(y), y.stride(0),
                          static_cast<float*>(mut(mean)), static_cast<float*>(mut(rstd)),
                          stream_of(x)),
           op);
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> op_layer_norm_backward(
    Tensor dy, Tensor x, std::optional<Tensor> weight, std::optional<Tensor> bias, Tensor mean,
    Tensor rstd, bool one_plus, bool need_x, bool need_weight, bool need_bias) {
  const char* op = "pkv_layer_norm_backward";
  check_norm_x(x, op, "x");
  check_norm_x(dy, op, "dy");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() &&
                  dy.device() == x.device(),
              op, ": dy must be like x");
  for (const Tensor* t : {&mean, &rstd})
    TORCH_CHECK(t->device() == x.device() && t->scalar_type() == at::kFloat &&
                    t->is_contiguous() && t->numel() == x.size(0),
                op, ": mean / rstd must be the fp32 [rows] pkv_layer_norm returned");
  const int dt = type_code(x, op);
  const c10::cuda::CUDAGuard g(x.device());
  const NormParams p = norm_params(op, x, weight, bias);
  TORCH_CHECK((!need_weight || p.w.defined()) && (!need_bias || p.b.defined()), op,
              ": no weight / bias to differentiate");
  const Tensor xx = dense_rows(x), dd = dense_rows(dy);
  Tensor dx, dw, db;
  if (need_x) dx = at::empty(x.sizes(), x.options());
  if (need_weight) dw = at::empty(p.w.sizes(), p.w.options());
  if (need_bias) db = at::empty(p.b.sizes(), p.b.options());
  if (x.size(0) == 0) {  // no rows: the sums are zero
    if (need_weight) dw.zero_();
    if (need_bias) db.zero_();
    return {dx, dw, db};
  }
  int64_t bytes = 0;
  Tensor ws;
  if (need_weight || need_bias) {
    bytes = pkv_layer_norm_workspace_bytes(x.size(0), x.size(1), p.groups);
    ws = at::empty({bytes}, x.options().dtype(at::kByte));
  }
  check_rc(pkv_layer_norm_backward(
               ptr(dd), dd.stride(0), ptr(xx), xx.stride(0), ptr(p.w),
               static_cast<const float*>(ptr(mean)), static_cast<const float*>(ptr(rstd)), dt,
               p.wtype, x.size(0), x.size(1), p.groups, one_plus, mut(dx),
               need_x ? dx.stride(0) : 0, mut(dw), mut(db), mut(ws), bytes, stream_of(x)),
           op);
  return {dx, dw, db};
}

// ---- rotary positions --------------------------------------------------------
Tensor dense_heads(const Tensor& x) { return x.stride(2) == 1 || x.size(2) == 1 ? x : x.contiguous(); }

std::tuple<Tensor, Tensor> op_rotary(Tensor q, std::optional<Tensor> k, Tensor positions,
                                     Tensor inv_freq, std::optional<Tensor> axis, bool half,
                                     double scale, bool inverse) {
  const char* op = "pkv_rotary";
  TORCH_CHECK(q.is_cuda() && q.dim() == 3, op, ": q must be a [tokens, heads, dim] CUDA tensor");
  const int dt = type_code(q, op);
  const bool two = k.has_value() && k->defined();
  if (two)
    TORCH_CHECK(k->dim() == 3 && k->size(0) == q.size(0) && k->size(2) == q.size(2) &&
                    k->scalar_type() == q.scalar_type() && k->device() == q.device(),
                op, ": k must match q's tokens, head size, type and device");
  const int64_t T = q.size(0), D = q.size(2);
  TORCH_CHECK(positions.device() == q.device() && positions.scalar_type() == at::kLong &&
                  positions.dim() == 2 && positions.size(0) == T && positions.is_contiguous() &&
                  positions.size(1) >= 1 && positions.size(1) <= 4,
              op, ": positions must be contiguous int64 [tokens, axes] on q's device, 1-4 axes");
  TORCH_CHECK(inv_freq.device() == q.device() && inv_freq.scalar_type() == at::kDouble &&
                  inv_freq.dim() == 1 && inv_freq.is_contiguous() && 2 * inv_freq.size(0) <= D,
              op, ": inv_freq must be contiguous float64 [pairs] on q's device, 2 * pairs <= ", D);
  const bool have_axis = axis.has_value() && axis->defined();
  if (have_axis)
    TORCH_CHECK(axis->device() == q.device() && axis->scalar_type() == at::kInt &&
                    axis->dim() == 1 && axis->is_contiguous() &&
                    axis->size(0) == inv_freq.size(0),
                op, ": axis must be contiguous int32 [pairs] on q's device");
  TORCH_CHECK(have_axis || positions.size(1) == 1, op, ": ", positions.size(1),
              " position axes need axis");
  TORCH_CHECK(D <= 65536 && q.size(1) <= 65536 && (!two || k->size(1) <= 65536), op,
              ": too many heads or dims");
  const c10::cuda::CUDAGuard g(q.device());
  const Tensor qq = dense_heads(q);
  const Tensor qo = at::empty(q.sizes(), q.options());
  Tensor kk, ko;
  if (two) {
    kk = dense_heads(*k);
    ko = at::empty(k->sizes(), k->options());
  }
  check_rc(pkv_rotary(ptr(qq), qq.stride(0), qq.stride(1), q.numel() ? int(q.size(1)) : 0,
                      mut(qo), qo.stride(0), qo.stride(1), ptr(kk), two ? kk.stride(0) : 0,
                      two ? kk.stride(1) : 0, two && k->numel() ? int(k->size(1)) : 0, mut(ko),
                      two ? ko.stride(0) : 0, two ? ko.stride(1) : 0, dt, T, int(D),
                      static_cast<const int64_t*>(ptr(positions)), int(positions.size(1)),
                      static_cast<const double*>(ptr(inv_freq)),
                      have_axis ? static_cast<const int32_t*>(ptr(*axis)) : nullptr,
                      int(inv_freq.size(0)), half, float(scale), inverse, stream_of(q)),
           op);
  return {qo, ko};
}

}  // namespace
}  // namespace pkv_torch

using namespace pkv_torch;

TORCH_LIBRARY_FRAGMENT(adahead, m) {
  m.def("pkv_layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool one_plus, "
        "bool stats) -> (Tensor, Tensor, Tensor)");
  m.def("pkv_layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor mean, "
        "Tensor rstd, bool one_plus, bool need_x, bool need_weight, bool need_bias) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("pkv_rotary(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, Tensor? axis, "
        "bool half, float scale, bool inverse) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(adahead, CUDA, m) {
  m.impl("pkv_layer_norm", op_layer_norm);
  m.impl("pkv_layer_norm_backward", op_layer_norm_backward);
  m.impl("pkv_rotary", op_rotary);
}
