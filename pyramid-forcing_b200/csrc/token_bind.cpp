// torch glue of the token-path ops (layer norm, rotary positions, block-sparse
// attention): checks the
// tensors and calls one extern "C" entry point of libpkv.so on the current
// CUDA stream.  A fragment of the `adahead` library registered in
// adahead_bind.cpp.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "../../include/pkv.h"

namespace pkv_torch {
namespace {

using at::Tensor;

// The registered op of a kernel below.  The autograd kernels call it rather than the
// CUDA body, so that dispatch modes, fake tensors and tensor subclasses see the call.
template <typename F>
c10::TypedOperatorHandle<F> registered(const char* name, F&) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

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
  Tensor mean, rstd;
  if (stats) {
    mean = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
    rstd = at::empty_like(mean);
  }
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

bool wants_grad(const std::optional<Tensor>& t) {
  return t.has_value() && t->defined() && t->requires_grad();
}

// Layer norm over the last dimension of any x, with its gradient.
Tensor norm_rows(const Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) > 0, "pkv_layer_norm: x has no channels");
  return x.dim() == 2 ? x
                      : x.reshape_symint({x.sym_numel() / x.sym_size(-1), x.sym_size(-1)});
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void refuse_twice(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op,
              ": the gradient is not differentiable (no create_graph)");
}

// A dual tensor does not require a gradient by itself: without this its tangent
// would be lost.
void refuse_forward(const char* op, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op,
                ": forward-mode derivatives are not implemented");
}
const Tensor& or_none(const std::optional<Tensor>& t) {
  static const Tensor none;
  return t.has_value() ? *t : none;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, Tensor x, std::optional<Tensor> weight,
                        std::optional<Tensor> bias, double eps, bool one_plus) {
    at::AutoDispatchBelowADInplaceOrView guard;  // (a tracked view may not be changed in place)
    const Tensor rows = norm_rows(x);
    static const auto op = registered("adahead::pkv_layer_norm", op_layer_norm);
    auto [y, mean, rstd] = op.call(rows, weight, bias, eps, one_plus, true);
    ctx->save_for_backward({x, weight.value_or(Tensor()), bias.value_or(Tensor()), mean, rstd});
    ctx->saved_data["one_plus"] = one_plus;
    return y.view_symint(x.sym_sizes());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_twice("pkv_norm");
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto op =
        registered("adahead::pkv_layer_norm_backward", op_layer_norm_backward);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const bool need_w = w.defined() && ctx->needs_input_grad(1);
    const bool need_b = b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1);
    auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    auto [dx, dw, db] = op.call(
        norm_rows(grads[0]), norm_rows(x), opt(w), opt(b), saved[3], saved[4],
        ctx->saved_data["one_plus"].toBool(), ctx->needs_input_grad(0), need_w, need_b);
    if (dx.defined()) dx = dx.view_symint(x.sym_sizes());
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

Tensor op_norm(Tensor x, std::optional<Tensor> weight, std::optional<Tensor> bias, double eps,
               bool one_plus) {
  return std::get<0>(op_layer_norm(norm_rows(x), weight, bias, eps, one_plus, false))
      .view(x.sizes());
}

Tensor op_norm_autograd(Tensor x, std::optional<Tensor> weight, std::optional<Tensor> bias,
                        double eps, bool one_plus) {
  refuse_forward("pkv_norm", {&x, &or_none(weight), &or_none(bias)});
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(weight) || wants_grad(bias)))
    return LayerNormFn::apply(x, weight, bias, eps, one_plus);
  at::AutoDispatchBelowADInplaceOrView guard;
  static const auto op = registered("adahead::pkv_norm", op_norm);
  return op.call(x, weight, bias, eps, one_plus);
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

// Rotary positions of q and k [..., heads, D], with their gradients.
Tensor rot_rows(const Tensor& x) {
  TORCH_CHECK(x.dim() >= 3, "pkv_rotary: q and k must be [..., heads, dim]");
  c10::SymInt n = 1;
  for (int64_t i = 0; i < x.dim() - 2; ++i) n *= x.sym_size(i);
  return x.dim() == 3 ? x : x.reshape_symint({n, x.sym_size(-2), x.sym_size(-1)});
}

// Positions of any leading shape and whole-number type as int64 [tokens, axes].
Tensor pos_rows(const Tensor& q, const Tensor& positions, int64_t axes) {
  const c10::SymInt per = q.sym_size(-2) * q.sym_size(-1);
  const c10::SymInt n = per > 0 ? q.sym_numel() / per : c10::SymInt(0);
  Tensor p = positions.scalar_type() == at::kLong ? positions : positions.to(at::kLong);
  TORCH_CHECK(axes >= 1 && (per == 0 || p.sym_numel() == n * axes),
              "pkv_rotary: positions must hold ", axes, " axes for each of ", n, " tokens");
  if (p.dim() != 2 || p.sym_size(1) != axes) p = p.reshape_symint({p.sym_numel() / axes, axes});
  return p.contiguous();
}

std::tuple<Tensor, Tensor> op_rotary_apply(Tensor q, std::optional<Tensor> k, Tensor positions,
                                           int64_t axes, Tensor inv_freq,
                                           std::optional<Tensor> axis, bool half, double scale) {
  TORCH_CHECK(q.dim() >= 3, "pkv_rotary: q must be [..., heads, dim]");
  const bool two = k.has_value() && k->defined();
  positions = pos_rows(q, positions, axes);
  auto [qo, ko] = op_rotary(rot_rows(q), two ? std::optional<Tensor>(rot_rows(*k)) : std::nullopt,
                            positions, inv_freq, axis, half, scale, false);
  return {qo.view(q.sizes()), two ? ko.view(k->sizes()) : ko};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, Tensor q, std::optional<Tensor> k,
                               Tensor positions, int64_t axes, Tensor inv_freq,
                               std::optional<Tensor> axis, bool half, double scale) {
    TORCH_CHECK(q.dim() >= 3, "pkv_rotary: q must be [..., heads, dim]");
    at::AutoDispatchBelowADInplaceOrView guard;  // (a tracked view may not be changed in place)
    positions = pos_rows(q, positions, axes);
    const bool two = k.has_value() && k->defined();
    static const auto op = registered("adahead::pkv_rotary", op_rotary);
    auto [qo, ko] =
        op.call(rot_rows(q), two ? std::optional<Tensor>(rot_rows(*k)) : std::nullopt, positions,
                inv_freq, axis, half, scale, false);
    qo = qo.view_symint(q.sym_sizes());
    if (two) ko = ko.view_symint(k->sym_sizes());
    ctx->save_for_backward({positions, inv_freq, axis.value_or(Tensor())});
    ctx->saved_data["half"] = half;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["k"] = two;
    ctx->set_materialize_grads(false);
    if (!two) return {qo};
    return {qo, ko};
  }
  // the transpose of a rotation: the same turn the other way
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_twice("pkv_rotary_apply");
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto op = registered("adahead::pkv_rotary", op_rotary);
    const auto saved = ctx->get_saved_variables();
    const bool two = ctx->saved_data["k"].toBool();
    Tensor dq = grads[0], dk = two ? grads[1] : Tensor();
    if (!ctx->needs_input_grad(0)) dq = Tensor();
    if (two && !ctx->needs_input_grad(1)) dk = Tensor();
    variable_list out(8);
    const Tensor first = dq.defined() ? dq : dk;
    if (!first.defined()) return out;
    const bool both = dq.defined() && dk.defined();
    auto [g0, g1] = op.call(
        rot_rows(first), both ? std::optional<Tensor>(rot_rows(dk)) : std::nullopt, saved[0],
        saved[1], saved[2].defined() ? std::optional<Tensor>(saved[2]) : std::nullopt,
        ctx->saved_data["half"].toBool(), ctx->saved_data["scale"].toDouble(), true);
    out[dq.defined() ? 0 : 1] = g0.view_symint(first.sym_sizes());
    if (both) out[1] = g1.view_symint(dk.sym_sizes());
    return out;
  }
};

std::tuple<Tensor, Tensor> op_rotary_autograd(Tensor q, std::optional<Tensor> k, Tensor positions,
                                              int64_t axes, Tensor inv_freq,
                                              std::optional<Tensor> axis, bool half,
                                              double scale) {
  refuse_forward("pkv_rotary_apply", {&q, &or_none(k), &inv_freq});
  TORCH_CHECK(!at::GradMode::is_enabled() || !inv_freq.requires_grad(),
              "pkv_rotary_apply: inv_freq has no gradient here; detach it");
  if (at::GradMode::is_enabled() && (q.requires_grad() || wants_grad(k))) {
    const variable_list r = RotaryFn::apply(q, k, positions, axes, inv_freq, axis, half, scale);
    return {r[0], r.size() > 1 ? r[1] : Tensor()};
  }
  at::AutoDispatchBelowADInplaceOrView guard;
  static const auto op = registered("adahead::pkv_rotary_apply", op_rotary_apply);
  return op.call(q, k, positions, axes, inv_freq, axis, half, scale);
}

// ---- block-sparse attention ----------------------------------------------------
struct SparseCall {
  Tensor q, k, v, cu;
  int64_t C, H, R, D, groups;
};

const uint16_t* u16(const Tensor& t) { return static_cast<const uint16_t*>(ptr(t)); }

// q [C * R, H, D], k / v [rows, D] (or anything that views so), cu int32.
SparseCall sparse_call(const char* op, const Tensor& q, const Tensor* k, const Tensor* v,
                       const Tensor& cu, int64_t num_chunks, int64_t rows, int64_t query_block,
                       int64_t block, int64_t top_k) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && q.scalar_type() == at::kBFloat16, op,
              ": q must be a bf16 [num_chunks * rows, H, D] CUDA tensor");
  SparseCall c;
  c.C = num_chunks;
  c.R = rows;
  c.H = q.size(1);
  c.D = q.size(2);
  TORCH_CHECK(num_chunks >= 0 && rows >= 0 && q.size(0) == num_chunks * rows, op,
              ": q has ", q.size(0), " rows, not ", num_chunks, " x ", rows);
  TORCH_CHECK(c.D == 64 || c.D == 128, op, ": head size must be 64 or 128");
  TORCH_CHECK(block == 64 || block == 128, op, ": block must be 64 or 128");
  TORCH_CHECK(query_block >= 1 && query_block <= 128, op, ": query_block must be 1 to 128");
  TORCH_CHECK(top_k >= 1 && top_k <= 1024, op, ": top_k must be 1 to 1024");
  TORCH_CHECK(num_chunks * c.H < (int64_t(1) << 31), op, ": too many segments");
  TORCH_CHECK(cu.device() == q.device() && cu.scalar_type() == at::kInt && cu.dim() == 1 &&
                  cu.numel() >= num_chunks * c.H + 1,
              op, ": cu_seqlens_k must be int32 [num_chunks * H + 1] on q's device");
  c.cu = cu.contiguous();
  for (const Tensor* t : {k, v}) {
    if (t == nullptr) continue;
    TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kBFloat16 &&
                    t->numel() % c.D == 0,
                op, ": k / v must be bf16 rows of q's head size on its device");
    Tensor f = t->reshape({t->numel() / c.D, c.D}).contiguous();
    // a view at an odd offset is copied: rows are read 16 bytes at a time
    if (reinterpret_cast<uintptr_t>(f.data_ptr()) % 16) f = f.clone();
    (t == k ? c.k : c.v) = f;
  }
  if (v != nullptr) TORCH_CHECK(c.k.size(0) == c.v.size(0), op, ": k and v rows differ");
  c.q = q;
  if (c.q.stride(2) != 1 || c.q.stride(0) % 8 || c.q.stride(1) % 8 || c.q.stride(0) <= 0 ||
      (c.q.stride(1) <= 0 && c.H > 1) || reinterpret_cast<uintptr_t>(c.q.data_ptr()) % 16)
    c.q = c.q.clone(at::MemoryFormat::Contiguous);
  c.groups = (rows + query_block - 1) / query_block;
  return c;
}

// The three steps over one checked call.
Tensor run_means(const char* op, const Tensor& k, int64_t D, const Tensor& cu, int64_t segs,
                 int64_t block, bool zero_rest) {
  const int64_t rows = pkv_block_rows(k.size(0), int(segs), int(block));
  const Tensor means = at::empty({rows, D}, k.options().dtype(at::kFloat));
  check_rc(pkv_block_means(u16(k), k.size(0), int(D), cu.data_ptr<int32_t>(), int(segs),
                           int(block), static_cast<float*>(mut(means)), rows, zero_rest,
                           stream_of(k)),
           op);
  return means;
}

Tensor run_select(const char* op, const SparseCall& c, const Tensor& means, int64_t kv_rows,
                  int64_t query_block, int64_t block, int64_t top_k) {
  TORCH_CHECK(means.device() == c.q.device() && means.scalar_type() == at::kFloat &&
                  means.dim() == 2 && means.size(1) == c.D && kv_rows >= 0 &&
                  means.size(0) >= pkv_block_rows(kv_rows, int(c.C * c.H), int(block)),
              op, ": means must be the fp32 table pkv_block_means gives for these keys");
  Tensor mm = means.contiguous();
  if (reinterpret_cast<uintptr_t>(mm.data_ptr()) % 16) mm = mm.clone();
  const Tensor blocks = at::empty({c.C * c.H, c.groups, top_k}, c.cu.options());
  check_rc(pkv_select_blocks(u16(c.q), c.q.stride(0), c.q.stride(1),
                             static_cast<const float*>(ptr(mm)), mm.size(0),
                             c.cu.data_ptr<int32_t>(), kv_rows, int(c.C), int(c.H), int(c.R),
                             int(c.D), int(query_block), int(block), int(top_k),
                             static_cast<int32_t*>(mut(blocks)), stream_of(c.q)),
           op);
  return blocks;
}

Tensor run_attention(const char* op, const SparseCall& c, const Tensor& blocks,
                     int64_t query_block, int64_t block, double scale,
                     const std::optional<Tensor>& status) {
  TORCH_CHECK(scale > 0.0, op, ": softmax_scale must be positive");
  int32_t* st = nullptr;
  if (status.has_value() && status->defined()) {
    TORCH_CHECK(status->device() == c.q.device() && status->scalar_type() == at::kInt &&
                    status->numel() >= 1,
                op, ": status must be int32 on q's device");
    st = status->data_ptr<int32_t>();
  }
  const Tensor out = at::empty({c.C * c.R, c.H, c.D}, c.q.options());
  check_rc(pkv_block_attention(u16(c.q), c.q.stride(0), c.q.stride(1), u16(c.k), u16(c.v),
                               c.k.size(0), c.cu.data_ptr<int32_t>(), int(c.C), int(c.H),
                               int(c.R), int(c.D), float(scale),
                               static_cast<const int32_t*>(ptr(blocks)), int(query_block),
                               int(block), int(blocks.size(2)), static_cast<uint16_t*>(mut(out)),
                               out.stride(0), out.stride(1), st, stream_of(c.q)),
           op);
  return out;
}

Tensor op_block_means(Tensor k, Tensor cu, int64_t block, bool zero_rest) {
  const char* op = "pkv_block_means";
  TORCH_CHECK(k.is_cuda() && k.dim() >= 2 && k.scalar_type() == at::kBFloat16, op,
              ": k must be a bf16 [rows, D] CUDA tensor");
  const int64_t D = k.size(-1);
  TORCH_CHECK(D == 64 || D == 128, op, ": head size must be 64 or 128");
  TORCH_CHECK(block == 64 || block == 128, op, ": block must be 64 or 128");
  TORCH_CHECK(cu.device() == k.device() && cu.scalar_type() == at::kInt && cu.dim() == 1 &&
                  cu.numel() >= 1 && cu.numel() < (int64_t(1) << 31),
              op, ": cu_seqlens_k must be int32 [segments + 1] on k's device");
  const c10::cuda::CUDAGuard g(k.device());
  Tensor kk = k.reshape({k.numel() / D, D}).contiguous();
  if (reinterpret_cast<uintptr_t>(kk.data_ptr()) % 16) kk = kk.clone();
  const Tensor cc = cu.contiguous();
  return run_means(op, kk, D, cc, cc.numel() - 1, block, zero_rest);
}

Tensor op_select_blocks(Tensor q, Tensor means, Tensor cu, int64_t kv_rows, int64_t num_chunks,
                        int64_t rows, int64_t top_k, int64_t query_block, int64_t block) {
  const char* op = "pkv_select_blocks";
  const c10::cuda::OptionalCUDAGuard g(q.is_cuda() ? std::optional<c10::Device>(q.device())
                                                   : std::nullopt);
  const SparseCall c =
      sparse_call(op, q, nullptr, nullptr, cu, num_chunks, rows, query_block, block, top_k);
  return run_select(op, c, means, kv_rows, query_block, block, top_k);
}

Tensor op_block_attention(Tensor q, Tensor k, Tensor v, Tensor cu, int64_t num_chunks,
                          int64_t rows, Tensor blocks, int64_t query_block, int64_t block,
                          double scale, std::optional<Tensor> status) {
  const char* op = "pkv_block_attention";
  TORCH_CHECK(blocks.dim() == 3, op, ": blocks must be [num_chunks * H, groups, top_k]");
  const c10::cuda::OptionalCUDAGuard g(q.is_cuda() ? std::optional<c10::Device>(q.device())
                                                   : std::nullopt);
  const SparseCall c =
      sparse_call(op, q, &k, &v, cu, num_chunks, rows, query_block, block, blocks.size(2));
  TORCH_CHECK(blocks.device() == q.device() && blocks.scalar_type() == at::kInt &&
                  blocks.size(0) == c.C * c.H && blocks.size(1) == c.groups,
              op, ": blocks must be int32 [", c.C * c.H, ", ", c.groups, ", top_k] on q's device");
  return run_attention(op, c, blocks.contiguous(), query_block, block, scale, status);
}

std::tuple<Tensor, Tensor> op_sparse_attention(Tensor q, Tensor k, Tensor v, Tensor cu,
                                               int64_t num_chunks, int64_t rows, int64_t top_k,
                                               int64_t query_block, int64_t block,
                                               std::optional<double> scale,
                                               std::optional<Tensor> means,
                                               std::optional<Tensor> status) {
  const char* op = "pkv_sparse_attention";
  const c10::cuda::OptionalCUDAGuard g(q.is_cuda() ? std::optional<c10::Device>(q.device())
                                                   : std::nullopt);
  const SparseCall c =
      sparse_call(op, q, &k, &v, cu, num_chunks, rows, query_block, block, top_k);
  const Tensor table = means.has_value() && means->defined()
                           ? *means
                           : run_means(op, c.k, c.D, c.cu, c.C * c.H, block, false);
  const Tensor blocks = run_select(op, c, table, c.k.size(0), query_block, block, top_k);
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt(double(c.D));
  return {run_attention(op, c, blocks, query_block, block, sc, status), blocks};
}

}  // namespace
}  // namespace pkv_torch

using namespace pkv_torch;

TORCH_LIBRARY_FRAGMENT(adahead, m) {
  m.def("pkv_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool one_plus) -> Tensor");
  m.def("pkv_rotary_apply(Tensor q, Tensor? k, Tensor positions, int axes, Tensor inv_freq, "
        "Tensor? axis, bool half, float scale) -> (Tensor, Tensor)");
  m.def("pkv_layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool one_plus, "
        "bool stats) -> (Tensor, Tensor, Tensor)");
  m.def("pkv_layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor mean, "
        "Tensor rstd, bool one_plus, bool need_x, bool need_weight, bool need_bias) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("pkv_rotary(Tensor q, Tensor? k, Tensor positions, Tensor inv_freq, Tensor? axis, "
        "bool half, float scale, bool inverse) -> (Tensor, Tensor)");
  m.def("pkv_block_means(Tensor k, Tensor cu_seqlens_k, int block, bool zero_rest) -> Tensor");
  m.def("pkv_select_blocks(Tensor q, Tensor means, Tensor cu_seqlens_k, int kv_rows, "
        "int num_chunks, int rows_per_chunk, int top_k, int query_block, int block) -> Tensor");
  m.def("pkv_block_attention(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens_k, int num_chunks, "
        "int rows_per_chunk, Tensor blocks, int query_block, int block, float softmax_scale, "
        "Tensor(a!)? status) -> Tensor");
  m.def("pkv_sparse_attention(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens_k, int num_chunks, "
        "int rows_per_chunk, int top_k, int query_block, int block, float? softmax_scale, "
        "Tensor? means, Tensor(a!)? status) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(adahead, CUDA, m) {
  m.impl("pkv_layer_norm", op_layer_norm);
  m.impl("pkv_layer_norm_backward", op_layer_norm_backward);
  m.impl("pkv_rotary", op_rotary);
  m.impl("pkv_block_means", op_block_means);
  m.impl("pkv_select_blocks", op_select_blocks);
  m.impl("pkv_block_attention", op_block_attention);
  m.impl("pkv_sparse_attention", op_sparse_attention);
  m.impl("pkv_norm", op_norm);
  m.impl("pkv_rotary_apply", op_rotary_apply);
}

TORCH_LIBRARY_IMPL(adahead, AutogradCUDA, m) {
  m.impl("pkv_norm", op_norm_autograd);
  m.impl("pkv_rotary_apply", op_rotary_autograd);
}

// Shapes only.
TORCH_LIBRARY_IMPL(adahead, Meta, m) {
  using Opt = std::optional<Tensor>;
  auto given = [](const Opt& t) { return t.has_value() && t->defined(); };
  auto like = [](const Tensor& t) { return at::empty_symint(t.sym_sizes(), t.options()); };
  m.impl("pkv_norm", [like](Tensor x, Opt, Opt, double, bool) { return like(x); });
  m.impl("pkv_layer_norm", [like](Tensor x, Opt, Opt, double, bool, bool stats) {
    Tensor mean, rstd;
    if (stats) {
      mean = at::empty_symint({x.sym_size(0)}, x.options().dtype(at::kFloat));
      rstd = at::empty_like(mean);
    }
    return std::tuple<Tensor, Tensor, Tensor>(like(x), mean, rstd);
  });
  m.impl("pkv_layer_norm_backward", [like, given](Tensor, Tensor x, Opt w, Opt b, Tensor, Tensor,
                                                  bool, bool need_x, bool need_weight,
                                                  bool need_bias) {
    TORCH_CHECK((!need_weight || given(w)) && (!need_bias || given(b)),
                "pkv_layer_norm_backward: no weight / bias to differentiate");
    return std::tuple<Tensor, Tensor, Tensor>(need_x ? like(x) : Tensor(),
                                              need_weight ? like(*w) : Tensor(),
                                              need_bias ? like(*b) : Tensor());
  });
  auto rotate = [like, given](const Tensor& q, const Opt& k) {
    return std::tuple<Tensor, Tensor>(like(q), given(k) ? like(*k) : Tensor());
  };
  m.impl("pkv_rotary", [rotate](Tensor q, Opt k, Tensor, Tensor, Opt, bool, double, bool) {
    return rotate(q, k);
  });
  m.impl("pkv_rotary_apply",
         [rotate](Tensor q, Opt k, Tensor, int64_t, Tensor, Opt, bool, double) {
           return rotate(q, k);
         });
  m.impl("pkv_block_means", [](Tensor k, Tensor cu, int64_t block, bool) {
    TORCH_CHECK(k.dim() >= 2 && (k.size(-1) == 64 || k.size(-1) == 128) &&
                    (block == 64 || block == 128),
                "pkv_block_means: head size and block must be 64 or 128");
    const c10::SymInt D = k.size(-1);
    return at::empty_symint({k.sym_numel() / D / block + cu.sym_numel() - 1, D},
                            k.options().dtype(at::kFloat));
  });
  auto lists = [](const Tensor& q, const Tensor& cu, int64_t chunks, int64_t rows, int64_t top_k,
                  int64_t query_block) {
    TORCH_CHECK(query_block >= 1, "query_block must be 1 to 128");
    return at::empty_symint({chunks * q.sym_size(1), (rows + query_block - 1) / query_block, top_k},
                            cu.options());
  };
  m.impl("pkv_select_blocks",
         [lists](Tensor q, Tensor, Tensor cu, int64_t, int64_t chunks, int64_t rows,
                 int64_t top_k, int64_t query_block, int64_t) {
           return lists(q, cu, chunks, rows, top_k, query_block);
         });
  m.impl("pkv_block_attention",
         [like](Tensor q, Tensor, Tensor, Tensor, int64_t, int64_t, Tensor, int64_t, int64_t,
                double, Opt) { return like(q); });
  m.impl("pkv_sparse_attention",
         [like, lists](Tensor q, Tensor, Tensor, Tensor cu, int64_t chunks, int64_t rows,
                       int64_t top_k, int64_t query_block, int64_t, std::optional<double>, Opt,
                       Opt) {
           return std::tuple<Tensor, Tensor>(like(q),
                                             lists(q, cu, chunks, rows, top_k, query_block));
         });
}
