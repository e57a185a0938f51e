// Torch front of the language-model operators around the loss (embedding,
// residual norm, 8-bit output layer, output-layer cross entropy): argument
// checks, outputs, workspaces, the current stream, and the autograd nodes
// (in C++: a small call spends most of its time on the host).  Registered in
// the module fw_radix_cuda next to the loss (fw_torch_binding.cpp).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <vector>

#include "../../include/fwloss_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

void ok(int rc, const char* what) { TORCH_CHECK(rc == FWB_OK, what, " failed: ", fw_error_string(rc)); }

void type_check(bool cond, const char* what) {
  if (!cond) throw py::type_error(what);
}

void value_check(bool cond, const char* what) {
  if (!cond) throw py::value_error(what);
}

void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

bool is_float(const Tensor& t) {
  return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kHalf;
}

int code(torch::ScalarType t) {
  return t == torch::kBFloat16 ? FWB_DTYPE_BF16 : t == torch::kHalf ? FWB_DTYPE_F16 : FWB_DTYPE_F32;
}

int code(const Tensor& t) { return code(t.scalar_type()); }

// Unit column stride and rows that do not overlap; copies otherwise.
Tensor rows_of(const Tensor& t) {
  return (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}

// [..., D] as rows of D.
Tensor rows_2d(const Tensor& t) { return rows_of(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }

int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

int32_t* status_of(const OptTensor& s, const Tensor& like) {
  if (!s.has_value()) return nullptr;
  TORCH_CHECK(s->device() == like.device() && s->scalar_type() == torch::kInt32 && s->numel() >= 1 &&
                  s->is_contiguous(),
              "status must be an int32 tensor on the inputs' device");
  return s->data_ptr<int32_t>();
}

// The status word of a later backward.  Not a saved variable: clearing it in
// between is its normal use.
void keep_status(AutogradContext* ctx, const OptTensor& s) {
  if (s.has_value()) ctx->saved_data["status"] = c10::IValue(*s);
}

OptTensor kept_status(AutogradContext* ctx) {
  const auto it = ctx->saved_data.find("status");
  return it == ctx->saved_data.end() ? OptTensor() : OptTensor(it->second.toTensor());
}

Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({n > 0 ? n : 1}, like.options().dtype(torch::kUInt8));
}

Tensor f32(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(torch::kFloat32)); }

bool recording(const Tensor& t) { return t.requires_grad(); }

// A result without a tangent would drop the operand's silently, whatever the grad mode.
void no_tangent(const Tensor& t, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), op, ": forward-mode differentiation is not implemented");
}

// The gradients have none of their own: a second derivative raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list marked;
  std::vector<size_t> at;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      auto t = grads[i].detach();
      t.set_requires_grad(true);
      marked.push_back(t);
      at.push_back(i);
    }
  if (marked.empty()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "this operator's gradient cannot be differentiated again", (int)marked.size());
  auto out = (*node)(std::move(marked));
  for (size_t k = 0; k < at.size(); ++k) grads[at[k]] = out[k];
  return grads;
}

// ---------------------------------------------------------------- embedding
Tensor embed_rows(const Tensor& ids, const Tensor& weight, double scale, const OptTensor& status) {
  const c10::cuda::CUDAGuard guard(weight.device());
  auto w = rows_of(weight);
  auto i = ids.contiguous();
  const int64_t T = i.numel(), V = w.size(0), D = w.size(1);
  c10::SmallVector<int64_t, 6> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(D);
  auto out = at::empty(shape, w.options());
  ok(fw_embed_rows(code(w), i.data_ptr<int64_t>(), T, w.data_ptr(), ld_of(w), V, D, (float)scale, out.data_ptr(), D,
                   status_of(status, w), stream()),
     "fw_embed_rows");
  return out;
}

Tensor embed_grad(const Tensor& ids, const Tensor& grad, int64_t V, double scale, int64_t padding,
                  const OptTensor& status) {
  const c10::cuda::CUDAGuard guard(grad.device());
  auto i = ids.contiguous();
  auto g = rows_2d(grad);
  const int64_t T = i.numel(), D = g.size(1);
  auto dw = at::empty({V, D}, g.options());
  const int64_t n = fw_embed_grad_workspace(T, V, D);
  Tensor ws;
  if (n > 0) ws = bytes(n, g);
  ok(fw_embed_grad(code(g), i.data_ptr<int64_t>(), T, g.data_ptr(), ld_of(g), V, D, (float)scale, padding,
                   dw.data_ptr(), n > 0 ? ws.data_ptr() : nullptr, n, status_of(status, g), stream()),
     "fw_embed_grad");
  return dw;
}

struct EmbedTokens : torch::autograd::Function<EmbedTokens> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding,
                        const OptTensor& status) {
    ctx->save_for_backward({ids});
    keep_status(ctx, status);
    ctx->saved_data["a"] = c10::IValue(std::vector<double>{(double)weight.size(0), scale, (double)padding});
    return embed_rows(ids, weight, scale, status);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const auto a = ctx->saved_data["a"].toDoubleVector();
    auto dw = embed_grad(saved[0], g[0].detach(), (int64_t)a[0], a[1], (int64_t)a[2], kept_status(ctx));
    return once({Tensor(), dw, Tensor(), Tensor(), Tensor()});
  }
};

Tensor embed_tokens(const Tensor& ids, const Tensor& weight, double scale, c10::optional<int64_t> padding,
                    const OptTensor& status) {
  type_check(weight.is_cuda(), "embed_tokens: weight must be a CUDA tensor (this build has no CPU path)");
  type_check(weight.dim() == 2 && is_float(weight) && weight.numel() > 0,
             "embed_tokens: weight must be a non-empty 2-D float32, bfloat16 or float16 tensor [V, D]");
  type_check(ids.scalar_type() == torch::kLong, "embed_tokens: tokens must be an int64 tensor");
  value_check(ids.device() == weight.device(), "embed_tokens: tokens must be on weight's device");
  value_check(!padding || (*padding >= 0 && *padding < weight.size(0)),
              "embed_tokens: padding_idx is outside the table");
  no_tangent(weight, "embed_tokens");
  const int64_t pad = padding.value_or(-1);
  if (at::GradMode::is_enabled() && recording(weight)) return EmbedTokens::apply(ids, weight, scale, pad, status);
  return embed_rows(ids, weight, scale, status);
}

Tensor embed_grad_checked(const Tensor& ids, const Tensor& grad, int64_t V, double scale, int64_t padding,
                          const OptTensor& status) {
  type_check(grad.is_cuda(), "embed_grad: grad must be a CUDA tensor (this build has no CPU path)");
  type_check(grad.dim() >= 1 && is_float(grad) && grad.size(-1) >= 1,
             "embed_grad: grad must be a float32, bfloat16 or float16 tensor [..., D]");
  type_check(ids.scalar_type() == torch::kLong, "embed_grad: tokens must be an int64 tensor");
  value_check(ids.device() == grad.device(), "embed_grad: tokens must be on grad's device");
  value_check(ids.sizes() == grad.sizes().slice(0, grad.dim() - 1), "embed_grad: grad must have the tokens' shape and D");
  value_check(V >= 1 && padding >= -1 && padding < V, "embed_grad: padding is outside the table (-1: none)");
  return embed_grad(ids, grad, V, scale, padding, status);
}

// ---------------------------------------------------------------- norm
void check_norm(const Tensor& x, const Tensor& weight, double eps, const OptTensor& residual) {
  type_check(x.is_cuda(), "rms_norm: x must be a CUDA tensor (this build has no CPU path)");
  type_check(x.dim() >= 1 && is_float(x) && x.size(-1) >= 1,
             "rms_norm: x must be a float32, bfloat16 or float16 tensor [..., D]");
  type_check(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == torch::kFloat32,
             "rms_norm: weight must have x's dtype or float32");
  value_check(weight.dim() == 1 && weight.size(0) == x.size(-1) && weight.device() == x.device(),
              "rms_norm: weight must have shape [D] on x's device");
  value_check(eps >= 0.0, "rms_norm: eps must not be negative");
  if (residual.has_value()) {
    type_check(residual->scalar_type() == x.scalar_type(), "rms_norm: residual must have x's dtype");
    value_check(residual->sizes() == x.sizes() && residual->device() == x.device(),
                "rms_norm: residual must have x's shape and device");
  }
}

struct Norm {
  Tensor y, rstd, sum;
};

Norm norm_forward(const Tensor& x_, const Tensor& weight, double eps, const OptTensor& residual, bool keep) {
  const c10::cuda::CUDAGuard guard(x_.device());
  auto x = rows_2d(x_);
  auto w = weight.contiguous();
  const int64_t rows = x.size(0), D = x.size(1);
  Norm out;
  out.y = at::empty(x_.sizes(), x.options());
  if (keep) out.rstd = f32({rows}, x);
  Tensor r;
  if (residual.has_value()) {
    r = rows_2d(*residual);
    out.sum = at::empty(x_.sizes(), x.options());
  }
  ok(fw_rms_norm(code(x), code(w), x.data_ptr(), ld_of(x), r.defined() ? r.data_ptr() : nullptr,
                 r.defined() ? ld_of(r) : D, w.data_ptr(), rows, D, (float)eps,
                 r.defined() ? out.sum.data_ptr() : nullptr, D, out.y.data_ptr(), D,
                 keep ? out.rstd.data_ptr<float>() : nullptr, stream()),
     "fw_rms_norm");
  return out;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                               double eps) {
    ctx->set_materialize_grads(false);
    auto n = norm_forward(x, weight, eps, residual, true);
    ctx->save_for_backward({n.sum.defined() ? n.sum : x, weight, n.rstd});
    if (n.sum.defined()) return {n.y, n.sum};
    return {n.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const bool has_r = g.size() > 1;
    const bool want_w = ctx->needs_input_grad(1);
    const Tensor &dy_ = g[0], dsum = has_r ? g[1] : Tensor();
    if (!dy_.defined())  // only the sum was used
      return {dsum, Tensor(), has_r ? dsum : Tensor(), Tensor()};
    const c10::cuda::CUDAGuard guard(dy_.device());
    auto dy = rows_2d(dy_), s = rows_2d(saved[0]);
    auto w = saved[1].contiguous();
    const int64_t rows = s.size(0), D = s.size(1);
    auto dx = at::empty(dy_.sizes(), s.options());
    Tensor o, parts, dw;
    if (dsum.defined()) o = rows_2d(dsum);
    const int64_t n = fw_rms_norm_grad_parts(rows);
    if (want_w) {
      parts = f32({n, D}, s);
      dw = at::empty({D}, w.options());
    }
    ok(fw_rms_norm_grad(code(s), code(w), dy.data_ptr(), ld_of(dy), s.data_ptr(), ld_of(s),
                        o.defined() ? o.data_ptr() : nullptr, o.defined() ? ld_of(o) : D, w.data_ptr(),
                        saved[2].data_ptr<float>(), rows, D, dx.data_ptr(), D,
                        want_w ? parts.data_ptr<float>() : nullptr, n, want_w ? dw.data_ptr() : nullptr, stream()),
       "fw_rms_norm_grad");
    return once({dx, dw, has_r ? dx : Tensor(), Tensor()});
  }
};

py::object rms_norm(const Tensor& x, const Tensor& weight, double eps, const OptTensor& residual) {
  check_norm(x, weight, eps, residual);
  no_tangent(x, "rms_norm");
  no_tangent(weight, "rms_norm");
  if (residual.has_value()) no_tangent(*residual, "rms_norm");
  if (at::GradMode::is_enabled() &&
      (recording(x) || recording(weight) || (residual.has_value() && recording(*residual)))) {
    auto out = RmsNorm::apply(x, weight, residual, eps);
    return out.size() == 1 ? py::cast(out[0]) : py::object(py::make_tuple(out[0], out[1]));
  }
  auto n = norm_forward(x, weight, eps, residual, false);
  return n.sum.defined() ? py::object(py::make_tuple(n.y, n.sum)) : py::cast(n.y);
}

// [rows, cols] int8 whose rows start on 16-byte boundaries
Tensor int8_rows(int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t ld = (cols + 15) / 16 * 16;
  auto t = at::empty({rows, ld}, like.options().dtype(torch::kInt8));
  return ld == cols ? t : t.narrow(1, 0, cols);
}

py::tuple rms_norm_int8(const Tensor& x_, const Tensor& weight, double eps, const OptTensor& residual) {
  check_norm(x_, weight, eps, residual);
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(x_.device());
  auto x = rows_2d(x_);
  auto w = weight.contiguous();
  const int64_t rows = x.size(0), D = x.size(1);
  auto q = int8_rows(rows, D, x);
  auto scale = f32(x_.sizes().slice(0, x_.dim() - 1), x);
  Tensor r, sum;
  if (residual.has_value()) {
    r = rows_2d(*residual);
    sum = at::empty(x_.sizes(), x.options());
  }
  ok(fw_rms_norm_int8(code(x), code(w), x.data_ptr(), ld_of(x), r.defined() ? r.data_ptr() : nullptr,
                      r.defined() ? ld_of(r) : D, w.data_ptr(), rows, D, (float)eps,
                      r.defined() ? sum.data_ptr() : nullptr, D, q.data_ptr<int8_t>(), (D + 15) / 16 * 16,
                      scale.data_ptr<float>(), stream()),
     "fw_rms_norm_int8");
  if (x_.dim() == 1)
    q = q.select(0, 0);
  else if (x_.dim() > 2)
    q = q.unflatten(0, x_.sizes().slice(0, x_.dim() - 1));
  return sum.defined() ? py::make_tuple(q, scale, sum) : py::make_tuple(q, scale);
}

py::tuple quantize_rows_int8(const Tensor& x_) {
  type_check(x_.is_cuda(), "quantize_rows_int8: x must be a CUDA tensor (this build has no CPU path)");
  type_check(x_.dim() == 2 && is_float(x_) && x_.size(1) >= 1,
             "quantize_rows_int8: x must be a 2-D float32, bfloat16 or float16 tensor [R, D]");
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(x_.device());
  auto x = rows_of(x_);
  const int64_t rows = x.size(0), D = x.size(1);
  auto q = int8_rows(rows, D, x);
  auto scale = f32({rows}, x);
  ok(fw_quantize_rows_int8(code(x), x.data_ptr(), ld_of(x), rows, D, q.data_ptr<int8_t>(), (D + 15) / 16 * 16,
                           scale.data_ptr<float>(), stream()),
     "fw_quantize_rows_int8");
  return py::make_tuple(q, scale);
}

// ---------------------------------------------------------------- 8-bit output layer
// Rows on 16-byte boundaries; copied there if they are not.
Tensor aligned_rows(const Tensor& t) {
  const int64_t K = t.size(1);
  const bool fits = (K == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || (t.stride(0) >= K && t.stride(0) % 16 == 0)) &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (fits) return t;
  auto c = int8_rows(t.size(0), K, t);
  c.copy_(t);
  return c;
}

int64_t int8_ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16; }

Tensor int8_linear(const Tensor& q_, const Tensor& q_scale, const Tensor& w_, const Tensor& w_scale,
                   at::ScalarType out_dtype, const OptTensor& status) {
  type_check(q_.is_cuda() && q_.scalar_type() == torch::kInt8, "int8_linear: q must be an int8 CUDA tensor");
  type_check(w_.is_cuda() && w_.scalar_type() == torch::kInt8, "int8_linear: weight must be an int8 CUDA tensor");
  type_check(q_scale.is_cuda() && w_scale.is_cuda() && q_scale.scalar_type() == torch::kFloat32 &&
                 w_scale.scalar_type() == torch::kFloat32,
             "int8_linear: q_scale and weight_scale must be float32 CUDA tensors");
  type_check(out_dtype == torch::kFloat32 || out_dtype == torch::kBFloat16 || out_dtype == torch::kHalf,
             "int8_linear: out_dtype must be float32, bfloat16 or float16");
  value_check(w_.device() == q_.device() && q_scale.device() == q_.device() && w_scale.device() == q_.device(),
              "int8_linear: all inputs must be on one device");
  value_check(w_.dim() == 2 && w_.numel() > 0 && q_.dim() >= 1 && q_.size(-1) == w_.size(1),
              "int8_linear: q [..., K] and weight [N, K] disagree");
  value_check(q_scale.sizes() == q_.sizes().slice(0, q_.dim() - 1) && w_scale.dim() == 1 &&
                  w_scale.size(0) == w_.size(0),
              "int8_linear: q_scale must have q's leading shape and weight_scale the shape [N]");
  value_check(w_.size(1) <= FWB_INT8_MAX_K, "int8_linear: K is at most 131071 (the sum is a 32-bit integer)");
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(q_.device());
  auto q = aligned_rows(q_.dim() == 2 ? q_ : q_.reshape({-1, q_.size(-1)})), w = aligned_rows(w_);
  auto qs = q_scale.contiguous(), ws = w_scale.contiguous();
  const int64_t T = q.size(0), K = q.size(1), N = w.size(0);
  c10::SmallVector<int64_t, 6> shape(q_.sizes().begin(), q_.sizes().end());
  shape.back() = N;
  auto out = at::empty(shape, q.options().dtype(out_dtype));
  ok(fw_int8_linear(code(out_dtype), q.data_ptr<int8_t>(), int8_ld(q), qs.data_ptr<float>(), w.data_ptr<int8_t>(),
                    int8_ld(w), ws.data_ptr<float>(), T, N, K, out.data_ptr(), N, status_of(status, q), stream()),
     "fw_int8_linear");
  return out;
}

// ---------------------------------------------------------------- cross entropy
struct Xent {
  Tensor loss, state;
};

Xent xent_forward(const Tensor& hidden, const Tensor& weight, const Tensor& target, int64_t ignore_index,
                  int64_t reduction, const OptTensor& status) {
  const c10::cuda::CUDAGuard guard(hidden.device());
  auto h = rows_of(hidden), w = rows_of(weight);
  auto y = target.contiguous();
  const int64_t B = h.size(0), D = h.size(1), V = w.size(0);
  auto loss = reduction == FWB_REDUCE_NONE ? f32({B}, h) : f32({}, h);
  const int64_t ns = fw_xent_state_bytes(B, D, V, w.data_ptr(), ld_of(w)), nw = fw_xent_workspace(B, D, V, 0);
  auto state = bytes(ns, h), ws = bytes(nw, h);
  ok(fw_xent_forward(code(h), h.data_ptr(), ld_of(h), w.data_ptr(), ld_of(w), y.data_ptr<int64_t>(), B, D, V,
                     ignore_index, (int)reduction, loss.data_ptr<float>(), state.data_ptr(), ns, ws.data_ptr(), nw,
                     status_of(status, h), stream()),
     "fw_xent_forward");
  return {loss, state};
}

struct LmHeadCrossEntropy : torch::autograd::Function<LmHeadCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& target,
                        int64_t ignore_index, int64_t reduction, const OptTensor& status) {
    auto x = xent_forward(hidden, weight, target, ignore_index, reduction, status);
    ctx->save_for_backward({weight, x.state});
    keep_status(ctx, status);
    ctx->saved_data["a"] = c10::IValue(std::vector<int64_t>{hidden.size(0), reduction});
    return x.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const auto a = ctx->saved_data["a"].toIntVector();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    auto w = rows_of(saved[0]);
    const Tensor& state = saved[1];
    auto go = g[0].detach().contiguous();
    const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const int64_t B = a[0], V = w.size(0), D = w.size(1);
    // A hook may have restored the weight off the 16-byte boundaries it was saved on; the state has no copy of it then.
    if (fw_xent_state_bytes(B, D, V, w.data_ptr(), ld_of(w)) > state.numel()) {
      auto c = at::empty({V, (D + 7) / 8 * 8}, w.options()).narrow(1, 0, D);
      c.copy_(w);
      w = c;
    }
    Tensor dh, dw;
    if (want_h) dh = at::empty({B, D}, w.options());
    if (want_w) dw = at::empty({V, D}, w.options());
    const int64_t nw = fw_xent_workspace(B, D, V, 1);
    auto ws = bytes(nw, w);
    const OptTensor status = kept_status(ctx);
    ok(fw_xent_backward(code(w), w.data_ptr(), ld_of(w), B, D, V, (int)a[1], go.data_ptr<float>(), state.data_ptr(),
                        state.numel(), ws.data_ptr(), nw, want_h ? dh.data_ptr() : nullptr,
                        want_w ? dw.data_ptr() : nullptr, status_of(status, w), stream()),
       "fw_xent_backward");
    return once({dh, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor lm_head_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& target, int64_t reduction,
                             int64_t ignore_index, const OptTensor& status) {
  type_check(hidden.is_cuda() && weight.is_cuda(),
             "lm_head_cross_entropy: hidden and weight must be CUDA tensors (this build has no CPU path)");
  type_check(hidden.dim() == 2 && weight.dim() == 2 && weight.numel() > 0,
             "lm_head_cross_entropy: hidden [B, D] and weight [V, D] must be matrices");
  type_check(hidden.scalar_type() == weight.scalar_type() &&
                 (hidden.scalar_type() == torch::kBFloat16 || hidden.scalar_type() == torch::kHalf),
             "lm_head_cross_entropy: hidden and weight must both be bfloat16 or both float16");
  value_check(hidden.size(1) == weight.size(1), "lm_head_cross_entropy: hidden and weight disagree on D");
  type_check(target.scalar_type() == torch::kLong, "lm_head_cross_entropy: target must be int64");
  value_check(target.dim() == 1 && target.size(0) == hidden.size(0),
              "lm_head_cross_entropy: target must have shape [B]");
  value_check(weight.device() == hidden.device() && target.device() == hidden.device(),
              "lm_head_cross_entropy: hidden, weight and target must be on one device");
  no_tangent(hidden, "lm_head_cross_entropy");
  no_tangent(weight, "lm_head_cross_entropy");
  if (at::GradMode::is_enabled() && (recording(hidden) || recording(weight)))
    return LmHeadCrossEntropy::apply(hidden, weight, target, ignore_index, reduction, status);
  return xent_forward(hidden, weight, target, ignore_index, reduction, status).loss;
}

}  // namespace

void register_lm_operators(pybind11::module_& m) {
  m.def("embed_tokens", &embed_tokens, "rows of a table, scaled (differentiable)");
  m.def("embed_grad", &embed_grad_checked, "gradient of embed_tokens in the table, deterministic");
  m.def("rms_norm", &rms_norm, "norm of a residual stream (differentiable)");
  m.def("rms_norm_int8", &rms_norm_int8, "(q, scale[, x + residual])");
  m.def("quantize_rows_int8", &quantize_rows_int8, "(q, scale)");
  m.def("int8_linear", &int8_linear, "8-bit output layer");
  m.def("lm_head_cross_entropy", &lm_head_cross_entropy, "softmax cross entropy of an output layer (differentiable)");
}
