// Torch front of the language-model operators around the loss (embedding,
// residual norm, 8-bit output layer, output-layer cross entropy): argument
// checks, outputs, workspaces and the current stream.  Registered in the
// module fw_radix_cuda next to the loss (fw_torch_binding.cpp).
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

#include "../../include/fwloss_b200.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void ok(int rc, const char* what) { TORCH_CHECK(rc == FWB_OK, what, " failed: ", fw_error_string(rc)); }

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

int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

int32_t* status_of(const OptTensor& s, const Tensor& like) {
  if (!s.has_value()) return nullptr;
  TORCH_CHECK(s->device() == like.device() && s->scalar_type() == torch::kInt32 && s->numel() >= 1 &&
                  s->is_contiguous(),
              "status must be an int32 tensor on the inputs' device");
  return s->data_ptr<int32_t>();
}

Tensor bytes(int64_t n, const Tensor& like) {
  return torch::empty({n > 0 ? n : 1}, like.options().dtype(torch::kUInt8));
}

void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// ---------------------------------------------------------------- embedding
Tensor embed_rows(Tensor ids, Tensor weight, double scale, OptTensor status) {
  const c10::cuda::CUDAGuard guard(weight.device());
  auto w = rows_of(weight);
  auto i = ids.contiguous();
  const int64_t T = i.numel(), V = w.size(0), D = w.size(1);
  auto shape = ids.sizes().vec();
  shape.push_back(D);
  auto out = torch::empty(shape, w.options());
  ok(fw_embed_rows(code(w), i.data_ptr<int64_t>(), T, w.data_ptr(), ld_of(w), V, D, (float)scale, out.data_ptr(), D,
                   status_of(status, w), stream()),
     "fw_embed_rows");
  return out;
}

Tensor embed_grad(Tensor ids, Tensor grad, int64_t V, double scale, int64_t padding, OptTensor status) {
  const c10::cuda::CUDAGuard guard(grad.device());
  const int64_t D = grad.size(-1);
  auto i = ids.contiguous();
  auto g = rows_of(grad.dim() == 2 ? grad : grad.reshape({i.numel(), D}));
  const int64_t T = i.numel();
  auto dw = torch::empty({V, D}, g.options());
  const int64_t n = fw_embed_grad_workspace(T, V, D);
  auto ws = bytes(n, g);
  ok(fw_embed_grad(code(g), i.data_ptr<int64_t>(), T, g.data_ptr(), ld_of(g), V, D, (float)scale, padding,
                   dw.data_ptr(), ws.data_ptr(), n, status_of(status, g), stream()),
     "fw_embed_grad");
  return dw;
}

// ---------------------------------------------------------------- norm
void check_norm(const Tensor& x, const OptTensor& residual, const Tensor& weight) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && is_float(x), "x must be a 2-D float32, bfloat16 or float16 CUDA tensor");
  TORCH_CHECK(weight.device() == x.device() && weight.dim() == 1 && weight.size(0) == x.size(1) &&
                  (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == torch::kFloat32),
              "weight must be [D] on x's device, in x's dtype or float32");
  if (residual.has_value())
    TORCH_CHECK(residual->device() == x.device() && residual->sizes() == x.sizes() &&
                    residual->scalar_type() == x.scalar_type(),
                "residual must match x");
}

// (y, rstd) or (y, rstd, sum)
std::vector<Tensor> rms_norm(Tensor x_, OptTensor residual, Tensor weight_, double eps) {
  check_norm(x_, residual, weight_);
  const c10::cuda::CUDAGuard guard(x_.device());
  auto x = rows_of(x_);
  auto w = weight_.contiguous();
  const int64_t rows = x.size(0), D = x.size(1);
  auto y = torch::empty({rows, D}, x.options());
  auto rstd = torch::empty({rows}, x.options().dtype(torch::kFloat32));
  std::vector<Tensor> out = {y, rstd};
  Tensor r;
  if (residual.has_value()) {
    r = rows_of(*residual);
    out.push_back(torch::empty({rows, D}, x.options()));
  }
  ok(fw_rms_norm(code(x), code(w), x.data_ptr(), ld_of(x), r.defined() ? r.data_ptr() : nullptr,
                 r.defined() ? ld_of(r) : D, w.data_ptr(), rows, D, (float)eps,
                 r.defined() ? out[2].data_ptr() : nullptr, D, y.data_ptr(), D, rstd.data_ptr<float>(), stream()),
     "fw_rms_norm");
  return out;
}

// (dx, dweight or nothing)
std::vector<Tensor> rms_norm_grad(Tensor dy_, Tensor sum_, OptTensor dsum, Tensor weight_, Tensor rstd,
                                  bool want_dweight) {
  check_norm(sum_, dsum, weight_);
  TORCH_CHECK(dy_.sizes() == sum_.sizes() && dy_.scalar_type() == sum_.scalar_type() && dy_.device() == sum_.device(),
              "dy must match the stored sum");
  const c10::cuda::CUDAGuard guard(sum_.device());
  auto dy = rows_of(dy_), s = rows_of(sum_);
  auto w = weight_.contiguous();
  const int64_t rows = s.size(0), D = s.size(1);
  TORCH_CHECK(rstd.is_cuda() && rstd.numel() == rows && rstd.scalar_type() == torch::kFloat32, "rstd must be [rows]");
  auto dx = torch::empty({rows, D}, s.options());
  Tensor o, parts, dw;
  if (dsum.has_value()) o = rows_of(*dsum);
  const int64_t n = fw_rms_norm_grad_parts(rows);
  if (want_dweight) {
    parts = torch::empty({n, D}, rstd.options());
    dw = torch::empty({D}, w.options());
  }
  ok(fw_rms_norm_grad(code(s), code(w), dy.data_ptr(), ld_of(dy), s.data_ptr(), ld_of(s),
                      o.defined() ? o.data_ptr() : nullptr, o.defined() ? ld_of(o) : D, w.data_ptr(),
                      rstd.data_ptr<float>(), rows, D, dx.data_ptr(), D,
                      want_dweight ? parts.data_ptr<float>() : nullptr, n, want_dweight ? dw.data_ptr() : nullptr,
                      stream()),
     "fw_rms_norm_grad");
  return want_dweight ? std::vector<Tensor>{dx, dw} : std::vector<Tensor>{dx};
}

// [rows, cols] int8 whose rows start on 16-byte boundaries
Tensor int8_rows(int64_t rows, int64_t cols, const Tensor& like) {
  return torch::empty({rows, (cols + 15) / 16 * 16}, like.options().dtype(torch::kInt8)).narrow(1, 0, cols);
}

// (q, scale) or (q, scale, sum)
std::vector<Tensor> rms_norm_int8(Tensor x_, OptTensor residual, Tensor weight_, double eps) {
  check_norm(x_, residual, weight_);
  const c10::cuda::CUDAGuard guard(x_.device());
  auto x = rows_of(x_);
  auto w = weight_.contiguous();
  const int64_t rows = x.size(0), D = x.size(1), ldq = (D + 15) / 16 * 16;
  auto q = int8_rows(rows, D, x);
  auto scale = torch::empty({rows}, x.options().dtype(torch::kFloat32));
  std::vector<Tensor> out = {q, scale};
  Tensor r;
  if (residual.has_value()) {
    r = rows_of(*residual);
    out.push_back(torch::empty({rows, D}, x.options()));
  }
  ok(fw_rms_norm_int8(code(x), code(w), x.data_ptr(), ld_of(x), r.defined() ? r.data_ptr() : nullptr,
                      r.defined() ? ld_of(r) : D, w.data_ptr(), rows, D, (float)eps,
                      r.defined() ? out[2].data_ptr() : nullptr, D, q.data_ptr<int8_t>(), ldq,
                      scale.data_ptr<float>(), stream()),
     "fw_rms_norm_int8");
  return out;
}

std::vector<Tensor> quantize_rows_int8(Tensor x_) {
  TORCH_CHECK(x_.is_cuda() && x_.dim() == 2 && is_float(x_) && x_.size(1) >= 1,
              "x must be a 2-D float32, bfloat16 or float16 CUDA tensor");
  const c10::cuda::CUDAGuard guard(x_.device());
  auto x = rows_of(x_);
  const int64_t rows = x.size(0), D = x.size(1);
  auto q = int8_rows(rows, D, x);
  auto scale = torch::empty({rows}, x.options().dtype(torch::kFloat32));
  ok(fw_quantize_rows_int8(code(x), x.data_ptr(), ld_of(x), rows, D, q.data_ptr<int8_t>(), (D + 15) / 16 * 16,
                           scale.data_ptr<float>(), stream()),
     "fw_quantize_rows_int8");
  return {q, scale};
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

Tensor int8_linear(Tensor q_, Tensor q_scale, Tensor w_, Tensor w_scale, torch::ScalarType out_dtype,
                   OptTensor status) {
  const c10::cuda::CUDAGuard guard(q_.device());
  auto q = aligned_rows(q_), w = aligned_rows(w_);
  auto qs = q_scale.contiguous(), ws = w_scale.contiguous();
  const int64_t T = q.size(0), K = q.size(1), N = w.size(0);
  auto out = torch::empty({T, N}, q.options().dtype(out_dtype));
  ok(fw_int8_linear(code(out_dtype), q.data_ptr<int8_t>(), int8_ld(q), qs.data_ptr<float>(), w.data_ptr<int8_t>(),
                    int8_ld(w), ws.data_ptr<float>(), T, N, K, out.data_ptr(), N, status_of(status, q), stream()),
     "fw_int8_linear");
  return out;
}

// ---------------------------------------------------------------- cross entropy
// (loss, state)
std::vector<Tensor> xent_forward(Tensor hidden_, Tensor weight_, Tensor target, int64_t ignore_index,
                                 int64_t reduction, OptTensor status) {
  const c10::cuda::CUDAGuard guard(hidden_.device());
  auto h = rows_of(hidden_), w = rows_of(weight_);
  auto y = target.contiguous();
  const int64_t B = h.size(0), D = h.size(1), V = w.size(0);
  auto f32 = h.options().dtype(torch::kFloat32);
  auto loss = reduction == FWB_REDUCE_NONE ? torch::empty({B}, f32) : torch::empty({}, f32);
  const int64_t ns = fw_xent_state_bytes(B, D, V, w.data_ptr(), ld_of(w)), nw = fw_xent_workspace(B, D, V, 0);
  auto state = bytes(ns, h), ws = bytes(nw, h);
  ok(fw_xent_forward(code(h), h.data_ptr(), ld_of(h), w.data_ptr(), ld_of(w), y.data_ptr<int64_t>(), B, D, V,
                     ignore_index, (int)reduction, loss.data_ptr<float>(), state.data_ptr(), ns, ws.data_ptr(), nw,
                     status_of(status, h), stream()),
     "fw_xent_forward");
  return {loss, state};
}

// (dhidden, dweight); an unwanted one is an empty tensor
std::vector<Tensor> xent_backward(Tensor weight_, int64_t B, Tensor grad_output, int64_t reduction, Tensor state,
                                  bool want_hidden, bool want_weight, OptTensor status) {
  const c10::cuda::CUDAGuard guard(weight_.device());
  auto w = rows_of(weight_);
  auto go = grad_output.to(torch::kFloat32).contiguous();
  const int64_t V = w.size(0), D = w.size(1);
  auto dh = want_hidden ? torch::empty({B, D}, w.options()) : Tensor();
  auto dw = want_weight ? torch::empty({V, D}, w.options()) : Tensor();
  const int64_t nw = fw_xent_workspace(B, D, V, 1);
  auto ws = bytes(nw, w);
  ok(fw_xent_backward(code(w), w.data_ptr(), ld_of(w), B, D, V, (int)reduction, go.data_ptr<float>(), state.data_ptr(),
                      state.numel(), ws.data_ptr(), nw, want_hidden ? dh.data_ptr() : nullptr,
                      want_weight ? dw.data_ptr() : nullptr, status_of(status, w), stream()),
     "fw_xent_backward");
  return {want_hidden ? dh : torch::empty({0}, w.options()), want_weight ? dw : torch::empty({0}, w.options())};
}

}  // namespace

void register_lm_operators(pybind11::module_& m) {
  m.def("embed_rows", &embed_rows, "rows of a table, scaled");
  m.def("embed_grad", &embed_grad, "gradient of embed_rows in the table, deterministic");
  m.def("rms_norm", &rms_norm, "(y, rstd[, x + residual])");
  m.def("rms_norm_grad", &rms_norm_grad, "(dx[, dweight])");
  m.def("rms_norm_int8", &rms_norm_int8, "(q, scale[, x + residual])");
  m.def("quantize_rows_int8", &quantize_rows_int8, "(q, scale)");
  m.def("int8_linear", [](Tensor q, Tensor qs, Tensor w, Tensor ws, py::object dtype, OptTensor status) {
    return int8_linear(q, qs, w, ws, reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type, status);
  }, "8-bit output layer");
  m.def("xent_forward", &xent_forward, "(loss, state)");
  m.def("xent_backward", &xent_backward, "(dhidden, dweight)");
}
