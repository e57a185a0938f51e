// Torch front of the operators that score tokens: checks, outputs, the current
// stream and the autograd nodes, as in fw_torch_lm.cpp.
#include "fw_torch_lm.h"

#include <cmath>

namespace {

// ---------------------------------------------------------------- log probabilities from logits
struct Scores {
  Tensor logp, entropy, top_logp, top_ids, state;
};

Scores score_forward(const Tensor& logits, const Tensor& tokens, int64_t k, double temperature, int64_t ignore_index,
                     const OptTensor& status, bool keep) {
  const c10::cuda::CUDAGuard guard(logits.device());
  auto z = rows_2d(logits);
  auto y = tokens.contiguous();
  const int64_t B = z.size(0), V = z.size(1);
  Scores out;
  out.logp = f32(tokens.sizes(), z);
  out.entropy = f32(tokens.sizes(), z);
  if (k > 0) {
    c10::SmallVector<int64_t, 6> shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(k);
    out.top_logp = f32(shape, z);
    out.top_ids = at::empty(shape, z.options().dtype(torch::kLong));
  }
  if (keep) out.state = f32({B, 4}, z);
  ok(fw_token_log_probs(code(z), z.data_ptr(), ld_of(z), y.data_ptr<int64_t>(), B, V, (float)(1.0 / temperature),
                        ignore_index, (int)k, out.logp.data_ptr<float>(), out.entropy.data_ptr<float>(),
                        k > 0 ? out.top_logp.data_ptr<float>() : nullptr,
                        k > 0 ? out.top_ids.data_ptr<int64_t>() : nullptr,
                        keep ? out.state.data_ptr<float>() : nullptr, status_of(status, z), stream()),
     "fw_token_log_probs");
  return out;
}

Tensor upstream(const Tensor& g) { return g.defined() ? g.detach().contiguous() : g; }

const float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t k,
                               double temperature, int64_t ignore_index, const OptTensor& status) {
    ctx->set_materialize_grads(false);
    auto s = score_forward(logits, tokens, k, temperature, ignore_index, status, true);
    ctx->save_for_backward({logits, s.state});
    ctx->saved_data["a"] = c10::IValue(temperature);
    if (k == 0) return {s.logp, s.entropy};
    ctx->mark_non_differentiable({s.top_logp, s.top_ids});
    return {s.logp, s.entropy, s.top_logp, s.top_ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    auto z = rows_2d(saved[0].detach());
    auto state = saved[1].contiguous();
    const Tensor dlogp = upstream(g[0]), dentropy = upstream(g[1]);
    const int64_t B = z.size(0), V = z.size(1);
    auto grad = at::empty(saved[0].sizes(), z.options());
    ok(fw_token_log_probs_grad(code(z), z.data_ptr(), ld_of(z), B, V, (float)(1.0 / ctx->saved_data["a"].toDouble()),
                               state.data_ptr<float>(), floats(dlogp), floats(dentropy), grad.data_ptr(), V, stream()),
       "fw_token_log_probs_grad");
    return once({grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

py::object token_log_probs(const Tensor& logits, const Tensor& tokens, int64_t k, double temperature,
                           int64_t ignore_index, const OptTensor& status) {
  type_check(logits.is_cuda(), "token_log_probs: logits must be a CUDA tensor (this build has no CPU path)");
  type_check(logits.dim() >= 1 && is_float(logits) && logits.size(-1) >= 1,
             "token_log_probs: logits must be a float32, bfloat16 or float16 tensor [..., V]");
  type_check(tokens.scalar_type() == torch::kLong, "token_log_probs: tokens must be an int64 tensor");
  value_check(tokens.device() == logits.device(), "token_log_probs: tokens must be on the logits' device");
  value_check(tokens.sizes() == logits.sizes().slice(0, logits.dim() - 1),
              "token_log_probs: tokens must have the logits' leading shape");
  value_check(k >= 0 && k <= FWB_TOP_MAX && k <= logits.size(-1),
              "token_log_probs: top_k must be between 0 and 32, and at most V");
  value_check(temperature > 0.0 && std::isfinite((float)temperature) && std::isfinite((float)(1.0 / temperature)) &&
                  (float)(1.0 / temperature) > 0.0f,
              "token_log_probs: temperature must be positive and finite, and so must its reciprocal");
  no_tangent(logits, "token_log_probs");
  if (at::GradMode::is_enabled() && recording(logits)) {
    auto out = TokenLogProbs::apply(logits, tokens, k, temperature, ignore_index, status);
    if (k == 0) return py::make_tuple(out[0], out[1]);
    return py::make_tuple(out[0], out[1], out[2], out[3]);
  }
  auto s = score_forward(logits, tokens, k, temperature, ignore_index, status, false);
  if (k == 0) return py::make_tuple(s.logp, s.entropy);
  return py::make_tuple(s.logp, s.entropy, s.top_logp, s.top_ids);
}

}  // namespace

void register_score_operators(pybind11::module_& m) {
  m.def("token_log_probs", &token_log_probs,
        "(logp, entropy[, top_logp, top_ids]) from logits (differentiable in the first two)");
}
