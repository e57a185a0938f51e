// Torch front of the operators that score tokens and end a training step: checks, outputs, the current
// stream and the autograd nodes, as in fw_torch_lm.cpp.
#include "fw_torch_lm.h"

#include <ATen/MemoryOverlap.h>

#include <algorithm>
#include <cmath>
#include <string>

namespace {

// A temperature whose reciprocal fp32 holds, with some room above.
bool fits(double temperature) {
  return temperature > 0.0 && std::isfinite((float)temperature) && std::isfinite(1.5f * (float)(1.0 / temperature)) &&
         (float)(1.0 / temperature) > 0.0f;
}

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
  value_check(fits(temperature),
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

// ---------------------------------------------------------------- log probabilities of an output layer
struct HeadScores {
  Tensor logp, entropy, state;
};

HeadScores head_forward(const Tensor& hidden, const Tensor& weight, const Tensor& tokens, double temperature,
                        int64_t ignore_index, const OptTensor& status) {
  const c10::cuda::CUDAGuard guard(hidden.device());
  auto h = rows_of(hidden), w = rows_of(weight);
  auto y = tokens.contiguous();
  const int64_t B = h.size(0), D = h.size(1), V = w.size(0);
  HeadScores out;
  out.logp = f32({B}, h);
  out.entropy = f32({B}, h);
  const int64_t ns = fw_lm_head_log_probs_state(B, D, V, w.data_ptr(), ld_of(w));
  const int64_t nw = fw_lm_head_log_probs_workspace(B, D, V, 0);
  out.state = bytes(ns, h);
  auto ws = bytes(nw, h);
  ok(fw_lm_head_log_probs(code(h), h.data_ptr(), ld_of(h), w.data_ptr(), ld_of(w), y.data_ptr<int64_t>(), B, D, V,
                          (float)(1.0 / temperature), ignore_index, out.logp.data_ptr<float>(),
                          out.entropy.data_ptr<float>(), out.state.data_ptr(), ns, ws.data_ptr(), nw,
                          status_of(status, h), stream()),
     "fw_lm_head_log_probs");
  return out;
}

struct LmHeadLogProbs : torch::autograd::Function<LmHeadLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& tokens,
                               double temperature, int64_t ignore_index, const OptTensor& status) {
    ctx->set_materialize_grads(false);
    auto s = head_forward(hidden, weight, tokens, temperature, ignore_index, status);
    ctx->save_for_backward({weight, s.state});
    keep_status(ctx, status);
    ctx->saved_data["rows"] = c10::IValue(hidden.size(0));
    ctx->saved_data["temperature"] = c10::IValue(temperature);
    return {s.logp, s.entropy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    const c10::cuda::CUDAGuard guard(saved[0].device());
    auto w = rows_of(saved[0].detach());
    const Tensor& state = saved[1];
    const Tensor dlogp = upstream(g[0]), dentropy = upstream(g[1]);
    const bool want_h = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const int64_t B = ctx->saved_data["rows"].toInt(), V = w.size(0), D = w.size(1);
    // A hook may have restored the weight off the 16-byte boundaries it was saved on; the state has no copy of it then.
    if (fw_lm_head_log_probs_state(B, D, V, w.data_ptr(), ld_of(w)) > state.numel()) {
      auto c = at::empty({V, (D + 7) / 8 * 8}, w.options()).narrow(1, 0, D);
      c.copy_(w);
      w = c;
    }
    Tensor dh, dw;
    if (want_h) dh = at::empty({B, D}, w.options());
    if (want_w) dw = at::empty({V, D}, w.options());
    const int64_t nw = fw_lm_head_log_probs_workspace(B, D, V, 1);
    auto ws = bytes(nw, w);
    const OptTensor status = kept_status(ctx);
    ok(fw_lm_head_log_probs_grad(code(w), w.data_ptr(), ld_of(w), B, D, V,
                                 (float)(1.0 / ctx->saved_data["temperature"].toDouble()), floats(dlogp),
                                 floats(dentropy), state.data_ptr(), state.numel(), ws.data_ptr(), nw,
                                 want_h ? dh.data_ptr() : nullptr, want_w ? dw.data_ptr() : nullptr,
                                 status_of(status, w), stream()),
       "fw_lm_head_log_probs_grad");
    return once({dh, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

py::tuple lm_head_log_probs(const Tensor& hidden, const Tensor& weight, const Tensor& tokens, double temperature,
                            int64_t ignore_index, const OptTensor& status) {
  type_check(hidden.is_cuda() && weight.is_cuda(),
             "lm_head_log_probs: hidden and weight must be CUDA tensors (this build has no CPU path)");
  type_check(hidden.dim() == 2 && weight.dim() == 2 && weight.numel() > 0,
             "lm_head_log_probs: hidden [B, D] and weight [V, D] must be matrices");
  type_check(hidden.scalar_type() == weight.scalar_type() &&
                 (hidden.scalar_type() == torch::kBFloat16 || hidden.scalar_type() == torch::kHalf),
             "lm_head_log_probs: hidden and weight must both be bfloat16 or both float16");
  value_check(hidden.size(1) == weight.size(1), "lm_head_log_probs: hidden and weight disagree on D");
  type_check(tokens.scalar_type() == torch::kLong, "lm_head_log_probs: tokens must be int64");
  value_check(tokens.dim() == 1 && tokens.size(0) == hidden.size(0), "lm_head_log_probs: tokens must have shape [B]");
  value_check(weight.device() == hidden.device() && tokens.device() == hidden.device(),
              "lm_head_log_probs: hidden, weight and tokens must be on one device");
  value_check(fits(temperature), "lm_head_log_probs: temperature must be positive and finite, and so must its reciprocal");
  no_tangent(hidden, "lm_head_log_probs");
  no_tangent(weight, "lm_head_log_probs");
  if (at::GradMode::is_enabled() && (recording(hidden) || recording(weight))) {
    auto out = LmHeadLogProbs::apply(hidden, weight, tokens, temperature, ignore_index, status);
    return py::make_tuple(out[0], out[1]);
  }
  auto s = head_forward(hidden, weight, tokens, temperature, ignore_index, status);
  return py::make_tuple(s.logp, s.entropy);
}

// ---------------------------------------------------------------- gradient norm and clipping
struct List {
  std::vector<Tensor> held;  // copies that the pointers are to
  std::vector<const void*> in;
  std::vector<void*> out;
  std::vector<int64_t> numel;
  std::vector<int32_t> types, out_types;
  explicit List(size_t n) {
    in.reserve(n);
    out.reserve(n);
    numel.reserve(n);
    types.reserve(n);
    out_types.reserve(n);
  }
};

bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

[[noreturn]] void refuse_type(const char* op, const char* what) { throw py::type_error(std::string(op) + ": " + what); }

[[noreturn]] void refuse(const char* op, const char* what) { throw py::value_error(std::string(op) + ": " + what); }

void check_grads(const std::vector<Tensor>& grads, const char* op) {
  if (grads.empty()) refuse(op, "no tensors");
  const auto device = grads[0].device();
  for (const auto& t : grads) {
    if (!t.is_cuda()) refuse_type(op, "gradients must be CUDA tensors (this build has no CPU path)");
    if (t.layout() != torch::kStrided || !is_float(t))
      refuse_type(op, "gradients must be dense float32, bfloat16 or float16 tensors");
    if (t.device() != device) refuse(op, "gradients must be on one device");
    no_tangent(t, op);
  }
}

void check_max_norm(double max_norm) {
  value_check(max_norm >= 0.0 && !std::isnan(max_norm), "clip_grad_norm_: max_norm must not be negative");
}

Tensor norm_workspace(const std::vector<Tensor>& grads, int64_t* n) {
  *n = fw_grad_norm_workspace((int64_t)grads.size());
  return bytes(*n, grads[0]);
}

Tensor grad_norm(const std::vector<Tensor>& grads, const OptTensor& status) {
  check_grads(grads, "grad_norm");
  for (const auto& t : grads)
    value_check(!(at::GradMode::is_enabled() && t.requires_grad()),
                "grad_norm: not differentiable; pass gradients (p.grad), or detach");
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(grads[0].device());
  List l(grads.size());
  for (const auto& t : grads) {
    const bool as_is = dense(t);
    if (!as_is) l.held.push_back(t.contiguous());
    l.in.push_back(as_is ? t.data_ptr() : l.held.back().data_ptr());
    l.numel.push_back(t.numel());
    l.types.push_back(code(t));
  }
  int64_t nw;
  auto ws = norm_workspace(grads, &nw);
  auto norm = f32({}, grads[0]);
  ok(fw_grad_norm((int64_t)grads.size(), l.in.data(), l.numel.data(), l.types.data(), ws.data_ptr(), nw,
                  norm.data_ptr<float>(), status_of(status, grads[0]), stream()),
     "fw_grad_norm");
  return norm;
}

// Written ranges must not overlap each other, nor a range that is read for another tensor.
void check_overlaps(const List& l) {
  struct Range {
    uintptr_t lo, hi;
    bool written;
  };
  std::vector<Range> ranges;
  const auto size = [](int32_t type) { return type == FWB_DTYPE_F32 ? 4 : 2; };
  bool sorted = true;
  const auto add = [&](const void* p, int64_t bytes, bool written) {
    const auto lo = reinterpret_cast<uintptr_t>(p);
    if (!ranges.empty() && ranges.back().lo > lo) sorted = false;
    ranges.push_back({lo, lo + (uintptr_t)bytes, written});
  };
  for (size_t i = 0; i < l.in.size(); ++i) {
    if (l.numel[i] == 0) continue;
    add(l.out[i], l.numel[i] * size(l.out_types[i]), true);
    if (l.in[i] != l.out[i] || l.types[i] != l.out_types[i]) add(l.in[i], l.numel[i] * size(l.types[i]), false);
  }
  if (!sorted) std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t written = 0, read = 0;  // ends of the ranges so far
  for (const auto& r : ranges) {
    value_check(r.lo >= written && (!r.written || r.lo >= read),
                "clip_grad_norm_: tensors that are written overlap others (the same tensor twice?)");
    (r.written ? written : read) = std::max(r.written ? written : read, r.hi);
  }
}

// A tensor's memory: `lo` and what dims [stride, size] reach from there, in bytes, elements of `size`.
struct Memory {
  int64_t lo, hi, size;
  c10::SmallVector<std::pair<int64_t, int64_t>, 4> dims;
  explicit Memory(const Tensor& t) : lo((int64_t)reinterpret_cast<uintptr_t>(t.data_ptr())), size((int64_t)t.element_size()) {
    if (dense(t)) {
      dims.push_back({size, t.numel()});
    } else {
      for (int64_t d = 0; d < t.dim(); ++d)
        if (t.size(d) > 1 && t.stride(d) > 0) dims.push_back({t.stride(d) * size, t.size(d)});
    }
    hi = lo + size;
    for (const auto& d : dims) hi += d.first * (d.second - 1);
  }
};

// Whether two tensors have a byte in common.  Their elements are at lo + sum of stride * i: looked for is a set of
// indices whose distance is under an element's size, from the largest stride down, where a stride that both have counts
// as one with their difference as index; of every index only those values are tried from which the smaller strides
// reach.  Interleaved views take a few steps; where strides have nothing to do with each other it may be very many, and
// tensors that are not told apart in 2^16 steps count as overlapping.
bool meet(const Memory& a, const Memory& b) {
  if (a.lo >= b.hi || b.lo >= a.hi) return false;
  struct Step {
    int64_t stride, least, most;  // of the index
    int64_t under, over;          // what the strides behind it add at least and at most
  };
  c10::SmallVector<Step, 8> steps;
  const auto add = [&](int64_t stride, int64_t least, int64_t most) {
    for (auto& s : steps)
      if (s.stride == stride) {
        s.least += least, s.most += most;
        return;
      }
    steps.push_back({stride, least, most, 0, 0});
  };
  for (const auto& d : a.dims) add(d.first, 0, d.second - 1);
  for (const auto& d : b.dims) add(d.first, 1 - d.second, 0);
  std::sort(steps.begin(), steps.end(), [](const Step& x, const Step& y) { return x.stride > y.stride; });
  for (size_t i = steps.size(); i-- > 1;) {
    steps[i - 1].under = steps[i].under + steps[i].stride * steps[i].least;
    steps[i - 1].over = steps[i].over + steps[i].stride * steps[i].most;
  }
  const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0 ? 1 : 0); };
  int left = 1 << 16;
  const auto search = [&](auto&& self, size_t i, int64_t at) -> bool {  // at: a's place less b's, so far
    if (i == steps.size()) return at > -a.size && at < b.size;
    const Step& s = steps[i];
    const int64_t first = std::max(s.least, -floor_div(at + s.over + a.size - 1, s.stride));
    const int64_t last = std::min(s.most, floor_div(b.size - 1 - at - s.under, s.stride));
    for (int64_t k = first; k <= last; ++k)
      if (--left <= 0 || self(self, i + 1, at + s.stride * k)) return true;
    return false;
  };
  return search(search, 0, a.lo - b.lo);
}

// The same for results that are copied to where they belong (`back`), by their own memory.
void check_copied(const std::vector<Tensor>& grads, const std::vector<Tensor>& dest, const std::vector<bool>& copied) {
  struct Range {
    Memory memory;
    size_t tensor;
    bool written, copied;
  };
  std::vector<Range> ranges;
  ranges.reserve(2 * grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    if (grads[i].numel() == 0) continue;
    ranges.push_back({Memory(dest[i]), i, true, (bool)copied[i]});
    if (!grads[i].is_same(dest[i])) ranges.push_back({Memory(grads[i]), i, false, false});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& x, const Range& y) { return x.memory.lo < y.memory.lo; });
  std::vector<const Range*> open;  // those that reach the present one's start
  for (const auto& r : ranges) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Range* o) { return o->memory.hi <= r.memory.lo; }), open.end());
    for (const Range* o : open)
      if (o->tensor != r.tensor && (o->copied || r.copied) && meet(o->memory, r.memory))
        refuse("clip_grad_norm_", "tensors that are written overlap others (the same tensor twice?)");
    open.push_back(&r);
  }
}

Tensor clip_grad_norm_(const std::vector<Tensor>& grads, double max_norm, const c10::optional<std::vector<Tensor>>& out,
                       const OptTensor& norm_in, const OptTensor& status) {
  check_grads(grads, "clip_grad_norm_");
  check_max_norm(max_norm);
  const auto& dest = out.has_value() ? *out : grads;
  value_check(dest.size() == grads.size(), "clip_grad_norm_: out must have a tensor for every gradient");
  for (size_t i = 0; i < dest.size(); ++i) {
    const auto& t = dest[i];
    value_check(!t.requires_grad(), "clip_grad_norm_: written tensors must not require grad (pass p.grad, not p)");
    if (!out.has_value()) continue;
    value_check(!(at::GradMode::is_enabled() && grads[i].requires_grad()),
                "clip_grad_norm_: not differentiable; pass gradients (p.grad), or detach");
    type_check(t.is_cuda() && t.layout() == torch::kStrided && is_float(t),
               "clip_grad_norm_: out must hold dense float32, bfloat16 or float16 CUDA tensors");
    value_check(t.device() == grads[0].device() && t.sizes() == grads[i].sizes(),
                "clip_grad_norm_: out must have the gradients' shapes and device");
  }
  if (norm_in.has_value())
    value_check(norm_in->device() == grads[0].device() && norm_in->scalar_type() == torch::kFloat32 && norm_in->numel() == 1,
                "clip_grad_norm_: norm must be one float32 value on the gradients' device");
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(grads[0].device());
  List l(grads.size());
  std::vector<std::pair<Tensor, Tensor>> back;  // results that are copied to where they belong
  std::vector<bool> copied(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) {
    const auto &g = grads[i], &d = dest[i];
    l.numel.push_back(g.numel());
    l.types.push_back(code(g));
    l.out_types.push_back(code(d));
    if (dense(g) && (!out.has_value() || (dense(d) && (d.strides() == g.strides() || (d.is_contiguous() && g.is_contiguous()))))) {
      l.in.push_back(g.data_ptr());
      l.out.push_back(d.data_ptr());
      continue;
    }
    const Tensor from = dense(g) ? g : g.contiguous();
    Tensor to = out.has_value() ? d : from;
    if (!dense(to) || (to.strides() != from.strides() && !(to.is_contiguous() && from.is_contiguous())))
      to = at::empty_strided(from.sizes(), from.strides(), d.options());  // an element is where it is in `from`
    if (!to.is_same(d)) {
      back.emplace_back(d, to);
      copied[i] = true;
    }
    l.held.push_back(from);
    l.held.push_back(to);
    l.in.push_back(from.data_ptr());
    l.out.push_back(to.data_ptr());
  }
  for (const auto& b : back) at::assert_no_internal_overlap(b.first);
  check_overlaps(l);
  if (!back.empty()) check_copied(grads, dest, copied);
  if (norm_in.has_value()) {  // every CTA reads it, while others have begun to write
    const Memory at(*norm_in);
    for (const auto& t : dest)
      value_check(t.numel() == 0 || !meet(at, Memory(t)), "clip_grad_norm_: norm must not lie in a tensor that is written");
  }
  int64_t nw = 0;
  Tensor ws, norm;
  if (norm_in.has_value()) {
    norm = *norm_in;
  } else {
    ws = norm_workspace(grads, &nw);
    norm = f32({}, grads[0]);
  }
  ok(fw_grad_clip((int64_t)grads.size(), l.in.data(), l.out.data(), l.numel.data(), l.types.data(), l.out_types.data(),
                  (float)max_norm, norm_in.has_value() ? norm.data_ptr<float>() : nullptr,
                  ws.defined() ? ws.data_ptr() : nullptr, nw, norm.data_ptr<float>(), status_of(status, grads[0]), stream()),
     "fw_grad_clip");
  for (const auto& b : back) b.first.copy_(b.second);
  for (const auto& t : dest)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void register_score_operators(pybind11::module_& m) {
  m.def("token_log_probs", &token_log_probs,
        "(logp, entropy[, top_logp, top_ids]) from logits (differentiable in the first two)");
  m.def("lm_head_log_probs", &lm_head_log_probs, "(logp, entropy) of an output layer (differentiable)");
  m.def("grad_norm", &grad_norm, "global norm of many tensors");
  m.def("clip_grad_norm_", &clip_grad_norm_, "gradients clipped to a global norm, in place or into others; the norm");
}
