// Helpers shared by the torch fronts of the language-model operators
// (fw_torch_lm.cpp, fw_torch_score.cpp): argument checks, layouts, workspaces,
// status words and refusals of the autograd nodes.  Every file has its own copy.
#pragma once

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

inline void ok(int rc, const char* what) { TORCH_CHECK(rc == FWB_OK, what, " failed: ", fw_error_string(rc)); }

inline void type_check(bool cond, const char* what) {
  if (!cond) throw py::type_error(what);
}

inline void value_check(bool cond, const char* what) {
  if (!cond) throw py::value_error(what);
}

inline void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

inline bool is_float(const Tensor& t) {
  return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kHalf;
}

inline int code(torch::ScalarType t) {
  return t == torch::kBFloat16 ? FWB_DTYPE_BF16 : t == torch::kHalf ? FWB_DTYPE_F16 : FWB_DTYPE_F32;
}

inline int code(const Tensor& t) { return code(t.scalar_type()); }

// Unit column stride and rows that do not overlap; copies otherwise.
inline Tensor rows_of(const Tensor& t) {
  return (t.size(1) == 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}

// [..., D] as rows of D.
inline Tensor rows_2d(const Tensor& t) { return rows_of(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }

inline int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

inline int32_t* status_of(const OptTensor& s, const Tensor& like) {
  if (!s.has_value()) return nullptr;
  TORCH_CHECK(s->device() == like.device() && s->scalar_type() == torch::kInt32 && s->numel() >= 1 &&
                  s->is_contiguous(),
              "status must be an int32 tensor on the inputs' device");
  return s->data_ptr<int32_t>();
}

// The status word of a later backward.  Not a saved variable: clearing it in
// between is its normal use.
inline void keep_status(AutogradContext* ctx, const OptTensor& s) {
  if (s.has_value()) ctx->saved_data["status"] = c10::IValue(*s);
}

inline OptTensor kept_status(AutogradContext* ctx) {
  const auto it = ctx->saved_data.find("status");
  return it == ctx->saved_data.end() ? OptTensor() : OptTensor(it->second.toTensor());
}

inline Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({n > 0 ? n : 1}, like.options().dtype(torch::kUInt8));
}

inline Tensor f32(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(torch::kFloat32)); }

inline bool recording(const Tensor& t) { return t.requires_grad(); }

// A result without a tangent would drop the operand's silently, whatever the grad mode.
inline void no_tangent(const Tensor& t, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), op, ": forward-mode differentiation is not implemented");
}

// The gradients have none of their own: a second derivative raises.
inline variable_list once(variable_list grads) {
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

}  // namespace
