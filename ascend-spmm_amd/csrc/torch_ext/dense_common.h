// Helpers of the differentiable operators over FP16, BF16 and FP32 tensors.
#pragma once

#include "ext_common.h"

#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

inline int32_t dense_type_of(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kHalf: return SPMM_VALUE_F16;
    case at::kBFloat16: return SPMM_VALUE_BF16;
    case at::kFloat: return SPMM_VALUE_F32;
    default: TORCH_CHECK(false, op, " supports only FP16, BF16 and FP32 tensors, but got ", t.scalar_type());
  }
  return -1;
}

// `t` as rows of its last dimension: a view where its rows are contiguous and
// evenly apart, else a copy.
inline at::Tensor as_rows(const at::Tensor& t) {
  const int64_t width = t.size(-1);
  if (t.dim() == 2 && t.numel() == 0) return t;
  if (t.dim() == 2 && (t.stride(1) == 1 || width == 1) && (t.stride(0) >= width || t.size(0) <= 1)) return t;
  return t.contiguous().view({t.numel() / width, width});
}

inline int64_t row_stride(const at::Tensor& rows) {
  return rows.size(0) > 1 && rows.numel() > 0 ? rows.stride(0) : rows.size(1);
}

inline bool wants_grad(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
inline bool wants_grad(const c10::optional<at::Tensor>& t) { return t.has_value() && wants_grad(*t); }

// Forward-mode derivatives are refused: the kernels would drop them.
inline void check_no_tangent(const at::Tensor& t, const char* op) {
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), op,
              ": forward-mode derivatives are not supported");
}
