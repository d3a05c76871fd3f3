// Helpers shared by the translation units of custom_ops_lib.
#pragma once

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>

#include "../../../include/spmm_mi355x.h"

inline bool is_gpu(const at::Tensor& tensor) { return tensor.device().is_cuda(); }
#define TORCH_CHECK_GPU(tensor) \
  TORCH_CHECK(is_gpu(tensor), #tensor " must be a GPU tensor (MI355X build; reference: NPU tensor)")


inline int32_t index_type_of(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kInt) return SPMM_INDEX_I32;
  if (t.scalar_type() == at::kLong) return SPMM_INDEX_I64;
  TORCH_CHECK(false, name, " must be an int32 or int64 tensor, but got ", t.scalar_type());
  return -1;
}

// Maps a library status to the exception type the reference raises for the
// same condition (pybind11 turns these into ValueError / IndexError /
// OverflowError / RuntimeError).
inline void raise_status(spmm_status st, const char* what) {
  if (st == SPMM_OK) return;
  const std::string msg = std::string(what) + ": " + spmm_last_error();
  switch (st) {
    case SPMM_ERR_INVALID_ARGUMENT: throw std::invalid_argument(msg);
    case SPMM_ERR_OUT_OF_RANGE: throw std::out_of_range(msg);
    case SPMM_ERR_OVERFLOW: throw std::overflow_error(msg);
    default: TORCH_CHECK(false, msg);
  }
}

inline spmm_stream current_stream(const at::Tensor& t) {
  return reinterpret_cast<spmm_stream>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline at::Tensor workspace(const at::Tensor& like, size_t bytes) {
  return at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, like.options().dtype(at::kByte));
}


// Registers the dense operators (dense_ops.cpp) with the Python module.
void bind_dense_ops(pybind11::module_& m);
// And the operators around a layer of experts (expert_ops.cpp).
void bind_expert_ops(pybind11::module_& m);
