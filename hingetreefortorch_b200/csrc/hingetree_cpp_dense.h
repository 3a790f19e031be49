// What the operators on dense matrices (hingetree_cpp_dense.cpp, hingetree_cpp_answers.cpp) share.
#pragma once

#include "hingetree_cpp_ops.h"

namespace htx {

using OptionalTensor = std::optional<torch::Tensor>;

inline torch::Tensor given(const OptionalTensor &t) { return t.has_value() ? *t : torch::Tensor(); }
inline OptionalTensor optional(const torch::Tensor &t) { return t.defined() ? OptionalTensor(t) : std::nullopt; }
inline const void *pointer(const torch::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

inline void check_types(const torch::Tensor &x, std::initializer_list<const torch::Tensor *> others) {
  if (x.scalar_type() != torch::kFloat32 && x.scalar_type() != torch::kBFloat16 && x.scalar_type() != torch::kFloat16)
    bad_argument("Error: Unsupported data type. Only torch.float32, torch.bfloat16 and torch.float16 are supported.");
  for (const torch::Tensor *t : others) {
    if (!t->defined()) continue;
    if (t->scalar_type() != x.scalar_type()) bad_argument("Error: x, the weights and the biases are expected to have the same type.");
    if (t->device() != x.device()) bad_argument("Error: All tensors are expected to be on the same device.");
  }
}
// Rows of contiguous features, the first on 16 bytes; differentiable.
inline torch::Tensor as_rows(const torch::Tensor &x) {
  torch::Tensor rows = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  const bool contiguous = rows.is_contiguous();
  if (!contiguous && (rows.stride(1) != 1 || rows.stride(0) < rows.size(1))) rows = rows.contiguous();
  if (reinterpret_cast<uintptr_t>(rows.const_data_ptr()) % 16 != 0) rows = rows.clone(at::MemoryFormat::Contiguous);
  return rows;
}
inline torch::Tensor as_whole(const torch::Tensor &t) {
  if (!t.defined()) return t;
  const torch::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 != 0 ? c.clone(at::MemoryFormat::Contiguous) : c;
}

inline int type_code(const torch::Tensor &t) {
  return t.scalar_type() == torch::kFloat32 ? HT_DTYPE_F32 : t.scalar_type() == torch::kBFloat16 ? HT_DTYPE_BF16 : HT_DTYPE_F16;
}

}  // namespace htx
