// Shared by the C++ calls over the C ABI (sequence_ext.cpp, projection_ext.cpp):
// arguments that may be None, pointers and streams, checks, autograd's states.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <optional>
#include <tuple>
#include <vector>

#include "cpab_b200.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// An argument that may be None; the code below it takes an undefined tensor.
using MaybeTensor = std::optional<Tensor>;
[[maybe_unused]] Tensor given(const MaybeTensor &t) { return t.has_value() ? *t : Tensor(); }

[[maybe_unused]] void check(int status) {
  TORCH_CHECK(status == 0, "libcpab_b200: ", cpab_b200_last_error());
}

[[maybe_unused]] cpab_stream_t stream_of(const Tensor &t) {
  return reinterpret_cast<cpab_stream_t>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

[[maybe_unused]] const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
[[maybe_unused]] void *ptr_mut(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
[[maybe_unused]] const float *fptr(const Tensor &t) { return static_cast<const float *>(ptr(t)); }
[[maybe_unused]] float *fptr_mut(const Tensor &t) { return static_cast<float *>(ptr_mut(t)); }

[[maybe_unused]] int dtype_of(const Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case at::kFloat: return CPAB_F32;
    case at::kHalf: return CPAB_F16;
    case at::kBFloat16: return CPAB_BF16;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  }
}

[[maybe_unused]] void require(const Tensor &t, const Tensor &like, at::ScalarType dtype, at::IntArrayRef shape, const char *name) {
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", x on ", like.device());
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}

// Counts a write through a raw pointer as torch's own operations count theirs, so
// that a backward through the old value raises (an inference tensor has no count).
[[maybe_unused]] void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// No gradient of these gradients: refuse instead of treating them as constants.
[[maybe_unused]] void once(const char *name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " can be differentiated once only (create_graph=True)");
}

// Whether a forward-mode derivative flows into one of ts.
[[maybe_unused]] bool has_tangent(std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) return true;
  return false;
}

// Whether the call has to go through its node, which refuses forward mode.
[[maybe_unused]] bool needs_grad(std::initializer_list<const Tensor *> ts) {
  if (has_tangent(ts)) return true;
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

[[maybe_unused]] Tensor channels_adjacent(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// t [..., D] as rows of adjacent columns.
[[maybe_unused]] Tensor rows_of(const Tensor &t) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)});
  return channels_adjacent(r);
}

// Element i of a Python list of tensors (null where it is None and `maybe`),
// read in place: a step's lists hold every tensor of a network.
[[maybe_unused]] const Tensor *item(const pybind11::list &list, size_t i, const char *name, bool maybe = false) {
  PyObject *o = PyList_GET_ITEM(list.ptr(), (Py_ssize_t)i);
  if (maybe && o == Py_None) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " ", i, " is no tensor");
  return &THPVariable_Unpack(o);
}

}  // namespace
