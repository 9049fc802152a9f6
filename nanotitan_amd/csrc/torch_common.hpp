// What the torch bindings share: types, checks, streams and workspaces.
#pragma once

#include <torch/extension.h>

#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>

#include <tuple>

#include "nanotitan_moe.h"

namespace {

using torch::Tensor;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NT_F32;
    case at::kDouble: return NT_F64;
    case at::kHalf: return NT_F16;
    case at::kBFloat16: return NT_BF16;
    default:
      TORCH_CHECK(false, "unsupported dtype ", t,
                  " (expected float32, float64, float16 or bfloat16)");
  }
  return -1;
}
int dtype_code(const Tensor& t) { return dtype_code(t.scalar_type()); }

at::ScalarType scalar_of(int code) {
  switch (code) {
    case NT_F32: return at::kFloat;
    case NT_F64: return at::kDouble;
    case NT_F16: return at::kHalf;
    default: return at::kBFloat16;
  }
}

void check_status(int st, const char* what) {
  TORCH_CHECK(st == NT_OK, what, ": ", nt_strerror(st));
}

void check_device(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
}

void check_i32(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  check_device(t, name);
}

void check_f32(const Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kFloat, name, " must be float32");
  check_device(t, name);
}

// Every tensor of one call lives on the device of the first.
void check_same_device(const Tensor& first, std::initializer_list<const Tensor*> rest) {
  for (const Tensor* t : rest)
    TORCH_CHECK(t->device() == first.device(), "all tensors must be on the same device (",
                first.device(), " vs ", t->device(), ")");
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

Tensor workspace(const Tensor& like, size_t bytes) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

const float* f32_or_null(const c10::optional<Tensor>& t) {
  return t ? t->data_ptr<float>() : nullptr;
}
const void* ptr_or_null(const c10::optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }
void* out_or_null(const c10::optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

// Operators without a forward-mode derivative refuse dual tensors, in every grad
// mode: a kernel's output has no tangent, which torch would read as zero.
void refuse_tangents(std::initializer_list<const c10::optional<Tensor>*> ts, const char* what) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const auto* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(
        !t->has_value() || !(*t)->defined() || !(*t)->_fw_grad(/*level=*/0).defined(), what,
        " has no forward-mode derivative");
}

}  // namespace
