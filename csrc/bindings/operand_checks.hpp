// Checks of operands that the bindings of the forward-only and the packed operators share.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>

#include "../core/errors.hpp"
#include "../ops/serving.hpp"

namespace mccl {

namespace {

cudaStream_t stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
// at::empty on `like`'s device without the dispatcher: half a microsecond of the five that a small call takes.
at::Tensor empty_on(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}
void check_launch(cudaError_t rc, const char* what) {
  MCCL_CHECK_T(rc == cudaSuccess, CudaError, what << " failed: " << cudaGetErrorString(rc));
}
void need_on(const at::Tensor& t, const at::Tensor& like, const char* what) {
  MCCL_CHECK_TENSOR(t.defined() && t.is_cuda(), what << ": expected a CUDA tensor");
  MCCL_CHECK_TENSOR(t.device() == like.device(), what << ": on another device than the other operands");
}
void need_forward_only(const at::Tensor& t, const char* what) {
  MCCL_CHECK_TENSOR(!(at::GradMode::is_enabled() && t.requires_grad()), what << ": has no backward pass; call it under torch.no_grad()");
  MCCL_CHECK_TENSOR(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined()), what << ": has no forward-mode derivative; a tangent would be lost");
}
ops::Half16 half16(const at::Tensor& t, const char* what) {
  MCCL_CHECK_TENSOR(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf,
                    what << ": expected bf16 or fp16, got " << c10::toString(t.scalar_type()));
  return t.scalar_type() == at::kBFloat16 ? ops::Half16::bf16 : ops::Half16::fp16;
}
int as_int(int64_t v, const char* what) {
  MCCL_CHECK_TENSOR(v >= 0 && v <= std::numeric_limits<int>::max(), what << ": size out of range");
  return static_cast<int>(v);
}
// Whether 16-byte accesses of 16-bit elements stay on their boundaries: unit inner stride, the others multiples of 8 where they are used.
bool vector_rows(const at::Tensor& t) {
  if (t.numel() == 0) return true;
  const int64_t d = t.dim();
  if (t.size(d - 1) > 1 && t.stride(d - 1) != 1) return false;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < d; ++i)
    if (t.size(i) > 1 && t.stride(i) % 8 != 0) return false;
  return true;
}
// Whether a tensor has elements that are one place in memory (a dimension that was expanded), and whether two of the same sizes are the same places, all or, where
// both are without gaps, some.  (at::get_overlap_status and its like cost a small call a quarter of a microsecond.)
bool repeated(const at::Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return true;
  return false;
}
bool same_memory(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0) return false;
  const uintptr_t at_a = reinterpret_cast<uintptr_t>(a.data_ptr()), at_b = reinterpret_cast<uintptr_t>(b.data_ptr());
  const uintptr_t apart = at_a > at_b ? at_a - at_b : at_b - at_a;
  return apart == 0 || (apart < static_cast<uintptr_t>(a.nbytes()) && a.is_non_overlapping_and_dense() && b.is_non_overlapping_and_dense());
}
const int* need_int32(const at::Tensor& t, const at::Tensor& like, int64_t count, const char* what) {
  need_on(t, like, what);
  MCCL_CHECK_TENSOR(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), what << ": expected a contiguous one-dimensional int32 tensor");
  MCCL_CHECK_TENSOR(t.numel() == count, what << ": expected " << count << " elements, got " << t.numel());
  return t.data_ptr<int>();
}
ops::TokenView tokens_of(const at::Tensor& t, const char* what) {
  MCCL_CHECK_TENSOR(t.dim() == 3, what << ": expected [tokens, heads, head_dim]");
  MCCL_CHECK_TENSOR(vector_rows(t), what << ": needs a contiguous head_dim, strides that are multiples of 8 and a 16-byte aligned base");
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

}  // namespace

}  // namespace mccl
