// What the functs:: operators on GPU tensors share: checks of arguments, the stream of a device.
#pragma once
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include "../../../include/fxhip.h"

namespace functs {
namespace {
using at::Tensor;

#define FX_OK_OR_THROW(expr)                                             \
  do {                                                                   \
    int rc__ = (expr);                                                   \
    TORCH_CHECK(rc__ >= 0, "fxhip: ", fx_last_error(), " (", #expr, ")"); \
  } while (0)

void* streamOf(c10::Device dev) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream(); }
// (tensors made in inference mode carry no version)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void onGpu(const char* op, const Tensor& t, const char* name, c10::Device dev) {
  TORCH_CHECK(t.is_cuda(), op, " runs on the GPU only; ", name, " is a ", t.device(), " tensor");
  TORCH_CHECK(t.device() == dev, op, ": ", name, " is on ", t.device(), ", the others on ", dev);
}
void noGrad(const char* op, const Tensor& t, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), op, " has no backward pass: ", name, " requires a gradient");
  TORCH_CHECK(!t._fw_grad(0).defined(), op, " has no derivative: ", name, " carries a tangent");
}
int32_t sized(const char* op, int64_t n, const char* name) {
  TORCH_CHECK(n >= 0 && n <= INT32_MAX, op, ": ", name, " is out of range (", n, ")");
  return (int32_t)n;
}
Tensor ints(const char* op, const Tensor& t, const char* name, int64_t n, c10::Device dev) {
  onGpu(op, t, name, dev);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && (n < 0 || t.size(0) == n), op, ": ", name, " must be int32 [", n < 0 ? t.numel() : n,
              "], got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}
int dtypeOf(const char* op, at::ScalarType t, const char* name) {
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, op, ": ", name, " must be float32, float16 or bfloat16, got ", t);
  return t == at::kFloat ? FX_DT_F32 : t == at::kHalf ? FX_DT_F16 : FX_DT_BF16;
}
}  // namespace
}  // namespace functs
