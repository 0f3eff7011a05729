// Helpers of the binding files whose entry points are differentiable operators: Python's own error
// types, rows of a tensor, and what their C++ autograd nodes share.
#pragma once
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

namespace pca {

#define PCA_VALUE(cond, ...) \
  if (!(cond)) throw py::value_error(c10::str(__VA_ARGS__))
#define PCA_TYPE(cond, ...) \
  if (!(cond)) throw py::type_error(c10::str(__VA_ARGS__))

inline hipStream_t cur_stream() { return c10::hip::getCurrentHIPStream().stream(); }

// [..., n] as [rows][n] whose rows are contiguous in themselves, at any stride
inline at::Tensor rows_of(const at::Tensor& x) {
  auto r = x.dim() == 2 ? x : x.reshape({x.numel() / std::max<int64_t>(x.size(-1), 1), x.size(-1)});
  if ((r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < 0)) r = r.contiguous();
  return r;
}

// The nodes' gradients are not differentiable themselves: under create_graph they carry an error
// that a second derivative runs into (never a silent zero).
inline void once_differentiable(std::vector<at::Tensor>& grads, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  for (auto& g : grads)
    if (g.defined()) {
      auto node = std::make_shared<torch::autograd::DelayedError>(
          std::string(what) + " is differentiable once only", 1);
      g = (*node)({g.detach().requires_grad_(true)})[0];
    }
}

// No node here has a forward-mode derivative, and a dual tensor need not require grad: refused, never a
// result without its tangent.
inline void no_tangent(const at::Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), what,
                              " has no forward-mode derivative");
}

// debug mode: an asynchronous fault or launch error is raised at the operator that caused it
inline void debug_check(bool debug, const char* what) {
  if (!debug) return;
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = hipDeviceSynchronize();
  TORCH_CHECK(e == hipSuccess, "pytorch_cifar_amd ", what, ": ", hipGetErrorString(e));
}

// keeps a tensor of ones that a caller seeds backward passes with: nodes recognise it by address
bool is_unit_seed(const at::Tensor& g);

}  // namespace pca
