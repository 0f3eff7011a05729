// Bindings of distill.hip: host checks, outputs from the caching allocator, launches on the
// current stream of the tensors' own device (no host sync, hipGraph-capturable).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <cmath>

#include "distill.h"

namespace pca {
namespace {

using at::Tensor;
using c10::optional;

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

int logit_type(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  switch (t.scalar_type()) {
    case at::kFloat: return LOGIT_F32;
    case at::kBFloat16: return LOGIT_BF16;
    case at::kHalf: return LOGIT_F16;
    default: TORCH_CHECK(false, name, " must be fp32, bf16 or fp16, got ", t.scalar_type());
  }
}

// [R][V] rows with any stride between them
int check_rows(const Tensor& z, const char* name) {
  const int type = logit_type(z, name);
  TORCH_CHECK(z.dim() == 2, name, " must be [rows][classes]");
  TORCH_CHECK(z.size(1) >= 1 && z.size(1) <= kDistillMaxClasses, name, " has ", z.size(1),
              " classes: 1 to ", kDistillMaxClasses, " are supported");
  TORCH_CHECK(z.size(0) < (int64_t(1) << 31), name, " has too many rows");
  TORCH_CHECK(z.size(1) == 1 || z.stride(1) == 1, name, ": the classes of a row must be contiguous");
  TORCH_CHECK(z.size(0) <= 1 || z.stride(0) >= 0, name, ": negative row stride");
  return type;
}

void same_device(const Tensor& a, const Tensor& b, const char* name) {
  TORCH_CHECK(b.is_cuda() && b.device() == a.device(), name, " must be on ", a.device());
}

void check_temp(double t) {
  TORCH_CHECK(std::isfinite(t) && t > 0, "temperature must be positive and finite, got ", t);
}

std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& z, int64_t k, double temperature) {
  const int type = check_rows(z, "logits");
  const int64_t R = z.size(0);
  const int V = (int)z.size(1);
  TORCH_CHECK(k >= 1 && k <= std::min(V, kDistillMaxK), "k must be 1 to ",
              std::min(V, kDistillMaxK), ", got ", k);
  check_temp(temperature);
  c10::OptionalDeviceGuard guard(at::device_of(z));
  auto values = at::empty({R, k}, z.options());
  auto indices = at::empty({R, k}, z.options().dtype(at::kInt));
  auto lse = at::empty({R}, z.options().dtype(at::kFloat));
  if (R)
    top_logits_launch(z.data_ptr(), type, z.stride(0), R, V, (int)k, temperature,
                      values.data_ptr(), indices.data_ptr<int32_t>(), lse.data_ptr<float>(),
                      stream());
  return {values, indices, lse};
}

// reduction 0: a loss a row, 1: mean over the rows, 2: sum
std::tuple<Tensor, Tensor> distill(const Tensor& z, const Tensor& values, const Tensor& indices,
                                   const optional<Tensor>& lse, const optional<Tensor>& target,
                                   double temperature, double alpha, bool tail, int reduction,
                                   int64_t ignore_index, bool want_grad) {
  DistillArgs a{};
  a.type = check_rows(z, "logits");
  a.R = z.size(0);
  a.V = (int)z.size(1);
  a.ld = z.stride(0);
  a.value_type = logit_type(values, "values");
  TORCH_CHECK(values.dim() == 2 && values.size(0) == a.R && indices.sizes() == values.sizes(),
              "values and indices must be [rows][k] with the logits' rows");
  TORCH_CHECK(values.size(1) >= 1 && values.size(1) <= kDistillMaxK, "k must be 1 to ",
              kDistillMaxK, ", got ", values.size(1));
  TORCH_CHECK(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong,
              "indices must be int32 or int64");
  TORCH_CHECK(values.is_contiguous() && indices.is_contiguous(),
              "values and indices must be contiguous");
  same_device(z, values, "values");
  same_device(z, indices, "indices");
  a.K = (int)values.size(1);
  a.index64 = indices.scalar_type() == at::kLong;
  a.values = values.data_ptr();
  a.indices = indices.data_ptr();
  a.tail = tail;
  if (tail) {
    TORCH_CHECK(lse.has_value() && lse->defined(), "tail needs the teacher's lse");
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->numel() == a.R,
                "lse must be contiguous fp32 of one value a row");
    same_device(z, *lse, "lse");
    a.lse = lse->data_ptr<float>();
  }
  if (target.has_value() && target->defined()) {
    TORCH_CHECK(target->scalar_type() == at::kLong && target->is_contiguous() &&
                    target->numel() == a.R,
                "target must be contiguous int64 of one class a row");
    same_device(z, *target, "target");
    a.target = target->data_ptr<int64_t>();
  }
  check_temp(temperature);
  TORCH_CHECK(alpha >= 0 && alpha <= 1, "alpha must be in [0, 1], got ", alpha);
  TORCH_CHECK(a.target || alpha == 1, "alpha below 1 needs a target");
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "reduction");
  a.temp = temperature;
  a.alpha = alpha;
  a.ignore_index = ignore_index;
  a.grad_scale = reduction == 1 ? (float)(1.0 / std::max<int64_t>(a.R, 1)) : 1.f;

  c10::OptionalDeviceGuard guard(at::device_of(z));
  const auto f32 = z.options().dtype(at::kFloat);
  auto row_loss = at::empty({a.R}, f32);
  a.row_loss = row_loss.data_ptr<float>();
  a.z = z.data_ptr();
  Tensor dz;
  if (want_grad) {
    dz = at::empty({a.R, a.V}, z.options());
    a.dz = dz.data_ptr();
  }
  if (a.R) distill_launch(a, stream());
  if (reduction == 0) return {row_loss, dz};
  auto loss = at::empty({}, f32);
  // (no rows: the sum is 0, the mean 0 / 0)
  distill_sum_launch(a.row_loss, a.R, reduction == 2 ? 1.0 : 1.0 / (double)a.R,
                     loss.data_ptr<float>(), stream());
  return {loss, dz};
}

// dz[r][:] *= s (one value, or one a row), in place
void scale_rows_(const Tensor& dz, const Tensor& s) {
  const int type = check_rows(dz, "dz");
  TORCH_CHECK(dz.is_contiguous(), "dz must be contiguous");
  TORCH_CHECK(s.scalar_type() == at::kFloat && s.is_contiguous() &&
                  (s.numel() == 1 || s.numel() == dz.size(0)),
              "the factors must be contiguous fp32, one or one a row");
  same_device(dz, s, "the factors");
  c10::OptionalDeviceGuard guard(at::device_of(dz));
  if (dz.size(0))
    scale_rows_launch(dz.data_ptr(), type, dz.size(0), (int)dz.size(1), s.data_ptr<float>(),
                      s.numel() == 1 ? 0 : 1, stream());
}

}  // namespace

void register_distill(py::module& m) {
  m.def("top_logits", &top_logits, py::arg("logits"), py::arg("k"), py::arg("temperature"),
        "the k largest logits of each row, their classes and log sum exp(logits / temperature)");
  m.def("distill", &distill, py::arg("logits"), py::arg("values"), py::arg("indices"),
        py::arg("lse"), py::arg("target"), py::arg("temperature"), py::arg("alpha"),
        py::arg("tail"), py::arg("reduction"), py::arg("ignore_index"), py::arg("want_grad"),
        "loss against a teacher's top logits -> (loss, gradient for a unit seed)");
  m.def("scale_rows_", &scale_rows_, "rows scaled in place by one factor, or one each");
  m.attr("DISTILL_MAX_CLASSES") = kDistillMaxClasses;
  m.attr("DISTILL_MAX_K") = kDistillMaxK;
}

}  // namespace pca
