// Bindings of distill.hip: host checks, outputs from the caching allocator, launches on the
// current stream of the tensors' own device (no host sync, hipGraph-capturable). The loss's autograd
// node is C++: at the sizes of a CIFAR batch the step is bound by the host.
#include <cmath>
#include <mutex>

#include "bindings_util.h"
#include "distill.h"

namespace pca {
namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool is_logit_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 ||
         t.scalar_type() == at::kHalf;
}
int logit_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? LOGIT_F32
                                       : t.scalar_type() == at::kBFloat16 ? LOGIT_BF16 : LOGIT_F16;
}

void check_logits(const Tensor& z) {
  PCA_VALUE(z.is_cuda(), "logits must be a GPU tensor");
  PCA_VALUE(z.dim() >= 1, "logits must have a class dimension");
  PCA_TYPE(is_logit_type(z), "logits must be fp32, bf16 or fp16, got ", z.scalar_type());
  PCA_VALUE(z.size(-1) >= 1 && z.size(-1) <= kDistillMaxClasses, "logits has ", z.size(-1),
            " classes: 1 to ", kDistillMaxClasses, " are supported");
  PCA_VALUE(z.numel() / z.size(-1) < (int64_t(1) << 31), "logits has too many rows");
}

// (log2 e / T is an fp32 number)
void check_temp(double t) {
  PCA_VALUE(t >= kDistillMinTemp && t <= 1 / kDistillMinTemp,
            "temperature must be positive, 2^-64 to 2^64, got ", t);
}

// shape with the last dimension replaced by k (dropped for k = 0)
std::vector<int64_t> lead(const Tensor& z, int64_t k) {
  std::vector<int64_t> s(z.sizes().begin(), z.sizes().end() - 1);
  if (k) s.push_back(k);
  return s;
}

std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& logits, int64_t k, double temperature) {
  check_logits(logits);
  const int V = (int)logits.size(-1);
  PCA_VALUE(k >= 1 && k <= std::min(V, kDistillMaxK), "k must be 1 to ", std::min(V, kDistillMaxK),
            ", got ", k);
  check_temp(temperature);
  at::NoGradGuard no_grad;
  c10::OptionalDeviceGuard guard(at::device_of(logits));
  const Tensor z = rows_of(logits.detach());
  const int64_t R = z.size(0);
  auto values = at::empty(lead(logits, k), z.options());
  auto indices = at::empty(lead(logits, k), z.options().dtype(at::kInt));
  auto lse = at::empty(lead(logits, 0), z.options().dtype(at::kFloat));
  if (R)
    top_logits_launch(z.data_ptr(), logit_type(z), z.stride(0), R, V, (int)k, temperature,
                      values.data_ptr(), indices.data_ptr<int32_t>(), lse.data_ptr<float>(),
                      cur_stream());
  return {values, indices, lse};
}

struct Loss {
  double temperature, alpha;
  bool tail;
  int reduction;   // 0: a loss a row, 1: mean over the rows, 2: sum
  int64_t ignore_index;
};

// z [R][V] rows; the rest dense, one entry or K a row
DistillArgs args_of(const Tensor& z, const Tensor& values, const Tensor& indices, const Tensor& lse,
                    const Tensor& target, const Loss& l) {
  DistillArgs a{};
  a.type = logit_type(z);
  a.R = z.size(0);
  a.V = (int)z.size(1);
  a.ld = z.stride(0);
  a.z = z.data_ptr();
  a.K = (int)values.size(-1);
  a.value_type = logit_type(values);
  a.index64 = indices.scalar_type() == at::kLong;
  a.values = values.data_ptr();
  a.indices = indices.data_ptr();
  a.tail = l.tail;
  a.lse = l.tail ? lse.data_ptr<float>() : nullptr;
  a.target = target.defined() ? target.data_ptr<int64_t>() : nullptr;
  a.temp = l.temperature;
  a.alpha = l.alpha;
  a.ignore_index = l.ignore_index;
  a.grad_scale = l.reduction == 1 ? (float)(1.0 / std::max<int64_t>(a.R, 1)) : 1.f;
  return a;
}

// -> loss, gradient for a unit seed
std::tuple<Tensor, Tensor> distill(const Tensor& z, const Tensor& values, const Tensor& indices,
                                   const Tensor& lse, const Tensor& target, const Loss& l,
                                   bool want_grad) {
  DistillArgs a = args_of(z, values, indices, lse, target, l);
  const auto f32 = z.options().dtype(at::kFloat);
  auto row_loss = at::empty({a.R}, f32);
  a.row_loss = row_loss.data_ptr<float>();
  Tensor dz;
  if (want_grad) {
    dz = at::empty({a.R, a.V}, z.options());
    a.dz = dz.data_ptr();
  }
  if (a.R) distill_launch(a, cur_stream());
  if (l.reduction == 0) return {row_loss, dz};
  auto loss = at::empty({}, f32);
  // (no rows: the sum is 0, the mean 0 / 0)
  distill_sum_launch(a.row_loss, a.R, l.reduction == 2 ? 1.0 : 1.0 / (double)a.R,
                     loss.data_ptr<float>(), cur_stream());
  return {loss, dz};
}

// The capture that the current stream is in, 0: none.
int64_t capture() {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(cur_stream(), &status, &id) != hipSuccess) (void)hipGetLastError();
  return status == hipStreamCaptureStatusActive ? (int64_t)id : 0;
}

// The forward computes the gradient for a unit seed from the row it holds in registers and hands it
// to the backward, which computes the rows whose seed (read on the device) is not one again from the
// saved logits: the seed has to come before the rounding. A second backward of a retained graph
// computes all of them again, and so does one that is not in the forward's capture: a replay of
// either alone would find rows of another seed, or write over what was returned.
struct DistillFn : public torch::autograd::Function<DistillFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& values,
                        const Tensor& indices, const optional<Tensor>& lse_,
                        const optional<Tensor>& target_, const Loss& l, bool debug) {
    const Tensor lse = lse_.value_or(Tensor()), target = target_.value_or(Tensor());
    auto [loss, dz] = distill(rows_of(logits), values, indices, lse, target, l, true);
    ctx->save_for_backward({logits, values, indices, lse, target});
    ctx->saved_data["dz"] = dz;
    ctx->saved_data["capture"] = capture();
    ctx->saved_data["temperature"] = l.temperature;
    ctx->saved_data["alpha"] = l.alpha;
    ctx->saved_data["tail"] = l.tail;
    ctx->saved_data["reduction"] = (int64_t)l.reduction;
    ctx->saved_data["ignore_index"] = l.ignore_index;
    ctx->saved_data["debug"] = debug;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();   // (raises if the logits were changed)
    const Tensor& logits = saved[0];
    variable_list out(7);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::OptionalDeviceGuard guard(at::device_of(logits));
      auto& d = ctx->saved_data;
      Tensor dz;
      auto it = d.find("dz");
      const bool keep = it != d.end() && capture() == d["capture"].toInt();
      if (keep) {
        dz = it->second.toTensor();
        d.erase(it);
      }
      const bool unit = is_unit_seed(grads[0]);
      if (!keep || !unit) {
        const Loss l{d["temperature"].toDouble(), d["alpha"].toDouble(), d["tail"].toBool(),
                     (int)d["reduction"].toInt(), d["ignore_index"].toInt()};
        const Tensor z = rows_of(logits);
        DistillArgs a = args_of(z, saved[1], saved[2], saved[3], saved[4], l);
        const Tensor s = grads[0].reshape({-1}).contiguous();
        if (!unit) a.seed = s.data_ptr<float>();
        a.seed_rows = l.reduction == 0;
        a.keep = keep;
        if (!keep) dz = at::empty({a.R, a.V}, z.options());
        a.dz = dz.data_ptr();
        if (a.R) distill_launch(a, cur_stream());
      }
      debug_check(d["debug"].toBool(), "distill_loss backward");
      out[0] = dz.view(logits.sizes());
    }
    once_differentiable(out, "distill_loss");
    return out;
  }
};

Tensor distill_loss(const Tensor& logits, const Tensor& values, const Tensor& indices,
                    const optional<Tensor>& lse, const optional<Tensor>& target, double temperature,
                    double alpha, bool tail, const std::string& reduction, int64_t ignore_index,
                    bool debug) {
  check_logits(logits);
  check_temp(temperature);
  no_tangent(logits, "distill_loss");
  Loss l{temperature, alpha, tail,
         reduction == "none" ? 0 : reduction == "mean" ? 1 : reduction == "sum" ? 2 : -1,
         ignore_index};
  PCA_VALUE(l.reduction >= 0, "reduction must be \"none\", \"mean\" or \"sum\", got ", reduction);
  PCA_VALUE(alpha >= 0 && alpha <= 1, "alpha must be in [0, 1], got ", alpha);
  const bool labels = target.has_value() && target->defined();
  PCA_VALUE(labels || alpha == 1, "alpha below 1 needs a target");
  const auto rows = logits.sizes().slice(0, logits.dim() - 1);
  PCA_VALUE(values.dim() == logits.dim() && indices.sizes() == values.sizes() &&
                values.sizes().slice(0, values.dim() - 1) == rows,
            "top values ", values.sizes(), " and indices ", indices.sizes(), " do not fit logits ",
            logits.sizes());
  PCA_VALUE(values.size(-1) >= 1 && values.size(-1) <= kDistillMaxK, "1 to ", kDistillMaxK,
            " kept logits a row are supported, got ", values.size(-1));
  PCA_TYPE(is_logit_type(values) &&
               (indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong),
           "top values must be fp32, bf16 or fp16 and indices int32 or int64, got ",
           values.scalar_type(), ", ", indices.scalar_type());
  auto data = [&](const Tensor& t, const char* name) {
    PCA_VALUE(t.device() == logits.device(), name, " is on ", t.device(), ", the logits are on ",
              logits.device());
    PCA_VALUE(!t.requires_grad(), name, " requires grad: a teacher's answer is data, detach it");
    no_tangent(t, "distill_loss");
    return t.contiguous();
  };
  c10::OptionalDeviceGuard guard(at::device_of(logits));
  const Tensor v = data(values, "values"), i = data(indices, "indices");
  Tensor s, y;
  if (tail) {
    PCA_VALUE(lse.has_value() && lse->defined(), "tail=True needs the teacher's lse");
    PCA_VALUE(lse->scalar_type() == at::kFloat && lse->sizes() == rows, "lse must be fp32 of shape ",
              rows);
    s = data(*lse, "lse");
  }
  if (labels) {
    PCA_VALUE(target->scalar_type() == at::kLong && target->sizes() == rows,
              "target must be int64 of shape ", rows);
    y = data(*target, "target");
  }
  Tensor loss;
  if (at::GradMode::is_enabled() && logits.requires_grad())
    loss = DistillFn::apply(logits, v, i, s.defined() ? optional<Tensor>(s) : c10::nullopt,
                            y.defined() ? optional<Tensor>(y) : c10::nullopt, l, debug);
  else
    loss = std::get<0>(distill(rows_of(logits), v, i, s, y, l, false));
  debug_check(debug, "distill_loss");
  return l.reduction == 0 && logits.dim() != 2 ? loss.view(rows) : loss;
}

// never destroyed: their memory may outlive the allocator at exit. (Read by autograd's threads.)
struct Units {
  std::mutex lock;
  std::vector<Tensor> t;
};
Units& units() {
  static auto* u = new Units();
  return *u;
}

}  // namespace

bool is_unit_seed(const Tensor& g) {
  std::lock_guard<std::mutex> hold(units().lock);
  for (const Tensor& u : units().t)
    if (u.data_ptr() == g.data_ptr() && u.sizes() == g.sizes() &&
        u.scalar_type() == g.scalar_type())
      return true;
  return false;
}

void register_distill(py::module& m) {
  m.def("top_logits", &top_logits, py::arg("logits"), py::arg("k"), py::arg("temperature"),
        "the k largest logits of each row, their classes and log sum exp(logits / temperature)");
  m.def("distill_loss", &distill_loss, py::arg("logits"), py::arg("values"), py::arg("indices"),
        py::arg("lse"), py::arg("target"), py::arg("temperature"), py::arg("alpha"),
        py::arg("tail"), py::arg("reduction"), py::arg("ignore_index"), py::arg("debug"),
        "differentiable loss against a teacher's top logits");
  m.def("register_unit_seed", [](const Tensor& t) {
    std::lock_guard<std::mutex> hold(units().lock);
    units().t.push_back(t);
  },
        "a tensor of ones that is never written: backward passes seeded with it scale nothing");
}

}  // namespace pca
