// Bindings of gated.hip: host checks, outputs from the caching allocator, launches on the current
// stream of the tensors' own device (no host sync, hipGraph-capturable). The autograd node is C++:
// layers of a CIFAR batch's size are bound by the host.
#include "bindings_util.h"
#include "gated.h"

namespace pca {
namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMaxWidth = 1 << 19;

bool is_gated_type(at::ScalarType s) {
  return s == at::kFloat || s == at::kBFloat16 || s == at::kHalf;
}
int gated_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? GATED_F32
                                       : t.scalar_type() == at::kBFloat16 ? GATED_BF16 : GATED_F16;
}

int64_t piece(const Tensor& t) { return 16 / t.element_size(); }
int64_t whole(int64_t n, int64_t p) { return (n + p - 1) / p * p; }

// rows of whole 16-byte pieces at 16-byte addresses, which the tiles are loaded by; the largest
// offset inside a tile (256 rows) stays below 2^31 bytes
bool is_operand(const Tensor& t) {
  const int64_t es = t.element_size();
  return t.size(1) % piece(t) == 0 && (t.size(1) == 1 || t.stride(1) == 1) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
         (t.size(0) <= 1 || (t.stride(0) >= 0 && t.stride(0) * es % 16 == 0 &&
                             t.stride(0) * es < (1 << 22)));
}

// t [rows][n] itself if the products can read it, else a copy in the wanted type with its rows
// padded by zeros to whole pieces
Tensor operand(const Tensor& t, at::ScalarType want) {
  if (t.scalar_type() == want && is_operand(t)) return t;
  const Tensor src = t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous();
  const int64_t np = whole(t.size(1), 16 / (int64_t)c10::elementSize(want));
  auto out = at::empty({t.size(0), np}, t.options().dtype(want));
  if (t.size(0))
    gated_operand_launch(src.data_ptr(), gated_type(src), src.stride(0), t.size(0),
                         (int)t.size(1), out.data_ptr(), gated_type(out), (int)np, cur_stream());
  return out;
}

// both weights as operands of one row stride
std::pair<Tensor, Tensor> weights(const Tensor& wg, const Tensor& wu, at::ScalarType want) {
  Tensor g = operand(wg, want), u = operand(wu, want);
  if (g.size(0) > 1 && g.stride(0) != u.stride(0)) {
    g = g.contiguous();
    u = u.contiguous();
  }
  return {g, u};
}

void run(int form, const Tensor& like, bool out_f32, GatedArgs& a) {
  const int type = gated_type(like);
  a.splits = gated_splits(form, type, a.M, a.N, a.K, std::max(a.parts, 1));
  Tensor part;
  if (a.splits > 1) {
    part = at::empty({a.splits * gated_part_floats(form, a.M, a.N)},
                     like.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  gated_launch(form, type, out_f32, a, cur_stream());
}

// operands x [M][C'], wg / wu [F][C'] -> h [M][F] and, if wanted, the fp32 projections
std::tuple<Tensor, Tensor, Tensor> forward(const Tensor& x, const Tensor& wg, const Tensor& wu,
                                           int act, bool save) {
  const int64_t M = x.size(0), F = wg.size(0);
  auto h = at::empty({M, F}, x.options());
  Tensor g, u;
  if (save) {
    g = at::empty({M, F}, x.options().dtype(at::kFloat));
    u = at::empty({M, F}, x.options().dtype(at::kFloat));
  }
  if (M == 0) return {h, g, u};
  GatedArgs a{};
  a.q = x.data_ptr(), a.ldq = x.stride(0);
  a.p0 = wg.data_ptr(), a.p1 = wu.data_ptr(), a.ldp = wg.stride(0);
  a.M = (int)M, a.N = (int)F, a.K = (int)x.size(1);
  a.ncols = a.N;
  a.out0 = h.data_ptr();
  a.save_g = save ? g.data_ptr<float>() : nullptr;
  a.save_u = save ? u.data_ptr<float>() : nullptr;
  a.act = act;
  run(GATED_FWD, x, false, a);
  return {h, g, u};
}

// dh [M][F]; g, u of the forward; C the true width -> dx, dwg, dwu (undefined where not wanted);
// dw_f32: weight gradients in fp32
std::tuple<Tensor, Tensor, Tensor> backward(const Tensor& dh, const Tensor& x, const Tensor& wg,
                                            const Tensor& wu, const Tensor& g, const Tensor& u,
                                            int64_t C, int act, bool need_dx, bool need_dw,
                                            bool dw_f32) {
  const int64_t M = x.size(0), F = wg.size(0), Cp = x.size(1), Fp = whole(F, piece(x));
  Tensor dx, dwg, dwu;
  if (need_dx) dx = at::empty({M, C}, x.options());
  if (need_dw) {
    const auto opt = dw_f32 ? x.options().dtype(at::kFloat) : x.options();
    dwg = at::empty({F, C}, opt);
    dwu = at::empty({F, C}, opt);
  }
  if (M == 0) {
    if (need_dw) {
      dwg.zero_();
      dwu.zero_();
    }
    return {dx, dwg, dwu};
  }
  const int parts = gated_parts(gated_type(x), M, C, F);
  auto d = at::empty({M, 2 * parts * Fp}, x.options());
  gated_dact_launch(gated_type(x), g.data_ptr<float>(), u.data_ptr<float>(), dh.data_ptr(),
                    dh.stride(0), M, (int)F, (int)Fp, act, parts, d.data_ptr(), cur_stream());
  GatedArgs a{};
  a.q = d.data_ptr(), a.ldq = 2 * parts * Fp, a.qseg = Fp, a.parts = parts;
  a.N = (int)C, a.ncols = (int)Cp;
  if (need_dx) {
    GatedArgs b = a;
    b.p0 = wg.data_ptr(), b.p1 = wu.data_ptr(), b.ldp = wg.stride(0);
    b.M = (int)M, b.K = (int)F;
    b.out0 = dx.data_ptr();
    run(GATED_DX, x, false, b);
  }
  if (need_dw) {
    a.p0 = x.data_ptr(), a.ldp = x.stride(0);
    a.M = (int)F, a.mcols = (int)Fp, a.K = (int)M;
    a.out0 = dwg.data_ptr(), a.out1 = dwu.data_ptr();
    run(GATED_DW, x, dw_f32, a);
  }
  return {dx, dwg, dwu};
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = n;
  return s;
}

// The projections are kept in fp32 for the backward (8 bytes a hidden unit and row): computing them
// again would cost two of the forward's products, and 16-bit copies would add their rounding to
// every gradient.
struct GatedFn : public torch::autograd::Function<GatedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        int64_t act, bool debug) {
    const Tensor q = operand(rows_of(x), x.scalar_type());
    const auto [w0, w1] = weights(wg, wu, x.scalar_type());
    auto [h, g, u] = pca::forward(q, w0, w1, (int)act, true);
    ctx->save_for_backward({x, wg, wu, q, w0, w1, g, u});
    ctx->saved_data["act"] = act;
    ctx->saved_data["debug"] = debug;
    return h.view(with_last(x, wg.size(0)));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();   // (raises if an operand was changed)
    const Tensor &x = s[0], &wg = s[1];
    variable_list out(5);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      c10::OptionalDeviceGuard guard(at::device_of(x));
      auto [dx, dwg, dwu] = pca::backward(
          rows_of(grads[0]), s[3], s[4], s[5], s[6], s[7], wg.size(1),
          (int)ctx->saved_data["act"].toInt(), ctx->needs_input_grad(0),
          ctx->needs_input_grad(1) || ctx->needs_input_grad(2), wg.scalar_type() == at::kFloat);
      debug_check(ctx->saved_data["debug"].toBool(), "gated_linear backward");
      if (dx.defined()) out[0] = dx.view(x.sizes());
      out[1] = dwg;
      out[2] = dwu;
    }
    once_differentiable(out, "gated_linear");
    return out;
  }
};

// act(x Wg^T) * (x Wu^T) over the last dimension of x
Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act, bool debug) {
  PCA_VALUE(x.is_cuda(), "x must be a GPU tensor");
  PCA_TYPE(is_gated_type(x.scalar_type()), "x must be fp32, bf16 or fp16, got ", x.scalar_type());
  PCA_VALUE(x.dim() >= 1 && wg.dim() == 2 && wg.sizes() == wu.sizes(),
            "weights must be two [hidden, width] matrices, got ", wg.sizes(), " and ", wu.sizes());
  PCA_VALUE(x.size(-1) == wg.size(1), "x ", x.sizes(), " has ", x.size(-1),
            " features, the weights ", wg.size(1));
  PCA_VALUE(wg.size(0) >= 1 && wg.size(0) <= kMaxWidth && wg.size(1) >= 1 &&
                wg.size(1) <= kMaxWidth, "width and hidden must be 1 to ", kMaxWidth);
  PCA_TYPE(wg.scalar_type() == wu.scalar_type() &&
               (wg.scalar_type() == x.scalar_type() || wg.scalar_type() == at::kFloat),
           "weights must both be ", x.scalar_type(), " or fp32, got ", wg.scalar_type(), ", ",
           wu.scalar_type());
  PCA_VALUE(wg.device() == x.device() && wu.device() == x.device(), "weights are on ", wg.device(),
            " and ", wu.device(), ", x is on ", x.device());
  PCA_VALUE(x.numel() / x.size(-1) <= (int64_t(1) << 30), "x has more than 2^30 rows");
  for (const Tensor* t : {&x, &wg, &wu}) no_tangent(*t, "gated_linear");
  PCA_VALUE(act >= ACT_NONE && act <= ACT_SIGMOID, "activation");
  c10::OptionalDeviceGuard guard(at::device_of(x));
  Tensor h;
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wg.requires_grad() || wu.requires_grad())) {
    h = GatedFn::apply(x, wg, wu, act, debug);
  } else {
    const Tensor q = operand(rows_of(x), x.scalar_type());
    const auto [w0, w1] = weights(wg, wu, x.scalar_type());
    h = std::get<0>(forward(q, w0, w1, (int)act, false)).view(with_last(x, wg.size(0)));
  }
  debug_check(debug, "gated_linear");
  return h;
}

}  // namespace

void register_gated(py::module& m) {
  m.def("gated_linear", &gated_linear, py::arg("x"), py::arg("w_gate"), py::arg("w_up"),
        py::arg("act"), py::arg("debug"), "differentiable act(x Wg^T) * (x Wu^T)");
}

}  // namespace pca
