// Bindings of gated.hip: host checks, outputs from the caching allocator, launches on the current
// stream of the tensors' own device (no host sync, hipGraph-capturable).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "gated.h"

namespace pca {
namespace {

using at::Tensor;
using c10::optional;

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

int gated_type(at::ScalarType s, const char* name) {
  switch (s) {
    case at::kFloat: return GATED_F32;
    case at::kBFloat16: return GATED_BF16;
    case at::kHalf: return GATED_F16;
    default: TORCH_CHECK(false, name, " must be fp32, bf16 or fp16, got ", s);
  }
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

void check2d(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  gated_type(t.scalar_type(), name);
  TORCH_CHECK(t.dim() == 2 && t.size(1) >= 1, name, " must be [rows][columns]");
  TORCH_CHECK(t.size(0) < (int64_t(1) << 31) && t.size(1) <= (1 << 19), name, " is too large");
}

// t itself if the products can read it, else a copy in `like`'s type with its rows padded by zeros
// to whole pieces
Tensor gated_operand(const Tensor& t, const Tensor& like) {
  check2d(t, "operand");
  if (t.scalar_type() == like.scalar_type() && is_operand(t)) return t;
  c10::OptionalDeviceGuard guard(at::device_of(t));
  const Tensor src = t.size(1) == 1 || t.stride(1) == 1 ? t : t.contiguous();
  const int64_t np = whole(t.size(1), piece(like));
  auto out = at::empty({t.size(0), np}, t.options().dtype(like.scalar_type()));
  if (t.size(0))
    gated_operand_launch(src.data_ptr(), gated_type(t.scalar_type(), "operand"), src.stride(0),
                         t.size(0), (int)t.size(1), out.data_ptr(),
                         gated_type(like.scalar_type(), "like"), (int)np, stream());
  return out;
}

void check_operand(const Tensor& t, const Tensor& like, const char* name) {
  check2d(t, name);
  TORCH_CHECK(t.scalar_type() == like.scalar_type() && t.device() == like.device(), name,
              " must have the type and device of the rows");
  TORCH_CHECK(is_operand(t), name, " must come from gated_operand");
}

void run(int form, const Tensor& like, bool out_f32, GatedArgs& a) {
  const int type = gated_type(like.scalar_type(), "operand");
  a.splits = gated_splits(form, type, a.M, a.N, a.K);
  Tensor part;
  if (a.splits > 1) {
    part = at::empty({a.splits * gated_part_floats(form, a.M, a.N)},
                     like.options().dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  gated_launch(form, type, out_f32, a, stream());
}

// operands x [M][C'], wg / wu [F][C'] -> h [M][F] and, if wanted, the fp32 projections
std::tuple<Tensor, Tensor, Tensor> gated_fwd(const Tensor& x, const Tensor& wg, const Tensor& wu,
                                             int act, bool save) {
  check_operand(x, x, "x");
  check_operand(wg, x, "w_gate");
  check_operand(wu, x, "w_up");
  TORCH_CHECK(wg.sizes() == wu.sizes() && wg.size(1) == x.size(1), "weights must be [hidden][",
              x.size(1), "]");
  TORCH_CHECK(wg.size(0) >= 1 && wg.size(0) <= (1 << 19), "hidden units: 1 to ", 1 << 19);
  TORCH_CHECK(act >= ACT_NONE && act <= ACT_SIGMOID, "activation");
  c10::OptionalDeviceGuard guard(at::device_of(x));
  // (one row stride for both)
  const Tensor g0 = wg.stride(0) == wu.stride(0) ? wg : wg.contiguous();
  const Tensor u0 = wg.stride(0) == wu.stride(0) ? wu : wu.contiguous();
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
  a.p0 = g0.data_ptr(), a.p1 = u0.data_ptr(), a.ldp = g0.stride(0);
  a.M = (int)M, a.N = (int)F, a.K = (int)x.size(1);
  a.ncols = a.N;
  a.out0 = h.data_ptr();
  a.save_g = save ? g.data_ptr<float>() : nullptr;
  a.save_u = save ? u.data_ptr<float>() : nullptr;
  a.act = act;
  run(GATED_FWD, x, false, a);
  return {h, g, u};
}

// dh [M][F] any row stride; g, u of the forward; C the true width -> dx, dwg, dwu (undefined where
// not wanted); dw_f32: weight gradients in fp32
std::tuple<Tensor, Tensor, Tensor> gated_bwd(const Tensor& dh, const Tensor& x, const Tensor& wg,
                                             const Tensor& wu, const Tensor& g, const Tensor& u,
                                             int64_t C, int act, bool need_dx, bool need_dw,
                                             bool dw_f32) {
  check_operand(x, x, "x");
  check_operand(wg, x, "w_gate");
  check_operand(wu, x, "w_up");
  const int64_t M = x.size(0), F = wg.size(0), Cp = x.size(1), Fp = whole(F, piece(x));
  TORCH_CHECK(wg.sizes() == wu.sizes() && wg.size(1) == Cp && C >= 1 && C <= Cp &&
                  Cp == whole(C, piece(x)), "weights must be [hidden][", Cp, "]");
  for (const Tensor* t : {&g, &u})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 &&
                    t->size(0) == M && t->size(1) == F && t->device() == x.device(),
                "the projections must be the forward's");
  TORCH_CHECK(dh.scalar_type() == x.scalar_type() && dh.device() == x.device() && dh.dim() == 2 &&
                  dh.size(0) == M && dh.size(1) == F && (F == 1 || dh.stride(1) == 1),
              "dh must be [", M, "][", F, "] of the rows' type with contiguous rows");
  TORCH_CHECK(act >= ACT_NONE && act <= ACT_SIGMOID, "activation");
  c10::OptionalDeviceGuard guard(at::device_of(x));
  const int type = gated_type(x.scalar_type(), "x");
  Tensor dx, dwg, dwu;
  const auto wopt = dw_f32 ? x.options().dtype(at::kFloat) : x.options();
  if (need_dx) dx = at::empty({M, C}, x.options());
  if (need_dw) {
    dwg = at::empty({F, C}, wopt);
    dwu = at::empty({F, C}, wopt);
  }
  if (M == 0) {
    if (need_dw) {
      dwg.zero_();
      dwu.zero_();
    }
    return {dx, dwg, dwu};
  }
  auto d = at::empty({M, 2 * Fp}, x.options());
  gated_dact_launch(type, g.data_ptr<float>(), u.data_ptr<float>(), dh.data_ptr(), dh.stride(0), M,
                    (int)F, (int)Fp, act, d.data_ptr(), stream());
  GatedArgs a{};
  a.q = d.data_ptr(), a.ldq = 2 * Fp, a.qseg = Fp;
  a.N = (int)C, a.ncols = (int)Cp;
  if (need_dx) {
    GatedArgs b = a;
    const Tensor g0 = wg.stride(0) == wu.stride(0) ? wg : wg.contiguous();
    const Tensor u0 = wg.stride(0) == wu.stride(0) ? wu : wu.contiguous();
    b.p0 = g0.data_ptr(), b.p1 = u0.data_ptr(), b.ldp = g0.stride(0);
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

}  // namespace

void register_gated(py::module& m) {
  m.def("gated_operand", &gated_operand, py::arg("t"), py::arg("like"),
        "t as an operand of the gated products in the type of `like`: itself, or a padded copy");
  m.def("gated_fwd", &gated_fwd, py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("act"),
        py::arg("save"), "act(x Wg^T) * (x Wu^T) -> (h, fp32 projections if saved)");
  m.def("gated_bwd", &gated_bwd, py::arg("dh"), py::arg("x"), py::arg("w_gate"), py::arg("w_up"),
        py::arg("g"), py::arg("u"), py::arg("C"), py::arg("act"), py::arg("need_dx"),
        py::arg("need_dw"), py::arg("dw_f32"), "gradients of gated_fwd -> (dx, dw_gate, dw_up)");
}

}  // namespace pca
