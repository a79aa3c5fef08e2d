// PyTorch-ROCm operators of the norms around a block, on the C ABI of include/fsw.h: add_norm and rms_norm in bf16 and fp16, in
// `fused_mlp_module` and the dispatcher library `ASMLLM` (no counterpart in the reference).
#include <optional>
#include <tuple>

#include "bindings.h"

namespace {

typedef std::optional<Tensor> Maybe;

// x: [..., d]; rows are all dimensions but the last, which have to have one stride between them
void check_x(const Tensor& x, at::ScalarType want, const char* name) {
  check_type(x, want, name);
  TORCH_CHECK(x.dim() >= 1, name, " must have at least 1 dimension");
}

void check_weight(const Maybe& w, const Tensor& x, at::ScalarType want, const char* name) {
  if (!w) return;
  check_rows(*w, want, 1, name);
  TORCH_CHECK(w->size(0) == x.size(-1), name, " must be [", x.size(-1), "]");
}

void check_norm(const Tensor& x, const Tensor& y, const Maybe& gate, const Maybe& post, const Maybe& pre, at::ScalarType want) {
  check_x(x, want, "x");
  check_x(y, want, "y");
  TORCH_CHECK(x.sizes() == y.sizes(), "x and y must have the same shape");
  if (gate) {
    check_type(*gate, want, "gate");
    TORCH_CHECK(gate->sizes() == x.sizes() || (gate->dim() == 1 && gate->size(0) == x.size(-1)), "gate must be [d] or have the shape of x");
  }
  check_weight(post, x, want, "post_weight");
  check_weight(pre, x, want, "pre_weight");
}

// [rows, d] with contiguous channels; a copy only where the leading dimensions have no common stride
Tensor rows_of(const Tensor& t) {
  const int64_t d = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({d > 0 ? t.numel() / d : 0, d});
  return r.size(1) <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}
int64_t ld(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }
const void* data(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
void check_place(const Maybe& t, const Tensor& first, const char* name) {
  if (t) check_place(*t, first, name);
}

template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> add_norm(const Tensor& x, const Tensor& y, const Maybe& gate, const Maybe& post, const Maybe& pre, double scale,
                                    double eps) {
  check_norm(x, y, gate, post, pre, WANT);
  check_place(x, x, "x");
  check_place(y, x, "y");
  check_place(gate, x, "gate");
  check_place(post, x, "post_weight");
  check_place(pre, x, "pre_weight");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(x));
  const Tensor xr = rows_of(x), yr = rows_of(y);
  const bool per_row = gate && gate->sizes() == x.sizes() && x.dim() > 1;
  Tensor gr;
  if (gate) gr = per_row ? rows_of(*gate) : gate->contiguous();
  Tensor x_out = at::empty(x.sizes(), x.options()), h = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return {x_out, h};
  const int64_t M = xr.size(0), D = xr.size(1);
  const int rc = fsw_add_norm(code_of<WANT>(), M, D, xr.data_ptr(), ld(xr), yr.data_ptr(), ld(yr), gate ? gr.data_ptr() : nullptr,
                              per_row ? ld(gr) : 0, data(post), data(pre), (float)scale, (float)eps, x_out.data_ptr(), D, h.data_ptr(), D,
                              current_stream());
  check_rc(rc, "add_norm");
  return {x_out, h};
}

template <at::ScalarType WANT>
Tensor rms_norm(const Tensor& x, const Maybe& weight, double eps) {
  check_x(x, WANT, "x");
  check_weight(weight, x, WANT, "weight");
  check_place(x, x, "x");
  check_place(weight, x, "weight");
  const at::hip::OptionalHIPGuardMasqueradingAsCUDA device_guard(device_of(x));
  const Tensor xr = rows_of(x);
  Tensor h = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return h;
  const int64_t M = xr.size(0), D = xr.size(1);
  const int rc = fsw_add_norm(code_of<WANT>(), M, D, xr.data_ptr(), ld(xr), nullptr, 0, nullptr, 0, nullptr, data(weight), 1.0f, (float)eps,
                              nullptr, 0, h.data_ptr(), D, current_stream());
  check_rc(rc, "rms_norm");
  return h;
}

template <at::ScalarType WANT>
std::tuple<Tensor, Tensor> meta_add_norm(const Tensor& x, const Tensor& y, const Maybe& gate, const Maybe& post, const Maybe& pre, double,
                                         double) {
  check_norm(x, y, gate, post, pre, WANT);
  return {at::empty(x.sizes(), x.options()), at::empty(x.sizes(), x.options())};
}
template <at::ScalarType WANT>
Tensor meta_rms_norm(const Tensor& x, const Maybe& weight, double) {
  check_x(x, WANT, "x");
  check_weight(weight, x, WANT, "weight");
  return at::empty(x.sizes(), x.options());
}

constexpr auto BF = at::kBFloat16;
constexpr auto HF = at::kHalf;

}  // namespace

void bind_norms(pybind11::module_& m) {
  namespace py = pybind11;
  const char* add = "x' = x + scale * gate * norm(y) post_weight, h = norm(x') pre_weight; returns (x', h)";
  m.def("add_norm_bf16", &add_norm<BF>, add, py::arg("x"), py::arg("y"), py::arg("gate") = py::none(), py::arg("post_weight") = py::none(),
        py::arg("pre_weight") = py::none(), py::arg("scale") = 1.0, py::arg("eps") = 1e-5);
  m.def("add_norm_fp16", &add_norm<HF>, add, py::arg("x"), py::arg("y"), py::arg("gate") = py::none(), py::arg("post_weight") = py::none(),
        py::arg("pre_weight") = py::none(), py::arg("scale") = 1.0, py::arg("eps") = 1e-5);
  m.def("rms_norm_bf16", &rms_norm<BF>, "norm(x) weight, bf16", py::arg("x"), py::arg("weight") = py::none(), py::arg("eps") = 1e-5);
  m.def("rms_norm_fp16", &rms_norm<HF>, "norm(x) weight, fp16", py::arg("x"), py::arg("weight") = py::none(), py::arg("eps") = 1e-5);
}

TORCH_LIBRARY_FRAGMENT(ASMLLM, m) {
  for (const char* t : {"bf16", "fp16"}) {
    const std::string s(t);
    m.def(("add_norm_" + s + "(Tensor x, Tensor y, Tensor? gate=None, Tensor? post_weight=None, Tensor? pre_weight=None, "
           "float scale=1.0, float eps=1e-05) -> (Tensor, Tensor)").c_str());
    m.def(("rms_norm_" + s + "(Tensor x, Tensor? weight=None, float eps=1e-05) -> Tensor").c_str());
  }
}

TORCH_LIBRARY_IMPL(ASMLLM, CUDA, m) {
  m.impl("add_norm_bf16", &add_norm<BF>);
  m.impl("add_norm_fp16", &add_norm<HF>);
  m.impl("rms_norm_bf16", &rms_norm<BF>);
  m.impl("rms_norm_fp16", &rms_norm<HF>);
}

TORCH_LIBRARY_IMPL(ASMLLM, Meta, m) {
  m.impl("add_norm_bf16", &meta_add_norm<BF>);
  m.impl("add_norm_fp16", &meta_add_norm<HF>);
  m.impl("rms_norm_bf16", &meta_rms_norm<BF>);
  m.impl("rms_norm_fp16", &meta_rms_norm<HF>);
}
