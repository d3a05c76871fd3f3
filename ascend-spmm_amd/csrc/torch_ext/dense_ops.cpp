// The dense operators of a graph layer with typed nodes, as differentiable
// torch operators over the C ABI: layer_norm.  They check their tensors,
// allocate outputs and workspace on the tensors' device and launch on its
// current stream.  Gradients are not differentiable themselves.
#include "ext_common.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int32_t dense_type_of(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kHalf: return SPMM_VALUE_F16;
    case at::kBFloat16: return SPMM_VALUE_BF16;
    case at::kFloat: return SPMM_VALUE_F32;
    default: TORCH_CHECK(false, op, " supports only FP16, BF16 and FP32 tensors, but got ", t.scalar_type());
  }
  return -1;
}

// `t` as rows of its last dimension: a view where its rows are contiguous and
// evenly apart, else a copy.
at::Tensor as_rows(const at::Tensor& t) {
  const int64_t width = t.size(-1);
  if (t.dim() == 2 && (t.stride(1) == 1 || width == 1) && (t.stride(0) >= width || t.size(0) <= 1)) return t;
  return t.contiguous().view({width > 0 ? t.numel() / width : 0, width});
}

int64_t row_stride(const at::Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

bool wants_grad(const at::Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
bool wants_grad(const c10::optional<at::Tensor>& t) { return t.has_value() && wants_grad(*t); }

// ------------------------------------------------------------- layer_norm

void check_layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                      const c10::optional<at::Tensor>& bias) {
  TORCH_CHECK_GPU(x);
  TORCH_CHECK(x.dim() >= 1, "layer_norm: x must have at least one dimension");
  TORCH_CHECK(x.size(-1) >= 1, "layer_norm requires a last dimension of at least one element");
  dense_type_of(x, "layer_norm");
  for (const auto* p : {&weight, &bias}) {
    if (!p->has_value()) continue;
    const char* name = p == &weight ? "weight" : "bias";
    const at::Tensor& t = **p;
    TORCH_CHECK(t.device() == x.device(), "layer_norm: ", name, " must be on the same device as x");
    TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), "layer_norm: ", name, " must be a 1D Tensor of ", x.size(-1),
                " elements, but got ", t.sizes());
    TORCH_CHECK(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, "layer_norm: ", name,
                " must have the dtype of x or be FP32");
  }
  TORCH_CHECK(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(),
              "layer_norm: weight and bias must have the same dtype");
}

spmm_norm_desc norm_desc(const at::Tensor& rows, const c10::optional<at::Tensor>& weight,
                         const c10::optional<at::Tensor>& bias, double eps) {
  const int32_t type = dense_type_of(rows, "layer_norm");
  const at::Tensor& param = weight.has_value() ? *weight : bias.has_value() ? *bias : rows;
  return {rows.size(0), rows.size(1), row_stride(rows), rows.size(1), eps, type, dense_type_of(param, "layer_norm")};
}

at::Tensor contiguous_or_none(const c10::optional<at::Tensor>& t) { return t.has_value() ? t->contiguous() : at::Tensor(); }
const void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// y, and where `keep` is set the rows' mean and rstd.
at::Tensor layer_norm_forward(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                              const c10::optional<at::Tensor>& bias, double eps, bool keep, at::Tensor* mean,
                              at::Tensor* rstd) {
  c10::DeviceGuard guard(x.device());
  const at::Tensor rows = as_rows(x), w = contiguous_or_none(weight), b = contiguous_or_none(bias);
  const spmm_norm_desc d = norm_desc(rows, weight, bias, eps);
  at::Tensor y = at::empty(x.sizes(), x.options());
  if (keep) {
    *mean = at::empty({d.rows}, x.options().dtype(at::kFloat));
    *rstd = at::empty({d.rows}, x.options().dtype(at::kFloat));
  }
  raise_status(spmm_layer_norm_run(&d, rows.data_ptr(), data_or_null(w), data_or_null(b), y.data_ptr(),
                                   keep ? mean->data_ptr<float>() : nullptr, keep ? rstd->data_ptr<float>() : nullptr,
                                   current_stream(x)),
               "layer_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                            const c10::optional<at::Tensor>& bias, double eps) {
    at::Tensor mean, rstd;
    at::Tensor y = layer_norm_forward(x, weight, bias, eps, true, &mean, &rstd);
    ctx->save_for_backward({x, weight.has_value() ? *weight : at::Tensor(), bias.has_value() ? *bias : at::Tensor(),
                            mean, rstd});
    ctx->saved_data["eps"] = eps;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm: its gradient is not differentiable");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &mean = saved[3], &rstd = saved[4];
    c10::optional<at::Tensor> weight, bias;
    if (saved[1].defined()) weight = saved[1];
    if (saved[2].defined()) bias = saved[2];
    c10::DeviceGuard guard(x.device());
    const at::Tensor rows = as_rows(x), grad = as_rows(grads[0]), w = contiguous_or_none(weight);
    spmm_norm_desc d = norm_desc(rows, weight, bias, ctx->saved_data["eps"].toDouble());
    d.grad_stride = row_stride(grad);
    // Inputs that are tensors are numbered in order.
    size_t edge = 0;
    at::Tensor dx, dw, db;
    if (ctx->needs_input_grad(edge++)) dx = at::empty(x.sizes(), x.options());
    if (weight.has_value() && ctx->needs_input_grad(edge++)) dw = at::empty(weight->sizes(), weight->options());
    if (bias.has_value() && ctx->needs_input_grad(edge++)) db = at::empty(bias->sizes(), bias->options());
    size_t bytes = 0;
    raise_status(spmm_layer_norm_grad_workspace(&d, &bytes), "layer_norm");
    at::Tensor ws = workspace(x, dw.defined() || db.defined() ? bytes : 0);
    auto out = [](at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    raise_status(spmm_layer_norm_grad_run(&d, rows.data_ptr(), data_or_null(w), mean.data_ptr<float>(),
                                          rstd.data_ptr<float>(), grad.data_ptr(), out(dx), out(dw), out(db),
                                          ws.data_ptr(), bytes, current_stream(x)),
                 "layer_norm");
    return {dx, dw, db, at::Tensor()};
  }
};

at::Tensor layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                      const c10::optional<at::Tensor>& bias, double eps) {
  check_layer_norm(x, weight, bias);
  if (wants_grad(x) || wants_grad(weight) || wants_grad(bias)) return LayerNorm::apply(x, weight, bias, eps);
  return layer_norm_forward(x, weight, bias, eps, false, nullptr, nullptr);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(myops, m) {
  m.def("layer_norm(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> Tensor", &layer_norm);
}

void bind_dense_ops(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm,
        R"doc(
    Layer norm over the last dimension, on the GPU: (x - mean) / sqrt(var + eps)
    * weight + bias, statistics in FP32, one rounding to the type of x (FP16,
    BF16 or FP32).  weight and bias have that type or FP32, or are None.
    Differentiable with respect to x, weight and bias.
    )doc",
        pybind11::arg("x"), pybind11::arg("weight") = pybind11::none(), pybind11::arg("bias") = pybind11::none(),
        pybind11::arg("eps") = 1e-5);
}
