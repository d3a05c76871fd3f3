// The dense operators of a graph layer with typed nodes, as differentiable
// torch operators over the C ABI: layer_norm and grouped_matmul.  They check their tensors,
// allocate outputs and workspace on the tensors' device and launch on its
// current stream.  Gradients are not differentiable themselves.
#include "dense_common.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------- layer_norm

void check_layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                      const c10::optional<at::Tensor>& bias) {
  TORCH_CHECK_GPU(x);
  TORCH_CHECK(x.dim() >= 1, "layer_norm: x must have at least one dimension");
  TORCH_CHECK(x.size(-1) >= 1, "layer_norm requires a last dimension of at least one element");
  dense_type_of(x, "layer_norm");
  check_no_tangent(x, "layer_norm");
  for (const auto* p : {&weight, &bias}) {
    if (!p->has_value()) continue;
    check_no_tangent(**p, "layer_norm");
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

// ---------------------------------------------------------- grouped_matmul

// weight [groups, inner, width] whose matrices are contiguous, either as they
// are or transposed; a copy where they are neither.
at::Tensor grouped_weight(const at::Tensor& w, bool* transposed) {
  const int64_t k = w.size(1), n = w.size(2);
  const bool apart = w.size(0) <= 1 || w.stride(0) >= k * n;
  *transposed = false;
  if (apart && (w.stride(2) == 1 || n <= 1) && (w.stride(1) == n || k <= 1)) return w;
  if (apart && (w.stride(1) == 1 || k <= 1) && (w.stride(2) == k || n <= 1)) {
    *transposed = true;
    return w;
  }
  return w.contiguous();
}

// Rows for the grouped products, whose row strides are below 2^22.
at::Tensor as_grouped_rows(const at::Tensor& t) {
  const at::Tensor rows = as_rows(t);
  return row_stride(rows) < (int64_t(1) << 22) ? rows : rows.contiguous();
}

void check_grouped(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& offsets) {
  TORCH_CHECK_GPU(x);
  TORCH_CHECK_GPU(weight);
  TORCH_CHECK_GPU(offsets);
  TORCH_CHECK(x.dim() == 2, "grouped_matmul: x must be a 2D Tensor, but got: ", x.dim());
  TORCH_CHECK(weight.dim() == 3, "grouped_matmul: weight must be a 3D Tensor, but got: ", weight.dim());
  TORCH_CHECK(offsets.dim() == 1, "grouped_matmul: offsets must be a 1D Tensor, but got: ", offsets.dim());
  dense_type_of(x, "grouped_matmul");
  check_no_tangent(x, "grouped_matmul");
  check_no_tangent(weight, "grouped_matmul");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "grouped_matmul: weight must have the dtype of x");
  TORCH_CHECK(weight.size(1) == x.size(1), "grouped_matmul: x has ", x.size(1), " columns, but weight takes ",
              weight.size(1));
  TORCH_CHECK(offsets.size(0) == weight.size(0) + 1, "grouped_matmul: offsets must hold one entry more than weight has "
              "matrices (", weight.size(0) + 1, "), but got ", offsets.size(0));
  index_type_of(offsets, "offsets");
  TORCH_CHECK(weight.device() == x.device() && offsets.device() == x.device(),
              "grouped_matmul: weight and offsets must be on the same device as x");
}

spmm_grouped_desc grouped_desc(const at::Tensor& rows, const at::Tensor& weight, bool transposed,
                               const at::Tensor& offsets) {
  const int64_t k = weight.size(1), n = weight.size(2);
  return {rows.size(0), weight.size(0), k, n, row_stride(rows), n, weight.size(0) > 1 ? weight.stride(0) : k * n,
          transposed ? 1 : 0, index_type_of(offsets, "offsets"), dense_type_of(rows, "grouped_matmul")};
}

at::Tensor grouped_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& offsets) {
  c10::DeviceGuard guard(x.device());
  bool transposed;
  const at::Tensor rows = as_grouped_rows(x), w = grouped_weight(weight, &transposed), off = offsets.contiguous();
  const spmm_grouped_desc d = grouped_desc(rows, w, transposed, off);
  at::Tensor out = at::empty({d.rows, d.width}, x.options());
  size_t bytes = 0;
  raise_status(spmm_grouped_workspace(&d, &bytes), "grouped_matmul");
  at::Tensor ws = workspace(x, bytes);
  raise_status(spmm_grouped_run(&d, rows.data_ptr(), w.data_ptr(), off.data_ptr(), out.data_ptr(), ws.data_ptr(), bytes,
                                current_stream(x)),
               "grouped_matmul");
  return out;
}

struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const at::Tensor& offsets) {
    ctx->save_for_backward({x, weight, offsets});
    return grouped_forward(x, weight, offsets);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "grouped_matmul: its gradient is not differentiable");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1];
    c10::DeviceGuard guard(x.device());
    bool transposed;
    const at::Tensor rows = as_grouped_rows(x), grad = as_grouped_rows(grads[0]), w = grouped_weight(weight, &transposed);
    const at::Tensor off = saved[2].contiguous();
    spmm_grouped_desc d = grouped_desc(rows, w, transposed, off);
    d.grad_stride = row_stride(grad);
    at::Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
    // In weight's storage order, as its gradient is added to it.
    if (ctx->needs_input_grad(1))
      dw = transposed ? at::empty({d.groups, d.width, d.inner}, x.options()).transpose(1, 2)
                      : at::empty({d.groups, d.inner, d.width}, x.options());
    size_t bytes = 0;
    raise_status(spmm_grouped_grad_workspace(&d, &bytes), "grouped_matmul");
    at::Tensor ws = workspace(x, bytes);
    raise_status(spmm_grouped_grad_run(&d, rows.data_ptr(), w.data_ptr(), off.data_ptr(), grad.data_ptr(),
                                       dx.defined() ? dx.data_ptr() : nullptr, dw.defined() ? dw.data_ptr() : nullptr,
                                       ws.data_ptr(), bytes, current_stream(x)),
                 "grouped_matmul");
    return {dx, dw, at::Tensor()};
  }
};

at::Tensor grouped_matmul(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& offsets) {
  check_grouped(x, weight, offsets);
  if (wants_grad(x) || wants_grad(weight)) return GroupedMatmul::apply(x, weight, offsets);
  return grouped_forward(x, weight, offsets);
}

// ----------------------------------------------------------- orthogonalize

// coefficients: a, b, c of every step.
at::Tensor orthogonalize(const at::Tensor& update, const std::vector<double>& coefficients, double eps, bool precise) {
  TORCH_CHECK_GPU(update);
  TORCH_CHECK(update.dim() >= 2, "orthogonalize: update must have at least two dimensions, but got: ", update.dim());
  TORCH_CHECK(coefficients.size() % 3 == 0, "orthogonalize: coefficients must hold three values for each step");
  TORCH_CHECK(!wants_grad(update), "orthogonalize is not differentiable: call it under torch.no_grad()");
  check_no_tangent(update, "orthogonalize");
  c10::DeviceGuard guard(update.device());
  const at::Tensor u = update.contiguous();
  const int64_t rows = u.size(-2), width = u.size(-1);
  int64_t batch = 1;
  for (int64_t i = 0; i + 2 < u.dim(); ++i) batch *= u.size(i);
  const spmm_orthogonalize_desc d{batch, rows, width, static_cast<int64_t>(coefficients.size() / 3),
                                  coefficients.data(), eps, dense_type_of(u, "orthogonalize"), precise ? 1 : 0};
  at::Tensor out = at::empty(u.sizes(), u.options());
  size_t bytes = 0;
  raise_status(spmm_orthogonalize_workspace(&d, &bytes), "orthogonalize");
  at::Tensor ws = workspace(u, bytes);
  raise_status(spmm_orthogonalize_run(&d, u.data_ptr(), out.data_ptr(), ws.data_ptr(), bytes, current_stream(u)),
               "orthogonalize");
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(myops, m) {
  m.def("layer_norm(Tensor x, Tensor? weight=None, Tensor? bias=None, float eps=1e-05) -> Tensor", &layer_norm);
  m.def("grouped_matmul(Tensor x, Tensor weight, Tensor offsets) -> Tensor", &grouped_matmul);
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
  m.def("grouped_matmul", &grouped_matmul,
        R"doc(
    Products of row groups with their own matrices, on the GPU: out[r] = x[r] @
    weight[g] for offsets[g] <= r < offsets[g + 1].  x [rows, inner], weight
    [groups, inner, width] (its matrices contiguous or transposed), offsets
    [groups + 1] int32 or int64, ascending, on the GPU; groups may be empty, and
    rows outside of all groups become zero.  FP16, BF16 or FP32, sums in FP32.
    Differentiable with respect to x and weight.
    )doc",
        pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("offsets"));
  m.def("orthogonalize", &orthogonalize, "Newton-Schulz steps on matrix updates (GPU)", pybind11::arg("update"),
        pybind11::arg("coefficients"), pybind11::arg("eps"), pybind11::arg("precise") = false);
}
