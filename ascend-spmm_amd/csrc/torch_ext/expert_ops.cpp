// The operators around a layer of experts, as differentiable torch operators
// over the C ABI: embedding, route, the packing of rows for experts, and
// log_probs.  They check their tensors, allocate outputs and workspace on the
// tensors' device and launch on its current stream.  Gradients are not
// differentiable themselves.
#include "dense_common.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// `t` as `rows` rows of its last dimension: a view where its rows are contiguous
// and evenly apart, else a copy.
at::Tensor flat_rows(const at::Tensor& t, int64_t rows) {
  const at::Tensor flat = t.dim() == 2 ? t : t.reshape({rows, t.size(-1)});
  const int64_t width = flat.size(1);
  if ((flat.stride(1) == 1 || width <= 1) && (flat.stride(0) >= width || rows <= 1)) return flat;
  return flat.contiguous();
}

// Rows of an n-dimensional tensor whose last dimension is the row.
int64_t leading(const at::Tensor& t) {
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  return rows;
}

std::vector<int64_t> leading_sizes(const at::Tensor& t, int64_t last) {
  std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end() - 1);
  sizes.push_back(last);
  return sizes;
}

// Scratch of the library's calls, and its address: none where none is needed.
at::Tensor scratch(const at::Tensor& like, size_t bytes) { return bytes > 0 ? workspace(like, bytes) : at::Tensor(); }
void* scratch_data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_differentiable_once(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": its gradient is not differentiable");
}

// -------------------------------------------------------------- embedding

spmm_embedding_desc embedding_desc(int64_t count, const at::Tensor& weight, int64_t weight_stride, int64_t grad_stride,
                                   const at::Tensor& ids, double scale) {
  return {count,  weight.size(0), weight.size(1), weight_stride, grad_stride, scale, index_type_of(ids, "ids"),
          dense_type_of(weight, "embedding")};
}

at::Tensor embedding_forward(const at::Tensor& weight, const at::Tensor& ids, double scale) {
  c10::DeviceGuard guard(weight.device());
  const at::Tensor table = flat_rows(weight, weight.size(0)), index = ids.contiguous();
  std::vector<int64_t> sizes(ids.sizes().begin(), ids.sizes().end());
  sizes.push_back(weight.size(1));
  at::Tensor out = at::empty(sizes, weight.options());
  const spmm_embedding_desc d = embedding_desc(ids.numel(), table, row_stride(table), table.size(1), index, scale);
  raise_status(spmm_embedding_run(&d, table.data_ptr(), index.data_ptr(), out.data_ptr(), current_stream(weight)),
               "embedding");
  return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& weight, const at::Tensor& ids, double scale) {
    // The gradient needs the table's sizes alone.
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["width"] = weight.size(1);
    return embedding_forward(weight, ids, scale);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_differentiable_once("embedding");
    const at::Tensor ids = ctx->get_saved_variables()[0].contiguous();
    const at::Tensor grad = flat_rows(grads[0], ids.numel());
    c10::DeviceGuard guard(grad.device());
    at::Tensor dweight =
        at::empty({ctx->saved_data["rows"].toInt(), ctx->saved_data["width"].toInt()}, grad.options());
    const spmm_embedding_desc d = embedding_desc(ids.numel(), dweight, dweight.size(1), row_stride(grad), ids,
                                                 ctx->saved_data["scale"].toDouble());
    size_t bytes = 0;
    raise_status(spmm_embedding_grad_workspace(&d, &bytes), "embedding");
    at::Tensor ws = scratch(grad, bytes);
    raise_status(spmm_embedding_grad_run(&d, ids.data_ptr(), grad.data_ptr(), dweight.data_ptr(), scratch_data(ws), bytes,
                                         current_stream(grad)),
                 "embedding");
    return {dweight, at::Tensor(), at::Tensor()};
  }
};

at::Tensor embedding(const at::Tensor& weight, const at::Tensor& ids, double scale) {
  TORCH_CHECK_GPU(weight);
  TORCH_CHECK_GPU(ids);
  TORCH_CHECK(weight.dim() == 2, "embedding: weight must be a 2D Tensor, but got: ", weight.dim());
  dense_type_of(weight, "embedding");
  index_type_of(ids, "ids");
  check_no_tangent(weight, "embedding");
  TORCH_CHECK(ids.device() == weight.device(), "embedding: ids must be on the same device as weight");
  if (wants_grad(weight)) return Embedding::apply(weight, ids, scale);
  return embedding_forward(weight, ids, scale);
}

// ------------------------------------------------------------------ route

struct RouteOptions {
  int64_t top_k, score, groups, top_groups;
  bool renormalize;
  double scale;
};

spmm_route_desc route_desc(const at::Tensor& rows, const RouteOptions& o) {
  return {rows.size(0), rows.size(1),  row_stride(rows),           o.top_k, o.groups,
          o.top_groups, o.scale,       static_cast<int32_t>(o.score), o.renormalize ? 1 : 0,
          dense_type_of(rows, "route")};
}

std::tuple<at::Tensor, at::Tensor> route_forward(const at::Tensor& logits, const c10::optional<at::Tensor>& bias,
                                                 const RouteOptions& o, at::Tensor* stats) {
  c10::DeviceGuard guard(logits.device());
  const at::Tensor rows = flat_rows(logits, leading(logits));
  const at::Tensor b = bias.has_value() ? bias->contiguous() : at::Tensor();
  const spmm_route_desc d = route_desc(rows, o);
  // Before the outputs of that size are allocated; the rest is checked below.
  TORCH_CHECK_VALUE(o.top_k >= 1 && o.top_k <= 64, "route: top_k must be 1 to 64, but got ", o.top_k);
  at::Tensor weights = at::empty(leading_sizes(logits, o.top_k), logits.options().dtype(at::kFloat));
  at::Tensor experts = at::empty(leading_sizes(logits, o.top_k), logits.options().dtype(at::kInt));
  if (stats != nullptr && o.score == SPMM_SCORE_SOFTMAX && !o.renormalize)
    *stats = at::empty({d.rows, 2}, weights.options());
  raise_status(spmm_route_run(&d, rows.data_ptr(), b.defined() ? b.data_ptr<float>() : nullptr,
                              weights.data_ptr<float>(), experts.data_ptr<int32_t>(),
                              stats != nullptr && stats->defined() ? stats->data_ptr<float>() : nullptr,
                              current_stream(logits)),
               "route");
  return {weights, experts};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const c10::optional<at::Tensor>& bias,
                               int64_t top_k, int64_t score, int64_t groups, int64_t top_groups, bool renormalize,
                               double scale) {
    at::Tensor stats;
    auto [weights, experts] =
        route_forward(logits, bias, {top_k, score, groups, top_groups, renormalize, scale}, &stats);
    ctx->save_for_backward({logits, weights, experts, stats});
    ctx->saved_data["ints"] = std::vector<int64_t>{top_k, score, groups, top_groups, renormalize ? 1 : 0};
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["bias"] = bias.has_value();
    ctx->mark_non_differentiable({experts});
    ctx->set_materialize_grads(false);  // the ids' would be zeros, filled by a launch
    return {weights, experts};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_differentiable_once("route");
    if (!grads[0].defined()) return variable_list(8);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor& logits = saved[0];
    c10::DeviceGuard guard(logits.device());
    const at::Tensor rows = flat_rows(logits, leading(logits)), grad = grads[0].contiguous();
    const std::vector<int64_t> o = ctx->saved_data["ints"].toIntVector();
    const spmm_route_desc d =
        route_desc(rows, {o[0], o[1], o[2], o[3], o[4] != 0, ctx->saved_data["scale"].toDouble()});
    at::Tensor dlogits = at::empty(logits.sizes(), logits.options());
    raise_status(spmm_route_grad_run(&d, rows.data_ptr(), saved[2].data_ptr<int32_t>(), saved[1].data_ptr<float>(),
                                     saved[3].defined() ? saved[3].data_ptr<float>() : nullptr,
                                     grad.data_ptr<float>(), dlogits.data_ptr(), current_stream(logits)),
                 "route");
    return {dlogits, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor> route(const at::Tensor& logits, int64_t top_k, int64_t score,
                                         const c10::optional<at::Tensor>& bias, int64_t groups, int64_t top_groups,
                                         bool renormalize, double scale) {
  TORCH_CHECK_GPU(logits);
  TORCH_CHECK(logits.dim() >= 1, "route: logits must have at least one dimension");
  dense_type_of(logits, "route");
  check_no_tangent(logits, "route");
  if (bias.has_value()) {
    check_no_tangent(*bias, "route");
    TORCH_CHECK(bias->device() == logits.device(), "route: bias must be on the same device as logits");
    TORCH_CHECK(bias->scalar_type() == at::kFloat, "route: bias must be FP32, but got ", bias->scalar_type());
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == logits.size(-1), "route: bias must be a 1D Tensor of ",
                logits.size(-1), " elements, but got ", bias->sizes());
    TORCH_CHECK(!wants_grad(*bias), "route: bias decides the choice alone and has no gradient: detach it");
  }
  if (wants_grad(logits)) {
    const variable_list out = Route::apply(logits, bias, top_k, score, groups, top_groups, renormalize, scale);
    return {out[0], out[1]};
  }
  return route_forward(logits, bias, {top_k, score, groups, top_groups, renormalize, scale}, nullptr);
}

// ---------------------------------------------------- rows packed for experts

std::tuple<at::Tensor, at::Tensor> expert_plan(const at::Tensor& experts, int64_t count) {
  TORCH_CHECK_GPU(experts);
  TORCH_CHECK(experts.dim() == 1 || experts.dim() == 2, "ExpertPlan: experts must be a 1D or 2D Tensor, but got: ",
              experts.dim());
  const int32_t type = index_type_of(experts, "experts");
  TORCH_CHECK(experts.dim() == 1 || (experts.size(1) >= 1 && experts.size(1) <= 64),
              "ExpertPlan takes 1 to 64 choices a row, but got ", experts.size(1));
  c10::DeviceGuard guard(experts.device());
  const at::Tensor ids = experts.contiguous();
  size_t bytes = 0;
  raise_status(spmm_expert_plan_workspace(ids.numel(), count, &bytes), "ExpertPlan");
  const auto i32 = ids.options().dtype(at::kInt);
  at::Tensor offsets = at::empty({count + 1}, i32);
  at::Tensor place = at::empty({ids.size(0), ids.dim() == 2 ? ids.size(1) : 1}, i32);
  at::Tensor ws = scratch(ids, bytes);
  raise_status(spmm_expert_plan_run(type, ids.data_ptr(), ids.numel(), count, offsets.data_ptr<int32_t>(),
                                    place.data_ptr<int32_t>(), scratch_data(ws), bytes, current_stream(ids)),
               "ExpertPlan");
  return {offsets, place};
}

void check_plan(const at::Tensor& place, const at::Tensor& offsets, const at::Tensor& like) {
  TORCH_CHECK_GPU(like);
  for (const at::Tensor* t : {&place, &offsets}) {
    TORCH_CHECK(t->device() == like.device(), "ExpertPlan: the plan is on another device than the tensor");
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), "ExpertPlan: the plan's tensors must be contiguous "
                "int32 tensors");
  }
  TORCH_CHECK(place.dim() == 2 && offsets.dim() == 1 && offsets.size(0) >= 2, "ExpertPlan: not a plan's tensors");
}

spmm_experts_desc experts_desc(const at::Tensor& place, const at::Tensor& offsets, const at::Tensor& like,
                               int64_t stride, int64_t grad_stride) {
  return {place.size(0), place.size(1), offsets.size(0) - 1, like.size(1), stride, grad_stride,
          dense_type_of(like, "ExpertPlan")};
}

at::Tensor pack_forward(const at::Tensor& x, const at::Tensor& place, const at::Tensor& offsets) {
  c10::DeviceGuard guard(x.device());
  const at::Tensor rows = flat_rows(x, x.size(0));
  at::Tensor packed = at::empty({place.numel(), x.size(1)}, x.options());
  const spmm_experts_desc d = experts_desc(place, offsets, rows, row_stride(rows), rows.size(1));
  raise_status(spmm_expert_pack_run(&d, rows.data_ptr(), place.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                                    packed.data_ptr(), current_stream(x)),
               "ExpertPlan");
  return packed;
}

struct ExpertPack : torch::autograd::Function<ExpertPack> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& place,
                            const at::Tensor& offsets) {
    ctx->save_for_backward({place, offsets});
    return pack_forward(x, place, offsets);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_differentiable_once("ExpertPlan");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &place = saved[0], &offsets = saved[1];
    c10::DeviceGuard guard(grads[0].device());
    const at::Tensor grad = flat_rows(grads[0], place.numel());
    at::Tensor dx = at::empty({place.size(0), grad.size(1)}, grad.options());
    const spmm_experts_desc d = experts_desc(place, offsets, grad, row_stride(grad), grad.size(1));
    raise_status(spmm_expert_pack_grad_run(&d, grad.data_ptr(), place.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                                           dx.data_ptr(), current_stream(grad)),
                 "ExpertPlan");
    return {dx, at::Tensor(), at::Tensor()};
  }
};

at::Tensor expert_pack(const at::Tensor& x, const at::Tensor& place, const at::Tensor& offsets) {
  check_plan(place, offsets, x);
  dense_type_of(x, "ExpertPlan");
  TORCH_CHECK(x.dim() == 2 && x.size(0) == place.size(0), "ExpertPlan: x must be a 2D Tensor of the plan's ",
              place.size(0), " rows, but got ", x.sizes());
  check_no_tangent(x, "ExpertPlan");
  if (wants_grad(x)) return ExpertPack::apply(x, place, offsets);
  return pack_forward(x, place, offsets);
}

at::Tensor restore_forward(const at::Tensor& y, const at::Tensor& weights, const at::Tensor& place,
                           const at::Tensor& offsets) {
  c10::DeviceGuard guard(y.device());
  const at::Tensor rows = flat_rows(y, y.size(0)), w = weights.contiguous();
  at::Tensor out = at::empty({place.size(0), y.size(1)}, y.options());
  const spmm_experts_desc d = experts_desc(place, offsets, rows, row_stride(rows), rows.size(1));
  raise_status(spmm_expert_restore_run(&d, rows.data_ptr(), w.data_ptr<float>(), place.data_ptr<int32_t>(),
                                       offsets.data_ptr<int32_t>(), out.data_ptr(), current_stream(y)),
               "ExpertPlan");
  return out;
}

struct ExpertRestore : torch::autograd::Function<ExpertRestore> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& weights,
                            const at::Tensor& place, const at::Tensor& offsets) {
    ctx->save_for_backward({y, weights, place, offsets});
    return restore_forward(y, weights, place, offsets);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_differentiable_once("ExpertPlan");
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &y = saved[0], &place = saved[2], &offsets = saved[3];
    c10::DeviceGuard guard(y.device());
    const at::Tensor rows = flat_rows(y, y.size(0)), w = saved[1].contiguous();
    const at::Tensor grad = flat_rows(grads[0], place.size(0));
    at::Tensor dy, dw;
    if (ctx->needs_input_grad(0)) dy = at::empty(y.sizes(), y.options());
    if (ctx->needs_input_grad(1)) dw = at::empty(w.sizes(), w.options());
    const spmm_experts_desc d = experts_desc(place, offsets, rows, row_stride(rows), row_stride(grad));
    raise_status(spmm_expert_restore_grad_run(&d, rows.data_ptr(), w.data_ptr<float>(), place.data_ptr<int32_t>(),
                                              offsets.data_ptr<int32_t>(), grad.data_ptr(),
                                              dy.defined() ? dy.data_ptr() : nullptr,
                                              dw.defined() ? dw.data_ptr<float>() : nullptr, current_stream(y)),
                 "ExpertPlan");
    return {dy, dw, at::Tensor(), at::Tensor()};
  }
};

at::Tensor expert_restore(const at::Tensor& y, const at::Tensor& weights, const at::Tensor& place,
                          const at::Tensor& offsets) {
  check_plan(place, offsets, y);
  dense_type_of(y, "ExpertPlan");
  TORCH_CHECK(y.dim() == 2 && y.size(0) == place.numel(), "ExpertPlan: results must be a 2D Tensor of the plan's ",
              place.numel(), " packed rows, but got ", y.sizes());
  TORCH_CHECK(weights.device() == y.device(), "ExpertPlan: weights must be on the same device as the results");
  TORCH_CHECK(weights.scalar_type() == at::kFloat, "ExpertPlan: weights must be FP32, but got ", weights.scalar_type());
  TORCH_CHECK(weights.sizes() == place.sizes(), "ExpertPlan: weights must have one entry for each choice (",
              place.sizes(), "), but got ", weights.sizes());
  check_no_tangent(y, "ExpertPlan");
  check_no_tangent(weights, "ExpertPlan");
  if (wants_grad(y) || wants_grad(weights)) return ExpertRestore::apply(y, weights, place, offsets);
  return restore_forward(y, weights, place, offsets);
}

// -------------------------------------------------------------- log_probs

spmm_log_probs_desc log_probs_desc(const at::Tensor& rows, const at::Tensor& targets, int64_t top) {
  return {rows.size(0), rows.size(1), row_stride(rows), top, index_type_of(targets, "targets"),
          dense_type_of(rows, "log_probs")};
}

// logp, entropy, top log probabilities, top ids.
variable_list log_probs_forward(const at::Tensor& logits, const at::Tensor& targets, int64_t top, at::Tensor* stats) {
  c10::DeviceGuard guard(logits.device());
  const at::Tensor rows = flat_rows(logits, leading(logits)), t = targets.contiguous();
  const spmm_log_probs_desc d = log_probs_desc(rows, t, top);
  size_t bytes = 0;
  raise_status(spmm_log_probs_workspace(&d, &bytes), "log_probs");
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor logp = at::empty(targets.sizes(), f32), entropy = at::empty(targets.sizes(), f32);
  at::Tensor values = at::empty(leading_sizes(logits, top), f32);
  at::Tensor ids = at::empty(leading_sizes(logits, top), f32.dtype(at::kInt));
  if (stats != nullptr) *stats = at::empty({d.rows, 2}, f32);
  at::Tensor ws = scratch(logits, bytes);
  raise_status(spmm_log_probs_run(&d, rows.data_ptr(), t.data_ptr(), logp.data_ptr<float>(), entropy.data_ptr<float>(),
                                  values.data_ptr<float>(), ids.data_ptr<int32_t>(),
                                  stats != nullptr ? stats->data_ptr<float>() : nullptr, scratch_data(ws), bytes,
                                  current_stream(logits)),
               "log_probs");
  return {logp, entropy, values, ids};
}

struct LogProbs : torch::autograd::Function<LogProbs> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& targets, int64_t top) {
    at::Tensor stats;
    variable_list out = log_probs_forward(logits, targets, top, &stats);
    ctx->save_for_backward({logits, targets, out[1], stats});
    ctx->mark_non_differentiable({out[2], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_differentiable_once("log_probs");
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(3);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor& logits = saved[0];
    c10::DeviceGuard guard(logits.device());
    const at::Tensor rows = flat_rows(logits, leading(logits)), targets = saved[1].contiguous();
    const at::Tensor entropy = saved[2].contiguous();
    const at::Tensor glogp = grads[0].defined() ? grads[0].contiguous() : at::Tensor();
    const at::Tensor gentropy = grads[1].defined() ? grads[1].contiguous() : at::Tensor();
    const spmm_log_probs_desc d = log_probs_desc(rows, targets, 0);
    at::Tensor dlogits = at::empty(logits.sizes(), logits.options());
    raise_status(spmm_log_probs_grad_run(&d, rows.data_ptr(), targets.data_ptr(), saved[3].data_ptr<float>(),
                                         entropy.data_ptr<float>(),
                                         glogp.defined() ? glogp.data_ptr<float>() : nullptr,
                                         gentropy.defined() ? gentropy.data_ptr<float>() : nullptr,
                                         dlogits.data_ptr(), current_stream(logits)),
                 "log_probs");
    return {dlogits, at::Tensor(), at::Tensor()};
  }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> log_probs(const at::Tensor& logits,
                                                                     const at::Tensor& targets, int64_t top) {
  TORCH_CHECK_GPU(logits);
  TORCH_CHECK_GPU(targets);
  TORCH_CHECK(logits.dim() >= 1, "log_probs: logits must have at least one dimension");
  dense_type_of(logits, "log_probs");
  index_type_of(targets, "targets");
  check_no_tangent(logits, "log_probs");
  TORCH_CHECK(targets.device() == logits.device(), "log_probs: targets must be on the same device as logits");
  TORCH_CHECK(targets.sizes() == logits.sizes().slice(0, logits.dim() - 1), "log_probs: targets must have one entry for "
              "each row of logits (", logits.sizes().slice(0, logits.dim() - 1), "), but got ", targets.sizes());
  const variable_list out = wants_grad(logits) ? LogProbs::apply(logits, targets, top)
                                               : log_probs_forward(logits, targets, top, nullptr);
  return {out[0], out[1], out[2], out[3]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(myops, m) {
  m.def("embedding(Tensor weight, Tensor ids, float scale=1.0) -> Tensor", &embedding);
  m.def("route(Tensor logits, int top_k, int score=0, Tensor? bias=None, int groups=1, int top_groups=1, "
        "bool renormalize=True, float scale=1.0) -> (Tensor, Tensor)", &route);
  m.def("expert_plan(Tensor experts, int count) -> (Tensor, Tensor)", &expert_plan);
  m.def("expert_pack(Tensor x, Tensor place, Tensor offsets) -> Tensor", &expert_pack);
  m.def("expert_restore(Tensor results, Tensor weights, Tensor place, Tensor offsets) -> Tensor", &expert_restore);
  m.def("log_probs(Tensor logits, Tensor targets, int top=0) -> (Tensor, Tensor, Tensor, Tensor)", &log_probs);
}

void bind_expert_ops(pybind11::module_& m) {
  m.def("embedding", &embedding,
        R"doc(
    Rows of a table by ids, on the GPU: scale * weight[ids], of shape ids.shape +
    [width], and a row of zeros for an id outside of the table.  weight [rows,
    width] FP16, BF16 or FP32, ids int32 or int64.  Differentiable with respect
    to weight; its gradient adds in FP32 in the order of the ids, so that it
    repeats exactly.  A weight whose rows are not contiguous is copied whole by
    each call.
    )doc",
        pybind11::arg("weight"), pybind11::arg("ids"), pybind11::arg("scale") = 1.0);
  m.def("log_probs", &log_probs,
        R"doc(
    Log probabilities of given classes, on the GPU: for each row of logits
    [..., classes] (FP16, BF16 or FP32) and each target [...] (int32 or int64)
    returns the log probability of the target (0 for one outside of the classes),
    the entropy, and the log probabilities [..., top] and ids (int32) of the `top`
    likeliest classes, best first, ties to the lowest id.  Results are FP32.
    Classes with a logit of -inf or NaN are none of the likeliest: id -1, -inf.  A
    row of -inf alone has -inf, entropy 0 and no gradient.  The log probability of
    the target and the entropy are differentiable with respect to logits.
    )doc",
        pybind11::arg("logits"), pybind11::arg("targets"), pybind11::arg("top") = 0);
  m.def("route", &route, "Experts of rows from a router's logits (GPU)");
  m.def("expert_plan", &expert_plan, "Offsets and places of rows sorted by expert (GPU)");
  m.def("expert_pack", &expert_pack, "Rows at the places of their choices (GPU)");
  m.def("expert_restore", &expert_restore, "Weighted sums of the choices' rows (GPU)");
}
