// What stands around a layer's blocks, in the `flashMoeLauncher` extension: checks of the tensors, the autograd nodes, and the
// C ABI's calls on the current stream. `flash_distributed_moe_amd/flashLayerOp.py` is the Python surface above them.
#include "tensorChecks.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool differentiated(std::initializer_list<const at::Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
void refuse_second_derivatives(const char* name) {
  // Under create_graph the gradients would be taken for constants by whoever differentiates them again.
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivatives (create_graph=True)");
}
at::TensorOptions plain(const at::Tensor& like) { return like.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous); }

// ------------------------------------------------------------------ the router's choice
// Logits as rows, which may lie apart; copied where a row's values do.
Rows logit_rows(const at::Tensor& t, const char* name) {
  const int64_t width = t.size(-1), rows = t.numel() / width;
  at::Tensor flat = t.dim() == 2 ? t : t.reshape({rows, width});
  if (flat.numel() > 0 && (flat.stride(1) != 1 || (rows > 1 && (flat.stride(0) < width || flat.stride(0) > kMaxStride))))
    flat = flat.clone(at::MemoryFormat::Contiguous);
  return {flat, rows <= 1 ? width : flat.stride(0), int_size(rows, name)};
}

FlashMoeRouteDesc describe(const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
  TORCH_CHECK(logits.defined() && logits.is_cuda(), "logits must be a CUDA tensor (ROCm)");
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) >= 1, "logits must be [..., E]");
  FlashMoeRouteDesc d{};
  d.dtype = dtype_of(logits, "logits");
  d.experts = int_size(logits.size(-1), "E");
  TORCH_CHECK(d.experts <= 256, "E must be at most 256, not ", d.experts);
  TORCH_CHECK(top_k >= 1 && top_k <= std::min(d.experts, 32), "top_k must be 1 to min(E, 32), not ", top_k);
  d.top_k = static_cast<int>(top_k);
  d.renormalize = renormalize;
  if (mask.has_value()) {
    check_device(*mask, "mask", logits);
    TORCH_CHECK(mask->scalar_type() == at::kBool, "mask must be bool");
    TORCH_CHECK(mask->sizes() == logits.sizes().slice(0, logits.dim() - 1), "mask must have the logits' leading dimensions");
  }
  return d;
}

struct Routed {
  at::Tensor weights, experts, counts, balance, zed, totals, mask;
};
Routed route_forward(const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
  refuse_tangent(logits, "logits");
  const FlashMoeRouteDesc d = describe(logits, top_k, renormalize, mask);
  const DeviceGuard guard(logits.device());
  const Rows rows = logit_rows(logits, "logits");
  Routed r;
  if (mask.has_value()) r.mask = mask->contiguous();
  auto sizes = logits.sizes().vec();
  sizes.back() = top_k;
  const auto floats = plain(logits).dtype(at::kFloat), ints = plain(logits).dtype(at::kInt);
  r.weights = at::empty(sizes, floats), r.experts = at::empty(sizes, ints);
  r.counts = at::empty({d.experts}, ints), r.totals = at::empty({2}, ints);
  r.balance = at::empty({}, floats), r.zed = at::empty({}, floats);
  size_t bytes = 0;
  check_hip(flashMoeRouteBytes(&d, rows.count, &bytes), "flashMoeRouteBytes");
  at::Tensor work;
  if (bytes > 0) work = bytes_on(logits, bytes);
  check_hip(flashMoeRoute(&d, pointer(rows.t), rows.stride, static_cast<unsigned char*>(pointer(r.mask)), rows.count,
                          static_cast<float*>(pointer(r.weights)), static_cast<int*>(pointer(r.experts)), r.counts.data_ptr<int>(),
                          r.totals.data_ptr<int>(), r.balance.data_ptr<float>(), r.zed.data_ptr<float>(), pointer(work),
                          current_stream()),
            "flashMoeRoute");
  return r;
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
    const Routed r = route_forward(logits, top_k, renormalize, mask);
    ctx->save_for_backward({logits, r.mask, r.experts, r.counts, r.totals});
    ctx->saved_data["top_k"] = top_k;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->mark_non_differentiable({r.experts, r.counts});
    ctx->set_materialize_grads(false);
    return {r.weights, r.experts, r.counts, r.balance, r.zed};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_derivatives("route");
    const auto kept = ctx->get_saved_variables();
    const at::Tensor &logits = kept[0], &mask = kept[1];
    const FlashMoeRouteDesc d = describe(logits, ctx->saved_data["top_k"].toInt(), ctx->saved_data["renormalize"].toBool(), c10::nullopt);
    const DeviceGuard guard(logits.device());
    const Rows rows = logit_rows(logits, "logits");
    at::Tensor dw = grads[0].defined() ? grads[0].contiguous() : at::Tensor();
    at::Tensor out = at::empty(logits.sizes(), plain(logits));
    const auto floats = [](const at::Tensor& t) { return static_cast<const float*>(pointer(t)); };
    check_hip(flashMoeRouteBackward(&d, pointer(rows.t), rows.stride, static_cast<unsigned char*>(pointer(mask)), rows.count,
                                    static_cast<int*>(pointer(kept[2])), kept[3].data_ptr<int>(), kept[4].data_ptr<int>(), floats(dw),
                                    floats(grads[3]), floats(grads[4]), pointer(out), d.experts, current_stream()),
              "flashMoeRouteBackward");
    return {out, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

variable_list route(const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
  TORCH_CHECK(logits.defined(), "logits tensor is undefined");
  if (!differentiated({&logits})) {
    Routed r = route_forward(logits, top_k, renormalize, mask);
    return {r.weights, r.experts, r.counts, r.balance, r.zed};
  }
  if (logits.is_cuda()) {
    const DeviceGuard guard(logits.device());
    if (capturing()) check_capture_behind(logits, "logits");
  }
  return Route::apply(logits, top_k, renormalize, mask);
}

}  // namespace

void bind_layer(py::module_& m) {
  m.def("route", &route, py::arg("logits"), py::arg("top_k"), py::arg("renormalize"), py::arg("mask"),
        py::call_guard<py::gil_scoped_release>());
}
