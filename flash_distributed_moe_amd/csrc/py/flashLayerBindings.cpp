// What stands around a layer's blocks, in the `flashMoeLauncher` extension: checks of the tensors, the autograd nodes, and the
// C ABI's calls on the current stream. `flash_distributed_moe_amd/flashLayerOp.py` is the Python surface above them.
#include <ATen/hip/EmptyTensor.h>

#include "tensorChecks.h"

#include <torch/csrc/autograd/python_variable.h>

// A number of a call. A tensor of one value would be taken for the number that it holds, and whoever learns it would get no gradient.
struct Number {
  double value;
};
namespace pybind11::detail {
template <>
struct type_caster<Number> {
  PYBIND11_TYPE_CASTER(Number, const_name("float"));
  bool load(handle source, bool convert) {
    TORCH_CHECK(PyFloat_Check(source.ptr()) || !THPVariable_Check(source.ptr()) || !at::GradMode::is_enabled() ||
                    !THPVariable_Unpack(source.ptr()).requires_grad(),
                "the scales and eps are numbers: there is no gradient of a tensor in their place");
    make_caster<double> number;
    if (!number.load(source, convert)) return false;
    value.value = cast_op<double>(number);
    return true;
  }
};
}  // namespace pybind11::detail

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
// An upstream gradient; torch's zeros without memory are as good as none.
at::Tensor upstream(const at::Tensor& t) { return t.defined() && t._is_zerotensor() ? at::Tensor() : t; }
// New memory on `like`'s device, without gaps. (Past the dispatcher, which takes as long again: the smallest calls are
// bound by the host, and make up to six of these.)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt));
}
at::Tensor fresh(const at::Tensor& like) { return fresh(like.sizes(), like.scalar_type(), like); }
at::Tensor fresh_bytes(size_t bytes, const at::Tensor& like) { return fresh({static_cast<int64_t>(bytes)}, at::kByte, like); }

// ------------------------------------------------------------------ the router's choice
// Logits as rows, which may lie apart; copied where a row's values do.
Rows logit_rows(const at::Tensor& t, const char* name) {
  const int64_t width = t.size(-1), rows = t.numel() / width;
  at::Tensor flat = t.dim() == 2 ? t : t.reshape({rows, width});
  if (flat.numel() > 0 && (flat.stride(1) != 1 || flat.is_neg() || (rows > 1 && (flat.stride(0) < width || flat.stride(0) > kMaxStride))))
    flat = flat.clone(at::MemoryFormat::Contiguous);
  return {flat, rows <= 1 ? width : flat.stride(0), int_size(rows, name)};
}

FlashMoeRouteDesc describe(const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
  TORCH_CHECK(logits.defined() && logits.is_cuda(), "logits must be a CUDA tensor (ROCm)");
  check_memory(logits, "logits");
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
  at::Tensor weights, experts, counts, balance, zed, kept, mask;
};
Routed route_forward(const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask, bool keep) {
  refuse_tangent(logits, "logits");
  const FlashMoeRouteDesc d = describe(logits, top_k, renormalize, mask);
  const DeviceGuard guard(logits.device());
  const Rows rows = logit_rows(logits, "logits");
  Routed r;
  if (mask.has_value()) r.mask = mask->contiguous();
  auto sizes = logits.sizes().vec();
  sizes.back() = top_k;
  r.weights = fresh(sizes, at::kFloat, logits), r.experts = fresh(sizes, at::kInt, logits);
  r.counts = fresh({d.experts}, at::kInt, logits);
  if (keep) r.kept = fresh({2 + d.experts}, at::kInt, logits);
  r.balance = fresh({}, at::kFloat, logits), r.zed = fresh({}, at::kFloat, logits);
  size_t bytes = 0;
  check_hip(flashMoeRouteBytes(&d, rows.count, &bytes), "flashMoeRouteBytes");
  at::Tensor work;
  if (bytes > 0) work = fresh_bytes(bytes, logits);
  check_hip(flashMoeRoute(&d, pointer(rows.t), rows.stride, static_cast<unsigned char*>(pointer(r.mask)), rows.count,
                          static_cast<float*>(pointer(r.weights)), static_cast<int*>(pointer(r.experts)), r.counts.data_ptr<int>(),
                          r.balance.data_ptr<float>(), r.zed.data_ptr<float>(), static_cast<int*>(pointer(r.kept)), pointer(work),
                          current_stream()),
            "flashMoeRoute");
  return r;
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
    const Routed r = route_forward(logits, top_k, renormalize, mask, true);
    // the counts are kept apart: a caller may well add those of other ranks to what is returned
    ctx->save_for_backward({logits, r.mask, r.experts, r.kept, r.weights});
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
    // as they are in memory: torch may hand a gradient over that is negated when it is read
    const auto plain = [](const at::Tensor& given) {
      const at::Tensor t = upstream(given);
      return !t.defined() ? t : t.is_neg() ? t.contiguous().resolve_neg() : t.contiguous();
    };
    const at::Tensor dw = plain(grads[0]), db = plain(grads[3]), dz = plain(grads[4]);
    at::Tensor out = fresh(logits);
    const auto floats = [](const at::Tensor& t) { return static_cast<const float*>(pointer(t)); };
    check_hip(flashMoeRouteBackward(&d, pointer(rows.t), rows.stride, static_cast<unsigned char*>(pointer(mask)), rows.count,
                                    floats(kept[4]), static_cast<int*>(pointer(kept[2])), kept[3].data_ptr<int>(), floats(dw), floats(db),
                                    floats(dz), pointer(out), d.experts, current_stream()),
              "flashMoeRouteBackward");
    return {out, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

variable_list route(const at::Tensor& logits, int64_t top_k, bool renormalize, const OptTensor& mask) {
  TORCH_CHECK(logits.defined(), "logits tensor is undefined");
  if (!differentiated({&logits})) {
    Routed r = route_forward(logits, top_k, renormalize, mask, false);
    return {r.weights, r.experts, r.counts, r.balance, r.zed};
  }
  if (logits.is_cuda()) {
    const DeviceGuard guard(logits.device());
    if (capturing()) check_capture_behind(logits, "logits");
  }
  return Route::apply(logits, top_k, renormalize, mask);
}

// ------------------------------------------------------------------ the norms around a block
void check_vector(const at::Tensor& t, const char* name, const at::Tensor& x) {
  if (!t.defined()) return;
  check_device(t, name, x);
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have x's dtype");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), name, " must be [H] with H = ", x.size(-1));
  check_packed(t, name);
}

// How a gate is shared among x's rows: its leading dimensions are x's up to some one, and ones from there.
void describe_gate(FlashMoeNormDesc& d, const at::Tensor& gate, const at::Tensor& x, int64_t rows) {
  check_device(gate, "gate", x);
  TORCH_CHECK(gate.scalar_type() == x.scalar_type(), "gate must have x's dtype");
  TORCH_CHECK(gate.dim() >= 1 && gate.dim() <= x.dim(), "gate must not have more dimensions than x");
  const int64_t width = gate.size(-1), missing = x.dim() - gate.dim();
  TORCH_CHECK(width == x.size(-1) || width == 1, "gate's last dimension must be x's or 1");
  int64_t own = 1;
  bool shared = false;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) {
    const int64_t n = i < missing ? 1 : gate.size(i - missing);
    TORCH_CHECK(n == x.size(i) ? !shared || n == 1 : n == 1,
                "gate's leading dimensions must be x's up to some one, and 1 from there");
    if (n != x.size(i)) shared = true;
    own *= n;
  }
  TORCH_CHECK(width != 1 || own == rows, "a gate of one value a token must have x's leading dimensions");
  d.gate = width == 1 ? FLASH_MOE_GATE_TOKEN : own == 1 ? FLASH_MOE_GATE_CHANNEL : own == rows ? FLASH_MOE_GATE_FULL : FLASH_MOE_GATE_GROUP;
  d.shared = d.gate == FLASH_MOE_GATE_GROUP && rows > 0 ? static_cast<int>(rows / own) : 1;
}

struct NormInputs {
  at::Tensor x, branch, post, gate, next;
};
at::Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
struct NormCall {
  FlashMoeNormDesc d;
  Rows x, branch;
  at::Tensor gate;
};
NormCall prepare(const NormInputs& in, double alpha, double beta, double eps) {
  TORCH_CHECK(in.x.defined() && in.x.is_cuda(), "x must be a CUDA tensor (ROCm)");
  TORCH_CHECK(in.x.dim() >= 1, "x must be [..., H]");
  NormCall c{};
  c.d.dtype = dtype_of(in.x, "x");
  c.d.hidden = int_size(in.x.size(-1), "H");
  TORCH_CHECK(c.d.hidden >= 8 && c.d.hidden % 8 == 0 && c.d.hidden <= 8192, "H must be a multiple of 8, at most 8192, not ", c.d.hidden);
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  c.d.eps = eps, c.d.residual_scale = alpha, c.d.branch_scale = beta;
  check_vector(in.post, "post_weight", in.x);
  check_vector(in.next, "the next norm's weight", in.x);
  c.x = rows_of(in.x, "x");
  if (in.branch.defined()) {
    check_device(in.branch, "branch", in.x);
    TORCH_CHECK(in.branch.sizes() == in.x.sizes() && in.branch.scalar_type() == in.x.scalar_type(), "branch must have x's shape and dtype");
    c.branch = rows_of(in.branch, "branch");
  }
  if (in.gate.defined()) {
    describe_gate(c.d, in.gate, in.x, c.x.count);
    if (c.x.count == 0 && c.d.gate != FLASH_MOE_GATE_CHANNEL) c.d.gate = FLASH_MOE_GATE_NONE;  // no rows to have one
    c.gate = in.gate.contiguous();
    if (!begins_on_16(c.gate) || c.gate.is_neg()) c.gate = c.gate.clone();
    if (c.d.gate != FLASH_MOE_GATE_NONE) c.d.gate_values = c.gate.data_ptr();
  }
  c.d.post_weight = pointer(in.post), c.d.next_weight = pointer(in.next);
  return c;
}

// (y, h, kept), undefined where there is none
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_forward(const NormInputs& in, double alpha, double beta, double eps, bool keep) {
  refuse_tangent(in.x, "x");
  refuse_tangent(in.branch, "branch");
  refuse_tangent(in.post, "post_weight");
  refuse_tangent(in.gate, "gate");
  refuse_tangent(in.next, "the next norm's weight");
  TORCH_CHECK(in.x.defined() && in.x.is_cuda(), "x must be a CUDA tensor (ROCm)");
  check_memory(in.x, "x");
  const DeviceGuard guard(in.x.device());
  const NormCall c = prepare(in, alpha, beta, eps);
  at::Tensor y, h, kept;
  if (in.branch.defined()) y = fresh(in.x);
  if (in.next.defined()) h = fresh(in.x);
  if (keep) kept = fresh({2, c.x.count}, at::kFloat, in.x);
  check_hip(flashMoeBlockNorm(&c.d, pointer(c.x.t), c.x.stride, pointer(c.branch.t), c.branch.stride, c.x.count, pointer(y), pointer(h),
                              static_cast<float*>(pointer(kept)), current_stream()),
            "flashMoeBlockNorm");
  return {y, h, kept};
}

struct BlockNorm : torch::autograd::Function<BlockNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& branch, const OptTensor& post,
                               const OptTensor& gate, const OptTensor& next, double alpha, double beta, double eps) {
    const NormInputs in{x, or_none(branch), or_none(post), or_none(gate), or_none(next)};
    const auto [y, h, kept] = norm_forward(in, alpha, beta, eps, true);
    ctx->save_for_backward({in.x, in.branch, in.post, in.gate, in.next, kept});
    ctx->saved_data["alpha"] = alpha;
    ctx->saved_data["beta"] = beta;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    if (!y.defined()) return {h};
    if (!h.defined()) return {y};
    return {y, h};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_derivatives("block_norm and block_join");
    const auto kept = ctx->get_saved_variables();
    const NormInputs in{kept[0], kept[1], kept[2], kept[3], kept[4]};
    const DeviceGuard guard(in.x.device());
    const NormCall c = prepare(in, ctx->saved_data["alpha"].toDouble(), ctx->saved_data["beta"].toDouble(), ctx->saved_data["eps"].toDouble());
    const at::Tensor dy = in.branch.defined() ? upstream(grads[0]) : at::Tensor(), dh = in.next.defined() ? upstream(grads.back()) : at::Tensor();
    Rows dys{}, dhs{};
    if (dy.defined()) dys = rows_of(dy, "dy");
    if (dh.defined()) dhs = rows_of(dh, "dh");
    variable_list out(8);
    for (int i = 0, present = 0; i < 5; ++i)  // inputs that are not there have no place in the node
      if (kept[i].defined() && ctx->needs_input_grad(present++)) out[i] = fresh(kept[i]);
    void* dgate = pointer(out[3]);
    if (dgate != nullptr && c.d.gate == FLASH_MOE_GATE_NONE) out[3].zero_(), dgate = nullptr;
    size_t bytes = 0;
    check_hip(flashMoeBlockNormBytes(&c.d, c.x.count, &bytes), "flashMoeBlockNormBytes");
    const at::Tensor work = fresh_bytes(bytes, in.x);
    check_hip(flashMoeBlockNormBackward(&c.d, pointer(c.x.t), c.x.stride, pointer(c.branch.t), c.branch.stride, pointer(dys.t), dys.stride,
                                        pointer(dhs.t), dhs.stride, c.x.count, static_cast<float*>(pointer(kept[5])), pointer(work),
                                        pointer(out[0]), pointer(out[1]), pointer(out[2]), dgate, pointer(out[4]), current_stream()),
              "flashMoeBlockNormBackward");
    return out;
  }
};

variable_list block_norm(const at::Tensor& x, const OptTensor& branch, const OptTensor& post, const OptTensor& gate, const OptTensor& next,
                         Number residual_scale, Number branch_scale, Number epsilon) {
  const NormInputs in{x, or_none(branch), or_none(post), or_none(gate), or_none(next)};
  const double alpha = residual_scale.value, beta = branch_scale.value, eps = epsilon.value;
  TORCH_CHECK(in.x.defined(), "x tensor is undefined");
  if (!differentiated({&in.x, &in.branch, &in.post, &in.gate, &in.next})) {
    const auto [y, h, kept] = norm_forward(in, alpha, beta, eps, false);
    if (!y.defined()) return {h};
    if (!h.defined()) return {y};
    return {y, h};
  }
  if (x.is_cuda()) {
    const DeviceGuard guard(x.device());
    if (capturing()) {
      check_capture_behind(in.x, "x");
      check_capture_behind(in.branch, "branch");
      check_capture_behind(in.post, "post_weight");
      check_capture_behind(in.gate, "gate");
      check_capture_behind(in.next, "the next norm's weight");
    }
  }
  return BlockNorm::apply(x, branch, post, gate, next, alpha, beta, eps);
}

// ------------------------------------------------------------------ adapters beside a projection
// Whether two sets of rows share no memory: behind one another, or columns of the same rows side by side.
bool apart(const Rows& a, const Rows& b) {
  if (a.count == 0 || b.count == 0) return true;
  const int64_t size = a.t.element_size(), wa = a.t.size(-1) * size, wb = b.t.size(-1) * size;
  const int64_t pa = reinterpret_cast<int64_t>(a.t.data_ptr()), pb = reinterpret_cast<int64_t>(b.t.data_ptr());
  const int64_t la = a.stride * size, lb = b.stride * size;
  if (pa + (a.count - 1) * la + wa <= pb || pb + (b.count - 1) * lb + wb <= pa) return true;
  if (la != lb) return false;
  const int64_t d = ((pb - pa) % la + la) % la;
  return d >= wa && d + wb <= la;
}

// Whether rows end before t begins, or begin behind its last value; t may have gaps.
bool behind(const Rows& a, const at::Tensor& t) {
  if (a.count == 0 || t.numel() == 0) return true;
  int64_t values = 1;
  for (int64_t i = 0; i < t.dim(); ++i) values += (t.size(i) - 1) * t.stride(i);
  const int64_t size = a.t.element_size(), pa = reinterpret_cast<int64_t>(a.t.data_ptr()), pt = reinterpret_cast<int64_t>(t.data_ptr());
  return pa + ((a.count - 1) * a.stride + a.t.size(-1)) * size <= pt || pt + values * t.element_size() <= pa;
}

at::Tensor add_adapters(const at::Tensor& y, const at::Tensor& x, const at::Tensor& down, const at::Tensor& up, const at::Tensor& scales,
                        const at::Tensor& ids, const OptTensor& out) {
  for (const at::Tensor* t : {&y, &x, &down, &up, &scales}) refuse_tangent(*t, "an input");
  if (out.has_value()) refuse_tangent(*out, "out");
  TORCH_CHECK(!differentiated({&y, &x, &down, &up, &scales}), "adapters have no backward pass: detach the inputs or use torch.no_grad()");
  TORCH_CHECK(x.defined() && x.is_cuda(), "x must be a CUDA tensor (ROCm)");
  check_memory(x, "x");
  check_device(y, "y", x);
  check_device(down, "down", x);
  check_device(up, "up", x);
  check_device(scales, "scales", x);
  check_device(ids, "ids", x);
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>{y, "y"}, {x, "x"}, {down, "down"}, {up, "up"}})
    TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bfloat16");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous(), "scales must be float32 without gaps");
  TORCH_CHECK(!scales.is_neg(), "scales must not be a negated view");
  TORCH_CHECK(ids.scalar_type() == at::kInt, "ids must be int32");
  TORCH_CHECK(down.dim() == 3 && up.dim() == 3 && scales.dim() == 1 && down.size(0) == up.size(0) && down.size(0) == scales.size(0) &&
                  down.size(1) == up.size(2),
              "adapters must be down [adapters, r, K], up [adapters, N, r] and scales [adapters]");
  check_packed(down, "down");
  check_packed(up, "up");
  FlashMoeAdapterDesc d{};
  d.adapters = int_size(down.size(0), "adapters"), d.rank = int_size(down.size(1), "rank");
  d.n = int_size(up.size(1), "N"), d.k = int_size(down.size(2), "K");
  TORCH_CHECK(d.adapters >= 1 && d.adapters <= 1000, "1 to 1000 adapters, not ", d.adapters);
  TORCH_CHECK(d.rank >= 8 && d.rank <= 128 && d.rank % 8 == 0, "the rank must be a multiple of 8, at most 128, not ", d.rank);
  TORCH_CHECK(d.n >= 8 && d.n % 8 == 0 && d.k >= 8 && d.k % 8 == 0, "N and K must be multiples of 8, not ", d.n, " and ", d.k);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == d.k, "x must be [..., K] with K = ", d.k);
  TORCH_CHECK(y.dim() == x.dim() && y.size(-1) == d.n, "y must be [..., N] with N = ", d.n);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  TORCH_CHECK(y.sizes().slice(0, y.dim() - 1) == lead && ids.sizes() == lead, "x, y and ids must have the same leading dimensions");
  d.down = down.data_ptr(), d.up = up.data_ptr(), d.scales = scales.data_ptr<float>();
  const DeviceGuard guard(x.device());
  const Rows xs = rows_of(x, "x"), ys = rows_of(y, "y");
  at::Tensor result;
  Rows outs;
  if (out.has_value()) {
    result = *out;
    check_device(result, "out", x);
    TORCH_CHECK(result.sizes() == y.sizes() && result.scalar_type() == y.scalar_type(), "out must have y's shape and dtype");
    TORCH_CHECK(!result.requires_grad() || !at::GradMode::is_enabled(), "out requires a gradient");
    outs = rows_of(result, "out");
    TORCH_CHECK(outs.t.data_ptr() == result.data_ptr(), "out must have rows without gaps that begin on 16 bytes");
    const bool itself = result.is_same(y) || (pointer(ys.t) == pointer(outs.t) && ys.stride == outs.stride);
    TORCH_CHECK(itself || apart(outs, ys), "out must be y or apart from it");
    TORCH_CHECK(apart(outs, xs), "out must be apart from x");
    for (const at::Tensor* t : {&down, &up, &scales, &ids}) TORCH_CHECK(behind(outs, *t), "out must be apart from the adapters and ids");
  } else {
    result = fresh(y);
    outs = rows_of(result, "out");
  }
  const at::Tensor which = ids.contiguous();
  size_t bytes = 0;
  check_hip(flashMoeAdapterBytes(&d, xs.count, &bytes), "flashMoeAdapterBytes");
  const at::Tensor work = fresh_bytes(bytes, x);
  check_hip(flashMoeAdapterAdd(&d, pointer(xs.t), xs.stride, pointer(ys.t), ys.stride, static_cast<int*>(pointer(which)), xs.count,
                               pointer(outs.t), outs.stride, pointer(work), current_stream()),
            "flashMoeAdapterAdd");
  if (out.has_value() && !result.is_inference()) torch::autograd::impl::bump_version(result);  // for whoever saved what was there
  return result;
}

}  // namespace

void bind_layer(py::module_& m) {
  m.def("route", &route, py::arg("logits"), py::arg("top_k"), py::arg("renormalize"), py::arg("mask"),
        py::call_guard<py::gil_scoped_release>());
  m.def("block_norm", &block_norm, py::arg("x"), py::arg("branch"), py::arg("post_weight"), py::arg("gate"), py::arg("next_weight"),
        py::arg("residual_scale"), py::arg("branch_scale"), py::arg("eps"), py::call_guard<py::gil_scoped_release>());
  m.def("add_adapters", &add_adapters, py::arg("y"), py::arg("x"), py::arg("down"), py::arg("up"), py::arg("scales"), py::arg("ids"),
        py::arg("out"), py::call_guard<py::gil_scoped_release>());
}
