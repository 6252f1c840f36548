// The dense gated feed-forward block and MXFP4 in the `flashMoeLauncher` extension: checks of the
// tensors, outputs and workspaces from torch's allocator, and the C ABI's calls on the current stream.
// `flash_distributed_moe_amd/flashFfnOp.py` is the Python surface above them.
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <hip/hip_runtime.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <limits>

#include "../../../include/flash_moe.h"

namespace py = pybind11;

namespace {

using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
using OptTensor = c10::optional<at::Tensor>;

void* current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

void check_hip(int e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, " failed: ", hipGetErrorString(static_cast<hipError_t>(e)), " (hipError_t ", e, ")");
}

void check_device(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.defined(), name, " tensor is undefined");
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (ROCm)");
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device(), ", not on ", t.device());
}

// A dual tensor's result would come back without a tangent, which stands for a zero one.
void refuse_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!t.defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), name,
              " carries a tangent: there are no forward-mode derivatives here");
}

int dtype_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, " must be float32 or bfloat16");
  return t.scalar_type() == at::kFloat ? FLASH_MOE_F32 : FLASH_MOE_BF16;
}

int int_size(int64_t v, const char* name) {
  TORCH_CHECK(v >= 0 && v <= std::numeric_limits<int>::max(), name, " is too large: ", v);
  return static_cast<int>(v);
}

bool begins_on_16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A weight or code tensor as the kernels read it: without gaps. (One that is a view into something
// larger, at an odd place, is refused rather than copied at every call.)
void check_packed(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(begins_on_16(t), name, " must begin on 16 bytes");
}

// t [..., width] as rows whose distance the kernels can take; copied where it cannot.
struct Rows {
  at::Tensor t;
  int64_t stride;
  int count;
};
constexpr int64_t kMaxStride = 1 << 20;
Rows rows_of(const at::Tensor& t, const char* name) {
  const int64_t width = t.size(-1), rows = width > 0 ? t.numel() / width : 0;
  at::Tensor flat = t.dim() == 2 ? t : t.reshape({rows, width});
  int64_t stride = flat.stride(0);
  const bool apart = rows <= 1 || (stride >= width && stride <= kMaxStride && stride * flat.element_size() % 16 == 0);
  if (flat.numel() > 0 && (flat.stride(1) != 1 || !apart || !begins_on_16(flat)))
    flat = flat.clone(at::MemoryFormat::Contiguous);
  stride = rows <= 1 ? width : flat.stride(0);
  return {flat, stride, int_size(rows, name)};
}

at::Tensor bytes_on(const at::Tensor& like, size_t bytes) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte).requires_grad(false));
}
void* pointer(const at::Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

// The description of a block, from its weights. x is used for its device and dtype.
FlashMoeFfnDesc describe(const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2, const OptTensor& s13,
                         const OptTensor& s2, int activation) {
  TORCH_CHECK(x.defined() && x.is_cuda(), "x must be a CUDA tensor (ROCm)");
  TORCH_CHECK(x.dim() >= 1, "x must be [..., hidden]");
  check_device(w13, "w13", x);
  check_device(w2, "w2", x);
  TORCH_CHECK(w13.dim() == 2 && w2.dim() == 2, "weights must be [2I, H] and [H, I]");
  FlashMoeFfnDesc d{};
  const bool mx = s13.has_value();
  TORCH_CHECK(mx == s2.has_value(), "both weights must be MXFP4, or neither");
  const int64_t per = mx ? 2 : 1;
  d.dtype = dtype_of(x, "x");
  d.hidden = int_size(w2.size(0), "hidden");
  d.intermediate = int_size(w2.size(1) * per, "intermediate");
  d.activation = activation;
  d.weights = mx ? FLASH_MOE_FFN_MXFP4 : FLASH_MOE_FFN_ROW_MAJOR;
  TORCH_CHECK(w13.size(0) == 2 * w2.size(1) * per && w13.size(1) * per == w2.size(0), "weights must be [2I, H] and [H, I]");
  TORCH_CHECK(x.size(-1) == d.hidden, "x must be [..., hidden] with hidden = ", d.hidden);
  check_packed(w13, "w13");
  check_packed(w2, "w2");
  if (mx) {
    TORCH_CHECK(w13.scalar_type() == at::kByte && w2.scalar_type() == at::kByte, "MXFP4 codes must be uint8");
    check_device(*s13, "w13 scales", x);
    check_device(*s2, "w2 scales", x);
    TORCH_CHECK(s13->scalar_type() == at::kByte && s2->scalar_type() == at::kByte, "MXFP4 scales must be uint8");
    TORCH_CHECK(s13->dim() == 2 && s13->size(0) == w13.size(0) && s13->size(1) * 16 == w13.size(1) && s2->dim() == 2 &&
                    s2->size(0) == w2.size(0) && s2->size(1) * 16 == w2.size(1),
                "MXFP4 scales must be [rows, k / 32]");
    TORCH_CHECK(s13->is_contiguous() && s2->is_contiguous(), "MXFP4 scales must be contiguous");
    TORCH_CHECK(d.dtype == FLASH_MOE_BF16, "MXFP4 weights take bfloat16 x");
    d.w13_scales = s13->data_ptr();
    d.w2_scales = s2->data_ptr();
  } else {
    TORCH_CHECK(w13.scalar_type() == x.scalar_type() && w2.scalar_type() == x.scalar_type(),
                "x and the weights must share one dtype");
  }
  d.w13 = w13.data_ptr();
  d.w2 = w2.data_ptr();
  return d;
}

// (y, saved): saved is undefined unless `save`
std::tuple<at::Tensor, at::Tensor> ffn_forward(const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2,
                                               const OptTensor& s13, const OptTensor& s2, int activation, bool save) {
  refuse_tangent(x, "x");
  refuse_tangent(w13, "w13");
  refuse_tangent(w2, "w2");
  const FlashMoeFfnDesc d = describe(x, w13, w2, s13, s2, activation);
  const DeviceGuard guard(x.device());
  const Rows rows = rows_of(x, "x");
  size_t saved_bytes = 0, work_bytes = 0;
  check_hip(flashMoeFfnBytes(&d, rows.count, save ? &saved_bytes : nullptr, save ? nullptr : &work_bytes, nullptr),
            "flashMoeFfnBytes");
  if (save) check_hip(flashMoeFfnSavingBytes(&d, rows.count, &work_bytes), "flashMoeFfnSavingBytes");
  at::Tensor y = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
  at::Tensor saved, work;
  if (save) saved = bytes_on(x, saved_bytes);
  if (work_bytes > 0) work = bytes_on(x, work_bytes);
  check_hip(flashMoeFfnForward(&d, pointer(rows.t), rows.stride, pointer(y), d.hidden, rows.count, pointer(saved),
                               pointer(work), current_stream()),
            "flashMoeFfnForward");
  return {y, saved};
}

// (dx, dw13, dw2), undefined where not asked for
std::tuple<at::Tensor, at::Tensor, at::Tensor> ffn_backward(const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2,
                                                            int activation, const at::Tensor& dy, const at::Tensor& saved,
                                                            bool want_dx, bool want_dw13, bool want_dw2) {
  const FlashMoeFfnDesc d = describe(x, w13, w2, c10::nullopt, c10::nullopt, activation);
  check_device(dy, "dy", x);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "dy must have x's shape and dtype");
  const DeviceGuard guard(x.device());
  const Rows rows = rows_of(x, "x"), grad = rows_of(dy, "dy");
  size_t saved_bytes = 0, work_bytes = 0;
  check_hip(flashMoeFfnBytes(&d, rows.count, &saved_bytes, nullptr, &work_bytes), "flashMoeFfnBytes");
  check_device(saved, "saved", x);
  TORCH_CHECK(saved.scalar_type() == at::kByte && saved.is_contiguous() &&
                  static_cast<size_t>(saved.numel()) >= saved_bytes,
              "saved is not what a forward pass of this block and batch left");
  const auto plain = x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor dx, dw13, dw2, work;
  if (want_dx) dx = at::empty(x.sizes(), plain);
  if (want_dw13) dw13 = at::empty(w13.sizes(), plain);
  if (want_dw2) dw2 = at::empty(w2.sizes(), plain);
  if (want_dx || want_dw13) work = bytes_on(x, work_bytes);
  check_hip(flashMoeFfnBackward(&d, pointer(rows.t), rows.stride, pointer(grad.t), grad.stride, rows.count, pointer(saved),
                                pointer(work), pointer(dx), d.hidden, pointer(dw13), pointer(dw2), current_stream()),
            "flashMoeFfnBackward");
  return {dx, dw13, dw2};
}

// A gradient of a leaf is accumulated on the stream on which its accumulator was made, by the first graph of it
// that is still alive. Captured into a HIP graph, a backward pass that finds an accumulator of another
// stream would make that stream wait inside the capture, and the process ends. So the forward pass that
// would lead there is refused.
void check_capture(const at::Tensor& leaf, const char* name) {
  if (!leaf.requires_grad() || !leaf.is_leaf()) return;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!accumulator) return;
  const auto stream = accumulator->stream();
  TORCH_CHECK(!stream.has_value() || *stream == c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().unwrap(), name,
              " is part of an autograd graph made on another stream that is still alive: drop it before a step is captured");
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w13,
                            const at::Tensor& w2, int64_t activation) {
    auto [y, saved] = ffn_forward(x, w13, w2, c10::nullopt, c10::nullopt, static_cast<int>(activation), true);
    ctx->save_for_backward({x, w13, w2, saved});
    ctx->saved_data["activation"] = activation;
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    // Under create_graph the gradients would be taken for constants by whoever differentiates them again.
    TORCH_CHECK(!at::GradMode::is_enabled(), "gated_ffn has no second derivatives (create_graph=True)");
    const auto kept = ctx->get_saved_variables();
    auto [dx, dw13, dw2] =
        ffn_backward(kept[0], kept[1], kept[2], static_cast<int>(ctx->saved_data["activation"].toInt()), grads[0], kept[3],
                     ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2));
    return {dx, dw13, dw2, at::Tensor()};
  }
};

at::Tensor gated_ffn(const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2, int activation) {
  TORCH_CHECK(x.defined() && w13.defined() && w2.defined(), "x or a weight tensor is undefined");
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || w13.requires_grad() || w2.requires_grad()))
    return std::get<0>(ffn_forward(x, w13, w2, c10::nullopt, c10::nullopt, activation, false));
  if (x.is_cuda()) {
    const DeviceGuard guard(x.device());
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    check_hip(hipStreamIsCapturing(static_cast<hipStream_t>(current_stream()), &capturing), "hipStreamIsCapturing");
    if (capturing != hipStreamCaptureStatusNone) {
      check_capture(x, "x");
      check_capture(w13, "w13");
      check_capture(w2, "w2");
    }
  }
  return GatedFfn::apply(x, w13, w2, static_cast<int64_t>(activation));
}

std::tuple<at::Tensor, at::Tensor> mxfp4_quantize(const at::Tensor& x) {
  TORCH_CHECK(x.defined() && x.is_cuda(), "x must be a CUDA tensor (ROCm)");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0 && x.size(-1) % 32 == 0, "x must be [..., K], K a multiple of 32");
  const int dtype = dtype_of(x, "x"), k = int_size(x.size(-1), "K");
  const DeviceGuard guard(x.device());
  const Rows rows = rows_of(x, "x");
  auto sizes = x.sizes().vec();
  const auto bytes = x.options().dtype(at::kByte).requires_grad(false).memory_format(at::MemoryFormat::Contiguous);
  sizes.back() = k / 2;
  at::Tensor codes = at::empty(sizes, bytes);
  sizes.back() = k / 32;
  at::Tensor scales = at::empty(sizes, bytes);
  check_hip(flashMoeMxfp4Quantize(dtype, pointer(rows.t), rows.stride, rows.count, k, pointer(codes), pointer(scales),
                                  current_stream()),
            "flashMoeMxfp4Quantize");
  return {codes, scales};
}

// codes [..., K / 2] and scales [..., K / 32]; returns K
int check_mxfp4(const at::Tensor& codes, const at::Tensor& scales, const char* name) {
  TORCH_CHECK(codes.defined() && codes.is_cuda(), name, " codes must be a CUDA tensor (ROCm)");
  check_device(scales, "scales", codes);
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, name, " codes and scales must be uint8");
  TORCH_CHECK(codes.dim() >= 1 && codes.dim() == scales.dim() && codes.size(-1) > 0 && codes.size(-1) == scales.size(-1) * 16,
              name, " must be codes [..., K / 2] and scales [..., K / 32]");
  for (int64_t i = 0; i + 1 < codes.dim(); ++i)
    TORCH_CHECK(codes.size(i) == scales.size(i), name, " codes and scales must have the same rows");
  check_packed(codes, name);
  TORCH_CHECK(scales.is_contiguous(), name, " scales must be contiguous");
  return int_size(codes.size(-1) * 2, "K");
}

at::Tensor mxfp4_dequantize(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
  const int k = check_mxfp4(codes, scales, "MXFP4");
  TORCH_CHECK(dtype == at::kFloat || dtype == at::kBFloat16, "dtype must be float32 or bfloat16");
  const DeviceGuard guard(codes.device());
  auto sizes = codes.sizes().vec();
  sizes.back() = k;
  at::Tensor out = at::empty(sizes, codes.options().dtype(dtype));
  check_hip(flashMoeMxfp4Dequantize(dtype == at::kFloat ? FLASH_MOE_F32 : FLASH_MOE_BF16, pointer(codes), pointer(scales),
                                    int_size(codes.numel() * 2 / k, "rows"), k, pointer(out), k, current_stream()),
            "flashMoeMxfp4Dequantize");
  return out;
}

at::Tensor mxfp4_linear(const at::Tensor& x, const OptTensor& x_scales, const at::Tensor& codes, const at::Tensor& scales) {
  refuse_tangent(x, "x");
  const int k = check_mxfp4(codes, scales, "weights");
  TORCH_CHECK(codes.dim() == 2, "weights must be MXFP4 [N, K]");
  check_device(x, "x", codes);
  const DeviceGuard guard(codes.device());
  const bool mx = x_scales.has_value();
  Rows rows;
  if (mx) {
    TORCH_CHECK(check_mxfp4(x, *x_scales, "x") == k, "x must have K = ", k, " values a row");
    rows = {x, k, int_size(x.numel() * 2 / k, "rows")};
  } else {
    TORCH_CHECK(x.scalar_type() == at::kBFloat16, "x must be bfloat16 or MXFP4");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) == k, "x must be [..., K] with K = ", k);
    rows = rows_of(x, "x");
  }
  const int n = int_size(codes.size(0), "N");
  auto sizes = x.sizes().vec();
  sizes.back() = n;
  at::Tensor y = at::empty(sizes, codes.options().dtype(at::kBFloat16));
  const int format = mx ? static_cast<int>(FLASH_MOE_MXFP4) : static_cast<int>(FLASH_MOE_BF16);
  size_t work_bytes = 0;
  check_hip(flashMoeMxfp4LinearBytes(format, rows.count, n, k, &work_bytes), "flashMoeMxfp4LinearBytes");
  at::Tensor work;
  if (work_bytes > 0) work = bytes_on(codes, work_bytes);
  check_hip(flashMoeMxfp4Linear(format, pointer(rows.t), mx ? x_scales->data_ptr() : nullptr, rows.stride, rows.count,
                                pointer(codes), pointer(scales), n, k, pointer(y), n, pointer(work), current_stream()),
            "flashMoeMxfp4Linear");
  return y;
}

}  // namespace

void bind_ffn(py::module_& m) {
  m.attr("ACT_SILU") = static_cast<int>(FLASH_MOE_ACT_SILU);
  m.attr("ACT_GELU_TANH") = static_cast<int>(FLASH_MOE_ACT_GELU_TANH);
  m.def("gated_ffn", &gated_ffn, py::arg("x"), py::arg("w13"), py::arg("w2"), py::arg("activation"),
        py::call_guard<py::gil_scoped_release>());
  m.def("gated_ffn_mxfp4",
        [](const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w2, const at::Tensor& w13_scales, const at::Tensor& w2_scales,
           int activation) { return std::get<0>(ffn_forward(x, w13, w2, w13_scales, w2_scales, activation, false)); },
        py::arg("x"), py::arg("w13"), py::arg("w2"), py::arg("w13_scales"), py::arg("w2_scales"), py::arg("activation"));
  m.def("mxfp4_quantize", &mxfp4_quantize, py::arg("x"));
  m.def("mxfp4_dequantize",
        [](const at::Tensor& codes, const at::Tensor& scales, const py::object& dtype) {
          return mxfp4_dequantize(codes, scales, torch::python::detail::py_object_to_dtype(dtype));
        },
        py::arg("codes"), py::arg("scales"), py::arg("dtype"));
  m.def("mxfp4_linear", &mxfp4_linear, py::arg("x"), py::arg("x_scales"), py::arg("codes"), py::arg("scales"));
}
