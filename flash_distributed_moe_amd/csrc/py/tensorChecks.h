// Checks of tensors and small helpers that the extension's bindings share.
#pragma once
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
#include <unordered_set>
#include <vector>

#include "../../../include/flash_moe.h"

namespace py = pybind11;

namespace {

using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
using OptTensor = c10::optional<at::Tensor>;

[[maybe_unused]] void* current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

[[maybe_unused]] void check_hip(int e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, " failed: ", hipGetErrorString(static_cast<hipError_t>(e)), " (hipError_t ", e, ")");
}

// Tensors that stand for others (of a subclass that wraps one, or inside a functional transform) have none: their addresses are null,
// which stands for an argument that is left out, or for a view of them a number that is no address.
[[maybe_unused]] void check_memory(const at::Tensor& t, const char* name) {
  const c10::StorageImpl* memory = t.unsafeGetTensorImpl()->unsafe_storage().unsafeGetStorageImpl();
  TORCH_CHECK((memory != nullptr && memory->data() != nullptr) || t.numel() == 0, name,
              " has no memory of its own (a tensor subclass, or a tensor inside a functional transform)");
}

[[maybe_unused]] void check_device(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.defined(), name, " tensor is undefined");
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (ROCm)");
  check_memory(t, name);
  TORCH_CHECK(t.device() == like.device(), name, " must be on ", like.device(), ", not on ", t.device());
}

// A dual tensor's result would come back without a tangent, which stands for a zero one.
[[maybe_unused]] void refuse_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!t.defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), name,
              " carries a tangent: there are no forward-mode derivatives here");
}

[[maybe_unused]] int dtype_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, " must be float32 or bfloat16");
  return t.scalar_type() == at::kFloat ? FLASH_MOE_F32 : FLASH_MOE_BF16;
}

[[maybe_unused]] int int_size(int64_t v, const char* name) {
  TORCH_CHECK(v >= 0 && v <= std::numeric_limits<int>::max(), name, " is too large: ", v);
  return static_cast<int>(v);
}

[[maybe_unused]] bool begins_on_16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A weight or code tensor as the kernels read it: without gaps. (One that is a view into something
// larger, at an odd place, or that is negated when it is read, is refused rather than copied at every call.)
[[maybe_unused]] void check_packed(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(!t.is_neg(), name, " must not be a negated view");
  TORCH_CHECK(begins_on_16(t), name, " must begin on 16 bytes");
}

// t [..., width] as rows whose distance the kernels can take; copied where it cannot, or where torch keeps the values negated.
struct Rows {
  at::Tensor t;
  int64_t stride;
  int count;
};
constexpr int64_t kMaxStride = 1 << 20;
[[maybe_unused]] Rows rows_of(const at::Tensor& t, const char* name) {
  const int64_t width = t.size(-1), rows = width > 0 ? t.numel() / width : 0;
  if (t.is_contiguous() && begins_on_16(t) && !t.is_neg() && (rows <= 1 || (width <= kMaxStride && width * t.element_size() % 16 == 0)))
    return {t, width, int_size(rows, name)};
  at::Tensor flat = t.dim() == 2 ? t : t.reshape({rows, width});
  int64_t stride = flat.stride(0);
  const bool apart = rows <= 1 || (stride >= width && stride <= kMaxStride && stride * flat.element_size() % 16 == 0);
  if (flat.numel() > 0 && (flat.stride(1) != 1 || !apart || !begins_on_16(flat) || flat.is_neg()))
    flat = flat.clone(at::MemoryFormat::Contiguous);
  stride = rows <= 1 ? width : flat.stride(0);
  return {flat, stride, int_size(rows, name)};
}

[[maybe_unused]] at::Tensor bytes_on(const at::Tensor& like, size_t bytes) {
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte).requires_grad(false));
}
[[maybe_unused]] void* pointer(const at::Tensor& t) {
  if (!t.defined() || t.numel() == 0) return nullptr;
  check_memory(t, "a tensor");
  return t.data_ptr();
}

// A gradient of a leaf is accumulated on the stream on which its accumulator was made, by the first graph of it
// that is still alive. Captured into a HIP graph, a backward pass that finds an accumulator of another
// stream would make that stream wait inside the capture, and the process ends. So the forward pass that
// would lead there is refused.
[[maybe_unused]] void check_capture(const at::Tensor& leaf, const char* name) {
  if (!leaf.requires_grad() || !leaf.is_leaf()) return;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(leaf);
  if (!accumulator) return;
  const auto stream = accumulator->stream();
  TORCH_CHECK(!stream.has_value() || *stream == c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().unwrap(), name,
              " is part of an autograd graph made on another stream that is still alive: drop it before a step is captured");
}

// The same for whatever graph leads to `t`: its nodes run their backward passes on the streams of their forward passes.
// Looked at under capture only, where the graphs are those of one step.
[[maybe_unused]] void check_capture_behind(const at::Tensor& t, const char* name) {
  if (!t.defined() || !t.requires_grad()) return;
  check_capture(t, name);
  const auto here = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().unwrap();
  std::vector<torch::autograd::Node*> todo{t.grad_fn().get()};
  std::unordered_set<torch::autograd::Node*> seen{nullptr};
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    if (!seen.insert(node).second) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream.has_value() || *stream == here, name,
                " leads to an autograd graph made on another stream that is still alive: drop it before a step is captured");
    for (const auto& edge : node->next_edges()) todo.push_back(edge.function.get());
  }
}

// Whether the current stream is being captured.
[[maybe_unused]] bool capturing() {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  check_hip(hipStreamIsCapturing(static_cast<hipStream_t>(current_stream()), &status), "hipStreamIsCapturing");
  return status != hipStreamCaptureStatusNone;
}

}  // namespace
