// Element types of the fine-tuning kernels: bf16, fp16 and fp32 values that
// are read and written 16 bytes at a time and computed on in fp32.
#pragma once

#include <hip/hip_runtime.h>

#include <unordered_set>

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/StreamGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace elem {

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// elements of one 16-byte access
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// N elements from any element on, past the caches where NT is set: one access
// of 4, 8 or 16 bytes (two of 16) also where it does not start on as many.
// That costs little: 134M bf16 values at an odd offset take 8 % longer to pack.
template <bool NT, int N, typename T>
__device__ __forceinline__ vec<T, N> load(const T* p) {
  typedef int Words __attribute__((ext_vector_type(N * sizeof(T) / 4),
                                   aligned(sizeof(T)), may_alias));
  const Words* w = (const Words*)p;
  if (!NT) return __builtin_bit_cast(vec<T, N>, *w);
  return __builtin_bit_cast(vec<T, N>, __builtin_nontemporal_load(w));
}
template <bool NT, int N, typename T>
__device__ __forceinline__ void store(T* p, const vec<T, N>& v) {
  typedef int Words __attribute__((ext_vector_type(N * sizeof(T) / 4),
                                   aligned(sizeof(T)), may_alias));
  const Words w = __builtin_bit_cast(Words, v);
  if (!NT) *(Words*)p = w;
  else __builtin_nontemporal_store(w, (Words*)p);
}

// Tensors up to this size stay in the 256 MB last-level cache next to what is
// made of them; larger ones go past it.
constexpr long kCached = 128L << 20;

inline hipStream_t stream() {
  return at::hip::getCurrentHIPStream().stream();
}

// The legacy default stream takes no capture.
inline bool is_capturing(const c10::Stream& s) {
  if (s.id() == 0) return false;
  const c10::StreamGuard guard(s);
  return c10::hip::currentStreamCaptureStatusMayInitCtx() !=
         c10::hip::CaptureStatus::None;
}

// A node of an autograd graph belongs to the stream on which it was recorded,
// a leaf's to the one on which a graph first reached the leaf, for as long as
// any graph that does lives.  A backward captured elsewhere would wait there
// on an event of the capture, which ends the process: a call whose gradients
// reach such a node is refused in the forward, before anything is recorded.
inline void check_capture(std::initializer_list<at::Tensor> inputs) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() ==
      c10::hip::CaptureStatus::None)
    return;
  std::vector<torch::autograd::Node*> next;
  std::unordered_set<torch::autograd::Node*> seen;
  std::vector<std::shared_ptr<torch::autograd::Node>> leaves;
  const auto reach = [&](torch::autograd::Node* node) {
    if (node && seen.insert(node).second) next.push_back(node);
  };
  for (const at::Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad()) continue;
    if (t.is_leaf()) {
      leaves.push_back(torch::autograd::impl::try_get_grad_accumulator(t));
      reach(leaves.back().get());
    } else {
      reach(t.grad_fn().get());
    }
  }
  while (!next.empty()) {
    torch::autograd::Node* node = next.back();
    next.pop_back();
    const auto at = node->stream();
    TORCH_CHECK(!at || is_capturing(*at),
                "Stoke -- a graph capture with gradients that reach an "
                "autograd graph of another stream: drop that graph (its "
                "outputs and losses) before the capture");
    for (const auto& edge : node->next_edges()) reach(edge.function.get());
  }
}

// A forward-mode tangent would be dropped where a kernel runs without an
// autograd node: an input that carries one is refused.  (The node itself
// refuses it too.)
inline bool has_tangent(const at::Tensor& t) {
  return t.defined() && t._fw_grad(/*level=*/0).defined();
}
inline bool has_tangent(const std::optional<at::Tensor>& t) {
  return t && has_tangent(*t);
}
template <typename... Inputs>
void refuse_tangents(const char* what, const Inputs&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...), "Stoke -- ", what,
                              " has no forward-mode derivative on the GPU");
}

// Gradients of a kernel without a derivative of its own: a second backward
// through them raises instead of being taken for zero.
inline torch::autograd::variable_list once_differentiable(
    torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "Stoke -- a fused operator was differentiated twice",
      (int64_t)grads.size());
  return (*node)(std::move(grads));
}

}  // namespace elem

// Runs `...` with T bound to the device type of a torch scalar type.
#define STOKE_ELEM_SWITCH(DTYPE, WHAT, ...)                              \
  switch (DTYPE) {                                                       \
    case at::kBFloat16: { using T = __bf16; __VA_ARGS__; break; }        \
    case at::kHalf: { using T = _Float16; __VA_ARGS__; break; }          \
    case at::kFloat: { using T = float; __VA_ARGS__; break; }            \
    default:                                                             \
      TORCH_CHECK(false, WHAT ": bf16, fp16 or fp32 tensors, got ",      \
                  DTYPE);                                                \
  }
