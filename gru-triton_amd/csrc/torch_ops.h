// What the torch side of the operators shares (torch_ops.cpp, torch_sequence_ops.cpp): checks of
// tensors, the device's stream, errors and what a backward returns.
#pragma once

#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/extension.h>

#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/gruscan.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void raise_for(int64_t rc) {
  if (rc >= 0) return;
  TORCH_CHECK_VALUE(rc != GS_ERR_INVALID, gs_last_error());
  TORCH_CHECK(false, gs_last_error());
}

// The tensors' device made current, and torch's stream there.
struct On {
  c10::hip::OptionalHIPGuard guard;
  hipStream_t stream;
  explicit On(const Tensor& t) {
    const auto d = t.device();
    if (d.index() != c10::hip::current_device()) guard.set_index(d.index());
    stream = c10::hip::getCurrentHIPStream(d.index()).stream();
  }
};

template <typename T>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor get(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

int dtype_of(const char* who, const char* name, const Tensor& t) {
  if (t.scalar_type() == torch::kFloat) return GS_DTYPE_F32;
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kBFloat16, who, ": ", name, " dtype must be float32 or bfloat16; got ",
                    t.scalar_type());
  return GS_DTYPE_BF16;
}

// A tangent of forward-mode differentiation would be lost without a word: the kernels read values
// alone, and a dual tensor need not require a gradient.
void check_no_tangent(const char* who, const char* name, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), who, ": forward-mode derivatives are not implemented; ", name,
                              " has a tangent");
}

void check_on(const char* who, const char* name, const Tensor& t, const Tensor& ref) {
  TORCH_CHECK_VALUE(t.is_cuda(), who, ": ", name, " must be a CUDA (HIP) tensor; got ", t.device());
  TORCH_CHECK_VALUE(t.device() == ref.device(), who, ": all tensors must be on ", ref.device(), "; ", name, " is on ",
                    t.device());
  check_no_tangent(who, name, t);
}

// Unit stride along the last dimension.
Tensor unit(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// A tensor written through its pointer counts as modified in place: autograd refuses graphs
// that saved it before, and what the package keeps per version of a weight is found anew.
void modified(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }
// Asked before the launch: a tensor made in inference mode has no version to count outside it.
void check_may_modify(const char* who, const char* name, const Tensor& t) {
  TORCH_CHECK(!t.is_inference() || c10::InferenceMode::is_enabled(), who, ": ", name,
              " was made in inference mode and cannot be updated in place outside it");
}

// f(n) for every node that the current backward reaches from `node` and runs: with inputs asked for
// (torch.autograd.grad) those on the way to them alone, else all.
template <typename F>
void each_reached(torch::autograd::Node* node, F&& f) {
  const auto* asked = torch::autograd::get_current_graph_task_exec_info();
  if (asked != nullptr && asked->empty()) asked = nullptr;
  std::vector<torch::autograd::Node*> left{node};
  std::unordered_set<torch::autograd::Node*> seen{node};
  while (!left.empty()) {
    const auto* at = left.back();
    left.pop_back();
    for (const auto& e : at->next_edges()) {
      torch::autograd::Node* next = e.function.get();
      if (next == nullptr || !seen.insert(next).second) continue;
      if (asked != nullptr) {
        const auto it = asked->find(next);
        if (it == asked->end() || !it->second.should_execute()) continue;
      }
      f(*next);
      left.push_back(next);
    }
  }
}

// What a captured backward goes on to runs on the stream that it was made on, which for the default one no capture can
// wait for: torch's engine would end the process there. That is so for a leaf's accumulator where an eager graph of
// the leaf is still alive, however many views, casts or products are between, and for a graph made before.
// Asked before a backward launches anything.
void check_capture(const char* who) {
  const auto node = torch::autograd::get_current_node();
  if (!node || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  each_reached(node.get(), [&](torch::autograd::Node& n) {
    const auto stream = n.stream();
    if (!stream.has_value() || stream->id() != 0) return;
    TORCH_CHECK(dynamic_cast<torch::autograd::AccumulateGrad*>(&n) == nullptr,
                who, ": an eager graph of the same leaves, made on the default stream, is alive (through an output or a loss); "
                "drop it before a backward is captured");
    TORCH_CHECK(false, who, ": a captured backward goes on into a graph that was made on the default stream (", n.name(),
                "); make all of it under the capture");
  });
}

// A backward's results. Where a graph of them is asked for (create_graph), it goes on to
// `from`, which they were computed from, through an error for whoever asks for a second
// derivative: without it that derivative would lack their terms and nobody would know.
variable_list once(const char* who, variable_list grads, const variable_list& from) {
  if (!torch::GradMode::is_enabled()) return grads;
  const size_t n = grads.size();
  grads.insert(grads.end(), from.begin(), from.end());
  grads = torch::autograd::DelayedError(std::string(who) + ": second derivatives are not implemented",
                                        (int64_t)grads.size())(std::move(grads));
  grads.resize(n);
  return grads;
}

Tensor scratch(int64_t bytes, const Tensor& like) {
  raise_for(bytes);
  return bytes ? torch::empty({bytes}, like.options().dtype(torch::kByte)) : Tensor();
}

// [..., n] as rows of unit stride.
Tensor rows(const Tensor& t) { return unit(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }

}  // namespace

void bind_sequence_ops(py::module_& m);
