// What the autograd nodes of the `hingetree_cpp` torch extension share.
#pragma once

#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "hingetree_cpp_ops.h"

namespace htx {

// Forward-mode derivatives count, with or without grad mode: the nodes refuse them, the plain forward would drop the tangents.
inline bool differentiated(std::initializer_list<const torch::Tensor *> tensors) {
  if (at::GradMode::is_enabled())
    for (const torch::Tensor *t : tensors)
      if (t->requires_grad()) return true;
  if (torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr)  // a dual level is open
    for (const torch::Tensor *t : tensors)
      if (t->_fw_grad(/*level=*/0).defined()) return true;
  return false;
}

// While torch.jit.trace records, what the extension computes by itself would end up in the trace as a constant.  A Python
// Function is recorded as an operation, so the call is made through one (_HingeTree.py, _Traced), which calls `name` again: then,
// and whenever the trace runs, straight through.
inline thread_local bool recording = false;
template <typename Compute, typename... Args>
torch::Tensor traceable(const std::string &name, Compute &&compute, const Args &...args) {
  if (!torch::jit::tracer::isTracing()) return compute(args...);
  if (recording) {  // the result stands for something the recorder has seen made
    const torch::Tensor out = compute(args...);
    torch::jit::tracer::setValueTrace(out, torch::jit::tracer::getValueTrace(at::empty({0}, out.options())));
    return out;
  }
  struct Recording {
    Recording() { recording = true; }
    ~Recording() { recording = false; }
  } scope;
  return pybind11::module_::import("hingetreefortorch_b200.HingeTree._HingeTree")
      .attr("_Traced")
      .attr("apply")(name, args...)
      .template cast<torch::Tensor>();
}

}  // namespace htx
