// The dense layers around a forest: gated_linear in front of one, linear_class_loss behind one, with their autograd nodes.  Not part of
// the reference's operator set (its pipelines put torch.nn modules there, README.md:110-129).
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/graph_task.h>

#include "hingetree_cpp_autograd.h"

namespace htx {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptionalTensor = std::optional<torch::Tensor>;

torch::Tensor given(const OptionalTensor &t) { return t.has_value() ? *t : torch::Tensor(); }
OptionalTensor optional(const torch::Tensor &t) { return t.defined() ? OptionalTensor(t) : std::nullopt; }
const void *pointer(const torch::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

void check_types(const torch::Tensor &x, std::initializer_list<const torch::Tensor *> others) {
  if (x.scalar_type() != torch::kFloat32 && x.scalar_type() != torch::kBFloat16 && x.scalar_type() != torch::kFloat16)
    bad_argument("Error: Unsupported data type. Only torch.float32, torch.bfloat16 and torch.float16 are supported.");
  for (const torch::Tensor *t : others) {
    if (!t->defined()) continue;
    if (t->scalar_type() != x.scalar_type()) bad_argument("Error: x, the weights and the biases are expected to have the same type.");
    if (t->device() != x.device()) bad_argument("Error: All tensors are expected to be on the same device.");
  }
}
void check_weight(const torch::Tensor &x, const torch::Tensor &w, const torch::Tensor &bias) {
  if (x.dim() < 1 || w.dim() != 2 || x.size(-1) != w.size(1) || w.size(0) < 1 || w.size(1) < 1)
    bad_argument("Error: x must be [..., features] and a weight [outputs, features], with one feature and one output at least.");
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != w.size(0))) bad_argument("Error: a bias must be [outputs].");
}

// Rows of contiguous features, the first on 16 bytes; differentiable.
torch::Tensor as_rows(const torch::Tensor &x) {
  torch::Tensor rows = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  const bool contiguous = rows.is_contiguous();
  if (!contiguous && (rows.stride(1) != 1 || rows.stride(0) < rows.size(1))) rows = rows.contiguous();
  if (reinterpret_cast<uintptr_t>(rows.const_data_ptr()) % 16 != 0) rows = rows.clone(at::MemoryFormat::Contiguous);
  return rows;
}
torch::Tensor as_whole(const torch::Tensor &t) {
  if (!t.defined()) return t;
  const torch::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 != 0 ? c.clone(at::MemoryFormat::Contiguous) : c;
}

ht_dense_problem problem_of(const torch::Tensor &x, const torch::Tensor &w, int activation) {
  ht_dense_problem p = {};
  p.dtype = x.scalar_type() == torch::kFloat32 ? HT_DTYPE_F32 : x.scalar_type() == torch::kBFloat16 ? HT_DTYPE_BF16 : HT_DTYPE_F16;
  p.activation = activation;
  p.rows = x.size(0), p.features = x.size(1), p.outputs = w.size(0);
  p.x_stride = x.size(0) > 1 ? x.stride(0) : x.size(1);
  return p;
}

void refuse_second_derivative(const char *op) {
  if (at::GradMode::is_enabled()) bad_runtime(std::string("Error: ") + op + " has no second derivative (create_graph).");
}

// A backward's workspace within the caller's limit; one that cannot be had counts as one beyond it.
template <typename Bytes>
torch::Tensor backward_workspace(ht_dense_problem &p, const torch::Tensor &like, Bytes &&bytes) {
  p.scratch_limit = std::min<int64_t>(std::max<int64_t>(backward_scratch_limit(), 1), (int64_t)1 << 29);
  for (;;) {
    const size_t need = bytes(&p, 1);
    try {
      return make_workspace(need, like);
    } catch (const c10::OutOfMemoryError &) {
      do {  // (a limit that changes nothing yet is no other attempt)
        if (p.scratch_limit <= 1) throw;
        p.scratch_limit = std::max<int64_t>(p.scratch_limit / 4, 1);
      } while (bytes(&p, 1) >= need);
    }
  }
}

// Room for the copies that a forward leaves for its backward, where the caller's settings and the device's memory admit it.
torch::Tensor room_to_keep(size_t bytes, const torch::Tensor &like) {
  if (bytes == 0 || !may_keep((int64_t)bytes)) return torch::Tensor();
  try {
    return fresh({(int64_t)bytes}, like, torch::kUInt8);
  } catch (const c10::OutOfMemoryError &) {
    return torch::Tensor();
  }
}
// Leaves a forward's copies to its node, with the distance of x's rows that their layout goes by.
void leave_kept(AutogradContext *ctx, const torch::Tensor &kept, const torch::Tensor &x) {
  if (!kept.defined()) return;
  ctx->saved_data["kept"] = kept;
  ctx->saved_data["kept_stride"] = problem_of(x, x, 0).x_stride;
}
// The copies of a node's forward; they go with the graph's buffers.  Not taken where a hook has given x other strides since.
torch::Tensor take_kept(AutogradContext *ctx, const ht_dense_problem &p) {
  const auto at = ctx->saved_data.find("kept");
  if (at == ctx->saved_data.end()) return torch::Tensor();
  const torch::Tensor kept = at->second.toTensor();
  if (!torch::autograd::get_current_graph_task_keep_graph()) ctx->saved_data.erase(at);
  return ctx->saved_data["kept_stride"].toInt() == p.x_stride ? kept : torch::Tensor();
}

// ---- gated projection ------------------------------------------------------------------------------------------------

int activation_code(const std::string &name) {
  if (name == "silu") return HT_ACTIVATION_SILU;
  if (name == "gelu") return HT_ACTIVATION_GELU;
  if (name == "relu") return HT_ACTIVATION_RELU;
  if (name == "sigmoid") return HT_ACTIVATION_SIGMOID;
  bad_argument("Error: the activation must be one of 'silu', 'gelu', 'relu' or 'sigmoid'.");
}

torch::Tensor gated_forward(const torch::Tensor &x, const torch::Tensor &wg, const torch::Tensor &wv, const torch::Tensor &bg,
                            const torch::Tensor &bv, int activation, torch::Tensor *kept = nullptr) {
  c10::DeviceGuard guard(x.device());
  const ht_dense_problem p = problem_of(x, wg, activation);
  if (kept != nullptr) *kept = room_to_keep(ht_gated_linear_kept_bytes(&p), x);
  torch::Tensor h = fresh({p.rows, p.outputs}, x);
  const torch::Tensor ws = make_workspace(ht_gated_linear_workspace_bytes(&p, 0), x);
  raise_status(ht_gated_linear_forward(&p, pointer(x), pointer(wg), pointer(wv), pointer(bg), pointer(bv), h.data_ptr(),
                                       kept != nullptr && kept->defined() ? kept->data_ptr() : nullptr, ws.data_ptr(), ws.numel(), long_lived_word(x), current_stream(x)),
               "gated linear");
  return h;
}

struct GatedNode : public torch::autograd::Function<GatedNode> {
  static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &wg, const torch::Tensor &wv,
                               const OptionalTensor &bg, const OptionalTensor &bv, int64_t activation) {
    ctx->save_for_backward({x, wg, wv, given(bg), given(bv)});
    ctx->saved_data["activation"] = activation;
    torch::Tensor kept;
    const torch::Tensor h = gated_forward(x, wg, wv, given(bg), given(bv), (int)activation, &kept);
    leave_kept(ctx, kept, x);
    return h;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    refuse_second_derivative("gated_linear");
    variable_list s = ctx->get_saved_variables();
    c10::DeviceGuard guard(s[0].device());
    const torch::Tensor x = as_rows(s[0]);  // (a hook on what is saved may have laid it out anew)
    for (int i = 1; i < 5; ++i) s[i] = as_whole(s[i]);
    ht_dense_problem p = problem_of(x, s[1], (int)ctx->saved_data["activation"].toInt());
    const torch::Tensor dh = as_whole(grads[0]);
    variable_list out(6);
    for (int i = 0, edge = 0; i < 5; ++i)  // a bias that is not there has no edge
      if (s[i].defined() && ctx->needs_input_grad(edge++)) out[i] = fresh(s[i].sizes(), s[i]);
    const torch::Tensor kept = take_kept(ctx, p), ws = backward_workspace(p, x, ht_gated_linear_workspace_bytes);
    auto to = [](const torch::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    raise_status(ht_gated_linear_backward(&p, pointer(x), pointer(s[1]), pointer(s[2]), pointer(s[3]), pointer(s[4]), pointer(dh), pointer(kept), to(out[0]),
                                          to(out[1]), to(out[2]), to(out[3]), to(out[4]), ws.data_ptr(), ws.numel(), long_lived_word(x),
                                          current_stream(x)),
                 "gated linear backward");
    return out;
  }
};

torch::Tensor gated_linear(const torch::Tensor &x_, const torch::Tensor &wg_, const torch::Tensor &wv_, const OptionalTensor &bg_,
                           const OptionalTensor &bv_, const std::string &activation) {
  const int act = activation_code(activation);
  const torch::Tensor bg0 = given(bg_), bv0 = given(bv_);
  check_types(x_, {&wg_, &wv_, &bg0, &bv0});
  check_weight(x_, wg_, bg0);
  check_weight(x_, wv_, bv0);
  if (wg_.size(0) != wv_.size(0)) bad_argument("Error: both weights must have the same number of outputs.");
  require_cuda(x_);
  const torch::Tensor x = as_rows(x_), wg = as_whole(wg_), wv = as_whole(wv_), bg = as_whole(bg0), bv = as_whole(bv0);
  const bool node = differentiated({&x, &wg, &wv}) || (bg.defined() && differentiated({&bg})) || (bv.defined() && differentiated({&bv}));
  const torch::Tensor h = node ? GatedNode::apply(x, wg, wv, optional(bg), optional(bv), (int64_t)act) : gated_forward(x, wg, wv, bg, bv, act);
  if (x_.dim() == 2) return h;
  std::vector<int64_t> sizes = x_.sizes().vec();
  sizes.back() = wg.size(0);
  return h.reshape(sizes);
}

// ---- class loss ------------------------------------------------------------------------------------------------------

int reduction_code(const std::string &name) {
  if (name == "none") return HT_REDUCTION_NONE;
  if (name == "mean") return HT_REDUCTION_MEAN;
  if (name == "sum") return HT_REDUCTION_SUM;
  bad_argument("Error: the reduction must be one of 'none', 'mean' or 'sum'.");
}

// {loss, what the backward needs of the softmax (with `keep`)}
std::pair<torch::Tensor, torch::Tensor> loss_forward(const torch::Tensor &x, const torch::Tensor &w, const torch::Tensor &bias,
                                                     const torch::Tensor &target, int64_t ignore, int reduction, bool keep,
                                                     torch::Tensor *kept = nullptr) {
  c10::DeviceGuard guard(x.device());
  const ht_dense_problem p = problem_of(x, w, 0);
  if (kept != nullptr) *kept = room_to_keep(ht_linear_class_loss_kept_bytes(&p), x);
  torch::Tensor loss = reduction == HT_REDUCTION_NONE ? fresh({p.rows}, x, torch::kFloat32) : fresh({}, x, torch::kFloat32);
  torch::Tensor stats = keep ? fresh({2 * p.rows + 2}, x, torch::kFloat32) : torch::Tensor();
  const torch::Tensor ws = make_workspace(ht_linear_class_loss_workspace_bytes(&p, 0), x);
  raise_status(ht_linear_class_loss_forward(&p, pointer(x), pointer(w), pointer(bias), target.const_data_ptr<int64_t>(), ignore, reduction,
                                            loss.data_ptr<float>(), keep ? stats.data_ptr<float>() : nullptr,
                                            kept != nullptr && kept->defined() ? kept->data_ptr() : nullptr, ws.data_ptr(), ws.numel(), long_lived_word(x), current_stream(x)),
               "class loss");
  return {loss, stats};
}

struct ClassLossNode : public torch::autograd::Function<ClassLossNode> {
  static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const torch::Tensor &w, const OptionalTensor &bias,
                               const torch::Tensor &target, int64_t ignore, int64_t reduction) {
    torch::Tensor kept;
    const auto result = loss_forward(x, w, given(bias), target, ignore, (int)reduction, true, &kept);
    leave_kept(ctx, kept, x);
    ctx->save_for_backward({x, w, given(bias), target, result.second});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    return result.first;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    refuse_second_derivative("linear_class_loss");
    variable_list s = ctx->get_saved_variables();
    c10::DeviceGuard guard(s[0].device());
    const torch::Tensor x = as_rows(s[0]);  // (a hook on what is saved may have laid it out anew)
    for (int i = 1; i < 5; ++i) s[i] = as_whole(s[i]);
    ht_dense_problem p = problem_of(x, s[1], 0);
    const torch::Tensor grad = grads[0].contiguous();
    variable_list out(6);
    for (int i = 0, edge = 0; i < 3; ++i)  // a bias that is not there has no edge
      if (s[i].defined() && ctx->needs_input_grad(edge++)) out[i] = fresh(s[i].sizes(), s[i]);
    const torch::Tensor kept = take_kept(ctx, p), ws = backward_workspace(p, x, ht_linear_class_loss_workspace_bytes);
    auto to = [](const torch::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
    raise_status(ht_linear_class_loss_backward(&p, pointer(x), pointer(s[1]), pointer(s[2]), s[3].const_data_ptr<int64_t>(),
                                               ctx->saved_data["ignore"].toInt(), (int)ctx->saved_data["reduction"].toInt(),
                                               grad.const_data_ptr<float>(), s[4].const_data_ptr<float>(), pointer(kept), to(out[0]), to(out[1]), to(out[2]),
                                               ws.data_ptr(), ws.numel(), long_lived_word(x), current_stream(x)),
                 "class loss backward");
    return out;
  }
};

torch::Tensor linear_class_loss(const torch::Tensor &x_, const torch::Tensor &w_, const OptionalTensor &bias_, const torch::Tensor &target_,
                                int64_t ignore, const std::string &reduction) {
  const int code = reduction_code(reduction);
  const torch::Tensor bias0 = given(bias_);
  check_types(x_, {&w_, &bias0});
  check_weight(x_, w_, bias0);
  if (target_.scalar_type() != torch::kInt64) bad_argument("Error: the targets are expected to be torch.int64.");
  if (target_.device() != x_.device()) bad_argument("Error: All tensors are expected to be on the same device.");
  if (target_.sizes() != x_.sizes().slice(0, x_.dim() - 1)) bad_argument("Error: x is [..., features]: there must be a target for each row of it.");
  require_cuda(x_);
  const torch::Tensor x = as_rows(x_), w = as_whole(w_), bias = as_whole(bias0), target = target_.reshape({-1}).contiguous();
  const bool node = differentiated({&x, &w}) || (bias.defined() && differentiated({&bias}));
  const torch::Tensor loss = node ? ClassLossNode::apply(x, w, optional(bias), target, ignore, (int64_t)code)
                                  : loss_forward(x, w, bias, target, ignore, code, false).first;
  return code == HT_REDUCTION_NONE && target_.dim() != 1 ? loss.reshape(target_.sizes()) : loss;
}

}  // namespace

void bind_dense(pybind11::module_ &m) {
  using pybind11::arg;
  m.def(
      "gated_linear",
      [](const torch::Tensor &x, const torch::Tensor &wg, const torch::Tensor &wv, const OptionalTensor &bg, const OptionalTensor &bv,
         const std::string &activation) {
        return traceable("gated_linear", [](auto &...a) { return gated_linear(a...); }, x, wg, wv, bg, bv, activation);
      },
      arg("x"), arg("gate_weight"), arg("value_weight"), arg("gate_bias") = pybind11::none(), arg("value_bias") = pybind11::none(),
      arg("activation") = "silu",
      "act(x @ gate_weight.T + gate_bias) * (x @ value_weight.T + value_bias) as one kernel, differentiable; x [..., features], weights "
      "[outputs, features], all of one type (float32, bfloat16 or float16).");
  m.def(
      "linear_class_loss",
      [](const torch::Tensor &x, const torch::Tensor &w, const OptionalTensor &bias, const torch::Tensor &target, int64_t ignore,
         const std::string &reduction) {
        return traceable("linear_class_loss", [](auto &...a) { return linear_class_loss(a...); }, x, w, bias, target, ignore, reduction);
      },
      arg("x"), arg("weight"), arg("bias"), arg("target"), arg("ignore_index") = -100, arg("reduction") = "mean",
      "Softmax cross entropy of the scores x @ weight.T + bias against target, the scores never in memory, differentiable; float32.");
}

}  // namespace htx
