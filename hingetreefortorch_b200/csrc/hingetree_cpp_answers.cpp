// Answers of a linear layer with many classes: weights as microscaled 4-bit numbers, class scores under them, a class drawn from scores.  Not
// part of the reference's operator set (its pipelines put torch.nn modules there, README.md:110-129).
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>

#include <cmath>

#include "hingetree_cpp_autograd.h"
#include "hingetree_cpp_dense.h"

namespace htx {

namespace {

int64_t blocks_of(int64_t features) { return (features + 31) / 32; }

void require_floating(const torch::Tensor &t) {
  if (t.scalar_type() != torch::kFloat32 && t.scalar_type() != torch::kBFloat16 && t.scalar_type() != torch::kFloat16)
    bad_argument("Error: Unsupported data type. Only torch.float32, torch.bfloat16 and torch.float16 are supported.");
}
void refuse_derivatives(const char *op, const torch::Tensor &t) {
  if (differentiated({&t})) bad_runtime(std::string("Error: ") + op + " has no derivative: call it under torch.no_grad(), or with detached tensors.");
}
// What returns several tensors is not recorded as an operation, and a recorded constant would be wrong.
void refuse_tracing(const char *op) {
  if (torch::jit::tracer::isTracing()) bad_runtime(std::string("Error: ") + op + " cannot be traced (torch.jit.trace).");
}

void check_packed(const torch::Tensor &codes, const torch::Tensor &scales, int64_t features) {
  if (codes.scalar_type() != torch::kUInt8 || scales.scalar_type() != torch::kUInt8) bad_argument("Error: the codes and scales are expected to be torch.uint8.");
  if (features < 1 || codes.dim() != 2 || scales.dim() != 2 || scales.size(0) < 1 || codes.size(0) != scales.size(0) || scales.size(1) != blocks_of(features) ||
      codes.size(1) != 16 * scales.size(1))
    bad_argument("Error: with blocks = features / 32, rounded up, the codes must be [outputs, 16 blocks] and the scales [outputs, blocks].");
  if (codes.device() != scales.device()) bad_argument("Error: All tensors are expected to be on the same device.");
}

std::vector<torch::Tensor> pack_mx4(const torch::Tensor &weight) {
  require_floating(weight);
  if (weight.dim() != 2 || weight.size(0) < 1 || weight.size(1) < 1) bad_argument("Error: a weight must be [outputs, features], with one of each at least.");
  require_cuda(weight);
  refuse_tracing("pack_mx4");
  c10::DeviceGuard guard(weight.device());
  const bool rows = weight.stride(1) == 1 && (weight.size(0) == 1 || weight.stride(0) >= weight.size(1));
  const torch::Tensor w = rows || weight.size(1) == 1 ? weight.detach() : weight.detach().contiguous();
  const int64_t outputs = w.size(0), features = w.size(1), blocks = blocks_of(features), stride = outputs > 1 ? w.stride(0) : features;
  if (stride < features) return pack_mx4(weight.detach().contiguous());  // (rows that lie on one another)
  torch::Tensor codes = fresh({outputs, 16 * blocks}, w, torch::kUInt8), scales = fresh({outputs, blocks}, w, torch::kUInt8);
  raise_status(ht_mx4_pack(type_code(w), w.const_data_ptr(), stride, outputs, features, codes.data_ptr(), scales.data_ptr(), current_stream(w)), "pack_mx4");
  return {codes, scales};
}

torch::Tensor unpack_mx4(const torch::Tensor &codes_, const torch::Tensor &scales_, int64_t features, torch::ScalarType type) {
  if (type != torch::kFloat32 && type != torch::kBFloat16 && type != torch::kFloat16)
    bad_argument("Error: Unsupported data type. Only torch.float32, torch.bfloat16 and torch.float16 are supported.");
  check_packed(codes_, scales_, features);
  require_cuda(codes_);
  c10::DeviceGuard guard(codes_.device());
  const torch::Tensor codes = as_whole(codes_), scales = as_whole(scales_);
  torch::Tensor w = fresh({codes.size(0), features}, codes, type);
  raise_status(ht_mx4_unpack(type_code(w), codes.const_data_ptr(), scales.const_data_ptr(), codes.size(0), features, w.data_ptr(), features, current_stream(w)),
               "unpack_mx4");
  return w;
}

torch::Tensor linear_mx4(const torch::Tensor &x_, const torch::Tensor &codes_, const torch::Tensor &scales_, const OptionalTensor &bias_) {
  const torch::Tensor bias0 = given(bias_);
  check_types(x_, {&bias0});
  if (x_.dim() < 1) bad_argument("Error: x must be [..., features].");
  check_packed(codes_, scales_, x_.size(-1));
  if (bias0.defined() && (bias0.dim() != 1 || bias0.size(0) != codes_.size(0))) bad_argument("Error: a bias must be [outputs].");
  if (codes_.device() != x_.device()) bad_argument("Error: All tensors are expected to be on the same device.");
  require_cuda(x_);
  refuse_derivatives("linear_mx4", x_);
  if (bias0.defined()) refuse_derivatives("linear_mx4", bias0);
  c10::DeviceGuard guard(x_.device());
  const torch::Tensor x = as_rows(x_), codes = as_whole(codes_), scales = as_whole(scales_), bias = as_whole(bias0);
  ht_dense_problem p = {};
  p.dtype = type_code(x);
  p.rows = x.size(0), p.features = x.size(1), p.outputs = codes.size(0);
  p.x_stride = x.size(0) > 1 ? x.stride(0) : x.size(1);
  torch::Tensor y = fresh({p.rows, p.outputs}, x);
  size_t bytes = ht_linear_mx4_workspace_bytes(&p);
  torch::Tensor ws;
  if (bytes > 0) {  // (an allocation is a fifth of a small call)
    try {
      ws = make_workspace(bytes, x);
    } catch (const c10::OutOfMemoryError &) {  // without decoded weights
      p.scratch_limit = 1;
      const size_t least = ht_linear_mx4_workspace_bytes(&p);
      if (least >= bytes) throw;
      bytes = least;
      if (bytes > 0) ws = make_workspace(bytes, x);
    }
  }
  raise_status(ht_linear_mx4(&p, x.const_data_ptr(), codes.const_data_ptr(), scales.const_data_ptr(), pointer(bias), y.data_ptr(), bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                             long_lived_word(x), current_stream(x)),
               "linear_mx4");
  if (x_.dim() == 2) return y;
  std::vector<int64_t> sizes = x_.sizes().vec();
  sizes.back() = p.outputs;
  return y.reshape(sizes);
}

// A bound of sample_classes: one number for all rows, or a tensor with one a row.
struct Bound {
  double number = 0.0;
  int64_t count = 0;  // of one that is a whole number: not every one is a double
  torch::Tensor rows;
};
Bound bound_of(const pybind11::object &value, const char *name, torch::ScalarType type, const torch::Tensor &uniform) {
  Bound b;
  if (THPVariable_Check(value.ptr())) {
    const torch::Tensor t = pybind11::cast<torch::Tensor>(value);
    if (t.scalar_type() != type || t.sizes() != uniform.sizes())
      bad_argument(std::string("Error: ") + name + " must be a number, or a " + (type == torch::kInt64 ? "torch.int64" : "torch.float32") +
                   " tensor with one for each row.");
    if (t.device() != uniform.device()) bad_argument("Error: All tensors are expected to be on the same device.");
    refuse_derivatives("sample_classes", t);
    b.rows = t.detach().contiguous();
    return b;
  }
  try {
    if (type == torch::kInt64)
      b.count = pybind11::cast<int64_t>(value);
    else
      b.number = pybind11::cast<double>(value);
  } catch (const pybind11::cast_error &) {
    bad_argument(std::string("Error: ") + name + " must be a number or a tensor with one for each row.");
  }
  return b;
}

std::vector<torch::Tensor> sample_classes(const torch::Tensor &scores_, const torch::Tensor &uniform_, const pybind11::object &temperature,
                                          const pybind11::object &top_k, const pybind11::object &top_p, const pybind11::object &min_p) {
  require_floating(scores_);
  if (scores_.dim() < 1 || scores_.size(-1) < 1) bad_argument("Error: scores must be [..., classes], with one class at least.");
  if (uniform_.scalar_type() != torch::kFloat32) bad_argument("Error: the random numbers are expected to be torch.float32.");
  if (uniform_.sizes() != scores_.sizes().slice(0, scores_.dim() - 1)) bad_argument("Error: scores are [..., classes]: there must be a random number for each row of them.");
  if (uniform_.device() != scores_.device()) bad_argument("Error: All tensors are expected to be on the same device.");
  const Bound t = bound_of(temperature, "temperature", torch::kFloat32, uniform_), k = bound_of(top_k, "top_k", torch::kInt64, uniform_),
              p = bound_of(top_p, "top_p", torch::kFloat32, uniform_), least = bound_of(min_p, "min_p", torch::kFloat32, uniform_);
  if (!t.rows.defined() && !(t.number >= 0.0 && std::isfinite(t.number))) bad_argument("Error: the temperature must be finite, and 0 at the least.");
  if (!k.rows.defined() && k.count < 0) bad_argument("Error: top_k must be 0 (all classes) or more.");
  if (!p.rows.defined() && !(p.number >= 0.0 && p.number <= 1.0)) bad_argument("Error: top_p must be between 0 and 1.");
  if (!least.rows.defined() && !(least.number >= 0.0 && least.number <= 1.0)) bad_argument("Error: min_p must be between 0 and 1.");
  require_cuda(scores_);
  refuse_derivatives("sample_classes", scores_);
  refuse_derivatives("sample_classes", uniform_);
  refuse_tracing("sample_classes");
  c10::DeviceGuard guard(scores_.device());
  torch::Tensor scores = scores_.dim() == 2 ? scores_ : scores_.reshape({-1, scores_.size(-1)});
  if (scores.size(1) > 1 && scores.stride(1) != 1) scores = scores.contiguous();
  if (scores.size(0) > 1 && scores.stride(0) < scores.size(1)) scores = scores.contiguous();
  const torch::Tensor uniform = uniform_.detach().contiguous();
  ht_sample_problem problem = {};
  problem.dtype = type_code(scores);
  problem.rows = scores.size(0), problem.classes = scores.size(1);
  problem.stride = scores.size(0) > 1 ? scores.stride(0) : scores.size(1);
  problem.temperature = t.number, problem.top_p = p.number, problem.min_p = least.number;
  problem.top_k = k.count;
  auto rows_of = [](const Bound &b) { return b.rows.defined() ? b.rows.const_data_ptr<float>() : nullptr; };
  problem.row_temperature = rows_of(t), problem.row_top_p = rows_of(p), problem.row_min_p = rows_of(least);
  problem.row_top_k = k.rows.defined() ? k.rows.const_data_ptr<int64_t>() : nullptr;
  torch::Tensor drawn = fresh(uniform_.sizes(), scores, torch::kInt64), log_probs = fresh(uniform_.sizes(), scores, torch::kFloat32);
  raise_status(ht_sample_classes(&problem, scores.const_data_ptr(), uniform.const_data_ptr<float>(), drawn.data_ptr<int64_t>(), log_probs.data_ptr<float>(),
                                 current_stream(scores)),
               "sample_classes");
  return {drawn, log_probs};
}

}  // namespace

void bind_answers(pybind11::module_ &m) {
  using pybind11::arg;
  m.def("pack_mx4", &pack_mx4, arg("weight"),
        "Weights [outputs, features] (float32, bfloat16 or float16) as microscaled 4-bit numbers: [codes, scales], uint8.");
  m.def(
      "unpack_mx4",
      [](const torch::Tensor &codes, const torch::Tensor &scales, int64_t features, const pybind11::object &dtype) {
        refuse_tracing("unpack_mx4");
        if (!THPDtype_Check(dtype.ptr())) bad_argument("Error: dtype must be a torch.dtype.");
        return unpack_mx4(codes, scales, features, reinterpret_cast<THPDtype *>(dtype.ptr())->scalar_type);
      },
      arg("codes"), arg("scales"), arg("features"), arg("dtype"), "The values that packed weights stand for, [outputs, features].");
  m.def(
      "linear_mx4",
      [](const torch::Tensor &x, const torch::Tensor &codes, const torch::Tensor &scales, const OptionalTensor &bias) {
        return traceable("linear_mx4", [](auto &...a) { return linear_mx4(a...); }, x, codes, scales, bias);
      },
      arg("x"), arg("codes"), arg("scales"), arg("bias") = pybind11::none(),
      "x @ W.T + bias under packed weights W; x [..., features], float32, bfloat16 or float16; no derivative.");
  m.def("sample_classes", &sample_classes, arg("scores"), arg("uniform"), arg("temperature"), arg("top_k"), arg("top_p"), arg("min_p"),
        "[class, logarithm of its share] drawn from each row of scores with its number of uniform.");
}

}  // namespace htx
