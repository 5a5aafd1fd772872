// Python surface of the transformer operators (core/transformer.hpp).
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cmath>
#include <optional>
#include <string>

#include "transformer.hpp"

namespace py = pybind11;
using lmp::autograd::AttentionPlan;
using lmp::autograd::Variable;
using lmp::tensor::Scalar;
using lmp::tensor::Tensor;
namespace ag = lmp::autograd;
namespace tops = lmp::tensor::ops;

void bind_transformer(py::module_& m) {
  m.def(
      "layer_norm",
      [](const Variable& x, const Variable* w, const Variable* b, Scalar eps) {
        return ag::ops::layer_norm(x, w, b, eps);
      },
      py::arg("x"), py::arg("w").none(true) = py::none(), py::arg("b").none(true) = py::none(),
      py::arg("eps") = 1e-5,
      "(x - mean) / sqrt(var + eps) * w + b over the last axis, in one kernel; w and b may be "
      "left out.");

  py::class_<AttentionPlan>(m, "AttentionPlan",
                            "A packed batch for attention(): the lengths of its sequences' queries "
                            "and keys, the heads, and whether query i sees only keys up to "
                            "i + keys - queries.")
      .def(py::init([](const std::vector<int64_t>& q, const std::optional<std::vector<int64_t>>& k,
                       int64_t heads, std::optional<int64_t> kv_heads, int64_t head_dim,
                       bool causal) {
             const int64_t kv = kv_heads.value_or(heads);
             if (heads < 0 || kv < 0 || head_dim < 0)
               throw py::value_error("attention plan: negative heads or head_dim");
             return AttentionPlan(q, k ? *k : q, size_t(heads), size_t(kv), size_t(head_dim),
                                  causal);
           }),
           py::arg("q_lengths"), py::arg("k_lengths") = py::none(), py::kw_only(),
           py::arg("heads"), py::arg("kv_heads") = py::none(), py::arg("head_dim"),
           py::arg("causal") = true)
      .def_readonly("heads", &AttentionPlan::heads)
      .def_readonly("kv_heads", &AttentionPlan::kv_heads)
      .def_readonly("head_dim", &AttentionPlan::head_dim)
      .def_readonly("queries", &AttentionPlan::queries)
      .def_readonly("keys", &AttentionPlan::keys)
      .def_readonly("causal", &AttentionPlan::causal);

  const auto scale_of = [](const AttentionPlan& plan, std::optional<Scalar> scale) {
    return scale.value_or(1 / std::sqrt(Scalar(plan.head_dim)));
  };
  m.def(
      "attention",
      [scale_of](const Variable& q, const Variable& k, const Variable& v, const AttentionPlan& plan,
                 std::optional<Scalar> scale) {
        return ag::ops::attention(q, k, v, plan, scale_of(plan, scale));
      },
      py::arg("q"), py::arg("k"), py::arg("v"), py::arg("plan"), py::arg("scale") = py::none(),
      "softmax(scale q k^T + mask) v of the plan's packed batch, q [queries, heads * head_dim], k "
      "and v [keys, kv_heads * head_dim]; scale is 1 / sqrt(head_dim) unless given.");
  m.def(
      "attention_qkv",
      [scale_of](const Variable& rows, const AttentionPlan& plan, std::optional<Scalar> scale) {
        return ag::ops::attention_qkv(rows, plan, scale_of(plan, scale));
      },
      py::arg("rows"), py::arg("plan"), py::arg("scale") = py::none(),
      "attention() with q, k and v side by side in the rows of one projection: "
      "[queries, (heads + 2 kv_heads) * head_dim].");

  m.def(
      "rotary",
      [](const Variable& x, const Variable& positions, const Tensor& frequencies, int64_t heads,
         int64_t head_dim, bool interleaved, Scalar scale) {
        if (heads < 0 || head_dim < 0) throw py::value_error("rotary: negative heads or head_dim");
        return ag::ops::rotary(x, positions.data(), frequencies,
                               {size_t(heads), size_t(head_dim), interleaved, scale});
      },
      py::arg("x"), py::arg("positions"), py::arg("frequencies"), py::kw_only(), py::arg("heads"),
      py::arg("head_dim"), py::arg("interleaved") = false, py::arg("scale") = 1.0,
      "x [rows, columns] with the pairs of its first heads * head_dim columns turned by "
      "positions[row] * frequencies[pair]; layers.Rotary holds the frequencies.");
  m.def(
      "_dropout",
      [](const Variable& x, const Variable* residual, Scalar rate, uint64_t seed, Tensor state) {
        return ag::ops::dropout(x, residual, rate, seed, state);
      },
      py::arg("x"), py::arg("residual").none(true), py::arg("rate"), py::arg("seed"),
      py::arg("state"));
  m.def(
      "gated_linear",
      [](const Variable& x, const Variable& w, const Variable* b, const std::string& gate) {
        static const char* const names[] = {"silu", "gelu", "gelu_tanh", "relu", "sigmoid"};
        for (int i = 0; i < 5; ++i)
          if (gate == names[i]) return ag::ops::gated_linear(x, w, b, i);
        throw py::value_error("gated_linear: unknown gate '" + gate +
                              "' (silu, gelu, gelu_tanh, relu or sigmoid)");
      },
      py::arg("x"), py::arg("w"), py::arg("b").none(true) = py::none(), py::arg("gate") = "silu",
      "act(a) * u for [a | u] = x @ w + b: the gate's columns of w first, then as many more.");
  m.def(
      "linear_cross_entropy",
      [](const Variable& x, const Variable& w, const Variable* b, const Variable& targets,
         const Variable* weights) {
        if (weights && weights->requires_grad() && ag::is_grad_enabled())
          throw py::value_error("linear_cross_entropy: the weights take no gradient");
        return ag::ops::linear_cross_entropy(x, w, b, targets.data(),
                                             weights ? weights->data() : Tensor());
      },
      py::arg("x"), py::arg("w"), py::arg("b").none(true), py::arg("targets"),
      py::arg("weights").none(true) = py::none(),
      "The softmax cross entropies of the rows of x @ w + b against targets (int64; a negative one "
      "is not counted), summed with weights (finite, without a gradient) or averaged over what counts, "
      "of shape [1].  Logits are held in pieces of 512 MB at most, and the gradients are formed with the "
      "losses.");
  m.def(
      "linear_cross_entropy_rows",
      [](const Variable& x, const Variable& w, const Variable* b, const Variable& targets) {
        return Variable(ag::ops::linear_cross_entropy_rows(x, w, b, targets.data()), false);
      },
      py::arg("x"), py::arg("w"), py::arg("b").none(true), py::arg("targets"),
      "The cross entropy of each row, without a gradient (scoring).");

  // One AdamW step over lists of tensors (optim.AdamW): per parameter (p, g, m,
  // v, m_scale, v_scale, decay), the scales None for states of 32 bits.
  m.def("_adamw", [](int bits, const py::list& params, Scalar lr, Scalar beta1, Scalar beta2,
                     Scalar eps, uint64_t seed, Tensor step) {
    std::vector<tops::AdamWParam> list;
    list.reserve(params.size());
    const auto tensor = [](const py::handle& h) { return h.is_none() ? Tensor() : h.cast<Tensor>(); };
    for (const py::handle& h : params) {
      const auto t = h.cast<py::tuple>();
      if (t.size() != 7) throw py::value_error("adamw: seven entries per parameter");
      list.push_back({tensor(t[0]), tensor(t[1]), tensor(t[2]), tensor(t[3]), tensor(t[4]),
                      tensor(t[5]), t[6].cast<Scalar>()});
    }
    tops::adamw(bits, list, {lr, beta1, beta2, eps, seed}, step);
  });
  m.def("_adamw_decode", &tops::adamw_decode);
}
