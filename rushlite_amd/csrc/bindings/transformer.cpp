// Python surface of the transformer operators (core/transformer.hpp).
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cmath>
#include <optional>

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
