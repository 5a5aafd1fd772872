#include "transformer.hpp"

#include "lmp_hip_transformer.h"

namespace lmp::tensor::ops {

LMP_DEFINE_DISPATCH(layer_norm_fn, layer_norm_stub)
LMP_DEFINE_DISPATCH(layer_norm_backward_fn, layer_norm_backward_stub)
LMP_DEFINE_DISPATCH(attention_fn, attention_stub)
LMP_DEFINE_DISPATCH(attention_backward_fn, attention_backward_stub)
LMP_DEFINE_DISPATCH(rotary_fn, rotary_stub)
LMP_DEFINE_DISPATCH(dropout_fn, dropout_stub)
LMP_DEFINE_DISPATCH(dropout_backward_fn, dropout_backward_stub)
LMP_DEFINE_DISPATCH(gated_linear_fn, gated_linear_stub)
LMP_DEFINE_DISPATCH(gated_linear_backward_fn, gated_linear_backward_stub)
LMP_DEFINE_DISPATCH(linear_cross_entropy_fn, linear_cross_entropy_stub)
LMP_DEFINE_DISPATCH(adamw_fn, adamw_stub)
LMP_DEFINE_DISPATCH(adamw_decode_fn, adamw_decode_stub)

void adamw(int bits, const std::vector<AdamWParam>& params, const AdamWHyper& hyper, Tensor& step) {
  LMP_CHECK(bits == 32 || bits == 8) << "adamw: states have 32 or 8 bits, not " << bits;
  LMP_CHECK(step.type() == DataType::Int64 && step.numel() == 2)
      << "adamw: step must be an int64 tensor of 2 values";
  for (size_t i = 0; i < params.size(); ++i) {
    const AdamWParam& p = params[i];
    const auto is = [&](const Tensor& t, DataType type, size_t n) {
      return t.defined() && t.device() == step.device() && t.type() == type && t.numel() == n;
    };
    const size_t n = p.p.numel(), blocks = (n + LMP_ADAMW_BLOCK - 1) / LMP_ADAMW_BLOCK;
    LMP_CHECK(is(p.p, DataType::Float32, n) && is(p.g, DataType::Float32, n) &&
              p.g.shape() == p.p.shape())
        << "adamw: parameter " << i << " and its gradient must be float32 of one shape on the "
        << "device of the step";
    const bool states = bits == 32
                            ? is(p.m, DataType::Float32, n) && is(p.v, DataType::Float32, n)
                            : is(p.m, DataType::Int32, (n + 3) / 4) &&
                                  is(p.v, DataType::Int32, (n + 3) / 4) &&
                                  is(p.m_scale, DataType::Float32, blocks) &&
                                  is(p.v_scale, DataType::Float32, blocks);
    LMP_CHECK(states) << "adamw: the states of parameter " << i << " do not fit it";
  }
  adamw_stub()(step.device(), bits, params, hyper, step);
}

Tensor adamw_decode(bool signed_codes, const Tensor& codes, const Tensor& scales, size_t n) {
  LMP_CHECK(codes.type() == DataType::Int32 && codes.numel() == (n + 3) / 4 &&
            scales.type() == DataType::Float32 && scales.device() == codes.device() &&
            scales.numel() == (n + LMP_ADAMW_BLOCK - 1) / LMP_ADAMW_BLOCK)
      << "adamw_decode: the codes and scales do not hold " << n << " values";
  return adamw_decode_stub()(codes.device(), signed_codes, codes, scales, n);
}

}  // namespace lmp::tensor::ops

namespace lmp::autograd {

namespace tops = tensor::ops;
using tensor::empty;

AttentionPlan::AttentionPlan(const std::vector<int64_t>& q_lengths,
                             const std::vector<int64_t>& k_lengths, size_t heads_, size_t kv_heads_,
                             size_t head_dim_, bool causal_)
    : heads(heads_), kv_heads(kv_heads_), head_dim(head_dim_), causal(causal_) {
  LMP_CHECK(q_lengths.size() == k_lengths.size())
      << "attention plan: one query length and one key length per sequence";
  void* p = nullptr;
  hip_ok(lmp_k_attention_plan_create(&p, q_lengths.size(), q_lengths.data(), k_lengths.data(),
                                     heads, kv_heads, head_dim, causal ? 1 : 0),
         "lmp_k_attention_plan_create");
  handle_ = std::shared_ptr<const void>(
      p, [](const void* q) { lmp_k_attention_plan_destroy(const_cast<void*>(q)); });
  for (int64_t n : q_lengths) queries += size_t(n);
  for (int64_t n : k_lengths) keys += size_t(n);
}

namespace ops {
namespace {

using Backward = std::function<void(const Variable& out, variable_list& ins)>;

struct TransformerFunction : Function {
  Backward fn;
  variable_list apply(const variable_list& g) override {
    LMP_INTERNAL_ASSERT(g.size() == 1) << "Output size mismatch.";
    fn(g[0], *saved_inputs);
    return {};
  }
};

bool wants_grad(const variable_list& inputs) {
  if (!is_grad_enabled()) return false;
  for (const Variable& v : inputs)
    if (v.requires_grad()) return true;
  return false;
}

Variable result(const Tensor& data, variable_list inputs, const char* name, Backward bw) {
  const bool rg = wants_grad(inputs);
  Variable out = Variable::op_result(data, rg);
  if (rg) {
    auto f = std::make_shared<TransformerFunction>();
    f->name = name;
    f->saved_inputs = std::make_unique<variable_list>(std::move(inputs));
    f->fn = std::move(bw);
    out.set_grad_fn(std::move(f));
  }
  return out;
}

Tensor empty_like(const Tensor& t) { return empty(t.shape(), t.device(), t.type()); }

void check_rows(const Variable& v, const char* what, size_t rows, size_t width) {
  const Tensor& t = v.data();
  LMP_CHECK(t.type() == DataType::Float32) << "attention: " << what << " must be float32";
  LMP_CHECK(t.shape().size() == 2 && t.shape()[0] == rows && t.shape()[1] == width)
      << "attention: " << what << " has shape " << t.shape() << ", the plan's is ["
      << rows << ", " << width << "]";
}

}  // namespace

Variable layer_norm(const Variable& x, const Variable* w, const Variable* b, Scalar eps) {
  const Tensor& xt = x.data();
  LMP_CHECK(xt.type() == DataType::Float32 || xt.type() == DataType::Float64)
      << "layer_norm: x must be float32 or float64";
  LMP_CHECK(!xt.shape().empty() && xt.shape().back() > 0) << "layer_norm: rows of no values";
  for (const Variable* v : {w, b})
    LMP_CHECK(!v || (v->data().type() == xt.type() && v->data().device() == xt.device() &&
                     v->data().shape() == std::vector<size_t>{xt.shape().back()}))
        << "layer_norm: weight and bias must be of x's type and device, with the size of its last "
        << "axis";
  variable_list ins{x};
  const int wi = w ? int(ins.size()) : -1;
  if (w) ins.push_back(*w);
  const int bi = b ? int(ins.size()) : -1;
  if (b) ins.push_back(*b);
  const tops::LayerNormOut out = tops::layer_norm_stub()(
      xt.device(), xt, w ? w->data() : Tensor(), b ? b->data() : Tensor(), eps, wants_grad(ins));
  return result(out.y, std::move(ins), "LayerNormBackward",
                [mean = out.mean, rstd = out.rstd, wi, bi](const Variable& y, variable_list& in) {
                  const Tensor& xt = in[0].data();
                  const Tensor w = wi >= 0 ? in[wi].data() : Tensor();
                  const std::vector<size_t> row{xt.shape().back()};
                  const auto fresh = [&](int i) {
                    return i >= 0 && in[i].requires_grad() ? empty(row, xt.device(), xt.type())
                                                           : Tensor();
                  };
                  Tensor dx = in[0].requires_grad() ? empty_like(xt) : Tensor();
                  Tensor dw = fresh(wi), db = fresh(bi);
                  tops::layer_norm_backward_stub()(xt.device(), y.grad(), xt, w, mean, rstd, &dx,
                                                   &dw, &db);
                  if (dx.defined()) in[0].incr_grad_owned(dx);
                  if (dw.defined()) in[wi].incr_grad_owned(dw);
                  if (db.defined()) in[bi].incr_grad_owned(db);
                });
}

Variable attention(const Variable& q, const Variable& k, const Variable& v,
                   const AttentionPlan& plan, Scalar scale) {
  const size_t qw = plan.heads * plan.head_dim, kw = plan.kv_heads * plan.head_dim;
  check_rows(q, "q", plan.queries, qw);
  check_rows(k, "k", plan.keys, kw);
  check_rows(v, "v", plan.keys, kw);
  const DeviceType dev = q.data().device();
  LMP_CHECK(k.data().device() == dev && v.data().device() == dev)
      << "attention: q, k and v must be on one device";
  Tensor o = empty(q.data().shape(), dev, DataType::Float32), lse;
  const bool rg = wants_grad({q, k, v});
  if (rg) lse = empty({plan.queries, plan.heads}, dev, DataType::Float32);
  tensor::keep_for_graph(plan.handle());
  tops::attention_stub()(dev, plan.handle().get(), tops::Rows{q.data(), qw, 0},
                         tops::Rows{k.data(), kw, 0}, tops::Rows{v.data(), kw, 0}, scale, o,
                         rg ? &lse : nullptr);
  return result(o, {q, k, v}, "AttentionBackward",
                [handle = plan.handle(), lse, scale, qw, kw](const Variable& out, variable_list& in) {
                  const Tensor dq = empty_like(in[0].data()), dk = empty_like(in[1].data()),
                               dv = empty_like(in[2].data());
                  tensor::keep_for_graph(handle);
                  tops::attention_backward_stub()(
                      dq.device(), handle.get(), tops::Rows{in[0].data(), qw, 0},
                      tops::Rows{in[1].data(), kw, 0}, tops::Rows{in[2].data(), kw, 0}, scale,
                      out.data(), lse, out.grad(), tops::Rows{dq, qw, 0}, tops::Rows{dk, kw, 0},
                      tops::Rows{dv, kw, 0});
                  if (in[0].requires_grad()) in[0].incr_grad_owned(dq);
                  if (in[1].requires_grad()) in[1].incr_grad_owned(dk);
                  if (in[2].requires_grad()) in[2].incr_grad_owned(dv);
                });
}

Variable attention_qkv(const Variable& rows, const AttentionPlan& plan, Scalar scale) {
  LMP_CHECK(plan.queries == plan.keys)
      << "attention_qkv: the plan has " << plan.queries << " queries and " << plan.keys << " keys";
  const size_t qw = plan.heads * plan.head_dim, kw = plan.kv_heads * plan.head_dim;
  const size_t width = qw + 2 * kw;
  check_rows(rows, "rows", plan.queries, width);
  const DeviceType dev = rows.data().device();
  Tensor o = empty({plan.queries, qw}, dev, DataType::Float32), lse;
  const bool rg = wants_grad({rows});
  if (rg) lse = empty({plan.queries, plan.heads}, dev, DataType::Float32);
  tensor::keep_for_graph(plan.handle());
  const auto slice = [width, qw, kw](const Tensor& t, int i) {
    return tops::Rows{t, width, i == 0 ? 0 : i == 1 ? qw : qw + kw};
  };
  tops::attention_stub()(dev, plan.handle().get(), slice(rows.data(), 0), slice(rows.data(), 1),
                         slice(rows.data(), 2), scale, o, rg ? &lse : nullptr);
  return result(o, {rows}, "AttentionBackward",
                [handle = plan.handle(), lse, scale, slice](const Variable& out, variable_list& in) {
                  const Tensor& t = in[0].data();
                  const Tensor d = empty_like(t);
                  tensor::keep_for_graph(handle);
                  tops::attention_backward_stub()(t.device(), handle.get(), slice(t, 0),
                                                  slice(t, 1), slice(t, 2), scale, out.data(), lse,
                                                  out.grad(), slice(d, 0), slice(d, 1),
                                                  slice(d, 2));
                  in[0].incr_grad_owned(d);
                });
}

Variable rotary(const Variable& x, const Tensor& positions, const Tensor& frequencies,
                const tops::RotaryShape& shape) {
  const Tensor& xt = x.data();
  LMP_CHECK(xt.type() == DataType::Float32 || xt.type() == DataType::Float64)
      << "rotary: x must be float32 or float64";
  LMP_CHECK(xt.shape().size() == 2) << "rotary: x must have two axes, not " << xt.shape();
  LMP_CHECK(positions.type() == DataType::Int64 && positions.numel() == xt.shape()[0] &&
            positions.device() == xt.device())
      << "rotary: positions must be int64 on x's device, one for each of its "
      << xt.shape()[0] << " rows";
  LMP_CHECK(frequencies.type() == DataType::Float64 && frequencies.device() == xt.device())
      << "rotary: frequencies must be float64 on x's device";
  LMP_CHECK(2 * frequencies.numel() <= shape.head_dim)
      << "rotary: " << frequencies.numel() << " pairs do not fit heads of " << shape.head_dim;
  // Inputs made before a capture are read at every replay.
  for (const Tensor* t : {&positions, &frequencies})
    tensor::keep_for_graph(tensor::detail::UnsafeTensorAccessor::getImpl(*t));
  const Tensor y = tops::rotary_stub()(xt.device(), xt, positions, frequencies, shape, false);
  return result(y, {x}, "RotaryBackward",
                [positions, frequencies, shape](const Variable& out, variable_list& in) {
                  in[0].incr_grad_owned(tops::rotary_stub()(out.data().device(), out.grad(),
                                                            positions, frequencies, shape, true));
                });
}

Variable dropout(const Variable& x, const Variable* residual, Scalar rate, uint64_t seed,
                 Tensor state) {
  const Tensor& xt = x.data();
  LMP_CHECK(xt.type() == DataType::Float32 || xt.type() == DataType::Float64)
      << "dropout: x must be float32 or float64";
  LMP_CHECK(!residual || (residual->data().type() == xt.type() &&
                          residual->data().device() == xt.device() &&
                          residual->data().shape() == xt.shape()))
      << "dropout: the residual must be of x's type, device and shape";
  LMP_CHECK(state.type() == DataType::Int64 && state.numel() == 2 && state.device() == xt.device())
      << "dropout: the generator is not on x's device";
  variable_list ins{x};
  if (residual) ins.push_back(*residual);
  Tensor used;
  if (x.requires_grad() && wants_grad(ins)) used = empty({1}, xt.device(), DataType::Int64);
  tensor::keep_for_graph(tensor::detail::UnsafeTensorAccessor::getImpl(state));
  const Tensor y = tops::dropout_stub()(xt.device(), xt, residual ? residual->data() : Tensor(),
                                        rate, seed, state, &used);
  return result(y, std::move(ins), "DropoutBackward",
                [rate, seed, used](const Variable& out, variable_list& in) {
                  if (in[0].requires_grad())
                    in[0].incr_grad_owned(tops::dropout_backward_stub()(
                        out.data().device(), out.grad(), rate, seed, used));
                  if (in.size() > 1 && in[1].requires_grad()) in[1].incr_grad(out.grad());
                });
}

namespace {

// x [rows, in], w [in, width], b [width], all float32 on one device.
void check_linear(const char* name, const Variable& x, const Variable& w, const Variable* b) {
  const Tensor &xt = x.data(), &wt = w.data();
  const auto fits = [&](const Tensor& t) {
    return t.type() == DataType::Float32 && t.device() == xt.device();
  };
  LMP_CHECK(fits(xt) && fits(wt) && (!b || fits(b->data())))
      << name << ": x, the weights and the bias must be float32 on one device";
  LMP_CHECK(xt.shape().size() == 2 && wt.shape().size() == 2 && xt.shape()[1] == wt.shape()[0])
      << name << ": x " << xt.shape() << " and weights " << wt.shape() << " do not multiply";
  LMP_CHECK(!b || b->data().shape() == std::vector<size_t>{wt.shape()[1]})
      << name << ": the bias must have " << wt.shape()[1] << " values";
}

}  // namespace

Variable gated_linear(const Variable& x, const Variable& w, const Variable* b, int gate) {
  check_linear("gated_linear", x, w, b);
  LMP_CHECK(w.data().shape()[1] % 2 == 0)
      << "gated_linear: the weights' columns are the gate's and as many more, not "
      << w.data().shape()[1];
  variable_list ins{x, w};
  if (b) ins.push_back(*b);
  const tops::GatedOut out = tops::gated_linear_stub()(
      x.data().device(), gate, x.data(), w.data(), b ? b->data() : Tensor(), wants_grad(ins));
  return result(out.h, std::move(ins), "GatedLinearBackward",
                [gate, pre = out.pre](const Variable& h, variable_list& in) {
                  Tensor d[3];
                  for (size_t i = 0; i < in.size(); ++i)
                    if (in[i].requires_grad()) d[i] = empty_like(in[i].data());
                  tops::gated_linear_backward_stub()(h.data().device(), gate, h.grad(),
                                                     in[0].data(), in[1].data(), pre, &d[0], &d[1],
                                                     &d[2]);
                  for (size_t i = 0; i < in.size(); ++i)
                    if (d[i].defined()) in[i].incr_grad_owned(d[i]);
                });
}

namespace {

void check_targets(const Variable& x, const Tensor& targets, const Tensor& weights) {
  const size_t rows = x.data().shape()[0];
  LMP_CHECK(targets.type() == DataType::Int64 && targets.numel() == rows &&
            targets.device() == x.data().device())
      << "linear_cross_entropy: targets must be int64 on x's device, one for each of its " << rows
      << " rows";
  LMP_CHECK(!weights.defined() ||
            (weights.type() == DataType::Float32 && weights.numel() == rows &&
             weights.device() == x.data().device()))
      << "linear_cross_entropy: weights must be float32 on x's device, one for each of its " << rows
      << " rows";
  LMP_CHECK(rows > 0) << "linear_cross_entropy: no rows";
}

}  // namespace

Tensor linear_cross_entropy_rows(const Variable& x, const Variable& w, const Variable* b,
                                 const Tensor& targets) {
  check_linear("linear_cross_entropy", x, w, b);
  check_targets(x, targets, Tensor());
  tensor::keep_for_graph(tensor::detail::UnsafeTensorAccessor::getImpl(targets));
  Tensor none;
  return tops::linear_cross_entropy_stub()(x.data().device(), x.data(), w.data(),
                                           b ? b->data() : Tensor(), targets, Tensor(), &none,
                                           &none, &none);
}

Variable linear_cross_entropy(const Variable& x, const Variable& w, const Variable* b,
                              const Tensor& targets, const Tensor& weights) {
  check_linear("linear_cross_entropy", x, w, b);
  check_targets(x, targets, weights);
  const size_t rows = x.data().shape()[0];
  for (const Tensor* t : {&targets, &weights})
    if (t->defined())
      tensor::keep_for_graph(tensor::detail::UnsafeTensorAccessor::getImpl(*t));
  Tensor share;
  if (weights.defined()) {
    share = weights.reshape({rows});
  } else {
    const Tensor t = targets.reshape({rows});
    const Tensor counted =
        tops::ge(t, tensor::scalar_like(t, 0)) * tensor::scalar_like(x.data(), 1);
    share = counted / tops::clamp(tops::sum(counted, 0), 1, double(rows));
  }
  variable_list ins{x, w};
  if (b) ins.push_back(*b);
  Tensor d[3];
  const bool rg = wants_grad(ins);
  if (rg) {
    for (size_t i = 0; i < ins.size(); ++i)
      if (ins[i].requires_grad()) d[i] = empty_like(ins[i].data());
    // The bias' gradient rides with the weights'.
    if (d[2].defined() && !d[1].defined()) d[1] = empty_like(w.data());
  }
  const Tensor loss = tops::linear_cross_entropy_stub()(
      x.data().device(), x.data(), w.data(), b ? b->data() : Tensor(), targets,
      rg ? share : Tensor(), &d[0], &d[1], &d[2]);
  return result(tops::sum(tops::mul(loss, share), 0), std::move(ins), "LinearCrossEntropyBackward",
                [d0 = d[0], d1 = d[1], d2 = d[2]](const Variable& out, variable_list& in) {
                  const Tensor* d[3] = {&d0, &d1, &d2};
                  for (size_t i = 0; i < in.size(); ++i)
                    if (in[i].requires_grad()) in[i].incr_grad(tops::mul(*d[i], out.grad()));
                });
}

}  // namespace ops
}  // namespace lmp::autograd
