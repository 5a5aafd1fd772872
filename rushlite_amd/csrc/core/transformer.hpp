// Transformer-training operators over tensors and variables: layer norm, packed
// attention, the AdamW step, rotary positions, dropout, gated linear layers and
// the cross entropy over a vocabulary (include/lmp_hip_transformer.h).  The
// reference has none of them; they run on the HIP device only, as every op here
// does.
#pragma once

#include <memory>
#include <vector>

#include "autograd.hpp"

namespace lmp::tensor::ops {

// y, and the rows' mean and rstd where `stats` (else left undefined).  w and b
// may be undefined (1 and 0).
struct LayerNormOut {
  Tensor y, mean, rstd;
};
using layer_norm_fn = LayerNormOut (*)(const Tensor& x, const Tensor& w, const Tensor& b,
                                       Scalar eps, bool stats);
// Writes those of dx, dw and db that are defined.
using layer_norm_backward_fn = void (*)(const Tensor& g, const Tensor& x, const Tensor& w,
                                        const Tensor& mean, const Tensor& rstd, Tensor* dx,
                                        Tensor* dw, Tensor* db);

// Rows of `ld` values, of which the heads' vectors start `at` values in.
struct Rows {
  Tensor t;
  size_t ld = 0, at = 0;
};
using attention_fn = void (*)(const void* plan, const Rows& q, const Rows& k, const Rows& v,
                              Scalar scale, Tensor& o, Tensor* lse);
using attention_backward_fn = void (*)(const void* plan, const Rows& q, const Rows& k,
                                       const Rows& v, Scalar scale, const Tensor& o,
                                       const Tensor& lse, const Tensor& g, const Rows& dq,
                                       const Rows& dk, const Rows& dv);

struct AdamWParam {
  Tensor p, g, m, v, m_scale, v_scale;  // scales undefined for states of 32 bits
  Scalar decay = 0;
};
struct AdamWHyper {
  Scalar lr, beta1, beta2, eps;
  uint64_t seed;
};
using adamw_fn = void (*)(int bits, const std::vector<AdamWParam>& params, const AdamWHyper& hyper,
                          Tensor& step);
using adamw_decode_fn = Tensor (*)(bool signed_codes, const Tensor& codes, const Tensor& scales,
                                   size_t n);

// Pairs of the first heads * head_dim columns turned by position x frequency.
struct RotaryShape {
  size_t heads, head_dim;
  bool interleaved;
  Scalar scale;
};
using rotary_fn = Tensor (*)(const Tensor& x, const Tensor& positions, const Tensor& frequencies,
                             const RotaryShape& shape, bool inverse);

// The call's number goes to *used where `used` is defined.
using dropout_fn = Tensor (*)(const Tensor& x, const Tensor& residual, Scalar rate, uint64_t seed,
                              Tensor& state, Tensor* used);
using dropout_backward_fn = Tensor (*)(const Tensor& g, Scalar rate, uint64_t seed,
                                       const Tensor& used);

// h, and [a | u] where `keep` (else left undefined); bias may be undefined.
struct GatedOut {
  Tensor h, pre;
};
using gated_linear_fn = GatedOut (*)(int gate, const Tensor& x, const Tensor& w, const Tensor& bias,
                                     bool keep);
// Writes those of dx, dw and db that are defined.
using gated_linear_backward_fn = void (*)(int gate, const Tensor& g, const Tensor& x,
                                          const Tensor& w, const Tensor& pre, Tensor* dx,
                                          Tensor* dw, Tensor* db);

// The losses of the rows; with `weights` defined also those of dx, dw and db that
// are defined, of the weighted sum.
using linear_cross_entropy_fn = Tensor (*)(const Tensor& x, const Tensor& w, const Tensor& bias,
                                           const Tensor& targets, const Tensor& weights, Tensor* dx,
                                           Tensor* dw, Tensor* db);

LMP_DECLARE_DISPATCH(layer_norm_fn, layer_norm_stub)
LMP_DECLARE_DISPATCH(rotary_fn, rotary_stub)
LMP_DECLARE_DISPATCH(dropout_fn, dropout_stub)
LMP_DECLARE_DISPATCH(dropout_backward_fn, dropout_backward_stub)
LMP_DECLARE_DISPATCH(gated_linear_fn, gated_linear_stub)
LMP_DECLARE_DISPATCH(gated_linear_backward_fn, gated_linear_backward_stub)
LMP_DECLARE_DISPATCH(linear_cross_entropy_fn, linear_cross_entropy_stub)
LMP_DECLARE_DISPATCH(layer_norm_backward_fn, layer_norm_backward_stub)
LMP_DECLARE_DISPATCH(attention_fn, attention_stub)
LMP_DECLARE_DISPATCH(attention_backward_fn, attention_backward_stub)
LMP_DECLARE_DISPATCH(adamw_fn, adamw_stub)
LMP_DECLARE_DISPATCH(adamw_decode_fn, adamw_decode_stub)

// One AdamW step: every p (float32, updated in place) by its g and states.
// States of 32 bits are float32 of p's size; of 8 bits they are int32 tensors
// of ceil(n / 4) values holding n codes, with float32 scales of
// ceil(n / LMP_ADAMW_BLOCK) values.  `step` is an int64 tensor of 2 values.
void adamw(int bits, const std::vector<AdamWParam>& params, const AdamWHyper& hyper, Tensor& step);
// The n values a state of 8 bits stands for.
Tensor adamw_decode(bool signed_codes, const Tensor& codes, const Tensor& scales, size_t n);

}  // namespace lmp::tensor::ops

namespace lmp::autograd {

// The work lists of a packed batch (lmp_k_attention_plan_create).  Graphs that
// record calls with a plan keep its lists.
class AttentionPlan {
 public:
  AttentionPlan(const std::vector<int64_t>& q_lengths, const std::vector<int64_t>& k_lengths,
                size_t heads, size_t kv_heads, size_t head_dim, bool causal);
  const std::shared_ptr<const void>& handle() const { return handle_; }
  size_t heads, kv_heads, head_dim, queries = 0, keys = 0;
  bool causal;

 private:
  std::shared_ptr<const void> handle_;
};

namespace ops {
// (x - mean) / sqrt(var + eps) * w + b over the last axis; w and b of that
// axis' size, or null for 1 and 0.
Variable layer_norm(const Variable& x, const Variable* w, const Variable* b, Scalar eps);
// softmax(scale q k^T + mask) v of a packed batch: q [queries, heads * dim], k
// and v [keys, kv_heads * dim].
Variable attention(const Variable& q, const Variable& k, const Variable& v,
                   const AttentionPlan& plan, Scalar scale);
// x [rows, columns] with the pairs of its first heads * head_dim columns turned by
// positions[row] * frequencies[pair] (int64 and float64 tensors); a head's first
// 2 * frequencies values turn.
Variable rotary(const Variable& x, const Tensor& positions, const Tensor& frequencies,
                const tensor::ops::RotaryShape& shape);
// residual + (kept ? x / (1 - rate) : 0); `state` (two int64) counts the calls.
Variable dropout(const Variable& x, const Variable* residual, Scalar rate, uint64_t seed,
                 Tensor state);
// act(a) u for [a | u] = x w + b.
Variable gated_linear(const Variable& x, const Variable& w, const Variable* b, int gate);
// The cross entropies of the rows of x w + b against targets (int64), without a gradient.
Tensor linear_cross_entropy_rows(const Variable& x, const Variable& w, const Variable* b,
                                 const Tensor& targets);
// Their sum weighted by `weights` ([rows] float32; undefined: the mean over the rows whose
// targets are not negative), of shape [1].  The gradients are formed with the losses.
Variable linear_cross_entropy(const Variable& x, const Variable& w, const Variable* b,
                              const Tensor& targets, const Tensor& weights);
// The same with q, k and v side by side in the rows of one projection:
// [queries, (heads + 2 kv_heads) * dim].
Variable attention_qkv(const Variable& rows, const AttentionPlan& plan, Scalar scale);
}  // namespace ops

}  // namespace lmp::autograd
