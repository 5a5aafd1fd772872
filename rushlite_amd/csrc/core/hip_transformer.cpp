// `*_hip` adapters of the transformer operators over
// include/lmp_hip_transformer.h, registered as hip_backend.cpp's are.
#include "lmp_hip_transformer.h"
#include "transformer.hpp"

namespace lmp::tensor::hip {
namespace {

using namespace ops;

void* at(const Tensor& t) {
  return t.defined() ? detail::UnsafeTensorAccessor::getImpl(t)->data() : nullptr;
}
float* f32(const Rows& r) {
  float* p = static_cast<float*>(at(r.t));
  return p ? p + r.at : nullptr;
}
float* f32(const Tensor& t) { return static_cast<float*>(at(t)); }
void count_launch() { ++backend_stats().eager_launches; }

LayerNormOut layer_norm_hip(const Tensor& x, const Tensor& w, const Tensor& b, Scalar eps,
                            bool stats) {
  const size_t n = x.shape().back(), rows = x.numel() / n;
  LayerNormOut out{empty(x.shape(), x.device(), x.type()), {}, {}};
  if (stats) {
    out.mean = empty({rows}, x.device(), x.type());
    out.rstd = empty({rows}, x.device(), x.type());
  }
  if (rows) count_launch();
  hip_ok(lmp_k_layer_norm(int(x.type()), rows, n, at(x), n, at(w), at(b), eps, at(out.y), n,
                          at(out.mean), at(out.rstd)),
         "lmp_k_layer_norm");
  return out;
}

void layer_norm_backward_hip(const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& mean,
                             const Tensor& rstd, Tensor* dx, Tensor* dw, Tensor* db) {
  const size_t n = x.shape().back(), rows = x.numel() / n;
  count_launch();
  hip_ok(lmp_k_layer_norm_backward(int(x.type()), rows, n, at(g), n, at(x), n, at(w), at(mean),
                                   at(rstd), at(*dx), n, at(*dw), at(*db)),
         "lmp_k_layer_norm_backward");
}

void attention_hip(const void* plan, const Rows& q, const Rows& k, const Rows& v, Scalar scale,
                   Tensor& o, Tensor* lse) {
  count_launch();
  hip_ok(lmp_k_attention_f32(plan, f32(q), q.ld, f32(k), k.ld, f32(v), v.ld, scale, f32(o),
                             o.shape()[1], lse ? f32(*lse) : nullptr),
         "lmp_k_attention_f32");
}

void attention_backward_hip(const void* plan, const Rows& q, const Rows& k, const Rows& v,
                            Scalar scale, const Tensor& o, const Tensor& lse, const Tensor& g,
                            const Rows& dq, const Rows& dk, const Rows& dv) {
  count_launch();
  hip_ok(lmp_k_attention_backward_f32(plan, f32(q), q.ld, f32(k), k.ld, f32(v), v.ld, scale, f32(o),
                                      o.shape()[1], f32(lse), f32(g), g.shape()[1], f32(dq), dq.ld,
                                      f32(dk), dk.ld, f32(dv), dv.ld),
         "lmp_k_attention_backward_f32");
}

void adamw_hip(int bits, const std::vector<AdamWParam>& params, const AdamWHyper& h, Tensor& step) {
  std::vector<lmp_adamw_tensor> list;
  list.reserve(params.size());
  for (const AdamWParam& p : params) {
    // The gradient too: formed before the capture, nothing else may hold it at a replay.
    for (const Tensor* t : {&p.p, &p.g, &p.m, &p.v, &p.m_scale, &p.v_scale})
      if (t->defined()) keep_for_graph(detail::UnsafeTensorAccessor::getImpl(*t));
    list.push_back({f32(p.p), f32(p.g), at(p.m), at(p.v), f32(p.m_scale), f32(p.v_scale),
                    p.p.numel(), p.decay});
  }
  keep_for_graph(detail::UnsafeTensorAccessor::getImpl(step));
  count_launch();
  hip_ok(lmp_k_adamw_f32(bits, list.size(), list.data(), h.lr, h.beta1, h.beta2, h.eps, h.seed,
                         static_cast<int64_t*>(at(step))),
         "lmp_k_adamw_f32");
}

Tensor adamw_decode_hip(bool signed_codes, const Tensor& codes, const Tensor& scales, size_t n) {
  Tensor out = empty({n}, codes.device(), DataType::Float32);
  if (n) count_launch();
  hip_ok(lmp_k_adamw_decode(signed_codes ? 1 : 0, at(codes), f32(scales), n, f32(out)),
         "lmp_k_adamw_decode");
  return out;
}

}  // namespace

constexpr DeviceType kHip = DeviceType::HIP;
LMP_REGISTER_DISPATCH(layer_norm_stub, kHip, layer_norm_hip)
LMP_REGISTER_DISPATCH(layer_norm_backward_stub, kHip, layer_norm_backward_hip)
LMP_REGISTER_DISPATCH(attention_stub, kHip, attention_hip)
LMP_REGISTER_DISPATCH(attention_backward_stub, kHip, attention_backward_hip)
LMP_REGISTER_DISPATCH(adamw_stub, kHip, adamw_hip)
LMP_REGISTER_DISPATCH(adamw_decode_stub, kHip, adamw_decode_hip)

}  // namespace lmp::tensor::hip
