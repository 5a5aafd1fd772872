// Packed attention: plans, checks and launches.  The kernels and their
// mathematics: attention_f32.hpp.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <new>
#include <string>

#include "common.hpp"
#include "lmp_hip_transformer.h"

#include "attention_f32.hpp"

namespace lmp_hip {
namespace {

struct AttentionPlan {
  int64_t heads, kv_heads, dim;
  bool causal;
  int64_t queries, keys, parts;
  double pairs;
  int rows_count, keys_count, joins_count;
  char* device = nullptr;  // the lists, one after another
  const AttnItem *rows, *key_items;
  const AttnJoin* joins;
};

// Calls f with the ND blocks of 16 columns that hold `dim`.
template <class F>
void with_dim(int64_t dim, F&& f) {
  using std::integral_constant;
  const int64_t nd = (dim + 15) / 16;
  if (nd <= 1) f(integral_constant<int, 1>{});
  else if (nd <= 2) f(integral_constant<int, 2>{});
  else if (nd <= 4) f(integral_constant<int, 4>{});
  else if (nd <= 5) f(integral_constant<int, 5>{});
  else if (nd <= 6) f(integral_constant<int, 6>{});
  else if (nd <= 8) f(integral_constant<int, 8>{});
  else f(integral_constant<int, 16>{});
}

// Grids stay below 2^32 threads; workgroups take further items in turn.
uint32_t grid_of(int64_t work) { return uint32_t(std::clamp<int64_t>(work, 1, int64_t(1) << 22)); }

struct Scratch {  // returned to the pool when the call ends, in stream order
  void* p = nullptr;
  ~Scratch() { if (p) scratch_free(p); }
  bool get(size_t bytes) { return bytes == 0 || (p = scratch_alloc(bytes)) != nullptr; }
};

AttnArgs common_args(const AttentionPlan& plan, double scale) {
  AttnArgs a{};
  a.kv_heads = int(plan.kv_heads);
  a.group = int(plan.heads / plan.kv_heads);
  a.dim = int(plan.dim);
  a.causal = plan.causal;
  a.scale = float(scale);
  return a;
}

int forward(Runtime* rt, const AttentionPlan& plan, AttnArgs a) {
  if (plan.queries == 0) return LMP_OK;
  Scratch part;
  const size_t slots = size_t(plan.parts) * size_t(plan.kv_heads) * kAttnRows;
  if (!part.get(slots * size_t(plan.dim + 2) * sizeof(float))) return LMP_ERR_OOM;
  a.part_ml = static_cast<float*>(part.p);
  a.part = a.part_ml + slots * 2;
  a.items = plan.rows;
  a.count = plan.rows_count;
  const uint32_t grid = grid_of(int64_t(a.count) * plan.kv_heads);
  with_dim(plan.dim, [&](auto nd) {
    attention_rows<nd><<<dim3(grid), dim3(256), 0, rt->stream>>>(a);
  });
  LMP_LAUNCH_CHECK("attention_rows");
  if (plan.joins_count) {
    attention_join<<<dim3(grid_of(int64_t(plan.joins_count) * plan.kv_heads)), dim3(256), 0,
                     rt->stream>>>(a, plan.joins, plan.joins_count);
    LMP_LAUNCH_CHECK("attention_join");
  }
  return LMP_OK;
}

int backward(Runtime* rt, const AttentionPlan& plan, AttnArgs a, const float* o, int64_t o_ld,
             float* dq, int64_t dq_ld, float* dk, int64_t dk_ld, float* dv, int64_t dv_ld) {
  Scratch delta;
  if (!delta.get(size_t(plan.queries) * size_t(plan.heads) * sizeof(float))) return LMP_ERR_OOM;
  if (plan.queries) {
    attention_delta<<<dim3(grid_of((plan.queries * plan.heads + 15) / 16)), dim3(256), 0,
                      rt->stream>>>(plan.queries, int(plan.heads), int(plan.dim), o, o_ld, a.g,
                                    a.g_ld, static_cast<float*>(delta.p));
    LMP_LAUNCH_CHECK("attention_delta");
    a.delta = static_cast<const float*>(delta.p);
    a.items = plan.rows;
    a.count = plan.rows_count;
    a.o = dq;
    a.o_ld = dq_ld;
    const uint32_t grid = grid_of(int64_t(a.count) * plan.kv_heads);
    with_dim(plan.dim, [&](auto nd) {
      attention_back_rows<nd><<<dim3(grid), dim3(256), 0, rt->stream>>>(a);
    });
    LMP_LAUNCH_CHECK("attention_back_rows");
  }
  if (plan.keys) {
    a.items = plan.key_items;
    a.count = plan.keys_count;
    a.o = dv;
    a.o_ld = dv_ld;
    a.dk = dk;
    a.dk_ld = dk_ld;
    const uint32_t grid = grid_of(int64_t(a.count) * plan.kv_heads);
    with_dim(plan.dim, [&](auto nd) {
      attention_back_keys<nd><<<dim3(grid), dim3(256), 0, rt->stream>>>(a);
    });
    LMP_LAUNCH_CHECK("attention_back_keys");
  }
  return LMP_OK;
}

// Lengths and indices are 32-bit in the kernels, which step a few hundred past
// them.
constexpr int64_t kMostRows = (int64_t(1) << 31) - 65536;

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_attention_plan_create(void** out, size_t sequences, const int64_t* q_lengths,
                                           const int64_t* k_lengths, size_t heads, size_t kv_heads,
                                           size_t head_dim, int causal) {
  const std::string name = "lmp_k_attention_plan_create: ";
  if (!out) return fail(LMP_ERR_INVALID, name + "null out pointer");
  *out = nullptr;
  if (sequences && (!q_lengths || !k_lengths)) return fail(LMP_ERR_INVALID, name + "null lengths");
  if (!heads || !kv_heads || heads % kv_heads)
    return fail(LMP_ERR_INVALID, name + "heads (" + std::to_string(heads) +
                                     ") is not a multiple of kv_heads (" +
                                     std::to_string(kv_heads) + ")");
  if (!head_dim) return fail(LMP_ERR_INVALID, name + "head_dim is 0");
  if (head_dim > LMP_ATTENTION_MAX_DIM)
    return fail(LMP_ERR_UNSUPPORTED, name + "head_dim " + std::to_string(head_dim) + " is above " +
                                         std::to_string(LMP_ATTENTION_MAX_DIM));
  if (heads > 65536) return fail(LMP_ERR_UNSUPPORTED, name + "more than 65536 heads");
  int64_t queries = 0, keys = 0;
  for (size_t i = 0; i < sequences; ++i) {
    if (q_lengths[i] < 0 || k_lengths[i] < 0)
      return fail(LMP_ERR_INVALID, name + "sequence " + std::to_string(i) + ": negative length");
    if (q_lengths[i] > kMostRows || k_lengths[i] > kMostRows ||
        (queries += q_lengths[i]) > kMostRows / int64_t(heads) || (keys += k_lengths[i]) > kMostRows)
      return fail(LMP_ERR_UNSUPPORTED, name + "too many rows");
  }
  LMP_RUNTIME_OR_FAIL(rt);
  // Host memory can run out here; no exception crosses the C boundary.
  try {
    AttnLists lists = attn_lists(sequences, q_lengths, k_lengths, int64_t(heads),
                                 int64_t(kv_heads), causal != 0, int64_t(rt->cu_count) * 4);
    auto plan = std::make_unique<AttentionPlan>();
    plan->heads = int64_t(heads);
    plan->kv_heads = int64_t(kv_heads);
    plan->dim = int64_t(head_dim);
    plan->causal = causal != 0;
    plan->queries = lists.queries;
    plan->keys = lists.key_rows;
    plan->parts = lists.parts;
    plan->pairs = lists.pairs;
    plan->rows_count = int(lists.rows.size());
    plan->keys_count = int(lists.keys.size());
    plan->joins_count = int(lists.joins.size());
    std::string bytes;
    const auto add = [&](const auto& v) {
      const size_t at = bytes.size();
      bytes.append(reinterpret_cast<const char*>(v.data()), v.size() * sizeof(v[0]));
      bytes.resize((bytes.size() + 255) / 256 * 256);
      return at;
    };
    const size_t rows = add(lists.rows), key_items = add(lists.keys), joins = add(lists.joins);
    if (!bytes.empty()) {
      void* p = nullptr;
      if (int s = lmp_rt_malloc(&p, bytes.size())) return s;
      if (int s = lmp_rt_memcpy_h2d(p, bytes.data(), bytes.size())) {
        lmp_rt_free(p);
        return s;
      }
      plan->device = static_cast<char*>(p);
    }
    plan->rows = reinterpret_cast<const AttnItem*>(plan->device + rows);
    plan->key_items = reinterpret_cast<const AttnItem*>(plan->device + key_items);
    plan->joins = reinterpret_cast<const AttnJoin*>(plan->device + joins);
    *out = plan.release();
  } catch (const std::exception& e) {
    return fail(LMP_ERR_OOM, name + e.what());
  }
  return LMP_OK;
}

extern "C" int lmp_k_attention_plan_destroy(void* handle) {
  if (!handle) return LMP_OK;
  std::unique_ptr<AttentionPlan> plan(static_cast<AttentionPlan*>(handle));
  return plan->device ? lmp_rt_free(plan->device) : LMP_OK;
}

namespace {
// The operands both passes share.
int check_operands(const char* name, const AttentionPlan* plan, const float* q, size_t q_ld,
                   const float* k, size_t k_ld, const float* v, size_t v_ld, double scale) {
  if (!plan) return fail(LMP_ERR_INVALID, std::string(name) + ": null plan");
  if (!std::isfinite(scale)) return fail(LMP_ERR_INVALID, std::string(name) + ": scale is not finite");
  if ((plan->queries && !q) || (plan->keys && (!k || !v)))
    return fail(LMP_ERR_INVALID, std::string(name) + ": null buffer");
  const size_t qw = size_t(plan->heads * plan->dim), kw = size_t(plan->kv_heads * plan->dim);
  if (q_ld < qw || k_ld < kw || v_ld < kw)
    return fail(LMP_ERR_INVALID, std::string(name) + ": leading dimension below a row's heads");
  return LMP_OK;
}
}  // namespace

extern "C" int lmp_k_attention_f32(const void* handle, const float* q, size_t q_ld, const float* k,
                                   size_t k_ld, const float* v, size_t v_ld, double scale, float* o,
                                   size_t o_ld, float* lse) {
  const char* name = "lmp_k_attention_f32";
  const auto* plan = static_cast<const AttentionPlan*>(handle);
  if (int s = check_operands(name, plan, q, q_ld, k, k_ld, v, v_ld, scale)) return s;
  if (plan->queries && !o) return fail(LMP_ERR_INVALID, std::string(name) + ": null buffer");
  if (o_ld < size_t(plan->heads * plan->dim))
    return fail(LMP_ERR_INVALID, std::string(name) + ": leading dimension below a row's heads");
  LMP_RUNTIME_OR_FAIL(rt);
  AttnArgs a = common_args(*plan, scale);
  a.q = q;
  a.q_ld = int64_t(q_ld);
  a.k = k;
  a.k_ld = int64_t(k_ld);
  a.v = v;
  a.v_ld = int64_t(v_ld);
  a.o = o;
  a.o_ld = int64_t(o_ld);
  a.lse = lse;
  return forward(rt, *plan, a);
}

extern "C" int lmp_k_attention_backward_f32(const void* handle, const float* q, size_t q_ld,
                                            const float* k, size_t k_ld, const float* v,
                                            size_t v_ld, double scale, const float* o, size_t o_ld,
                                            const float* lse, const float* g, size_t g_ld,
                                            float* dq, size_t dq_ld, float* dk, size_t dk_ld,
                                            float* dv, size_t dv_ld) {
  const char* name = "lmp_k_attention_backward_f32";
  const auto* plan = static_cast<const AttentionPlan*>(handle);
  if (int s = check_operands(name, plan, q, q_ld, k, k_ld, v, v_ld, scale)) return s;
  if ((plan->queries && (!o || !lse || !g || !dq)) || (plan->keys && (!dk || !dv)))
    return fail(LMP_ERR_INVALID, std::string(name) + ": null buffer");
  const size_t qw = size_t(plan->heads * plan->dim), kw = size_t(plan->kv_heads * plan->dim);
  if (o_ld < qw || g_ld < qw || dq_ld < qw || dk_ld < kw || dv_ld < kw)
    return fail(LMP_ERR_INVALID, std::string(name) + ": leading dimension below a row's heads");
  LMP_RUNTIME_OR_FAIL(rt);
  AttnArgs a = common_args(*plan, scale);
  a.q = q;
  a.q_ld = int64_t(q_ld);
  a.k = k;
  a.k_ld = int64_t(k_ld);
  a.v = v;
  a.v_ld = int64_t(v_ld);
  a.g = g;
  a.g_ld = int64_t(g_ld);
  a.lse_in = lse;
  return backward(rt, *plan, a, o, int64_t(o_ld), dq, int64_t(dq_ld), dk, int64_t(dk_ld), dv,
                  int64_t(dv_ld));
}
