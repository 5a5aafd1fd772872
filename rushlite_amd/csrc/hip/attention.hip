// Packed attention: plans, checks and launches.  The kernels and their
// mathematics: attention_f32.hpp and attention_split.hpp.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <memory>
#include <new>
#include <string>

#include "common.hpp"
#include "lmp_hip_transformer.h"

#include "attention_split.hpp"

namespace lmp_hip {
namespace {

// A list on the device.
template <class T>
struct List {
  const T* at = nullptr;
  int count = 0;
};

struct AttentionPlan {
  int64_t heads, kv_heads, dim;
  bool causal;
  int64_t queries, keys, parts, q_parts, k_parts;
  double row_work, block_work;  // AttnLists'
  int64_t longest_q = 0, longest_k = 0;
  // Each sequence has one item of packed rows, so that a pass reads every key once,
  // and the keys and values pass the memory-side cache (kStreamBytes).
  bool keys_once;
  char* device = nullptr;  // the lists, one after another
  List<AttnItem> rows, key_items, q_blocks, k_blocks;
  List<AttnJoin> joins, q_joins, k_joins;
  List<AttnTile> q_tiles, k_tiles;
  List<AttnSeq> seqs;
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
  bool get(size_t bytes) {
    if (p) scratch_free(p);
    p = bytes ? scratch_alloc(bytes) : nullptr;
    return !bytes || p;
  }
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

// Whether the split-fp16 kernels run a pass: where they take less time by what
// both forms have to do.  The rates are a fit to batches on this card.  Over 160 (8 to
// 2048 queries, 64 to 8192 keys, 1 to 32 heads of 32, 64 and 128) the form it takes is
// 0.7% slower than the faster one on average, forward, and 2.6% backward; at worst 1.26
// times as slow, forward (4 sequences of 500, 16 heads of 32: 25 | 31), and 2.3
// times, backward (8 queries against each of 8 x 1024 keys, 8 heads of 128: 216 | 95).
// Others, fp32 | split in us: forward, one sequence of 1024, 4 heads of 128, 42 | 38;
// 16 heads on 4, 89 | 42; 8 queries against 8 x 8192 keys, 32 heads on 4, 149 | 304; 64
// queries, 895 | 400; backward, one sequence of 256, 4 heads of 64, 27 | 43; of 1024, 16
// heads of 64 on 4, 220 | 75; 8 queries against 8 x 8192 keys, 32 heads on 4, 1246 | 880.
bool split_form(const AttentionPlan& plan, double scale, bool back) {
  const double q_tiles = double(plan.q_tiles.count) * double(plan.heads),
               k_tiles = double(plan.k_tiles.count) * double(plan.kv_heads);
  // Grids stay below 2^32 threads; a scale of 0 leaves no power of two to divide.
  if (plan.dim > 128 || scale == 0 || !plan.queries || !plan.keys ||
      2 * (q_tiles + k_tiles) >= double(1 << 22) ||
      double(plan.seqs.count) * double(plan.kv_heads) >= double(1 << 22))
    return false;
  // In millions: the multiplications of one product in each form's steps, and the
  // bytes of a split operand's fragments.
  const double dim = double(plan.dim), f32 = plan.row_work * double(plan.kv_heads) * dim / 1e6,
               split = plan.block_work * double(plan.heads) * dim / 1e6,
               q = q_tiles * dim * 256 / 1e6, k = k_tiles * dim * 256 / 1e6;
  if (!back) return 10 + 0.077 * f32 > 20 + 0.011 * split + 0.22 * (q + 2 * k);
  // The fp32 kernels do not share out the keys of a row or the rows of a key.
  const double chain =
      double(plan.longest_k + plan.longest_q * (plan.heads / plan.kv_heads)) * dim / 1e3;
  return 13 + 0.27 * f32 + 0.46 * chain > 41 + 0.041 * split + 0.134 * (3 * q + 4 * k);
}

// Calls f with the ND of the split kernels that hold `dim` (at most 128).
template <class F>
void with_split_dim(int64_t dim, F&& f) {
  using std::integral_constant;
  const int64_t nd = (dim + 15) / 16;
  if (nd <= 2) f(integral_constant<int, 2>{});
  else if (nd <= 4) f(integral_constant<int, 4>{});
  else if (nd <= 5) f(integral_constant<int, 5>{});
  else if (nd <= 6) f(integral_constant<int, 6>{});
  else f(integral_constant<int, 8>{});
}

// The operands' fragments, exponents and marks in one allocation.
struct SplitOperands {
  Scratch memory;
  SplitAttnArgs args{};
  float* stats = nullptr;
  int32_t* any_mark = nullptr;
};

// Splits q, k, v (and g) for the forward or the backward kernels.  LMP_ERR_OOM
// leaves nothing launched.
int split_operands(Runtime* rt, const AttentionPlan& plan, const AttnArgs& a, double scale,
                   bool back, SplitOperands& out) {
  const int64_t qn = int64_t(plan.q_tiles.count) * plan.heads,
                kn = int64_t(plan.k_tiles.count) * plan.kv_heads;
  int status = LMP_OK;
  with_split_dim(plan.dim, [&](auto nd) {
    using F = Frag<nd>;
    size_t bytes = 0;
    const auto place = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    const size_t q_along = place(qn * F::ALONG), k_along = place(kn * F::ALONG);
    const size_t v_across = place(back ? 0 : kn * F::ACROSS), v_along = place(back ? kn * F::ALONG : 0);
    const size_t g_along = place(back ? qn * F::ALONG : 0);
    const size_t q_across = place(back ? qn * F::ACROSS : 0), g_across = place(back ? qn * F::ACROSS : 0);
    const size_t k_across = place(back ? kn * F::ACROSS : 0);
    const size_t exps = place((2 * qn + 2 * kn) * 4), marks = place((plan.seqs.count * plan.kv_heads + 1) * 4);
    const size_t stats = place(back ? qn * 256 : 0);
    if (!out.memory.get(bytes)) {
      status = LMP_ERR_OOM;
      return;
    }
    char* m = static_cast<char*>(out.memory.p);
    int32_t* e = reinterpret_cast<int32_t*>(m + exps);
    SplitAttnArgs& s = out.args;
    s.kv_heads = int(plan.kv_heads);
    s.group = int(plan.heads / plan.kv_heads);
    s.dim = int(plan.dim);
    s.causal = plan.causal;
    s.scale = float(scale);
    s.scale_log2e = std::fabs(float(scale)) * kLog2e;
    s.q_along = m + q_along;
    s.k_along = m + k_along;
    s.v_along = m + v_along;
    s.v_across = m + v_across;
    s.g_along = m + g_along;
    s.q_across = m + q_across;
    s.g_across = m + g_across;
    s.k_across = m + k_across;
    s.q_exp = e;
    s.k_exp = e + qn;
    s.v_exp = e + qn + kn;
    s.g_exp = back ? e + qn + 2 * kn : nullptr;
    s.marks = reinterpret_cast<const int32_t*>(m + marks);
    out.any_mark = reinterpret_cast<int32_t*>(m + marks) + plan.seqs.count * plan.kv_heads;
    out.stats = reinterpret_cast<float*>(m + stats);
    s.stats = out.stats;
    SplitArgs p{};
    p.dim = int(plan.dim);
    p.any_mark = out.any_mark;
    const auto add = [&](const float* x, int64_t ld, bool queries, float sign, char* along,
                         char* across, const int32_t* exponent) {
      const auto& tiles = queries ? plan.q_tiles : plan.k_tiles;
      if (tiles.count)
        p.op[p.count++] = {x, ld, tiles.at, tiles.count, int(queries ? plan.heads : plan.kv_heads),
                           sign, along, across, const_cast<int32_t*>(exponent),
                           nullptr, 0, nullptr, nullptr, nullptr};
    };
    add(a.q, a.q_ld, true, scale < 0 ? -1.0f : 1.0f, m + q_along, back ? m + q_across : nullptr, s.q_exp);
    add(a.k, a.k_ld, false, 1.0f, m + k_along, back ? m + k_across : nullptr, s.k_exp);
    add(a.v, a.v_ld, false, 1.0f, back ? m + v_along : nullptr, back ? nullptr : m + v_across, s.v_exp);
    if (back && plan.queries) {
      add(a.g, a.g_ld, true, 1.0f, m + g_along, m + g_across, s.g_exp);
      SplitOperand& g = p.op[p.count - 1];
      g.out = a.out;
      g.out_ld = a.out_ld;
      g.lse = a.lse_in;
      g.stats = out.stats;
      g.delta = a.delta;
    }
    attention_split<nd><<<dim3(uint32_t(qn + 2 * kn + (back ? qn : 0))), dim3(256), 0, rt->stream>>>(p);
    status = [&]() -> int {
      LMP_LAUNCH_CHECK("attention_split");
      attention_marks<<<dim3(uint32_t(plan.seqs.count * plan.kv_heads)), dim3(256), 0, rt->stream>>>(
          plan.seqs.at, s.kv_heads, s.group, s.q_exp, s.k_exp, s.v_exp, s.g_exp,
          const_cast<int32_t*>(s.marks), out.any_mark);
      LMP_LAUNCH_CHECK("attention_marks");
      return LMP_OK;
    }();
  });
  return status;
}

// Launches a split kernel with its stages of LDS, which pass 64 KiB.
template <class Kernel>
int launch_split(Runtime* rt, const char* name, Kernel kernel, int64_t grid, int threads,
                 int lds, const SplitAttnArgs& s) {
  LMP_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  kernel<<<dim3(uint32_t(grid)), dim3(threads), size_t(lds), rt->stream>>>(s);
  LMP_LAUNCH_CHECK(name);
  return LMP_OK;
}

// The fp32 kernels, over all rows or over the marked ones only (none as a rule:
// a small grid finds that out).
uint32_t f32_grid(const AttnArgs& a) {
  const int64_t work = int64_t(a.count) * a.kv_heads;
  return grid_of(a.marks ? std::min<int64_t>(work, 256) : work);
}
// Calls f with the ND of the columns and the waves of a backward workgroup: eight
// where two workgroups of four would leave compute units idle (columns past 128
// have no registers for them).
template <class F>
void with_back_form(Runtime* rt, const AttnArgs& a, F&& f) {
  using std::integral_constant;
  const bool few = int64_t(a.count) * a.kv_heads <= int64_t(rt->cu_count) * 2;
  with_dim(a.dim, [&](auto nd) {
    constexpr int most = nd <= 8 ? 8 : 4;
    if (few) f(nd, integral_constant<int, most>{});
    else f(nd, integral_constant<int, 4>{});
  });
}
int forward_f32(Runtime* rt, const AttentionPlan& plan, AttnArgs a) {
  a.items = plan.rows.at;
  a.count = plan.rows.count;
  with_dim(plan.dim, [&](auto nd) {
    if (plan.keys_once && !a.marks)
      attention_rows<nd, true><<<dim3(f32_grid(a)), dim3(256), 0, rt->stream>>>(a);
    else
      attention_rows<nd, false><<<dim3(f32_grid(a)), dim3(256), 0, rt->stream>>>(a);
  });
  LMP_LAUNCH_CHECK("attention_rows");
  return LMP_OK;
}

int forward(Runtime* rt, const AttentionPlan& plan, AttnArgs a, double scale) {
  if (plan.queries == 0) return LMP_OK;
  SplitOperands split;
  Scratch part;
  const auto parts = [&](int64_t n, int64_t heads, int64_t rows) {
    const size_t slots = size_t(n) * size_t(heads) * size_t(rows);
    if (!part.get(slots * size_t(plan.dim + 2) * sizeof(float))) return false;
    a.part_ml = static_cast<float*>(part.p);
    a.part = a.part_ml + slots * 2;
    return true;
  };
  // Without memory for the fragments the fp32 kernels, which need none, take over.
  int status = LMP_ERR_OOM;
  if (split_form(plan, scale, false) && parts(plan.q_parts, plan.heads, kAttnSplitRows))
    status = split_operands(rt, plan, a, scale, false, split);
  if (status != LMP_ERR_OOM) {
    if (status) return status;
    SplitAttnArgs& s = split.args;
    s.items = plan.q_blocks.at;
    s.count = plan.q_blocks.count;
    s.o = a.o;
    s.o_ld = a.o_ld;
    s.lse = a.lse;
    s.part = a.part;
    s.part_ml = a.part_ml;
    with_split_dim(plan.dim, [&](auto nd) {
      status = launch_split(rt, "attention_split_rows", attention_split_rows<nd>,
                            int64_t(s.count) * plan.heads, 256,
                            2 * (Frag<nd>::ALONG + Frag<nd>::ACROSS), s);
    });
    if (status) return status;
    if (plan.q_joins.count) {
      AttnArgs j = a;  // every head's rows by themselves
      j.kv_heads = int(plan.heads);
      j.group = 1;
      attention_join<kAttnSplitRows>
          <<<dim3(grid_of(int64_t(plan.q_joins.count) * plan.heads * (kAttnSplitRows / 16))),
             dim3(256), 0, rt->stream>>>(j, plan.q_joins.at, plan.q_joins.count);
      LMP_LAUNCH_CHECK("attention_join");
    }
    a.marks = s.marks;
    a.any_mark = split.any_mark;
    return forward_f32(rt, plan, a);
  }
  if (!parts(plan.parts, plan.kv_heads, kAttnRows)) return LMP_ERR_OOM;
  if (int s = forward_f32(rt, plan, a)) return s;
  if (plan.joins.count) {
    attention_join<kAttnRows>
        <<<dim3(grid_of(int64_t(plan.joins.count) * plan.kv_heads)), dim3(256), 0, rt->stream>>>(
            a, plan.joins.at, plan.joins.count);
    LMP_LAUNCH_CHECK("attention_join");
  }
  return LMP_OK;
}

int backward(Runtime* rt, const AttentionPlan& plan, AttnArgs a, double scale, const float* o,
             int64_t o_ld, float* dq, int64_t dq_ld, float* dk, int64_t dk_ld, float* dv,
             int64_t dv_ld) {
  Scratch delta;
  SplitOperands split;
  if (!delta.get(size_t(plan.queries) * size_t(plan.heads) * sizeof(float))) return LMP_ERR_OOM;
  a.delta = static_cast<float*>(delta.p);
  a.out = o;
  a.out_ld = o_ld;
  AttnArgs rows = a, keys = a;
  rows.items = plan.rows.at;
  rows.count = plan.rows.count;
  rows.o = dq;
  rows.o_ld = dq_ld;
  keys.items = plan.key_items.at;
  keys.count = plan.key_items.count;
  keys.o = dv;
  keys.o_ld = dv_ld;
  keys.dk = dk;
  keys.dk_ld = dk_ld;
  // Rows first, then keys; each one's parts are summed before the next needs the
  // memory.
  const size_t slot = size_t(kAttnSplitRows) * size_t(plan.dim) * sizeof(float);
  const size_t q_bytes = size_t(plan.q_parts) * size_t(plan.heads) * slot,
               k_bytes = size_t(plan.k_parts) * size_t(plan.kv_heads) * slot;
  Scratch part;
  int status = LMP_ERR_OOM;  // as in forward()
  if (split_form(plan, scale, true) && part.get(std::max(q_bytes, 2 * k_bytes)))
    status = split_operands(rt, plan, a, scale, true, split);
  if (status != LMP_ERR_OOM) {
    if (status) return status;
    SplitAttnArgs& s = split.args;
    s.part = static_cast<float*>(part.p);
    s.part_dk = int64_t(k_bytes / sizeof(float));
    const auto sum = [&](const SumArgs& p, int results) -> int {
      if (!p.count) return LMP_OK;
      const uint32_t grid = grid_of(int64_t(p.count) * p.heads * (kAttnSplitRows / 16));
      attention_sum<<<dim3(grid, uint32_t(results)), dim3(256), 0, rt->stream>>>(p);
      LMP_LAUNCH_CHECK("attention_sum");
      return LMP_OK;
    };
    with_split_dim(plan.dim, [&](auto nd) {
      using F = Frag<nd>;
      SplitAttnArgs r = s;
      r.items = plan.q_blocks.at;
      r.count = plan.q_blocks.count;
      r.o = dq;
      r.o_ld = dq_ld;
      status = launch_split(rt, "attention_split_back_rows", attention_split_back_rows<nd>,
                            int64_t(r.count) * plan.heads, 512,
                            4 * F::ALONG + 2 * F::ACROSS + 8 * 4096, r);
      if (!status)
        status = sum({plan.q_joins.at, plan.q_joins.count, int(plan.heads), int(plan.dim),
                      {r.part}, {dq}, {dq_ld}}, 1);
      if (status || !plan.keys) return;
      SplitAttnArgs k = s;
      k.items = plan.k_blocks.at;
      k.count = plan.k_blocks.count;
      k.scale = std::fabs(s.scale);  // q's parts carry its sign
      k.o = dv;
      k.o_ld = dv_ld;
      k.dk = dk;
      k.dk_ld = dk_ld;
      status = launch_split(rt, "attention_split_back_keys", attention_split_back_keys<nd>,
                            int64_t(k.count) * plan.kv_heads, 512,
                            4 * F::ALONG + 4 * F::ACROSS + 4 * 4096, k);
      if (!status)
        status = sum({plan.k_joins.at, plan.k_joins.count, int(plan.kv_heads), int(plan.dim),
                      {k.part, k.part + k.part_dk}, {dv, dk}, {dv_ld, dk_ld}}, 2);
    });
    if (status) return status;
    for (AttnArgs* x : {&rows, &keys}) {
      x->marks = s.marks;
      x->any_mark = split.any_mark;
    }
    const uint32_t grid = std::max(f32_grid(rows), f32_grid(keys));
    with_split_dim(plan.dim, [&](auto nd) {
      attention_back_marked<nd><<<dim3(grid), dim3(256), 0, rt->stream>>>(rows, keys);
    });
    LMP_LAUNCH_CHECK("attention_back_marked");
    return LMP_OK;
  }
  if (plan.queries) {
    with_back_form(rt, rows, [&](auto nd, auto waves) {
      attention_back_rows<nd, waves><<<dim3(f32_grid(rows)), dim3(waves * 64), 0, rt->stream>>>(rows);
    });
    LMP_LAUNCH_CHECK("attention_back_rows");
  }
  if (plan.keys) {
    with_back_form(rt, keys, [&](auto nd, auto waves) {
      attention_back_keys<nd, waves><<<dim3(f32_grid(keys)), dim3(waves * 64), 0, rt->stream>>>(keys);
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
                                 int64_t(kv_heads), causal != 0, int64_t(rt->cu_count));
    auto plan = std::make_unique<AttentionPlan>();
    plan->heads = int64_t(heads);
    plan->kv_heads = int64_t(kv_heads);
    plan->dim = int64_t(head_dim);
    plan->causal = causal != 0;
    plan->queries = lists.queries;
    plan->keys = lists.key_rows;
    plan->parts = lists.parts;
    plan->row_work = lists.row_work;
    plan->keys_once = uint64_t(lists.key_rows) * kv_heads * head_dim * 8 >= kStreamBytes;
    for (size_t i = 0; i < sequences; ++i) {
      plan->longest_q = std::max(plan->longest_q, q_lengths[i]);
      plan->longest_k = std::max(plan->longest_k, k_lengths[i]);
      plan->keys_once = plan->keys_once && q_lengths[i] * int64_t(heads / kv_heads) <= kAttnRows;
    }
    plan->block_work = lists.block_work;
    plan->q_parts = lists.q_parts;
    plan->k_parts = lists.k_parts;
    std::string bytes;
    // Appends a list; its place is an offset until the memory is there.
    const auto add = [&](const auto& v, auto& list) {
      using T = std::remove_cv_t<std::remove_pointer_t<decltype(list.at)>>;
      list.at = reinterpret_cast<const T*>(bytes.size());
      list.count = int(v.size());
      bytes.append(reinterpret_cast<const char*>(v.data()), v.size() * sizeof(T));
      bytes.resize((bytes.size() + 255) / 256 * 256);
    };
    const auto each = [&](auto&& f) {
      f(lists.rows, plan->rows);
      f(lists.keys, plan->key_items);
      f(lists.q_blocks, plan->q_blocks);
      f(lists.k_blocks, plan->k_blocks);
      f(lists.joins, plan->joins);
      f(lists.q_joins, plan->q_joins);
      f(lists.k_joins, plan->k_joins);
      f(lists.q_tiles, plan->q_tiles);
      f(lists.k_tiles, plan->k_tiles);
      f(lists.seqs, plan->seqs);
    };
    each(add);
    if (!bytes.empty()) {
      void* p = nullptr;
      if (int s = lmp_rt_malloc(&p, bytes.size())) return s;
      if (int s = lmp_rt_memcpy_h2d(p, bytes.data(), bytes.size())) {
        lmp_rt_free(p);
        return s;
      }
      plan->device = static_cast<char*>(p);
    }
    each([&](const auto&, auto& list) {
      using T = std::remove_cv_t<std::remove_pointer_t<decltype(list.at)>>;
      list.at = reinterpret_cast<const T*>(plan->device + reinterpret_cast<size_t>(list.at));
    });
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
  if (!std::isfinite(float(scale))) return fail(LMP_ERR_INVALID, std::string(name) + ": scale is not finite");
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
  return forward(rt, *plan, a, scale);
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
  return backward(rt, *plan, a, scale, o, int64_t(o_ld), dq, int64_t(dq_ld), dk, int64_t(dk_ld), dv,
                  int64_t(dv_ld));
}
