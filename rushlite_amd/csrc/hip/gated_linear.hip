// A gated linear layer: h = act(x Wg + bg) (x Wu + bu), both projections from one weight
// matrix [Wg | Wu], and its gradients.
//
//   pre = x W + b = [a | u],  h = act(a) u
//   d = [g u act'(a) | g act(a)],  dx = d W^T,  dW = x^T d,  db = the column sums of d
//
// Large layers run on the fp16 matrix cores (gemm_half.hpp): forward as one kernel, whose
// epilogue forms h; backward d in one pass, with the largest magnitudes and the column sums,
// then both products in one launch.  Smaller ones take the framework's fp32 products.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "gate.hpp"
#include "gemm_half.hpp"
#include "half_products.hpp"
#include "lmp_hip_transformer.h"
#include "strips.hpp"

namespace lmp_hip {
namespace {

constexpr int kThreads = 256;

struct GateArgs {
  int gate;
  int64_t rows;
  int hidden;
  const float* pre;
  int64_t ldpre;
  const float* g;
  int64_t ldg;
  float* out;  // h [rows, hidden] or d [rows, 2 hidden]
  int64_t ldo;
};

// h from pre, or (BACK) d from pre and g: columns over a workgroup's lanes, rows over the
// grid's y.
template <bool BACK>
__global__ __launch_bounds__(kThreads) void gate_rows(GateArgs a) {
  const int col = blockIdx.x * kThreads + threadIdx.x;
  if (col >= a.hidden) return;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float p = a.pre[row * a.ldpre + col], u = a.pre[row * a.ldpre + a.hidden + col];
    float act, slope;
    gate_of(a.gate, p, act, slope);
    if constexpr (BACK) {
      const float g = a.g[row * a.ldg + col];
      a.out[row * a.ldo + col] = g * u * slope;
      a.out[row * a.ldo + a.hidden + col] = g * act;
    } else {
      a.out[row * a.ldo + col] = act * u;
    }
  }
}

template <bool BACK>
int launch_gate(Runtime* rt, const GateArgs& a) {
  const uint32_t cols = uint32_t((int64_t(a.hidden) + kThreads - 1) / kThreads);
  const uint32_t rows = uint32_t(std::min<int64_t>(a.rows, 65535));
  gate_rows<BACK><<<dim3(cols, rows), dim3(kThreads), 0, rt->stream>>>(a);
  LMP_LAUNCH_CHECK("gate");
  return LMP_OK;
}

// ------------------------------------------------------- on the fp16 matrix cores

struct HalfGated {
  int gate, hidden;
  const float* bias;
  float* h;
  int64_t ldh;
  float* pre;
  int64_t ldpre;
};

// h (and pre) of a tile: its block columns are the gate's and the other half's by turns, so
// that a lane ends with both of a hidden value.
template <int NT, int MINB, class C>
__global__ __launch_bounds__(NT, MINB) void half_gated(HalfArgs g, HalfGated o) {
  static_assert(NT == C::THREADS, "one lane per thread of the configuration");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  hv16 acc[C::TM][C::TN];
  const HalfItem at = half_item(g, int(blockIdx.x));
  const int h0 = at.tile_n * (C::BN / 2);
  const int left = o.hidden - 1 - h0;
  const auto local = [&](int c) {
    const int block = c / 32;
    return min(block / 2 * 32 + c % 32, left) + (block & 1) * o.hidden;
  };
  const bool scaled = half_tile<C, false, false>(g, at, h0, local, smem, acc);
  const int wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % C::WN;
  const int col0 = h0 + wn * 32;
  const uint32_t* const tops[2] = {g.b_top + col0, g.b_top + o.hidden + col0};
  half_epilogue<C>(g, at, scaled, smem, tops, acc, [&](int row, int c4, hv4 (&v)[2]) {
    const int col = col0 + c4;
    if (row >= g.m || col >= o.hidden) return;
    if (o.bias) {
      v[0] = v[0] + load_four(o.bias, col, o.hidden);
      v[1] = v[1] + load_four(o.bias + o.hidden, col, o.hidden);
    }
    hv4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float act, slope;
      gate_of(o.gate, v[0][e], act, slope);
      h[e] = act * v[1][e];
    }
    store_four(o.h + row * o.ldh, col, o.hidden, h);
    if (o.pre) {
      float* p = o.pre + row * o.ldpre;
      store_four(p, col, o.hidden, v[0]);
      store_four(p + o.hidden, col, o.hidden, v[1]);
    }
  });
}

// d with its largest magnitudes, and (SUMS) the columns' sums of each strip of rows.
struct HalfGate {
  GateArgs a;
  StripShape s;
  uint32_t *row_top, *col_top;
  float* sums;  // [strips, 2 hidden]
};
template <bool SUMS>
__global__ __launch_bounds__(kStripThreads) void half_gate(HalfGate o) {
  const GateArgs& a = o.a;
  const int col = strip_col(), n = a.hidden;
  uint32_t top0[4] = {0, 0, 0, 0}, top1[4] = {0, 0, 0, 0};
  hv4 sum0 = hv4(0.0f), sum1 = hv4(0.0f);
  const int64_t end = strip_end(o.s);
#pragma unroll 2
  for (int64_t row = strip_begin(o.s); row < end; ++row) {
    const float* p = a.pre + row * a.ldpre;
    const hv4 x = load_four(p, col, n), u = load_four(p + n, col, n), g = load_four(a.g + row * a.ldg, col, n);
    hv4 d0, d1;
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float act, slope;
      gate_of(a.gate, x[e], act, slope);
      d0[e] = g[e] * u[e] * slope;
      d1[e] = g[e] * act;
      const uint32_t m0 = col + e < n ? magnitude(d0[e]) : 0, m1 = col + e < n ? magnitude(d1[e]) : 0;
      top0[e] = max(top0[e], m0);
      top1[e] = max(top1[e], m1);
      most = max(most, max(m0, m1));
    }
    float* out = a.out + row * a.ldo;
    store_four(out, col, n, d0);
    store_four(out + n, col, n, d1);
    if constexpr (SUMS) {
      sum0 = sum0 + d0;
      sum1 = sum1 + d1;
    }
    raise_row(o.row_top + row, most);
  }
  raise_cols(o.col_top, col, n, top0);
  raise_cols(o.col_top + n, col, n, top1);
  if constexpr (SUMS) {
    float* sums = o.sums + int64_t(blockIdx.y) * 2 * n;
    store_four(sums, col, n, sum0);
    store_four(sums + n, col, n, sum1);
  }
}

// From this many multiply-adds a product on, the fp16 matrix cores make up for the passes
// that find the largest magnitudes.
constexpr uint64_t kHalfWork = uint64_t(1) << 28;

bool use_half(size_t rows, size_t in, size_t hidden, size_t most_ld) {
  return half_fits(rows, in, 2 * hidden, std::max(most_ld, 2 * hidden)) && hidden >= 32 &&
         uint64_t(rows) * in * 2 * hidden >= kHalfWork;
}

}  // namespace
namespace {

int check_gated(const std::string& name, int gate, size_t rows, size_t in, size_t hidden) {
  if (gate < 0 || gate >= LMP_GATE_COUNT) return fail(LMP_ERR_INVALID, name + "unknown gate " + std::to_string(gate));
  if (in == 0 || hidden == 0) return fail(LMP_ERR_INVALID, name + "no inputs or no outputs");
  const size_t most = kGemmMaxExtent - 1;
  if (rows > most || in > most || hidden > most / 2)
    return fail(LMP_ERR_UNSUPPORTED, name + "dimension of 2^31 - 4096 or more");
  return LMP_OK;
}

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_gated_linear_f32(int gate, size_t rows, size_t in, size_t hidden, const float* x,
                                      size_t ldx, const float* w, size_t ldw, const float* bias, float* h,
                                      size_t ldh, float* pre, size_t ldpre) {
  const std::string name = "lmp_k_gated_linear_f32: ";
  if (int s = check_gated(name, gate, rows, in, hidden)) return s;
  if (rows == 0) return LMP_OK;
  if (!x || !w || !h) return fail(LMP_ERR_INVALID, name + "null buffer");
  if (ldx < in || ldw < 2 * hidden || ldh < hidden || (pre && ldpre < 2 * hidden))
    return fail(LMP_ERR_INVALID, name + "leading dimension too small");
  if (std::max({ldx, ldw, ldh, pre ? ldpre : 0}) >= kGemmMaxExtent)
    return fail(LMP_ERR_UNSUPPORTED, name + "dimension of 2^31 - 4096 or more");
  LMP_RUNTIME_OR_FAIL(rt);
  if (use_half(rows, in, hidden, std::max(ldx, ldw))) {
    const size_t of_x = half_tops_room(rows), of_w = half_tops_room(2 * hidden);
    uint32_t* tops = static_cast<uint32_t*>(scratch_alloc((of_x + of_w) * sizeof(uint32_t)));
    if (!tops) return LMP_ERR_OOM;
    const auto run = [&]() -> int {
      if (int s = clear_words(rt, tops, of_x + of_w)) return s;
      if (int s = half_tops(rt, x, rows, in, ldx, tops, nullptr)) return s;
      if (int s = half_tops(rt, w, in, 2 * hidden, ldw, nullptr, tops + of_x)) return s;
      // A tile of BN columns holds BN / 2 hidden values: the plan's columns are twice as many.
      const HalfPlan plan = half_plan(rt->cu_count, 0, int64_t(rows), 2 * int64_t(hidden), int64_t(in), false);
      if (plan.cfg < 0) return fail(LMP_ERR_UNSUPPORTED, name + "more tiles than a grid holds");
      const HalfArgs g = half_args(x, int(ldx), w, int(ldw), int(rows), int(2 * hidden), int(in), tops, tops + of_x, plan);
      const HalfGated o{gate, int(hidden), bias, h, int64_t(ldh), pre, int64_t(ldpre)};
      return with_half_cfg(plan.cfg, [&](auto cfg) -> int {
        using C = decltype(cfg);
        half_gated<C::THREADS, C::MINB, C><<<dim3(half_items(g)), dim3(C::THREADS), 0, rt->stream>>>(g, o);
        LMP_LAUNCH_CHECK("half_gated");
        return LMP_OK;
      });
    };
    const int rc = run();
    scratch_free(tops);
    return rc;
  }
  float* z = pre;
  if (!z) {
    z = static_cast<float*>(scratch_alloc(rows * 2 * hidden * sizeof(float)));
    if (!z) return LMP_ERR_OOM;
    ldpre = 2 * hidden;
  }
  int rc = bias ? lmp_k_linear_f32(0, 0, rows, 2 * hidden, in, x, ldx, w, ldw, bias, z, ldpre)
                : lmp_k_gemm_f32(0, 0, rows, 2 * hidden, in, x, ldx, w, ldw, z, ldpre, 0);
  if (rc == LMP_OK)
    rc = launch_gate<false>(rt, {gate, int64_t(rows), int(hidden), z, int64_t(ldpre), nullptr, 0, h, int64_t(ldh)});
  if (!pre) scratch_free(z);
  return rc;
}

extern "C" int lmp_k_gated_linear_backward_f32(int gate, size_t rows, size_t in, size_t hidden, const float* g,
                                               size_t ldg, const float* x, size_t ldx, const float* w,
                                               size_t ldw, const float* pre, size_t ldpre, float* dx,
                                               size_t lddx, float* dw, size_t lddw, float* db) {
  const std::string name = "lmp_k_gated_linear_backward_f32: ";
  if (int s = check_gated(name, gate, rows, in, hidden)) return s;
  if (!dx && !dw && !db) return LMP_OK;
  const size_t width = 2 * hidden;
  if (dw && lddw < width) return fail(LMP_ERR_INVALID, name + "leading dimension too small");
  if (rows) {
    if (!g || !pre || (dw && !x) || (dx && !w)) return fail(LMP_ERR_INVALID, name + "null buffer");
    if (ldg < hidden || ldpre < width || (dw && ldx < in) || (dx && (ldw < width || lddx < in)))
      return fail(LMP_ERR_INVALID, name + "leading dimension too small");
  }
  if (std::max({ldg, ldpre, dw ? std::max(ldx, lddw) : 0, dx ? std::max(ldw, lddx) : 0}) >= kGemmMaxExtent)
    return fail(LMP_ERR_UNSUPPORTED, name + "dimension of 2^31 - 4096 or more");
  LMP_RUNTIME_OR_FAIL(rt);
  if (rows == 0) {
    if (int s = clear_f32(rt, dw, in, width, lddw)) return s;
    return clear_f32(rt, db, 1, width, width);
  }
  if (use_half(rows, in, hidden, std::max(dw ? ldx : 0, dx ? ldw : 0))) {
    const StripShape strips = strips_of(rt, rows, hidden);
    const size_t of_d = (rows * width + 63) / 64 * 64, of_sums = db ? (size_t(strips.strips) * width + 63) / 64 * 64 : 0;
    const size_t of_x = half_tops_room(in), of_row = half_tops_room(rows), of_col = half_tops_room(width);
    const size_t of_tops = 2 * of_x + of_row + of_col;
    float* d = static_cast<float*>(scratch_alloc((of_d + of_sums + of_tops) * sizeof(float)));
    if (!d) return LMP_ERR_OOM;
    float* sums = d + of_d;
    uint32_t* x_col = reinterpret_cast<uint32_t*>(sums + of_sums);
    uint32_t *w_row = x_col + of_x, *d_row = w_row + of_x, *d_col = d_row + of_row;
    const auto run = [&]() -> int {
      if (int s = clear_words(rt, x_col, of_tops)) return s;
      if (dw)
        if (int s = half_tops(rt, x, rows, in, ldx, nullptr, x_col)) return s;
      if (dx)
        if (int s = half_tops(rt, w, in, width, ldw, w_row, nullptr)) return s;
      const HalfGate o{{gate, int64_t(rows), int(hidden), pre, int64_t(ldpre), g, int64_t(ldg), d, int64_t(width)},
                       strips, d_row, d_col, sums};
      if (db) half_gate<true><<<strip_grid(strips), dim3(kStripThreads), 0, rt->stream>>>(o);
      else half_gate<false><<<strip_grid(strips), dim3(kStripThreads), 0, rt->stream>>>(o);
      LMP_LAUNCH_CHECK("half_gate");
      if (db)
        if (int s = lmp_k_reduce(LMP_RED_SUM, LMP_FLOAT32, db, sums, 1, size_t(strips.strips), width)) return s;
      return half_backward(rt, {rows, in, width, d, width, d_row, d_col, x, ldx, x_col, w, ldw, w_row, dx, lddx, dw,
                                lddw, false});
    };
    const int rc = run();
    scratch_free(d);
    return rc;
  }
  float* d = static_cast<float*>(scratch_alloc(rows * width * sizeof(float)));
  if (!d) return LMP_ERR_OOM;
  const auto run = [&]() -> int {
    if (int s = launch_gate<true>(rt, {gate, int64_t(rows), int(hidden), pre, int64_t(ldpre), g, int64_t(ldg), d,
                                       int64_t(width)}))
      return s;
    if (dx && dw && db)
      return lmp_k_linear_backward_f32(rows, in, width, x, ldx, w, ldw, d, width, dx, lddx, 0, dw, lddw, 0, db, 0);
    if (dw) {
      const int s = db ? lmp_k_gemm_colsum_f32(1, 0, in, width, rows, x, ldx, d, width, dw, lddw, 0, db, 0)
                       : lmp_k_gemm_f32(1, 0, in, width, rows, x, ldx, d, width, dw, lddw, 0);
      if (s) return s;
    } else if (db) {
      if (int s = lmp_k_reduce(LMP_RED_SUM, LMP_FLOAT32, db, d, 1, rows, width)) return s;
    }
    return dx ? lmp_k_gemm_f32(0, 1, rows, in, width, d, width, w, ldw, dx, lddx, 0) : LMP_OK;
  };
  const int rc = run();
  scratch_free(d);
  return rc;
}
