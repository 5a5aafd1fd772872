// A gated linear layer: h = act(x Wg + bg) (x Wu + bu), both projections from one weight
// matrix [Wg | Wu], and its gradients.
//
//   pre = x W + b = [a | u],  h = act(a) u
//   d = [g u act'(a) | g act(a)],  dx = d W^T,  dW = x^T d,  db = the column sums of d
//
// Large layers run on the fp16 matrix cores (gemm_half.hpp), their columns 32 of the one half
// and 32 of the other by turns: forward the product's epilogue forms h; backward d is
// formed where it is split, and never held whole.  Smaller ones take the framework's fp32
// products.  12608 rows of 768 by 768 x 4096 take 0.95 to 0.98 ms forward and backward, of which the
// products would take 0.61 at the library's rate and the passes over pre, g and d 0.2.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "gate.hpp"
#include "gemm_half.hpp"
#include "half_backward.hpp"
#include "half_panels.hpp"
#include "half_products.hpp"
#include "lmp_hip_transformer.h"

namespace lmp_hip {
namespace {

constexpr int kThreads = 256;

struct GateArgs {
  int64_t rows;
  int hidden;
  const float* pre;
  int64_t ldpre;
  const float* g;
  int64_t ldg;
  float* out;  // h [rows, hidden] or d [rows, 2 hidden]
  int64_t ldo;
  int row_lanes;  // lanes of a row: a power of two
};

// h from pre, or (BACK) d from pre and g, four columns a lane.  Bound by memory: d of 5563 rows
// of 4672 takes 101 us, 520 MB at 5.1 TB/s.
template <int GATE, bool BACK>
__global__ __launch_bounds__(kThreads) void gate_rows(GateArgs a) {
  const int lane = threadIdx.x & (a.row_lanes - 1), each = kThreads / a.row_lanes, n = a.hidden;
  for (int64_t row = int64_t(blockIdx.x) * each + threadIdx.x / a.row_lanes; row < a.rows; row += int64_t(gridDim.x) * each)
    for (int col = (int(blockIdx.y) * a.row_lanes + lane) * 4; col < n; col += int(gridDim.y) * a.row_lanes * 4) {
      const float* p = a.pre + row * a.ldpre;
      const hv4 x = load_four(p, col, n), u = load_four(p + n, col, n);
      hv4 act, slope;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f, s;
        gate_at<GATE>(x[e], f, s);
        act[e] = f;
        slope[e] = s;
      }
      float* out = a.out + row * a.ldo;
      if constexpr (BACK) {
        const hv4 g = load_four(a.g + row * a.ldg, col, n);
        store_four(out, col, n, g * u * slope);
        store_four(out + n, col, n, g * act);
      } else {
        store_four(out, col, n, act * u);
      }
    }
}

template <bool BACK>
int launch_gate(Runtime* rt, int gate, GateArgs a) {
  a.row_lanes = 1;
  while (a.row_lanes < kThreads && a.row_lanes * 4 < a.hidden) a.row_lanes *= 2;
  const int64_t each = kThreads / a.row_lanes, groups = (a.rows + each - 1) / each;
  const int64_t across = std::min<int64_t>((int64_t(a.hidden) + kThreads * 4 - 1) / (kThreads * 4), 1024);
  const dim3 grid(uint32_t(std::min<int64_t>(groups, 65536)), uint32_t(across));
  with_gate(gate, [&](auto g) { gate_rows<decltype(g)::value, BACK><<<grid, dim3(kThreads), 0, rt->stream>>>(a); });
  LMP_LAUNCH_CHECK("gate");
  return LMP_OK;
}

// ------------------------------------------------------- on the fp16 matrix cores

// Columns by turns: how many there are, and what half and column of it column `col` is.
inline size_t turned_cols(size_t hidden) { return (hidden + 31) / 32 * 64; }
__device__ __forceinline__ int second_half(int col) { return col / 32 & 1; }
__device__ __forceinline__ int half_col(int col) { return col / 64 * 32 + col % 32; }

// A unit's eight columns: four of each half.
struct Turned {
  int64_t rows;
  int cols, hidden;
  __device__ __forceinline__ int column(int unit, int h) const { return unit / 8 * 64 + unit % 8 * 4 + 32 * h; }
  __device__ __forceinline__ int within(int unit) const { return unit * 4; }  // the first one's place in its half
  // Where a column is in the matrix itself, or -1.
  __device__ __forceinline__ int place(int col) const {
    const int c = half_col(col);
    return c < hidden ? c + second_half(col) * hidden : -1;
  }
};
struct GatedWeights : Turned {
  const float* w;
  int64_t ld;
  __device__ __forceinline__ void load(int64_t row, int unit, hv4 (&v)[2]) const {
    const float* p = w + row * ld;
    v[0] = load_four(p, within(unit), hidden);
    v[1] = load_four(p + hidden, within(unit), hidden);
  }
  __device__ __forceinline__ float value(int64_t row, int col) const {
    const int at = place(col);
    return at < 0 ? 0.0f : w[row * ld + at];
  }
};

// d, formed from pre and g.
template <int GATE>
struct GatedGradient : Turned {
  const float* pre;
  int64_t ldpre;
  const float* g;
  int64_t ldg;
  __device__ __forceinline__ void load(int64_t row, int unit, hv4 (&v)[2]) const {
    const float* p = pre + row * ldpre;
    const int c = within(unit);
    const hv4 a = load_four(p, c, hidden), u = load_four(p + hidden, c, hidden), gr = load_four(g + row * ldg, c, hidden);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float act, slope;
      gate_at<GATE>(a[e], act, slope);
      v[0][e] = gr[e] * u[e] * slope;
      v[1][e] = gr[e] * act;
    }
  }
};
// The same of any gate, for what is formed again.
struct AnyGatedGradient : Turned {
  const float* pre;
  int64_t ldpre;
  const float* g;
  int64_t ldg;
  int gate;
  __device__ __forceinline__ void load(int64_t row, int unit, hv4 (&v)[2]) const {
    with_gate(gate, [&](auto gt) {
      GatedGradient<decltype(gt)::value>{{rows, cols, hidden}, pre, ldpre, g, ldg}.load(row, unit, v);
    });
  }
  __device__ __forceinline__ float value(int64_t row, int col) const {
    const int c = half_col(col);
    if (c >= hidden) return 0.0f;
    const float a = pre[row * ldpre + c], u = pre[row * ldpre + hidden + c], gr = g[row * ldg + c];
    float act, slope;
    with_gate(gate, [&](auto gt) { gate_at<decltype(gt)::value>(a, act, slope); });
    return second_half(col) ? gr * act : gr * u * slope;
  }
};

struct HalfGated {
  int gate, hidden;
  const float* bias;
  float* h;
  int64_t ldh;
  float* pre;
  int64_t ldpre;
};

// h (and pre) of a tile: a lane ends with both halves of a hidden value.
template <int NT, int MINB, class C>
__global__ __launch_bounds__(NT, MINB) void half_gated(HalfArgs g, HalfGated o, RowsOf<MatrixSource> x, ColsOf<GatedWeights> w) {
  static_assert(NT == C::THREADS && C::TN == 2, "a wave has 32 columns of each half");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  const HalfItem at = half_item(g, int(blockIdx.x));
  const int wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % C::WN;
  const int col0 = at.tile_n * (C::BN / 2) + wn * 32;
  half_product<C>(g, at, smem, x, w, [&](int row, int c4, hv4 (&v)[2]) {
    const int col = col0 + c4;
    if (row >= g.m || col >= o.hidden) return;
    if (o.bias) {
      v[0] = v[0] + load_four(o.bias, col, o.hidden);
      v[1] = v[1] + load_four(o.bias + o.hidden, col, o.hidden);
    }
    hv4 h;
    with_gate(o.gate, [&](auto gate) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float act, slope;
        gate_at<decltype(gate)::value>(v[0][e], act, slope);
        h[e] = act * v[1][e];
      }
    });
    store_four(o.h + row * o.ldh, col, o.hidden, h);
    if (o.pre) {
      float* p = o.pre + row * o.ldpre;
      store_four(p, col, o.hidden, v[0]);
      store_four(p + o.hidden, col, o.hidden, v[1]);
    }
  });
}

// Whether the split products pay for reading x and w twice and writing their panels (12 bytes a
// value) and for their launches; forward they save a pass over pre besides (two where it is not
// kept, but what is kept does not change the results).  128 rows of 4096 by 4096 x 16384 take 160 us
// without them and 271 with them, 512 of 768 by 768 x 4096 39 and 36, 16384 of 64 by 64 x 2048 84 and 58.
bool half_forward_pays(size_t rows, size_t in, size_t hidden) {
  const double n = double(rows), d = double(in), w = 2 * double(hidden);
  return half_fits(rows, in, 2 * hidden) && hidden >= 32 &&
         half_saves_forward(n * d * w) + pass_time(4 * n * w) > 12 + pass_time(12 * (n * d + d * w));
}
// Backward they form d twice from pre and g and write it in two sets of panels: 20 bytes a value
// for 10.  16384 rows of 64 by 64 x 2048 take 143 us without them and 228 with them.
bool half_backward_pays(size_t rows, size_t in, size_t hidden) {
  const double n = double(rows), d = double(in), w = 2 * double(hidden);
  return half_fits(rows, in, 2 * hidden) && hidden >= 32 &&
         half_saves_backward(n * d * w) > 25 + pass_time(12 * (n * d + d * w) + 10 * n * w);
}

// The workspace as panels, their rows' magnitudes and, `tops` words on, marks.
HalfPanels panels_at(uint32_t* base, size_t panels, size_t k, size_t at, size_t tops) {
  return {reinterpret_cast<char*>(base + panels), int64_t(half_stride(k)), base + at, base + at + tops};
}

int gated_half(Runtime* rt, int gate, size_t rows, size_t in, size_t hidden, const float* x, size_t ldx,
               const float* w, size_t ldw, const float* bias, float* h, size_t ldh, float* pre, size_t ldpre) {
  const size_t cols = turned_cols(hidden);
  const HalfPlan plan = half_plan(rt->cu_count, 0, {int64_t(rows), int64_t(cols), int64_t(in), false, 2.0f}, {});
  if (plan.cfg < 0) return fail(LMP_ERR_UNSUPPORTED, "gated_linear: more tiles than a grid holds");
  HalfRoom room;
  const size_t at_x = room.take(half_tops_words(rows)), at_w = room.take(half_tops_words(cols)), tops = room.words;
  room.take(tops);
  const size_t x_panels = room.take(half_panel_words(rows, in)), w_panels = room.take(half_panel_words(cols, in));
  uint32_t* base = static_cast<uint32_t*>(scratch_alloc(room.words * sizeof(uint32_t)));
  if (!base) return LMP_ERR_OOM;
  const HalfPanels xr = panels_at(base, x_panels, in, at_x, tops), wc = panels_at(base, w_panels, in, at_w, tops), none{};
  const MatrixSource of_x{int64_t(rows), int(in), x, int64_t(ldx), nullptr};
  const GatedWeights of_w{{int64_t(in), int(cols), int(hidden)}, w, int64_t(ldw)};
  const auto run = [&]() -> int {
    if (int s = clear_words(rt, base, 2 * tops)) return s;
    if (int s = run_panel_jobs(rt, tops_job(rt, of_w, nullptr, wc.tops), tops_job(rt, of_x, xr.tops, nullptr))) return s;
    if (int s = run_panel_jobs(rt, pack_job(of_w, none, wc), pack_job(of_x, xr, none))) return s;
    const HalfArgs g = half_args(xr, wc, int(rows), int(cols), int(in), plan.cfg, 1);
    const HalfGated o{gate, int(hidden), bias, h, int64_t(ldh), pre, int64_t(ldpre)};
    return with_half_cfg(plan.cfg, [&](auto cfg) -> int {
      using C = decltype(cfg);
      half_gated<C::THREADS, C::MINB, C><<<dim3(half_items(g)), dim3(C::THREADS), 0, rt->stream>>>(g, o, {of_x}, {of_w});
      LMP_LAUNCH_CHECK("half_gated");
      return LMP_OK;
    });
  };
  const int rc = run();
  scratch_free(base);
  return rc;
}

int gated_half_backward(Runtime* rt, int gate, size_t rows, size_t in, size_t hidden, const float* g, size_t ldg,
                        const float* x, size_t ldx, const float* w, size_t ldw, const float* pre, size_t ldpre,
                        float* dx, size_t lddx, float* dw, size_t lddw, float* db) {
  const size_t cols = turned_cols(hidden), width = 2 * hidden;
  const size_t most = size_t(most_strips(rt, int64_t(rows), int64_t(cols)));
  HalfRoom room;
  const size_t at_dr = room.take(half_tops_words(rows)), at_dc = room.take(half_tops_words(cols));
  const size_t at_x = room.take(half_tops_words(in)), at_w = room.take(half_tops_words(in)), tops = room.words;
  room.take(tops);
  const size_t d_rows = room.take(dx ? half_panel_words(rows, cols) : 0);
  const size_t d_cols = room.take(dw ? half_panel_words(cols, rows) : 0);
  const size_t x_panels = room.take(dw ? half_panel_words(in, rows) : 0);
  const size_t w_panels = room.take(dx ? half_panel_words(in, cols) : 0);
  const size_t at_sums = room.take(db ? most * width : 0);
  uint32_t* base = static_cast<uint32_t*>(scratch_alloc(room.words * sizeof(uint32_t)));
  if (!base) return LMP_ERR_OOM;
  HalfPanels none{}, dr = none, dc = none, xc = none, wr = none;
  if (dx) dr = panels_at(base, d_rows, cols, at_dr, tops), wr = panels_at(base, w_panels, cols, at_w, tops);
  if (dw) dc = panels_at(base, d_cols, rows, at_dc, tops), xc = panels_at(base, x_panels, rows, at_x, tops);
  float* sums = db ? reinterpret_cast<float*>(base + at_sums) : nullptr;
  const MatrixSource of_x{dw ? int64_t(rows) : 0, int(in), x, int64_t(ldx), nullptr};
  const GatedWeights of_w{{dx ? int64_t(in) : 0, int(cols), int(hidden)}, w, int64_t(ldw)};
  size_t strips = 0;
  const auto run = [&]() -> int {
    if (int s = clear_words(rt, base, 2 * tops)) return s;
    if (int s = with_gate(gate, [&](auto gt) -> int {
          const GatedGradient<decltype(gt)::value> of_d{{int64_t(rows), int(cols), int(hidden)}, pre, int64_t(ldpre), g, int64_t(ldg)};
          auto job = tops_job(rt, of_d, dr.tops, dc.tops, sums);
          job.sums_ld = int64_t(width);
          strips = size_t(job.blocks / job.col_blocks);
          if (int e = run_panel_jobs(rt, job, tops_job(rt, of_w, wr.tops, nullptr), tops_job(rt, of_x, nullptr, xc.tops))) return e;
          if (!dx && !dw) return LMP_OK;
          return run_panel_jobs(rt, pack_job(of_d, dr, dc), pack_job(of_w, wr, none), pack_job(of_x, none, xc));
        }))
      return s;
    if (db)
      if (int s = lmp_k_reduce(LMP_RED_SUM, LMP_FLOAT32, db, sums, 1, strips, width)) return s;
    const AnyGatedGradient any{{int64_t(rows), int(cols), int(hidden)}, pre, int64_t(ldpre), g, int64_t(ldg), gate};
    return half_backward<AnyGatedGradient, GatedWeights>(
        rt, {rows, in, cols, dr, dc, xc, wr, dx, lddx, dw, lddw, false, hidden, of_x, any, of_w});
  };
  const int rc = run();
  scratch_free(base);
  return rc;
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
  // Where memory for the panels is short, the fp32 products take over.
  if (half_forward_pays(rows, in, hidden))
    if (int s = gated_half(rt, gate, rows, in, hidden, x, ldx, w, ldw, bias, h, ldh, pre, ldpre); s != LMP_ERR_OOM) return s;
  float* z = pre;
  if (!z) {
    z = static_cast<float*>(scratch_alloc(rows * 2 * hidden * sizeof(float)));
    if (!z) return LMP_ERR_OOM;
    ldpre = 2 * hidden;
  }
  int rc = bias ? lmp_k_linear_f32(0, 0, rows, 2 * hidden, in, x, ldx, w, ldw, bias, z, ldpre)
                : lmp_k_gemm_f32(0, 0, rows, 2 * hidden, in, x, ldx, w, ldw, z, ldpre, 0);
  if (rc == LMP_OK)
    rc = launch_gate<false>(rt, gate, {int64_t(rows), int(hidden), z, int64_t(ldpre), nullptr, 0, h, int64_t(ldh), 0});
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
  if (half_backward_pays(rows, in, hidden))
    if (int s = gated_half_backward(rt, gate, rows, in, hidden, g, ldg, x, ldx, w, ldw, pre, ldpre, dx, lddx, dw, lddw, db);
        s != LMP_ERR_OOM)
      return s;
  float* d = static_cast<float*>(scratch_alloc(rows * width * sizeof(float)));
  if (!d) return LMP_ERR_OOM;
  const auto run = [&]() -> int {
    if (int s = launch_gate<true>(rt, gate, {int64_t(rows), int(hidden), pre, int64_t(ldpre), g, int64_t(ldg), d,
                                             int64_t(width), 0}))
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
