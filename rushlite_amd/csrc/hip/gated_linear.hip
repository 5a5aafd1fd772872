// A gated linear layer: h = act(x Wg + bg) (x Wu + bu), both projections from one weight
// matrix [Wg | Wu], and its gradients.
//
//   pre = x W + b = [a | u],  h = act(a) u
//   d = [g u act'(a) | g act(a)],  dx = d W^T,  dW = x^T d,  db = the column sums of d
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "gate.hpp"
#include "lmp_hip_transformer.h"

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

__global__ __launch_bounds__(kThreads) void clear_rows(float* p, int64_t rows, int cols, int64_t ld) {
  const int64_t total = rows * cols;
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < total; i += int64_t(gridDim.x) * kThreads)
    p[i / cols * ld + i % cols] = 0.0f;
}

}  // namespace

// Zeros in `cols` columns of `rows` rows (the gradients of no rows).
int clear_f32(Runtime* rt, float* p, size_t rows, size_t cols, size_t ld) {
  if (!p || rows == 0 || cols == 0) return LMP_OK;
  const size_t groups = (rows * cols + kThreads - 1) / kThreads;
  clear_rows<<<dim3(uint32_t(std::min<size_t>(groups, 65536))), dim3(kThreads), 0, rt->stream>>>(
      p, int64_t(rows), int(cols), int64_t(ld));
  LMP_LAUNCH_CHECK("clear");
  return LMP_OK;
}

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
