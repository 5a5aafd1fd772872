// Softmax cross entropy of a linear layer's outputs over a vocabulary, with the gradients.
//
//   z = x W + b,  loss_i = log sum_v exp(z_iv) - z_i,t(i)
//   dz_iv = weight_i (exp(z_iv) / sum - [v = t(i)]),  dx = dz W^T,  dW = x^T dz,  db = its column sums
//
// The logits are never held whole: pieces of rows pass through one workspace.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "lmp_hip_transformer.h"

namespace lmp_hip {

int clear_f32(Runtime* rt, float* p, size_t rows, size_t cols, size_t ld);

namespace {

// Bytes of one piece's logits: well inside the 256 MB memory-side cache, so that what
// reads them after the product does not go to HBM.
constexpr size_t kPieceBytes = size_t(128) << 20;

struct LossArgs {
  int64_t rows;
  int vocab;
  float* z;  // [rows, vocab], contiguous: the logits, which the gradient replaces
  const int64_t* targets;
  const float* weights;
  float* loss;
  // The rows of x with zeros for those that are not counted: 0 x infinity would be NaN in dW.
  const float* x;
  int64_t ldx;
  int in;
  float* counted_x;  // [rows, in], or null
};

// A running maximum and the sum of exponents below it.
struct Softmax {
  float top, sum;
};
__device__ __forceinline__ Softmax joined(Softmax a, Softmax b) {
  // The larger one's own factor is exp(0); equal infinities too.
  const float top = fmaxf(a.top, b.top);
  const float fa = a.top == top ? 1.0f : expf(a.top - top), fb = b.top == top ? 1.0f : expf(b.top - top);
  return {top, a.sum * fa + b.sum * fb};
}

// One workgroup per row: loss and, with GRAD, dz in the place of z.
template <bool GRAD>
__global__ __launch_bounds__(1024) void loss_rows(LossArgs a) {
  __shared__ Softmax parts[16];
  const float low = -__builtin_huge_valf();
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float* z = a.z + row * a.vocab;
    const int64_t t = a.targets[row];
    const bool counted = t >= 0, known = t < a.vocab;
    if (a.counted_x)
      for (int i = threadIdx.x; i < a.in; i += 1024)
        a.counted_x[row * a.in + i] = counted ? a.x[row * a.ldx + i] : 0.0f;
    if (!counted) {
      if (GRAD)
        for (int v = threadIdx.x; v < a.vocab; v += 1024) z[v] = 0.0f;
      if (threadIdx.x == 0) a.loss[row] = 0.0f;
      continue;
    }
    Softmax s{low, 0.0f};
    bool nan = false;
    for (int v = threadIdx.x; v < a.vocab; v += 1024) {
      const float x = z[v];
      nan |= x != x;
      if (x > s.top) {
        s.sum = s.sum * expf(s.top - x) + 1.0f;
        s.top = x;
      } else if (x > low) {
        s.sum += expf(x - s.top);
      }
    }
    if (nan) s.sum = __builtin_nanf("");
    for (int off = 1; off < 64; off *= 2) {
      const Softmax o{__shfl_xor(s.top, off), __shfl_xor(s.sum, off)};
      s = joined(s, o);
    }
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    s = parts[0];
    for (int i = 1; i < 16; ++i) s = joined(s, parts[i]);
    const float zt = known ? z[t] : __builtin_nanf("");
    __syncthreads();  // z[t] and parts are read before they are written again
    if (threadIdx.x == 0) a.loss[row] = logf(s.sum) - (zt - s.top);
    if constexpr (GRAD) {
      const float w = a.weights ? a.weights[row] : 1.0f;
      const float f = known ? w / s.sum : __builtin_nanf("");
      for (int v = threadIdx.x; v < a.vocab; v += 1024) {
        const float p = expf(z[v] - s.top) * f;
        z[v] = v == t ? p - w : p;
      }
    }
  }
}

struct LossCall {
  size_t rows, in, vocab;
  const float* x;
  size_t ldx;
  const float* w;
  size_t ldw;
  const float* bias;
  const int64_t* targets;
  const float* weights;
  float* loss;
  float* dx;
  size_t lddx;
  float* dw;
  size_t lddw;
  float* db;
};

int check_loss(const std::string& name, const LossCall& c) {
  if (c.in == 0 || c.vocab == 0) return fail(LMP_ERR_INVALID, name + "no inputs or no vocabulary");
  const size_t most = kGemmMaxExtent - 1;
  if (std::max({c.rows, c.in, c.vocab, c.ldx, c.ldw, c.dx ? c.lddx : 0, c.dw ? c.lddw : 0}) > most)
    return fail(LMP_ERR_UNSUPPORTED, name + "dimension of 2^31 - 4096 or more");
  if (c.rows && (!c.x || !c.w || !c.targets || !c.loss)) return fail(LMP_ERR_INVALID, name + "null buffer");
  if ((c.rows && (c.ldx < c.in || c.ldw < c.vocab || (c.dx && c.lddx < c.in))) || (c.dw && c.lddw < c.vocab))
    return fail(LMP_ERR_INVALID, name + "leading dimension too small");
  return LMP_OK;
}

int run_loss(Runtime* rt, const LossCall& c) {
  if (c.rows == 0) {
    if (int s = clear_f32(rt, c.dw, c.in, c.vocab, c.lddw)) return s;
    return clear_f32(rt, c.db, 1, c.vocab, c.vocab);
  }
  const size_t fit = std::max<size_t>(256, kPieceBytes / (c.vocab * sizeof(float)));
  const size_t pieces = (c.rows + fit - 1) / fit, each = (c.rows + pieces - 1) / pieces;
  const size_t logits = (each * c.vocab + 3) / 4 * 4;
  float* z = static_cast<float*>(scratch_alloc((logits + (c.dw ? each * c.in : 0)) * sizeof(float)));
  if (!z) return LMP_ERR_OOM;
  float* counted_x = c.dw ? z + logits : nullptr;
  const auto piece = [&](size_t at, size_t n) -> int {
    const float* x = c.x + at * c.ldx;
    if (int s = c.bias ? lmp_k_linear_f32(0, 0, n, c.vocab, c.in, x, c.ldx, c.w, c.ldw, c.bias, z, c.vocab)
                       : lmp_k_gemm_f32(0, 0, n, c.vocab, c.in, x, c.ldx, c.w, c.ldw, z, c.vocab, 0))
      return s;
    const LossArgs a{int64_t(n), int(c.vocab), z, c.targets + at, c.weights ? c.weights + at : nullptr,
                     c.loss + at, x, int64_t(c.ldx), int(c.in), counted_x};
    const bool grad = c.dx || c.dw;
    const dim3 grid(uint32_t(std::min<size_t>(n, 65536)));
    if (grad) loss_rows<true><<<grid, dim3(1024), 0, rt->stream>>>(a);
    else loss_rows<false><<<grid, dim3(1024), 0, rt->stream>>>(a);
    LMP_LAUNCH_CHECK("loss_rows");
    if (!grad) return LMP_OK;
    const int more = at > 0;
    if (c.dw) {
      if (int s = c.db ? lmp_k_gemm_colsum_f32(1, 0, c.in, c.vocab, n, counted_x, c.in, z, c.vocab, c.dw, c.lddw, more, c.db, more)
                       : lmp_k_gemm_f32(1, 0, c.in, c.vocab, n, counted_x, c.in, z, c.vocab, c.dw, c.lddw, more))
        return s;
    }
    if (c.dx)
      return lmp_k_gemm_f32(0, 1, n, c.in, c.vocab, z, c.vocab, c.w, c.ldw, c.dx + at * c.lddx, c.lddx, 0);
    return LMP_OK;
  };
  int rc = LMP_OK;
  for (size_t at = 0; at < c.rows && rc == LMP_OK; at += each) rc = piece(at, std::min(each, c.rows - at));
  scratch_free(z);
  return rc;
}

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_linear_cross_entropy_f32(size_t rows, size_t in, size_t vocab, const float* x, size_t ldx,
                                              const float* w, size_t ldw, const float* bias,
                                              const int64_t* targets, float* loss) {
  const LossCall c{rows, in, vocab, x, ldx, w, ldw, bias, targets, nullptr, loss, nullptr, 0, nullptr, 0, nullptr};
  if (int s = check_loss("lmp_k_linear_cross_entropy_f32: ", c)) return s;
  if (rows == 0) return LMP_OK;
  LMP_RUNTIME_OR_FAIL(rt);
  return run_loss(rt, c);
}

extern "C" int lmp_k_linear_cross_entropy_grad_f32(size_t rows, size_t in, size_t vocab, const float* x,
                                                   size_t ldx, const float* w, size_t ldw, const float* bias,
                                                   const int64_t* targets, const float* weights, float* loss,
                                                   float* dx, size_t lddx, float* dw, size_t lddw, float* db) {
  const LossCall c{rows, in, vocab, x, ldx, w, ldw, bias, targets, weights, loss, dx, lddx, dw, lddw, db};
  if (int s = check_loss("lmp_k_linear_cross_entropy_grad_f32: ", c)) return s;
  if (db && !dw) return fail(LMP_ERR_INVALID, "lmp_k_linear_cross_entropy_grad_f32: db without dw");
  LMP_RUNTIME_OR_FAIL(rt);
  return run_loss(rt, c);
}
