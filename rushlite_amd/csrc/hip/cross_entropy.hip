// Softmax cross entropy of a linear layer's outputs over a vocabulary, with the gradients.
//
//   z = x W + b,  loss_i = log sum_v exp(z_iv) - z_i,t(i)
//   dz_iv = weight_i (exp(z_iv) / sum - [v = t(i)]),  dx = dz W^T,  dW = x^T dz,  db = its column sums
//
// Three ways.  A problem that fits one workgroup's LDS is one launch (tiny_loss).  Where the
// products are large enough they run on the fp16 matrix cores (gemm_half.hpp): the product's
// epilogue leaves a maximum and a sum of exponents per row and 64 columns, and for the losses
// alone no logits at all; with the gradients pieces of rows keep theirs, and dz is formed
// from them where it is split.  4096 x 1024 over 32768 words takes 2.63 to 2.71 ms, of which
// the three products would take 2.1 at the library's rate; scoring 8192 rows 1.52 to 1.59 ms of 1.4.
// Other sizes take the framework's fp32 products around a pass over the rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "common.hpp"
#include "gemm_half.hpp"
#include "half_backward.hpp"
#include "half_panels.hpp"
#include "half_products.hpp"
#include "lmp_hip_transformer.h"

namespace lmp_hip {
namespace {

// Bytes of one piece's logits, or of what the losses alone keep of them.  Each piece adds to dW
// once more: 4096 rows of 1024 over a vocabulary of 32768, 512 MB of logits, took 3.23 ms in pieces
// of 128 MB, 2.71 of 256, 2.57 of 512, 2.58 of 1024; a row more makes it two pieces, some 5%.
constexpr size_t kPieceBytes = size_t(512) << 20;

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

// e^x for x <= 0: 2^(x log2 e) with what rounding the product leaves out put back, so that
// it errs by two units, not by |x| of them.
__device__ __forceinline__ float exp_below(float x) {
  constexpr float kHi = 1.44269504088896341f, kLo = 1.925963033500e-8f, kLn2 = 0.69314718055994531f;
  const float t = x * kHi, e = __builtin_amdgcn_exp2f(t);
  const float rest = __builtin_fmaf(x, kHi, -t) + x * kLo;
  return t < -160.0f ? 0.0f : __builtin_fmaf(e, rest * kLn2, e);
}

// Loss and, with GRAD, dz in the place of z.  A row has the lanes of WAVES waves, which hold
// it in registers, QUADS times four logits each, or (QUADS 0) read it again from memory.
// Bound by memory there; short rows by the latency of their few loads and joins.
template <bool GRAD, int WAVES, int QUADS>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void loss_rows(LossArgs a) {
  __shared__ Softmax parts[16];
  constexpr int kLanes = 64 * WAVES, kRows = WAVES == 1 ? 4 : 1;
  const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, n = a.vocab;
  const float low = -__builtin_huge_valf();
  for (int64_t row = int64_t(blockIdx.x) * kRows + (WAVES == 1 ? threadIdx.x >> 6 : 0); row < a.rows;
       row += int64_t(gridDim.x) * kRows) {
    float* z = a.z + row * n;
    const int64_t t = a.targets[row];
    const bool counted = t >= 0, known = t < n;
    if (a.counted_x)
      for (int i = lane * 4; i < a.in; i += kLanes * 4)
        store_four(a.counted_x + row * a.in, i, a.in, counted ? load_four(a.x + row * a.ldx, i, a.in) : hv4(0.0f));
    if (!counted) {
      if (GRAD)
        for (int v = lane * 4; v < n; v += kLanes * 4) store_four(z, v, n, hv4(0.0f));
      if (lane == 0) a.loss[row] = 0.0f;
      continue;
    }
    const float zt = known ? z[t] : __builtin_nanf("");
    hv4 held[QUADS ? QUADS : 1];
    Softmax s{low, 0.0f};
    if constexpr (QUADS > 0) {
#pragma unroll
      for (int q = 0; q < QUADS; ++q) {
        const int v = (q * kLanes + lane) * 4;
        held[q] = hv4(low);
        if (v < n) held[q] = load_four(z, v, n);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (v + e >= n) held[q][e] = low;
          s.top = fmaxf(s.top, held[q][e]);
        }
      }
      // Of a lane with nothing but -inf the sum is 0; of +inf and NaN it is NaN.
      const float from = s.top > low ? s.top : 0.0f;
#pragma unroll
      for (int q = 0; q < QUADS; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) s.sum += exp_below(held[q][e] - from);
    } else {
      for (int v = lane * 4; v < n; v += kLanes * 4) {
        const hv4 x = load_four(z, v, n);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (v + e >= n) continue;
          const float top = fmaxf(s.top, x[e]), from = top > low ? top : 0.0f;
          s.sum = s.sum * exp_below(s.top - from) + exp_below(x[e] - from);
          s.top = top;
        }
      }
    }
    for (int off = 1; off < 64; off *= 2) s = joined(s, {__shfl_xor(s.top, off), __shfl_xor(s.sum, off)});
    if constexpr (WAVES > 1) {
      if ((lane & 63) == 0) parts[lane >> 6] = s;
      __syncthreads();
      s = parts[lane & (WAVES - 1)];
      for (int off = 1; off < WAVES; off *= 2) s = joined(s, {__shfl_xor(s.top, off), __shfl_xor(s.sum, off)});
      __syncthreads();  // z[t] and parts are read before they are written again
    }
    if (lane == 0) a.loss[row] = logf(s.sum) - (zt - s.top);
    if constexpr (GRAD) {
      const float w = a.weights ? a.weights[row] : 1.0f;
      const float f = known ? w / s.sum : __builtin_nanf("");
      const auto put = [&](int v, hv4 x) {
        if (v >= n) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = exp_below(x[e] - s.top) * f;
          x[e] = v + e == t ? p - w : p;
        }
        store_four(z, v, n, x);
      };
      if constexpr (QUADS > 0) {
#pragma unroll
        for (int q = 0; q < QUADS; ++q) put((q * kLanes + lane) * 4, held[q]);
      } else {
        for (int v = lane * 4; v < n; v += kLanes * 4) put(v, load_four(z, v, n));
      }
    }
  }
}
template <bool GRAD>
int launch_loss_rows(Runtime* rt, const LossArgs& a) {
  const auto go = [&](auto waves, auto quads) -> int {
    constexpr int W = decltype(waves)::value, each = W == 1 ? 4 : 1;
    loss_rows<GRAD, W, decltype(quads)::value>
        <<<dim3(uint32_t(std::min<int64_t>((a.rows + each - 1) / each, 65536))), dim3(W == 1 ? 256 : 64 * W), 0, rt->stream>>>(a);
    LMP_LAUNCH_CHECK("loss_rows");
    return LMP_OK;
  };
  using std::integral_constant;
  if (a.vocab <= 512) return go(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  if (a.vocab <= 4096) return go(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  if (a.vocab <= 8192) return go(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  if (a.vocab <= 32768) return go(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  return go(integral_constant<int, 16>{}, integral_constant<int, 0>{});
}

// --------------------------------------------------------------- one workgroup

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

// A problem that one workgroup holds in LDS: bound by latency, so everything in one launch.
// 32 x 64 over 10 words with the gradients takes 7.9 us, and 12.3 in three launches.
constexpr size_t kTinyFloats = 15360, kTinyWork = size_t(1) << 17;
bool tiny_fits(const LossCall& c) {
  return c.rows <= kTinyFloats && c.in <= kTinyFloats && c.vocab <= kTinyFloats &&
         c.rows * (c.in | 1) + (c.in + c.rows) * (c.vocab | 1) <= kTinyFloats && c.rows * c.in * c.vocab <= kTinyWork;
}
struct TinyLoss {
  int rows, in, vocab;
  const float* x;
  int64_t ldx;
  const float* w;
  int64_t ldw;
  const float* bias;
  const int64_t* targets;
  const float* weights;
  float *loss, *dx;
  int64_t lddx;
  float* dw;
  int64_t lddw;
  float* db;
};
__global__ __launch_bounds__(1024) void tiny_loss(TinyLoss a) {
  __shared__ float smem[kTinyFloats];
  const int xp = a.in | 1, wp = a.vocab | 1, tid = threadIdx.x;
  float *x = smem, *w = x + a.rows * xp, *z = w + a.in * wp;
  for (int i = tid; i < a.rows * a.in; i += 1024) {
    const int r = i / a.in, k = i % a.in;
    x[r * xp + k] = a.targets[r] < 0 ? 0.0f : a.x[r * a.ldx + k];
  }
  for (int i = tid; i < a.in * a.vocab; i += 1024) w[i / a.vocab * wp + i % a.vocab] = a.w[i / a.vocab * a.ldw + i % a.vocab];
  __syncthreads();
  for (int i = tid; i < a.rows * a.vocab; i += 1024) {
    const int r = i / a.vocab, v = i % a.vocab;
    float sum = 0.0f;
#pragma unroll 8
    for (int k = 0; k < a.in; ++k) sum = __builtin_fmaf(x[r * xp + k], w[k * wp + v], sum);
    z[r * wp + v] = a.bias ? sum + a.bias[v] : sum;
  }
  __syncthreads();
  const int lane = tid & 63;
  for (int r = tid >> 6; r < a.rows; r += 16) {
    const int64_t t = a.targets[r];
    const bool counted = t >= 0, known = t < a.vocab;
    const float low = -__builtin_huge_valf(), zt = counted && known ? z[r * wp + t] : __builtin_nanf("");
    float top = low, sum = 0.0f;
    for (int v = lane; v < a.vocab; v += 64) top = fmaxf(top, z[r * wp + v]);
    for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
    for (int v = lane; v < a.vocab; v += 64) sum += expf(z[r * wp + v] - top);
    for (int off = 1; off < 64; off *= 2) sum += __shfl_xor(sum, off);
    if (lane == 0) a.loss[r] = counted ? logf(sum) - (zt - top) : 0.0f;
    if (!a.dx && !a.dw) continue;
    const float weight = a.weights ? a.weights[r] : 1.0f, f = known ? weight / sum : __builtin_nanf("");
    for (int v = lane; v < a.vocab; v += 64) {
      const float p = expf(z[r * wp + v] - top) * f;
      z[r * wp + v] = !counted ? 0.0f : v == t ? p - weight : p;
    }
  }
  __syncthreads();
  if (a.dx)
    for (int i = tid; i < a.rows * a.in; i += 1024) {
      const int r = i / a.in, k = i % a.in;
      float sum = 0.0f;
#pragma unroll 8
      for (int v = 0; v < a.vocab; ++v) sum = __builtin_fmaf(z[r * wp + v], w[k * wp + v], sum);
      a.dx[r * a.lddx + k] = sum;
    }
  if (a.dw)
    for (int i = tid; i < a.in * a.vocab; i += 1024) {
      const int k = i / a.vocab, v = i % a.vocab;
      float sum = 0.0f;
#pragma unroll 8
      for (int r = 0; r < a.rows; ++r) sum = __builtin_fmaf(x[r * xp + k], z[r * wp + v], sum);
      a.dw[k * a.lddw + v] = sum;
    }
  if (a.db)
    for (int v = tid; v < a.vocab; v += 1024) {
      float sum = 0.0f;
      for (int r = 0; r < a.rows; ++r) sum += z[r * wp + v];
      a.db[v] = sum;
    }
}
int run_tiny_loss(Runtime* rt, const LossCall& c) {
  tiny_loss<<<dim3(1), dim3(1024), 0, rt->stream>>>(
      {int(c.rows), int(c.in), int(c.vocab), c.x, int64_t(c.ldx), c.w, int64_t(c.ldw), c.bias, c.targets, c.weights, c.loss,
       c.dx, int64_t(c.lddx), c.dw, int64_t(c.lddw), c.db});
  LMP_LAUNCH_CHECK("tiny_loss");
  return LMP_OK;
}

// ------------------------------------------------------- on the fp16 matrix cores

// The largest logit and the sum of exponents below it of a row's 64 columns, for each wave
// column of the tiles.
struct HalfLogits {
  const float* bias;
  float* z;      // [rows, vocab], or null
  Softmax* part;  // [rows, parts]
  int parts;
  const int64_t* targets;
  float* hit;  // [rows]: the target's logit
};

__device__ __forceinline__ float over_eight(float x, bool most) {
#define LMP_STEP(ctrl)                                                                                          \
  {                                                                                                             \
    const float y = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xF, 0xF, false)); \
    x = most ? fmaxf(x, y) : x + y;                                                                             \
  }
  LMP_STEP(0xB1);
  LMP_STEP(0x4E);
  LMP_STEP(0x141);
#undef LMP_STEP
  return x;
}

template <int NT, int MINB, class C>
__global__ __launch_bounds__(NT, MINB) void half_logits(HalfArgs g, HalfLogits o, RowsOf<MatrixSource> x, ColsOf<MatrixSource> w) {
  static_assert(NT == C::THREADS && C::TN == 2, "a wave has 64 columns");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  const HalfItem at = half_item(g, int(blockIdx.x));
  const int wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % C::WN, col0 = at.tile_n * C::BN + wn * 64;
  half_product<C>(g, at, smem, x, w, [&](int row, int c4, hv4 (&v)[2]) {
    const float low = -__builtin_huge_valf();
    const int64_t target = row < g.m ? o.targets[row] : -1;
    float top = low;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = col0 + 32 * j + c4;
      if (o.bias) v[j] = v[j] + load_four(o.bias, col, g.n);
      if (o.z && row < g.m) store_four(o.z + int64_t(row) * g.n, col, g.n, v[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (target == col + e && col + e < g.n) o.hit[row] = v[j][e];
        if (col + e >= g.n) v[j][e] = low;
        top = fmaxf(top, v[j][e]);  // of NaN the other one
      }
    }
    top = over_eight(top, true);
    const float from = top > low ? top : 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += exp_below(v[j][e] - from);
    sum = over_eight(sum, false);
    if (c4 == 0 && row < g.m) o.part[int64_t(row) * o.parts + at.tile_n * C::WN + wn] = {top, sum};
  });
}

// What the gradient of a row's logits needs: dz = e^(z - top) factor - [v = target] weight.
struct LossRow {
  float top, factor, weight;
  int target;  // -1: not counted, or past the vocabulary (whose factor is NaN)
};

// The rows' losses from their parts, a wave a row; with `info` what the gradient needs.
struct HalfRows {
  int64_t rows;
  int parts, vocab;
  const Softmax* part;
  const float* hit;
  const int64_t* targets;
  const float* weights;
  float* loss;
  LossRow* info;
};
__global__ __launch_bounds__(256) void half_loss_rows(HalfRows a) {
  const int lane = threadIdx.x & 63;
  for (int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); row < a.rows; row += int64_t(gridDim.x) * 4) {
    const int64_t t = a.targets[row];
    const Softmax* p = a.part + row * a.parts;
    Softmax s{-__builtin_huge_valf(), 0.0f};
    for (int i = lane; i < a.parts; i += 64) s = joined(s, p[i]);
    for (int off = 1; off < 64; off *= 2) s = joined(s, {__shfl_xor(s.top, off), __shfl_xor(s.sum, off)});
    if (lane) continue;
    const bool counted = t >= 0, known = t < a.vocab;
    const float nan = __builtin_nanf("");
    a.loss[row] = !counted ? 0.0f : known ? logf(s.sum) - (a.hit[row] - s.top) : nan;
    if (a.info) {
      const float w = !counted ? 0.0f : !known ? nan : a.weights ? a.weights[row] : 1.0f;
      a.info[row] = {s.top, w / s.sum, w, counted && known ? int(t) : counted ? -2 : -1};
    }
  }
}

// dz, formed from the logits.
struct LossGradient {
  int64_t rows;
  int cols;
  const float* z;  // [rows, cols]
  const LossRow* info;
  __device__ __forceinline__ void load(int64_t row, int unit, hv4 (&v)[2]) const {
    const LossRow r = info[row];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = column(unit, h);
      v[h] = load_four(z + row * cols, col, cols);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp_below(v[h][e] - r.top) * r.factor;
        v[h][e] = r.target == -1 || col + e >= cols ? 0.0f : col + e == r.target ? p - r.weight : p;
      }
    }
  }
  __device__ __forceinline__ int column(int unit, int h) const { return 8 * unit + 4 * h; }
  __device__ __forceinline__ int place(int col) const { return col; }
  __device__ __forceinline__ float value(int64_t row, int col) const {
    const LossRow r = info[row];
    const float p = exp_below(z[row * cols + col] - r.top) * r.factor;
    return r.target == -1 ? 0.0f : col == r.target ? p - r.weight : p;
  }
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

// Whether the split products pay for reading x and w twice, writing their panels (12 bytes a
// value, 16 with the gradients) and their launches.  They save the pass over the logits
// that the losses alone take, or cost 4 bytes a logit for the gradients' panels.  384 rows of
// 1024 over 32768 words take 265 us without them and 165 with them (586 and 463 with the
// gradients), 256 rows 150 and 139 (352 and 376), 64 rows 65 and 111.
bool half_pays(const LossCall& c) {
  const double n = double(c.rows), d = double(c.in), v = double(c.vocab), work = n * d * v;
  if (!half_fits(c.rows, c.in, c.vocab)) return false;
  if (!c.dx && !c.dw) return half_saves_forward(work) + pass_time(8 * n * v) > 12 + pass_time(12 * (n * d + d * v));
  return half_saves_forward(work) + half_saves_backward(work) > 25 + pass_time(16 * (n * d + d * v) + 4 * n * v);
}

int run_loss_half(Runtime* rt, const LossCall& c) {
  const bool grad = c.dx || c.dw;
  // Pieces of whole groups of panels: of logits, or for the losses alone of what is kept of 64 of them.
  const size_t row_bytes = grad ? c.vocab * sizeof(float) : (c.vocab + 63) / 64 * sizeof(Softmax);
  const size_t fit = std::max<size_t>(256, kPieceBytes / row_bytes / 256 * 256);
  const size_t pieces = (c.rows + fit - 1) / fit;
  const size_t each = pieces > 1 ? ((c.rows + pieces - 1) / pieces + 255) / 256 * 256 : c.rows;
  const HalfPlan plan = half_plan(rt->cu_count, 0, {int64_t(each), int64_t(c.vocab), int64_t(c.in), false, 2.0f}, {});
  if (plan.cfg < 0) return fail(LMP_ERR_UNSUPPORTED, "linear_cross_entropy: more tiles than a grid holds");
  const int bn = kHalfTiles[plan.cfg].bn, parts = int((c.vocab + bn - 1) / bn) * (bn / 64);
  const size_t strips = c.db ? size_t(most_strips(rt, int64_t(each), int64_t(c.vocab))) : 0;
  HalfRoom room;
  const size_t of_xr = room.take(half_tops_words(c.rows)), of_wc = room.take(half_tops_words(c.vocab));
  const size_t of_xc = room.take(c.dw ? half_tops_words(c.in) : 0), of_wr = room.take(c.dx ? half_tops_words(c.in) : 0);
  const size_t of_dr = room.take(grad ? half_tops_words(each) : 0), of_dc = room.take(grad ? half_tops_words(c.vocab) : 0);
  const size_t tops = room.words, of_marks = room.take(tops);
  const size_t at_part = room.take(each * size_t(parts) * 2), at_hit = room.take(each), at_info = room.take(grad ? each * 4 : 0);
  const size_t at_sums = room.take(strips * c.vocab), at_db = room.take(c.db ? c.vocab : 0);
  const size_t at_z = room.take(grad ? each * c.vocab : 0);
  const size_t at_xr = room.take(half_panel_words(c.rows, c.in)), at_wc = room.take(half_panel_words(c.vocab, c.in));
  const size_t at_xc = room.take(c.dw ? half_panel_words(c.in, c.rows) : 0);
  const size_t at_wr = room.take(c.dx ? half_panel_words(c.in, c.vocab) : 0);
  const size_t at_dr = room.take(c.dx ? half_panel_words(each, c.vocab) : 0);
  const size_t at_dc = room.take(c.dw ? half_panel_words(c.vocab, each) : 0);
  float* base = static_cast<float*>(scratch_alloc(room.words * sizeof(float)));
  if (!base) return LMP_ERR_OOM;
  uint32_t* words = reinterpret_cast<uint32_t*>(base);
  const auto panels = [&](size_t at, size_t k, size_t of) {
    return HalfPanels{reinterpret_cast<char*>(words + at), int64_t(half_stride(k)), words + of, words + of_marks + of};
  };
  const HalfPanels none{}, xr = panels(at_xr, c.in, of_xr), wc = panels(at_wc, c.in, of_wc);
  const HalfPanels xc = c.dw ? panels(at_xc, c.rows, of_xc) : none, wr = c.dx ? panels(at_wr, c.vocab, of_wr) : none;
  const MatrixSource of_w{int64_t(c.in), int(c.vocab), c.w, int64_t(c.ldw), nullptr};
  const auto piece = [&](size_t at, size_t n) -> int {
    const HalfPanels mine{xr.panels + int64_t(at / 64) * xr.stride, xr.stride, xr.tops + at, xr.marks + at};
    const HalfArgs g = half_args(mine, wc, int(n), int(c.vocab), int(c.in), plan.cfg, 1);
    float* z = grad ? base + at_z : nullptr;
    Softmax* part = reinterpret_cast<Softmax*>(base + at_part);
    LossRow* info = grad ? reinterpret_cast<LossRow*>(base + at_info) : nullptr;
    const HalfLogits o{c.bias, z, part, parts, c.targets + at, base + at_hit};
    const MatrixSource x{int64_t(n), int(c.in), c.x + at * c.ldx, int64_t(c.ldx), c.targets + at};
    if (int s = with_half_cfg(plan.cfg, [&](auto cfg) -> int {
          using C = decltype(cfg);
          half_logits<C::THREADS, C::MINB, C><<<dim3(half_items(g)), dim3(C::THREADS), 0, rt->stream>>>(g, o, {x}, {of_w});
          LMP_LAUNCH_CHECK("half_logits");
          return LMP_OK;
        }))
      return s;
    const HalfRows r{int64_t(n), parts, int(c.vocab), part, base + at_hit, c.targets + at,
                     c.weights ? c.weights + at : nullptr, c.loss + at, info};
    half_loss_rows<<<dim3(uint32_t(std::min<size_t>((n + 3) / 4, 65536))), dim3(256), 0, rt->stream>>>(r);
    LMP_LAUNCH_CHECK("half_loss_rows");
    if (!grad) return LMP_OK;
    if (at) {
      if (int s = clear_words(rt, words + of_dr, tops - of_dr)) return s;
      if (int s = clear_words(rt, words + of_marks + of_dr, tops - of_dr)) return s;
    }
    const HalfPanels dr = c.dx ? panels(at_dr, c.vocab, of_dr) : none, dc = c.dw ? panels(at_dc, n, of_dc) : none;
    const LossGradient of_d{int64_t(n), int(c.vocab), z, info};
    const auto job = tops_job(rt, of_d, dr.tops, dc.tops, c.db ? base + at_sums : nullptr);
    if (int s = run_panel_jobs(rt, job)) return s;
    if (c.db) {
      float* to = at ? base + at_db : c.db;
      const size_t mine_strips = size_t(job.blocks / job.col_blocks);
      if (int s = lmp_k_reduce(LMP_RED_SUM, LMP_FLOAT32, to, base + at_sums, 1, mine_strips, c.vocab)) return s;
      if (at)
        if (int s = lmp_k_add_inplace(LMP_FLOAT32, c.db, to, c.vocab)) return s;
    }
    if (int s = run_panel_jobs(rt, pack_job(of_d, dr, dc))) return s;
    HalfPanels xp = xc;  // K of dw from this piece's first row on
    if (c.dw) xp.panels += int64_t(at / kHalfK) * kHalfStep;
    return half_backward<LossGradient, MatrixSource>(
        rt, {n, c.in, c.vocab, dr, dc, xp, wr, c.dx ? c.dx + at * c.lddx : nullptr, c.lddx, c.dw, c.lddw, at > 0, 0, x, of_d, of_w});
  };
  const auto run = [&]() -> int {
    if (int s = clear_words(rt, words, 2 * tops)) return s;
    const MatrixSource of_x{int64_t(c.rows), int(c.in), c.x, int64_t(c.ldx), c.targets};
    if (int s = run_panel_jobs(rt, tops_job(rt, of_w, wr.tops, wc.tops), tops_job(rt, of_x, xr.tops, xc.tops))) return s;
    if (int s = run_panel_jobs(rt, pack_job(of_w, wr, wc), pack_job(of_x, xr, xc))) return s;
    for (size_t at = 0; at < c.rows; at += each)
      if (int s = piece(at, std::min(each, c.rows - at))) return s;
    return LMP_OK;
  };
  const int rc = run();
  scratch_free(base);
  return rc;
}

int run_loss(Runtime* rt, const LossCall& c) {
  if (c.rows == 0) {
    if (int s = clear_f32(rt, c.dw, c.in, c.vocab, c.lddw)) return s;
    return clear_f32(rt, c.db, 1, c.vocab, c.vocab);
  }
  if (tiny_fits(c)) return run_tiny_loss(rt, c);
  // Where memory is short, products that need none besides the logits' take over, and then
  // smaller pieces.
  if (half_pays(c))
    if (int s = run_loss_half(rt, c); s != LMP_ERR_OOM) return s;
  size_t each = 0, logits = 0;
  float* z = nullptr;
  for (size_t bytes = kPieceBytes;; bytes /= 4) {
    const size_t fit = std::max<size_t>(256, bytes / (c.vocab * sizeof(float))), pieces = (c.rows + fit - 1) / fit;
    each = (c.rows + pieces - 1) / pieces;
    logits = (each * c.vocab + 3) / 4 * 4;
    z = static_cast<float*>(scratch_alloc((logits + (c.dw ? each * c.in : 0)) * sizeof(float)));
    if (z) break;
    if (fit == 256) return LMP_ERR_OOM;
  }
  float* counted_x = c.dw ? z + logits : nullptr;
  const auto piece = [&](size_t at, size_t n) -> int {
    const float* x = c.x + at * c.ldx;
    if (int s = c.bias ? lmp_k_linear_f32(0, 0, n, c.vocab, c.in, x, c.ldx, c.w, c.ldw, c.bias, z, c.vocab)
                       : lmp_k_gemm_f32(0, 0, n, c.vocab, c.in, x, c.ldx, c.w, c.ldw, z, c.vocab, 0))
      return s;
    const LossArgs a{int64_t(n), int(c.vocab), z, c.targets + at, c.weights ? c.weights + at : nullptr,
                     c.loss + at, x, int64_t(c.ldx), int(c.in), counted_x};
    const bool grad = c.dx || c.dw;
    if (int s = grad ? launch_loss_rows<true>(rt, a) : launch_loss_rows<false>(rt, a)) return s;
    if (!grad) return LMP_OK;
    const int more = at > 0;
    if (c.dx && c.db)
      return lmp_k_linear_backward_f32(n, c.in, c.vocab, counted_x, c.in, c.w, c.ldw, z, c.vocab, c.dx + at * c.lddx, c.lddx,
                                       0, c.dw, c.lddw, more, c.db, more);
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
