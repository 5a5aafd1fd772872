// A layer's two gradient products on the fp16 matrix cores (gemm_half.hpp): dx = d w^T and
// dw (+)= x^T d in one launch, and where K is split a second one that adds the parts.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "gemm_half.hpp"
#include "half_panels.hpp"
#include "half_products.hpp"

namespace lmp_hip {
namespace {

// Where a product goes: C, or (splits > 1) the parts of each split, [split][m][n], scaled.  `hidden`:
// as HalfBackward's, of C's columns.
struct HalfOut {
  float* c;
  int64_t ldc;
  int accumulate, hidden;
  float* part;
};
// Where C holds column `col`, a multiple of 4, and where its run of columns ends.
__device__ __forceinline__ int place_of(const HalfOut& o, int col, int n, int& end) {
  end = n;
  if (!o.hidden) return col;
  const int second = col / 32 & 1;
  end = (1 + second) * o.hidden;
  return col / 64 * 32 + col % 32 + second * o.hidden;
}
__device__ __forceinline__ void put_four(const HalfOut& o, int64_t row, int col, int n, hv4 v) {
  int end;
  const int to = place_of(o, col, n, end);
  float* p = o.c + row * o.ldc;
  if (o.accumulate) v = load_four(p, to, end) + v;
  store_four(p, to, end, v);
}

template <class C, class A, class B>
__device__ __forceinline__ void half_plain(const HalfArgs& g, const HalfOut& o, const A& a, const B& b, int id, char* smem) {
  const HalfItem at = half_item(g, id);
  const int wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % C::WN, col0 = at.tile_n * C::BN + wn * C::TN * 32;
  if (g.splits > 1) {
    hv16 acc[C::TM][C::TN];
    half_sums<C, false>(g, at, smem, acc);
    __syncthreads();  // the stages have been read
    const hi4 none[C::TN] = {};
#pragma unroll
    for (int i = 0; i < C::TM; ++i)
      half_out<C, false>(g, at, smem, acc[i], i, none, 0, [&](int row, int c4, hv4 (&v)[C::TN]) {
        if (row >= g.m) return;
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
          store_four(o.part + (int64_t(at.split) * g.m + row) * g.n, col0 + 32 * j + c4, g.n, v[j]);
      });
    return;
  }
  half_product<C>(g, at, smem, a, b, [&](int row, int c4, hv4 (&v)[C::TN]) {
    if (row >= g.m) return;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) put_four(o, row, col0 + 32 * j + c4, g.n, v[j]);
  });
}

// One product: its panels, where it goes, and the operands themselves.
template <class A, class B>
struct HalfJob {
  HalfArgs g;
  HalfOut o;
  A a;
  B b;
};

// Two products in one grid, or one (the other has no tiles): the CUs that the first frees start
// on the second.
template <int NT, int MINB, class C, class W, class X>
__global__ __launch_bounds__(NT, MINB) void half_gemm(W dw, X dx, int dx_first) {
  static_assert(NT == C::THREADS, "one lane per thread of the configuration");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  const int of_dw = dw.g.tiles_m * dw.g.tiles_n * dw.g.splits, of_dx = dx.g.tiles_m * dx.g.tiles_n * dx.g.splits;
  const int id = int(blockIdx.x);
  if (dx_first ? id >= of_dx : id < of_dw) half_plain<C>(dw.g, dw.o, dw.a, dw.b, dx_first ? id - of_dx : id, smem);
  else half_plain<C>(dx.g, dx.o, dx.a, dx.b, dx_first ? id : id - of_dw, smem);
}

// C from the parts, added in their order, 64 x 64 of it a workgroup; what is too small or not
// finite is formed again as in half_tile.
struct FoldTile {
  static constexpr int WM = 2, WN = 2, TM = 1, TN = 1, BM = 64, BN = 64, THREADS = 512;  // four waves form whole tiles again
  static constexpr int EACH = 2, PITCH = 68, SMEM = 2 * 64 * 64 * 4;
};
template <class J>
__device__ __forceinline__ void fold_tile(const J& job, int64_t block, char* smem, HalfDoubt* doubt) {
  using C = FoldTile;
  const HalfArgs& g = job.g;
  const int across = (g.n + 63) / 64;
  const int64_t row0 = block / across * 64;
  const int col0 = int(block - block / across * across) * 64;
  const int r = threadIdx.x / 16, c4 = threadIdx.x % 16 * 4, col = col0 + c4;
  if (threadIdx.x == 0) doubt->count = 0;
  const int64_t stride = int64_t(g.m) * g.n;
  hv4 v[C::EACH];
  uint32_t a_top[C::EACH], a_marks[C::EACH];
  const hu4 b_top = *reinterpret_cast<const hu4*>(g.b_top + col), b_marks = *reinterpret_cast<const hu4*>(g.b_marks + col);
#pragma unroll
  for (int i = 0; i < C::EACH; ++i) {
    const int64_t row = row0 + r + 32 * i;
    a_top[i] = g.a_top[row];
    a_marks[i] = g.a_marks[row];
    v[i] = row < g.m && col < g.n ? load_four(job.o.part + row * g.n, col, g.n) : hv4(0.0f);
  }
#pragma unroll 4
  for (int s = 1; s < g.splits; ++s)
#pragma unroll
    for (int i = 0; i < C::EACH; ++i) {
      const int64_t row = row0 + r + 32 * i;
      if (row < g.m && col < g.n) v[i] = v[i] + load_four(job.o.part + s * stride + row * g.n, col, g.n);
    }
  __syncthreads();
  const float per_k = kHalfLeast / float(g.k);
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < C::EACH; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool inside = row0 + r + 32 * i < g.m && col + e < g.n;
      if (inside && half_doubtful(v[i][e], half_limit(a_top[i], a_marks[i], per_k), half_limit(b_top[e], b_marks[e], per_k)))
        found |= 1u << (4 * i + e);
      v[i][e] = ldexpf(v[i][e], -(half_exponent(a_top[i]) + half_exponent(b_top[e])));
    }
  note_doubts(doubt, found, uint32_t(r) << 16 | uint32_t(c4), 32 << 16, 1);
  __syncthreads();
  const int count = doubt->count;
  if (count > kHalfList) {
    hv16 acc[1];
    whole_blocks<C>(job.a, job.b, row0, col0, 0, smem, acc);
    float* t = reinterpret_cast<float*>(smem);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < C::WM * C::WN)
#pragma unroll
      for (int q = 0; q < 16; ++q)
        t[(wave / C::WN * 32 + 8 * (q / 4) + 4 * (lane >> 5) + q % 4) * C::PITCH + wave % C::WN * 32 + (lane & 31)] = acc[0][q];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C::EACH; ++i) v[i] = *reinterpret_cast<const hv4*>(t + (r + 32 * i) * C::PITCH + c4);
  } else {
#pragma unroll 1
    for (int p = 0; p < count; ++p) {
      const uint32_t where = doubt->at[p];
      const float sum = whole_sum<C::THREADS>(job.a, job.b, row0 + (where >> 16), col0 + (where & 0xffff), doubt->shares);
#pragma unroll
      for (int i = 0; i < C::EACH; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (where == (uint32_t(r + 32 * i) << 16 | uint32_t(c4 + e))) v[i][e] = sum;
    }
  }
#pragma unroll
  for (int i = 0; i < C::EACH; ++i)
    if (row0 + r + 32 * i < g.m && col < g.n) put_four(job.o, row0 + r + 32 * i, col, g.n, v[i]);
}
template <class W, class X>
__global__ __launch_bounds__(FoldTile::THREADS) void half_fold(W dw, X dx, int64_t of_dw) {
  __shared__ __attribute__((aligned(16))) char smem[FoldTile::SMEM];
  __shared__ HalfDoubt doubt;
  if (int64_t(blockIdx.x) < of_dw) fold_tile(dw, blockIdx.x, smem, &doubt);
  else fold_tile(dx, blockIdx.x - of_dw, smem, &doubt);
}

// Bytes of all parts of one product at most.
constexpr int64_t kHalfParts = int64_t(256) << 20;

// dx = d w^T and dw (+)= x^T d of a layer with x [rows, in] and w [in, width], each null
// where it is not wanted: d_rows [rows, width], w_rows [in, width], x_cols [in, rows], d_cols
// [width, rows]; and the sources of x, d and w.
template <class D, class W>
struct HalfBackward {
  size_t rows, in, width;
  HalfPanels d_rows, d_cols, x_cols, w_rows;
  float* dx;
  size_t lddx;
  float* dw;
  size_t lddw;
  bool dw_accumulate;
  // Not 0: the layer is gated, and its columns are 32 of the one half and 32 of the other by
  // turns, each half `hidden` columns long in dw.
  size_t hidden;
  MatrixSource x;
  D d;
  W w;
};

template <class D, class W>
int half_backward(Runtime* rt, const HalfBackward<D, W>& b) {
  const int rows = int(b.rows), in = int(b.in), width = int(b.width);
  HalfSize sizes[2];
  int jobs = 0;
  if (b.dw) sizes[jobs++] = {in, width, rows, true};
  if (b.dx) sizes[jobs++] = {rows, in, width, true};
  if (jobs == 0) return LMP_OK;
  const HalfPlan plan = half_plan(rt->cu_count, kHalfParts, sizes[0], sizes[1]);
  if (plan.cfg < 0) return fail(LMP_ERR_UNSUPPORTED, "gradient products: more tiles than a grid holds");
  HalfJob<ColsOf<MatrixSource>, ColsOf<D>> dw{{}, {}, {b.x}, {b.d}};
  HalfJob<RowsOf<D>, RowsOf<W>> dx{{}, {}, {b.d}, {b.w}};
  if (b.dw) {
    dw.g = half_args(b.x_cols, b.d_cols, in, width, rows, plan.cfg, plan.splits[0]);
    dw.o = {b.dw, int64_t(b.lddw), b.dw_accumulate ? 1 : 0, int(b.hidden), nullptr};
  }
  if (b.dx) {
    dx.g = half_args(b.d_rows, b.w_rows, rows, in, width, plan.cfg, plan.splits[jobs - 1]);
    dx.o = {b.dx, int64_t(b.lddx), 0, 0, nullptr};
  }
  const auto parts = [](const HalfArgs& g) { return g.splits > 1 ? size_t(g.splits) * size_t(g.m) * size_t(g.n) : 0; };
  HalfRoom room;
  const size_t at_dw = room.take(parts(dw.g)), at_dx = room.take(parts(dx.g));
  float* scratch = nullptr;
  if (room.words) {
    scratch = static_cast<float*>(scratch_alloc(room.words * sizeof(float)));
    if (!scratch) return LMP_ERR_OOM;
    dw.o.part = scratch + at_dw;
    dx.o.part = scratch + at_dx;
  }
  const auto run = [&]() -> int {
    if (int s = with_half_cfg(plan.cfg, [&](auto cfg) -> int {
          using C = decltype(cfg);
          half_gemm<C::THREADS, C::MINB, C><<<dim3(half_items(dw.g) + half_items(dx.g)), dim3(C::THREADS), 0, rt->stream>>>(
              dw, dx, plan.second_first ? 1 : 0);
          LMP_LAUNCH_CHECK("half_gemm");
          return LMP_OK;
        }))
      return s;
    const auto blocks = [](const HalfArgs& g) { return g.splits > 1 ? int64_t((g.m + 63) / 64) * ((g.n + 63) / 64) : 0; };
    const int64_t of_dw = blocks(dw.g), of_dx = blocks(dx.g);
    if (of_dw + of_dx) {
      half_fold<<<dim3(uint32_t(of_dw + of_dx)), dim3(FoldTile::THREADS), 0, rt->stream>>>(dw, dx, of_dw);
      LMP_LAUNCH_CHECK("half_fold");
    }
    return LMP_OK;
  };
  const int rc = run();
  if (scratch) scratch_free(scratch);  // stream-ordered: the fold reads it first
  return rc;
}

}  // namespace
}  // namespace lmp_hip
