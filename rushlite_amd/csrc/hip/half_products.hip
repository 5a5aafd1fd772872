// A layer's two gradient products on the fp16 matrix cores (gemm_half.hpp).
#include "half_products.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <utility>

#include "gemm_half.hpp"
#include "half_panels.hpp"

namespace lmp_hip {
namespace {

constexpr int kThreads = 256;

__global__ __launch_bounds__(kThreads) void clear_kernel(uint32_t* p, int64_t n) {
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < n; i += int64_t(gridDim.x) * kThreads) p[i] = 0;
}
__global__ __launch_bounds__(kThreads) void clear_rows(float* p, int64_t rows, int cols, int64_t ld) {
  const int64_t total = rows * cols;
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < total; i += int64_t(gridDim.x) * kThreads)
    p[i / cols * ld + i % cols] = 0.0f;
}

// Where a product goes: C, or (splits > 1) the parts of each split, [split][m][n].  `hidden`: as
// HalfBackward's, of C's columns.
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

template <class C>
__device__ __forceinline__ void half_plain(const HalfArgs& g, const HalfOut& o, int id, char* smem) {
  hv16 acc[C::TM][C::TN];
  const HalfItem at = half_item(g, id);
  half_tile<C>(g, at, smem, acc);
  const int wn = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % C::WN, col0 = at.tile_n * C::BN + wn * C::TN * 32;
  const bool partial = g.splits > 1;
  const bool add = !partial && o.accumulate;
  half_epilogue<C>(g, at, smem, acc, [&](int row, int c4, hv4 (&v)[C::TN]) {
    if (row >= g.m) return;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
      const int col = col0 + 32 * j + c4;
      if (partial) {
        store_four(o.part + (int64_t(at.split) * g.m + row) * g.n, col, g.n, v[j]);
        continue;
      }
      int end;
      const int to = place_of(o, col, g.n, end);
      float* p = o.c + row * o.ldc;
      if (add) v[j] = load_four(p, to, end) + v[j];
      store_four(p, to, end, v[j]);
    }
  });
}

// Two products in one grid, or one: the CUs that the first frees start on the second.
template <int NT, int MINB, class C>
__global__ __launch_bounds__(NT, MINB) void half_gemm(HalfArgs a, HalfOut ao, HalfArgs b, HalfOut bo) {
  static_assert(NT == C::THREADS, "one lane per thread of the configuration");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  const int first = a.tiles_m * a.tiles_n * a.splits, id = int(blockIdx.x);
  if (id < first) half_plain<C>(a, ao, id, smem);
  else half_plain<C>(b, bo, id - first, smem);
}

// C from the parts, added in their order; four values a lane.
struct HalfFold {
  HalfOut o;
  int m, n, splits;
  int64_t blocks;
};
__device__ __forceinline__ void fold_block(const HalfFold& f, int64_t block) {
  const int quads = (f.n + 3) / 4;
  const int64_t i = block * kThreads + threadIdx.x;
  if (i >= int64_t(f.m) * quads) return;
  const int row = int(i / quads), col = int(i - int64_t(row) * quads) * 4;
  const int64_t stride = int64_t(f.m) * f.n;
  const float* p = f.o.part + int64_t(row) * f.n;
  hv4 v = load_four(p, col, f.n);
#pragma unroll 4
  for (int s = 1; s < f.splits; ++s) v = v + load_four(p + s * stride, col, f.n);
  int end;
  const int to = place_of(f.o, col, f.n, end);
  float* c = f.o.c + row * f.o.ldc;
  if (f.o.accumulate) v = load_four(c, to, end) + v;
  store_four(c, to, end, v);
}
__global__ __launch_bounds__(kThreads) void half_fold(HalfFold a, HalfFold b) {
  const int64_t block = blockIdx.x;
  if (block < a.blocks) fold_block(a, block);
  else fold_block(b, block - a.blocks);
}

// Bytes of all parts of one product at most.
constexpr int64_t kHalfParts = int64_t(256) << 20;

struct HalfJob {
  HalfArgs g{};
  HalfOut o{};
};

}  // namespace

int clear_words(Runtime* rt, uint32_t* p, size_t n) {
  if (n == 0) return LMP_OK;
  clear_kernel<<<dim3(uint32_t(std::min<size_t>((n + 1023) / 1024, 4096))), dim3(kThreads), 0, rt->stream>>>(p, int64_t(n));
  LMP_LAUNCH_CHECK("clear");
  return LMP_OK;
}

int clear_f32(Runtime* rt, float* p, size_t rows, size_t cols, size_t ld) {
  if (!p || rows == 0 || cols == 0) return LMP_OK;
  const size_t groups = (rows * cols + kThreads - 1) / kThreads;
  clear_rows<<<dim3(uint32_t(std::min<size_t>(groups, 65536))), dim3(kThreads), 0, rt->stream>>>(
      p, int64_t(rows), int(cols), int64_t(ld));
  LMP_LAUNCH_CHECK("clear");
  return LMP_OK;
}

int half_backward(Runtime* rt, const HalfBackward& b) {
  const int rows = int(b.rows), in = int(b.in), width = int(b.width);
  HalfSize sizes[2];
  int jobs = 0;
  if (b.dw) sizes[jobs++] = {in, width, rows, true};
  if (b.dx) sizes[jobs++] = {rows, in, width, true};
  if (jobs == 0) return LMP_OK;
  const HalfPlan plan = half_plan(rt->cu_count, kHalfParts, sizes[0], sizes[1]);
  if (plan.cfg < 0) return fail(LMP_ERR_UNSUPPORTED, "gradient products: more tiles than a grid holds");
  HalfJob job[2];
  jobs = 0;
  if (b.dw) {
    job[jobs] = {half_args(b.x_cols, b.d_cols, in, width, rows, plan.cfg, plan.splits[jobs]),
                 {b.dw, int64_t(b.lddw), b.dw_accumulate ? 1 : 0, int(b.hidden), nullptr}};
    ++jobs;
  }
  if (b.dx) {
    job[jobs] = {half_args(b.d_rows, b.w_rows, rows, in, width, plan.cfg, plan.splits[jobs]),
                 {b.dx, int64_t(b.lddx), 0, 0, nullptr}};
    ++jobs;
  }
  if (plan.second_first) std::swap(job[0], job[1]);
  HalfRoom room;
  size_t at[2];
  for (int i = 0; i < 2; ++i)
    at[i] = room.take(job[i].g.splits > 1 ? size_t(job[i].g.splits) * size_t(job[i].g.m) * size_t(job[i].g.n) : 0);
  float* scratch = nullptr;
  if (room.words) {
    scratch = static_cast<float*>(scratch_alloc(room.words * sizeof(float)));
    if (!scratch) return LMP_ERR_OOM;
    for (int i = 0; i < 2; ++i) job[i].o.part = scratch + at[i];
  }
  const auto run = [&]() -> int {
    if (int s = with_half_cfg(plan.cfg, [&](auto cfg) -> int {
          using C = decltype(cfg);
          half_gemm<C::THREADS, C::MINB, C><<<dim3(half_items(job[0].g) + half_items(job[1].g)), dim3(C::THREADS), 0,
                                              rt->stream>>>(job[0].g, job[0].o, job[1].g, job[1].o);
          LMP_LAUNCH_CHECK("half_gemm");
          return LMP_OK;
        }))
      return s;
    const auto fold = [&](const HalfJob& j) {
      HalfFold f{j.o, j.g.m, j.g.n, j.g.splits, 0};
      if (j.g.splits > 1) f.blocks = (int64_t(f.m) * ((f.n + 3) / 4) + kThreads - 1) / kThreads;
      return f;
    };
    const HalfFold f0 = fold(job[0]), f1 = fold(job[1]);
    if (f0.blocks + f1.blocks) {
      half_fold<<<dim3(uint32_t(f0.blocks + f1.blocks)), dim3(kThreads), 0, rt->stream>>>(f0, f1);
      LMP_LAUNCH_CHECK("half_fold");
    }
    return LMP_OK;
  };
  const int rc = run();
  if (scratch) scratch_free(scratch);  // stream-ordered: the fold reads it first
  return rc;
}

}  // namespace lmp_hip
