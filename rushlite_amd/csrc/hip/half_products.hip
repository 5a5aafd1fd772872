// A layer's two gradient products on the fp16 matrix cores (gemm_half.hpp).
#include "half_products.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>

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

template <int NT, int MINB, class C>
__global__ __launch_bounds__(NT, MINB) void half_gemm(HalfArgs g, HalfOut o) {
  static_assert(NT == C::THREADS, "one lane per thread of the configuration");
  __shared__ __attribute__((aligned(1024))) char smem[C::SMEM];
  half_plain<C>(g, o, int(blockIdx.x), smem);
}

// A layer's weight gradient and input gradient in one grid: the CUs that the first frees
// start on the second.
template <int NT, int MINB, class CW, class CX>
__global__ __launch_bounds__(NT, MINB) void half_gemm_pair(HalfArgs w, HalfOut wo, HalfArgs x, HalfOut xo) {
  static_assert(NT == CW::THREADS && NT == CX::THREADS, "one workgroup size for both");
  __shared__ __attribute__((aligned(1024))) char smem[CW::SMEM > CX::SMEM ? CW::SMEM : CX::SMEM];
  const int of_w = w.tiles_m * w.tiles_n * w.splits, id = int(blockIdx.x);
  if (id < of_w) half_plain<CW>(w, wo, id, smem);
  else half_plain<CX>(x, xo, id - of_w, smem);
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
  HalfPlan plan;
  bool wanted = false;
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
  HalfJob w, x;
  const int64_t cus = rt->cu_count;
  const int rows = int(b.rows), in = int(b.in), width = int(b.width);
  if (b.dw) {
    w.wanted = true;
    w.plan = half_plan(cus, kHalfParts, in, width, rows, true);
    w.o = {b.dw, int64_t(b.lddw), b.dw_accumulate ? 1 : 0, int(b.hidden), nullptr};
  }
  if (b.dx) {
    x.wanted = true;
    x.plan = half_plan(cus, kHalfParts, rows, in, width, true);
    x.o = {b.dx, int64_t(b.lddx), 0, 0, nullptr};
  }
  if ((w.wanted && w.plan.cfg < 0) || (x.wanted && x.plan.cfg < 0))
    return fail(LMP_ERR_UNSUPPORTED, "gradient products: more tiles than a grid holds");
  if (w.wanted) w.g = half_args(b.x_cols, b.d_cols, in, width, rows, w.plan);
  if (x.wanted) x.g = half_args(b.d_rows, b.w_rows, rows, in, width, x.plan);
  size_t parts = 0;
  for (HalfJob* j : {&w, &x})
    if (j->wanted && j->g.splits > 1) parts += (size_t(j->g.splits) * size_t(j->g.m) * size_t(j->g.n) + 3) / 4 * 4;
  float* scratch = nullptr;
  if (parts) {
    scratch = static_cast<float*>(scratch_alloc(parts * sizeof(float)));
    if (!scratch) return LMP_ERR_OOM;
    float* p = scratch;
    for (HalfJob* j : {&w, &x})
      if (j->wanted && j->g.splits > 1) {
        j->o.part = p;
        p += (size_t(j->g.splits) * size_t(j->g.m) * size_t(j->g.n) + 3) / 4 * 4;
      }
  }
  const auto alone = [&](const HalfJob& j) {
    return with_half_cfg(j.plan.cfg, [&](auto cfg) -> int {
      using C = decltype(cfg);
      half_gemm<C::THREADS, C::MINB, C><<<dim3(half_items(j.g)), dim3(C::THREADS), 0, rt->stream>>>(j.g, j.o);
      LMP_LAUNCH_CHECK("half_gemm");
      return LMP_OK;
    });
  };
  const auto run = [&]() -> int {
    bool paired = false;
    if (w.wanted && x.wanted &&
        kHalfTiles[w.plan.cfg].threads == kHalfTiles[x.plan.cfg].threads &&
        bf3_pair_fits(half_items(w.g), half_items(x.g), kHalfTiles[w.plan.cfg].threads)) {
      paired = true;
      const int rc = with_half_cfg(w.plan.cfg, [&](auto cw) {
        return with_half_cfg(x.plan.cfg, [&](auto cx) -> int {
          using CW = decltype(cw);
          using CX = decltype(cx);
          if constexpr (CW::THREADS == CX::THREADS) {
            constexpr int kMinB = CW::MINB < CX::MINB ? CW::MINB : CX::MINB;
            half_gemm_pair<CW::THREADS, kMinB, CW, CX>
                <<<dim3(half_items(w.g) + half_items(x.g)), dim3(CW::THREADS), 0, rt->stream>>>(w.g, w.o, x.g, x.o);
            LMP_LAUNCH_CHECK("half_gemm_pair");
            return LMP_OK;
          } else {
            return fail(LMP_ERR_RUNTIME, "gradient products: workgroup sizes differ");
          }
        });
      });
      if (rc) return rc;
    }
    if (!paired && w.wanted)
      if (int s = alone(w)) return s;
    if (!paired && x.wanted)
      if (int s = alone(x)) return s;
    const auto fold = [&](const HalfJob& j) {
      HalfFold f{j.o, j.g.m, j.g.n, j.g.splits, 0};
      if (j.wanted && j.g.splits > 1) f.blocks = (int64_t(f.m) * ((f.n + 3) / 4) + kThreads - 1) / kThreads;
      return f;
    };
    const HalfFold fw = fold(w), fx = fold(x);
    if (fw.blocks + fx.blocks) {
      half_fold<<<dim3(uint32_t(fw.blocks + fx.blocks)), dim3(kThreads), 0, rt->stream>>>(fw, fx);
      LMP_LAUNCH_CHECK("half_fold");
    }
    return LMP_OK;
  };
  const int rc = run();
  if (scratch) scratch_free(scratch);  // stream-ordered: the fold reads it first
  return rc;
}

}  // namespace lmp_hip
