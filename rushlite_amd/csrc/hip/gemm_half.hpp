// fp32 products on the fp16 matrix cores, each operand in two fp16 parts.
//
// Why.  A value scaled by a power of two is x = h + m + r with h = fp16(x), m =
// fp16(x - h) and |r| <= 2^-22 |x|, so
//   a b = ah bh + ah bm + am bh + (am bm and what the r leave out: 3 x 2^-22 at most)
// is three fp16 MFMAs with fp32 accumulation, half of what three bf16 parts cost
// (gemm_bf3.hpp), with a product's error near that of rounding its operands: a sum's
// error is its own roundings'.
//
// Range.  Each row of A and each column of B has a power of two that takes its largest
// finite magnitude to [2^14, 2^15): values down to 2^-17 of the largest keep both parts
// whole, smaller ones lose at most 2^-40 of it.  The two powers leave the sum at the end,
// exactly.  An infinity keeps its sign in h and has m = 0; it leaves a sum that is not
// finite, and a workgroup that finds one forms its tile again with the parts h that are not
// finite left out of the two small products, where 0 x infinity would be NaN.
//
// Operands are split once, by kernels of their own (half_products.hip), into panels of 64
// rows of A, or columns of B:
//   [row / 64][k / 8][part][row % 64][k % 8], K filled up with zeros to a multiple of 32, rows to 256,
// so that 64 rows of one octet are a kilobyte in a row, which one wave's load takes to LDS
// as it is, and in which a fragment of an MFMA is one conflict-free 128-bit read a lane.
//
// Structure.  A workgroup owns a BM x BN tile, its waves TM x TN blocks of 32 x 32.  K
// advances 32 at a time through two LDS stages, each half's fragments read while the products
// of the half before run.  One barrier a step, in its middle: the stage has been read by
// then, the next one has arrived, and the loads of the one after it start, a whole step
// ahead of their use.  The LDS is busy for two thirds of a 256 x 256 step's MFMA cycles.
//
// Bound by the chip's power: random operands run at 397 TFLOP/s (8192 x 32768 over 1024,
// 1.19 PFLOP/s of fp16, the clock at 1.7 of 2.4 GHz) to 422 (1024 x 32768 over 4096), zeros at
// 654, and the library's fp16 product of the first at 1.18 PFLOP/s.  Splitting the operands in
// registers on their way to LDS, in every tile that reads them, took it to 350.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gemm_plan.hpp"
#include "half_products.hpp"

namespace lmp_hip {
namespace {

typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef float hv2 __attribute__((ext_vector_type(2)));
typedef float hv4 __attribute__((ext_vector_type(4)));
typedef float hv4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float hv16 __attribute__((ext_vector_type(16)));
typedef uint32_t hu4 __attribute__((ext_vector_type(4)));
typedef int hi4 __attribute__((ext_vector_type(4)));
typedef uint16_t hw8 __attribute__((ext_vector_type(8)));

// Kept out of the templates: a target builtin inside a kernel template keeps the host
// pass from emitting the kernel's launch stub.
__device__ __forceinline__ hv16 mfma_f16(hf8 a, hf8 b, hv16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// 16 bytes a lane from memory to LDS: lane l's to lds + 16 l.
__device__ __forceinline__ void panel_load(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const float*>(src), reinterpret_cast<float*>(lds), 16, 0, 0);
}
// This wave's loads and LDS accesses are done, and then the workgroup's.
__device__ __forceinline__ void panels_settled() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(7 << 4);
  asm volatile("s_barrier" ::: "memory");
}

// The exponent of a row's power of two from the bits of its largest finite magnitude: [2^14,
// 2^15) where that is at least 2^-112.  Smaller rows and rows of zeros take 2^126.
__device__ __forceinline__ int half_exponent(uint32_t top) { return min(141 - int(top >> 23), 126); }
__device__ __forceinline__ float power_of(int e) {
  return __builtin_bit_cast(float, uint32_t(e + 127) << 23);
}

template <int WM_, int WN_, int TM_, int TN_, int MINB_>
struct HalfCfg {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, MINB = MINB_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int A_PANELS = BM / 64, PANELS = (BM + BN) / 64;
  static constexpr int STAGE = PANELS * kHalfStep;
  static constexpr int LOADS = PANELS * 8 / NW;  // of a wave, a step
  static constexpr int SMEM = 2 * STAGE + 16;    // the stages and the flag of sums that are not finite
  static_assert((TM == 1 || TM % 2 == 0) && TN % 2 == 0, "a wave's blocks are whole panels, or half of one");
  static_assert(2 * STAGE >= NW * 16 * (32 * TN + 4) * 4, "the epilogue's wave tiles fit");
  static_assert(BM % 64 == 0 && BN % 64 == 0 && LOADS * NW == PANELS * 8, "whole panels, split evenly");
};

// A product op(A) [m, k] op(B) [k, n] of panels.  `a_top` and `b_top`: the bits of the
// largest finite magnitude of each row of op(A) and column of op(B), rounded up to 256 of them.
struct HalfArgs {
  const char *a, *b;
  int64_t a_stride, b_stride;  // bytes from panel to panel
  int m, n;
  int steps;  // 32-wide k steps
  const uint32_t *a_top, *b_top;
  int tiles_m, tiles_n;
  int splits, steps_per_split;
};

// Where a work item lies: its tile's origin in tiles, and its split of K.
struct HalfItem {
  int tile_m, tile_n, split;
};

// Consecutive ids go round the eight XCDs: each takes a contiguous run of (split, tile),
// so that its L2 sees one range of k and neighbouring tiles, in groups of eight tile rows.
__device__ __forceinline__ HalfItem half_item(const HalfArgs& g, int id) {
  const int ntiles = g.tiles_m * g.tiles_n, total = ntiles * g.splits;
  {
    const int q = total / 8, r = total % 8, x = id % 8;
    id = x * q + min(x, r) + id / 8;
  }
  const int split = id / ntiles, tile = id - split * ntiles;
  constexpr int kGroup = 8;
  const int per_group = kGroup * g.tiles_n, group = tile / per_group;
  const int gsize = min(g.tiles_m - group * kGroup, kGroup);
  const int in_group = tile - group * per_group;
  return {group * kGroup + in_group % gsize, in_group / gsize, split};
}

// The parts that are finite, zeros in place of the others.
__device__ __forceinline__ hf8 finite_parts(hf8 x) {
  const hw8 b = __builtin_bit_cast(hw8, x);
  hw8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (b[i] & 0x7c00) == 0x7c00 ? uint16_t(0) : b[i];
  return __builtin_bit_cast(hf8, r);
}

// The tile's sums, scaled by the powers of two of rows and columns, into acc: block (i, j)
// of the wave, register r: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32.
template <class C>
__device__ __forceinline__ void half_tile(const HalfArgs& g, const HalfItem& at, char* smem,
                                          hv16 (&acc)[C::TM][C::TN]) {
  constexpr int TM = C::TM, TN = C::TN;
  const int first = at.split * g.steps_per_split;
  const int steps = min(g.steps - first, g.steps_per_split);
  int* flag = reinterpret_cast<int*>(smem + 2 * C::STAGE);
  if (threadIdx.x == 0) *flag = 0;  // set after the K loop's barriers

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int li = lane & 31, lh = lane >> 5;

  // A wave's loads of a step: `unit` kilobytes from its own first one on.
  const char* src[C::LOADS];
#pragma unroll
  for (int i = 0; i < C::LOADS; ++i) {
    const int unit = wave * C::LOADS + i, panel = unit / 8;
    src[i] = (panel < C::A_PANELS ? g.a + (int64_t(at.tile_m) * C::A_PANELS + panel) * g.a_stride
                                  : g.b + (int64_t(at.tile_n) * (C::BN / 64) + panel - C::A_PANELS) * g.b_stride) +
             int64_t(first) * kHalfStep + unit % 8 * 1024;
  }
  char* const to = smem + wave * (C::LOADS * 1024);
  uint32_t ahead = lane * 16;  // of the next step to load
  const auto issue = [&](int stage) {
#pragma unroll
    for (int i = 0; i < C::LOADS; ++i) panel_load(src[i] + ahead, to + stage * C::STAGE + i * 1024);
    ahead += kHalfStep;
  };

  // Fragments of 16 k: A's blocks lie in panels of two, a part a kilobyte on, an octet two.
  const int a_at = lh * 2048 + wm * TM * 32 / 64 * kHalfStep + wm * TM * 32 % 64 * 16 + li * 16;
  const int b_at = C::A_PANELS * kHalfStep + lh * 2048 + wn * TN * 32 / 64 * kHalfStep + wn * TN * 32 % 64 * 16 + li * 16;
  struct Fragments {
    hf8 ah[TM], am[TM], bh[TN], bm[TN];
  };
  const auto read = [&](Fragments& f, const char* stage, int half) {
    const char* a = stage + half * 4096 + a_at;
    const char* b = stage + half * 4096 + b_at;
#pragma unroll
    for (int i = 0; i < TM; ++i) f.ah[i] = *reinterpret_cast<const hf8*>(a + i / 2 * kHalfStep + i % 2 * 512);
#pragma unroll
    for (int j = 0; j < TN; ++j) f.bm[j] = *reinterpret_cast<const hf8*>(b + 1024 + j / 2 * kHalfStep + j % 2 * 512);
#pragma unroll
    for (int j = 0; j < TN; ++j) f.bh[j] = *reinterpret_cast<const hf8*>(b + j / 2 * kHalfStep + j % 2 * 512);
#pragma unroll
    for (int i = 0; i < TM; ++i) f.am[i] = *reinterpret_cast<const hf8*>(a + 1024 + i / 2 * kHalfStep + i % 2 * 512);
  };
  const auto product = [&](const hf8 (&x)[TM], const hf8 (&y)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mfma_f16(x[i], y[j], acc[i][j]);
  };
  const auto products = [&](const Fragments& f) {
    product(f.ah, f.bm);
    product(f.am, f.bh);
    product(f.ah, f.bh);
  };
  // A half's products with the next half's reads among them: 0x8 MFMA, 0x100 LDS read.
  const auto order = [&]() {
    constexpr int READS = 2 * (TM + TN), MFMAS = 3 * TM * TN, EACH = MFMAS * 2 / 3 / READS > 0 ? MFMAS * 2 / 3 / READS : 1;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MFMAS - READS * EACH > 0 ? MFMAS - READS * EACH : 1, 0);
  };

#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = hv16(0.0f);
  issue(0);
  if (steps > 1) issue(1);
  panels_settled();
  Fragments f0, f1;
  read(f0, smem, 0);
  const auto step = [&](auto stage_c, int t) {
    constexpr int stage = decltype(stage_c)::value;
    const char* s = smem + stage * C::STAGE;
    read(f1, s, 1);
    products(f0);
    order();
    panels_settled();
    if (t + 2 < steps) issue(stage);
    read(f0, smem + (stage ^ 1) * C::STAGE, 0);  // after the last step: of no use
    products(f1);
    order();
  };
  int t = 0;
  while (t + 1 < steps) {
    step(std::integral_constant<int, 0>{}, t++);
    step(std::integral_constant<int, 1>{}, t++);
  }
  if (t < steps) step(std::integral_constant<int, 0>{}, t);

  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        top = max(top, __builtin_bit_cast(uint32_t, float(acc[i][j][r])) & 0x7fffffffu);
  if (top >= 0x7f800000u) *flag = 1;
  __syncthreads();
  if (!*flag) return;

#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = hv16(0.0f);
  ahead = lane * 16;
#pragma unroll 1
  for (int u = 0; u < steps; ++u) {
    issue(0);
    panels_settled();
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      read(f0, smem, half);
      product(f0.ah, f0.bh);
#pragma unroll
      for (int i = 0; i < TM; ++i) f0.ah[i] = finite_parts(f0.ah[i]);
#pragma unroll
      for (int j = 0; j < TN; ++j) f0.bh[j] = finite_parts(f0.bh[j]);
      product(f0.ah, f0.bm);
      product(f0.am, f0.bh);
    }
    panels_settled();
  }
}

// Calls f(row, column, values) for every four consecutive columns of the wave's rows: values
// [j] are block column j's at columns column + 32 j of the tile (so a lane has the same place
// of every block), unscaled.  Through a wave-private LDS tile of 16 rows (LDS requests
// of one wave complete in order).
template <class C, class F>
__device__ __forceinline__ void half_epilogue(const HalfArgs& g, const HalfItem& at, char* smem, hv16 (&acc)[C::TM][C::TN], F&& f) {
  constexpr int TM = C::TM, TN = C::TN, PITCH = 32 * TN + 4;
  static_assert(2 * C::STAGE >= C::NW * 16 * PITCH * 4, "the wave tiles fit");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int li = lane & 31, lh = lane >> 5;
  float* w = reinterpret_cast<float*>(smem) + wave * (16 * PITCH);
  const int c4 = 4 * (lane & 7);
  hi4 eb[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) eb[j][e] = half_exponent(g.b_top[at.tile_n * C::BN + wn * TN * 32 + j * 32 + c4 + e]);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 8; ++r)
          w[((r / 4) * 8 + lh * 4 + r % 4) * PITCH + j * 32 + li] = acc[i][j][8 * half + r];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int rr = q * 8 + (lane >> 3);
        const int row = at.tile_m * C::BM + (wm * TM + i) * 32 + half * 16 + rr;
        const int ea = half_exponent(g.a_top[row]);
        hv4 v[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          v[j] = *reinterpret_cast<const hv4*>(w + rr * PITCH + j * 32 + c4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = ldexpf(v[j][e], -(ea + eb[j][e]));
        }
        f(row, c4, v);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Four values of a row from `col` on, as far as the row's n go.
__device__ __forceinline__ void store_four(float* row, int col, int n, hv4 v) {
  if (col + 4 <= n) {
    *reinterpret_cast<hv4_any*>(row + col) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < n) row[col + e] = v[e];
  }
}

using HalfBig = HalfCfg<2, 4, 4, 2, 2>;   // 256 x 256, 8 waves of 128 x 64
using HalfWide = HalfCfg<4, 2, 2, 2, 2>;  // 256 x 128, 8 waves of 64 x 64
using HalfMid = HalfCfg<4, 2, 1, 2, 4>;   // 128 x 128, 8 waves of 32 x 64, two a CU
using HalfFlat = HalfCfg<2, 2, 1, 2, 2>;  // 64 x 128, 4 waves of 32 x 64, three a CU

// kHalfTiles is what these types are.
template <class C>
constexpr bool half_is(int cfg) {
  return kHalfTiles[cfg].bm == C::BM && kHalfTiles[cfg].bn == C::BN && kHalfTiles[cfg].threads == C::THREADS;
}
static_assert(half_is<HalfBig>(0) && half_is<HalfWide>(1) && half_is<HalfMid>(2) && half_is<HalfFlat>(3));
static_assert(HalfBig::TN == 2 && HalfWide::TN == 2 && HalfMid::TN == 2 && HalfFlat::TN == 2);

// Calls f with the configuration's type.
template <class F>
int with_half_cfg(int cfg, F&& f) {
  switch (cfg) {
    case 0: return f(HalfBig{});
    case 1: return f(HalfWide{});
    case 2: return f(HalfMid{});
    default: return f(HalfFlat{});
  }
}

// The launch arguments of a product.
inline HalfArgs half_args(const HalfPanels& a, const HalfPanels& b, int m, int n, int k, int cfg, int splits) {
  const HalfTile& t = kHalfTiles[cfg];
  const int steps = (k + kHalfK - 1) / kHalfK, each = (steps + splits - 1) / splits;
  return {a.panels, b.panels, a.stride, b.stride, m, n, steps, a.tops, b.tops, (m + t.bm - 1) / t.bm,
          (n + t.bn - 1) / t.bn, (steps + each - 1) / each, each};
}
inline uint32_t half_items(const HalfArgs& g) { return uint32_t(int64_t(g.tiles_m) * g.tiles_n * g.splits); }

}  // namespace
}  // namespace lmp_hip
