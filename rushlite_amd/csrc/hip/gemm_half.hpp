// fp32 products on the fp16 matrix cores, each operand in two fp16 parts.
//
// Why.  A value scaled by a power of two is x = h + m / 64 + r with h = fp16(x), m =
// fp16(64 (x - h)) and |r| <= 2^-22 |x|, so
//   a b = ah bh + (ah / 64) bm + am (bh / 64) + (what both m make and what the r leave out: 3 x 2^-22 at most)
// is three fp16 MFMAs with fp32 accumulation, half of what three bf16 parts cost
// (gemm_bf3.hpp), with a product's error near that of rounding its operands: a sum's
// error is its own roundings'.  The h / 64 are formed in registers.
//
// Range.  Each row of A and each column of B has a power of two that takes its largest
// finite magnitude to [2^14, 2^15).  Values down to 2^-8, 2^-23 of the largest, keep both
// parts whole.  Of a smaller one r, and what rounding h / 64 to fp16's smallest step costs its
// product with the other operand's m, are 2^-31 and 2^-30 + 2^-36 of the other value at most:
// 2^-19 of the product down to 2^-11.  The na and nb values of a sum's row and column that are
// smaller still (kHalfSmall) put it off by (na + nb) 2^15 (2^-31 + 2^-30 + 2^-36) < (na + nb) 2^-14.  So
// a sum of k products that is 2^8 (na + nb) / k or more errs by (4 k + 44) 2^-24 of its products'
// magnitudes at most, and by far less where the roundings go both ways; one that is less,
// where large values meet zeros, or that is not finite, is formed again in fp32 from the
// operands themselves: up to kHalfList of a tile one by one, and all of the tile by fp32 MFMAs
// where there are more.  The panels' kernel counts the small values.  One tile of 256 x 256 over
// 1024 normal values in 35 has any and looks at its sums; the others know before the K loop that
// they need not.  The second part's own power of two, which makes the small values 32 times
// fewer, takes 1% of 8192 x 32768 over 1024 and 2% of 12608 x 4096 over 768.
//
// Operands are split once, by kernels of their own (half_panels.hpp), into panels of 64
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
// Bound by the chip's power: random operands run at 385 TFLOP/s (8192 x 32768 over 1024,
// 1.16 PFLOP/s of fp16, the clock at 1.7 of 2.4 GHz) to 410 (1024 x 32768 over 4096), zeros ran
// at 654 before sums were looked after, and the library's fp16 product of the first at 1.18 PFLOP/s.  Splitting the operands in
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

// Kept out of the templates: a target builtin inside a kernel template keeps the host
// pass from emitting the kernel's launch stub.
__device__ __forceinline__ hv16 mfma_f16(hf8 a, hf8 b, hv16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ hv16 mfma_whole(float a, float b, hv16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
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

constexpr float kHalfSecond = 1.0f / 64;  // what m is a multiple of
// Values, scaled, below kHalfSmall are counted.  Sums are formed again below kHalfLeast times the share of
// such values, one by one up to kHalfList of a tile.
constexpr float kHalfSmall = 1.0f / 2048, kHalfLeast = 256.0f;
constexpr uint32_t kHalfInfinite = 1u << 31;  // the mark of a row that is not finite
constexpr int kHalfList = 32;
// What a tile has to form again, in LDS: whether any sum may be, whether any is, how many are, where
// (row << 16 | column in the tile), and the values, scaled as the others are.
struct HalfDoubt {
  int any, again, count;
  uint32_t at[kHalfList];
  float value[kHalfList];
  float shares[8];
};

template <int WM_, int WN_, int TM_, int TN_, int MINB_>
struct HalfCfg {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, MINB = MINB_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int A_PANELS = BM / 64, PANELS = (BM + BN) / 64;
  static constexpr int STAGE = PANELS * kHalfStep;
  static constexpr int LOADS = PANELS * 8 / NW;  // of a wave, a step
  // The stages, what is formed again, and what rows' and columns' sums may not be below.
  static constexpr int SMEM = 2 * STAGE + int(sizeof(HalfDoubt)) + (BM + BN) * 4;
  static_assert((TM == 1 || TM % 2 == 0) && TN % 2 == 0, "a wave's blocks are whole panels, or half of one");
  static_assert(2 * STAGE >= NW * 16 * (32 * TN + 4) * 4, "the epilogue's wave tiles fit");
  static_assert(BM + BN <= THREADS, "a lane each loads their limits");
  static_assert(BM % 64 == 0 && BN % 64 == 0 && LOADS * NW == PANELS * 8, "whole panels, split evenly");
};

// A product op(A) [m, k] op(B) [k, n] of panels.  `a_top` and `b_top`: the bits of the
// largest finite magnitude of each row of op(A) and column of op(B), rounded up to 256 of them;
// `a_marks` and `b_marks`: their marks (HalfPanels).
struct HalfArgs {
  const char *a, *b;
  int64_t a_stride, b_stride;  // bytes from panel to panel
  int m, n, k;
  int steps;  // 32-wide k steps
  const uint32_t *a_top, *b_top;
  const uint32_t *a_marks, *b_marks;
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

// An operand as the products' slow path reads it: rows of its source along K (RowsOf), or columns
// (ColsOf).  A source is as half_panels.hpp's passes take it, and has besides
//   float value(int64_t row, int col)   one value
// stage() puts 64 of K from k0 on, of N rows of the operand from row0 on, into t[k][N], zeros
// past the matrix; row0 and k0 are multiples of 64.
template <class S>
struct RowsOf {
  static constexpr bool ROWS = true;
  S s;
  __device__ __forceinline__ int64_t extent() const { return s.cols; }
  __device__ __forceinline__ float value(int64_t row, int64_t k) const { return s.value(row, int(k)); }
  template <int N, int NT>
  __device__ __forceinline__ void stage(float* t, int64_t row0, int64_t k0) const {
#pragma unroll 1
    for (int i = threadIdx.x; i < N * 8; i += NT) {
      const int r = i % N, unit = int(k0 / 8) + i / N;
      hv4 v[2] = {hv4(0.0f), hv4(0.0f)};
      if (row0 + r < s.rows && unit * 8 < s.cols) s.load(row0 + r, unit, v);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[(s.column(unit, h) + e - int(k0)) * N + r] = v[h][e];
    }
  }
};
template <class S>
struct ColsOf {
  static constexpr bool ROWS = false;
  S s;
  __device__ __forceinline__ int64_t extent() const { return s.rows; }
  __device__ __forceinline__ float value(int64_t row, int64_t k) const { return s.value(k, int(row)); }
  template <int N, int NT>
  __device__ __forceinline__ void stage(float* t, int64_t row0, int64_t k0) const {
#pragma unroll 1
    for (int i = threadIdx.x; i < 64 * (N / 8); i += NT) {
      const int k = i / (N / 8), unit = int(row0 / 8) + i % (N / 8);
      hv4 v[2] = {hv4(0.0f), hv4(0.0f)};
      if (k0 + k < s.rows && unit * 8 < s.cols) s.load(k0 + k, unit, v);
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<hv4*>(t + k * N + s.column(unit, h) - int(row0)) = v[h];
    }
  }
};

// Sum (row, col) in fp32 by the whole workgroup.
template <int NT, class A, class B>
__device__ __forceinline__ float whole_sum(const A& a, const B& b, int64_t row, int64_t col, float* shares) {
  float sum = 0.0f;
  if constexpr (A::ROWS && B::ROWS) {
#pragma unroll 2
    for (int unit = threadIdx.x; unit * 8 < a.s.cols; unit += NT) {
      hv4 x[2], y[2];
      a.s.load(row, unit, x);
      b.s.load(col, unit, y);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = __builtin_fmaf(x[h][e], y[h][e], sum);
    }
  } else {
#pragma unroll 4
    for (int64_t k = threadIdx.x; k < a.extent(); k += NT) sum = __builtin_fmaf(a.value(row, k), b.value(col, k), sum);
  }
  for (int off = 1; off < 64; off *= 2) sum += __shfl_xor(sum, off);
  if ((threadIdx.x & 63) == 0) shares[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = shares[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) sum += shares[w];
  __syncthreads();
  return sum;
}

// The sums of the waves' blocks (i, j) of C's tile at (row0, col0) in fp32, by way of (BM + BN) 256
// bytes of LDS.
template <class C, class A, class B>
__device__ __forceinline__ void whole_blocks(const A& a, const B& b, int64_t row0, int64_t col0, int i, char* smem,
                                             hv16 (&acc)[C::TN]) {
  float *ta = reinterpret_cast<float*>(smem), *tb = ta + 64 * C::BM;
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float* ra = ta + lh * C::BM + (wave % (C::WM * C::WN) / C::WN * C::TM + i) * 32 + li;
  const float* rb = tb + lh * C::BN + wave % C::WN * C::TN * 32 + li;
#pragma unroll
  for (int j = 0; j < C::TN; ++j) acc[j] = hv16(0.0f);
#pragma unroll 1
  for (int64_t k0 = 0; k0 < a.extent(); k0 += 64) {
    a.template stage<C::BM, C::THREADS>(ta, row0, k0);
    b.template stage<C::BN, C::THREADS>(tb, col0, k0);
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < 64; k += 2)
#pragma unroll
      for (int j = 0; j < C::TN; ++j) acc[j] = mfma_whole(ra[k * C::BM], rb[k * C::BN + 32 * j], acc[j]);
    __syncthreads();
  }
}

// A row's share of what a scaled sum may not be below, from its largest magnitude and its word of
// marks.  Rows of zeros, and those past the matrix, make sums of zero; all of a row that is not
// finite are formed again.
__device__ __forceinline__ float half_limit(uint32_t top, uint32_t marks, float per_k) {
  if (marks & kHalfInfinite) return 1e38f;
  return top ? float(marks) * per_k : -1e37f;
}

// Whether a sum is to be formed again, by its row's and its column's limit.
__device__ __forceinline__ bool half_doubtful(float sum, float row, float col) {
  const float above = fabsf(sum) - col;
  return !(above >= row && above < __builtin_huge_valf());
}

// Lists what a lane found: bit b of `found` is at + b / 4 four + b % 4 one, in the list's terms.
__device__ __forceinline__ void note_doubts(HalfDoubt* d, uint32_t found, uint32_t at, uint32_t four, uint32_t one) {
  if (!found) return;
  int i = atomicAdd(&d->count, __popc(found));
  for (; found && i < kHalfList; ++i, found &= found - 1) {
    const uint32_t b = __ffs(int(found)) - 1;
    d->at[i] = at + b / 4 * four + b % 4 * one;
  }
}

template <class C>
__device__ __forceinline__ HalfDoubt* half_doubt(char* smem) {
  return reinterpret_cast<HalfDoubt*>(smem + 2 * C::STAGE);
}
// The tile's limits: its rows', then its columns'.
template <class C>
__device__ __forceinline__ float* half_limits(char* smem) {
  return reinterpret_cast<float*>(smem + 2 * C::STAGE + sizeof(HalfDoubt));
}

// The tile's sums, scaled by the powers of two of rows and columns, into acc: block (i, j)
// of the wave, register r: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32.  With LIMITS
// also what its rows' and columns' sums may not be below, into LDS.
template <class C, bool LIMITS>
__device__ __forceinline__ void half_sums(const HalfArgs& g, const HalfItem& at, char* smem,
                                          hv16 (&acc)[C::TM][C::TN]) {
  constexpr int TM = C::TM, TN = C::TN;
  const int first = at.split * g.steps_per_split;
  const int steps = min(g.steps - first, g.steps_per_split);
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
    for (int j = 0; j < TN; ++j) f.bh[j] = *reinterpret_cast<const hf8*>(b + j / 2 * kHalfStep + j % 2 * 512);
#pragma unroll
    for (int j = 0; j < TN; ++j) f.bm[j] = *reinterpret_cast<const hf8*>(b + 1024 + j / 2 * kHalfStep + j % 2 * 512);
#pragma unroll
    for (int i = 0; i < TM; ++i) f.am[i] = *reinterpret_cast<const hf8*>(a + 1024 + i / 2 * kHalfStep + i % 2 * 512);
  };
  const auto product = [&](const hf8 (&x)[TM], const hf8 (&y)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mfma_f16(x[i], y[j], acc[i][j]);
  };
  const auto products = [&](Fragments& f) {
    product(f.ah, f.bh);
#pragma unroll
    for (int i = 0; i < TM; ++i) f.ah[i] = f.ah[i] * _Float16(kHalfSecond);
#pragma unroll
    for (int j = 0; j < TN; ++j) f.bh[j] = f.bh[j] * _Float16(kHalfSecond);
    product(f.ah, f.bm);
    product(f.am, f.bh);
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
  const int mine = threadIdx.x;
  const bool of_a = mine < C::BM, limited = LIMITS && mine < C::BM + C::BN;
  uint32_t top = 0, marks = 0;
  if (limited) {
    const int64_t row = of_a ? int64_t(at.tile_m) * C::BM + mine : int64_t(at.tile_n) * C::BN + mine - C::BM;
    top = (of_a ? g.a_top : g.b_top)[row];
    marks = (of_a ? g.a_marks : g.b_marks)[row];
  }
  issue(0);
  if (steps > 1) issue(1);
  if (limited) {
    const float limit = half_limit(top, marks, kHalfLeast / float(g.k));
    half_limits<C>(smem)[mine] = limit;
    if (limit > 0.0f) half_doubt<C>(smem)->any = 1;
    if (marks & kHalfInfinite) half_doubt<C>(smem)->again = 1;
  }
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
}

// The same, and how many of them are too small or not finite: up to kHalfList are formed again and
// listed.
template <class C, class A, class B>
__device__ __forceinline__ int half_tile(const HalfArgs& g, const HalfItem& at, char* smem, hv16 (&acc)[C::TM][C::TN],
                                         const A& a, const B& b) {
  constexpr int TM = C::TM, TN = C::TN;
  HalfDoubt* doubt = half_doubt<C>(smem);
  if (threadIdx.x == 0) doubt->any = doubt->again = doubt->count = 0;
  __syncthreads();
  half_sums<C, true>(g, at, smem, acc);
  if (!doubt->any) {  // as the K loop's first barrier left it
    __syncthreads();  // the stages have been read
    return 0;
  }

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row_at = wave / C::WN * TM * 32 + 4 * (lane >> 5), col_at = wave % C::WN * TN * 32 + (lane & 31);
  const float *row_limits = half_limits<C>(smem) + row_at, *col_limits = half_limits<C>(smem) + C::BM + col_at;
  float col_limit[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) col_limit[j] = col_limits[32 * j];
  bool again = false;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const hv4 limits = *reinterpret_cast<const hv4*>(row_limits + 32 * i + 8 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float above = fabsf(acc[i][0][4 * q + e]) - col_limit[0];
#pragma unroll
        for (int j = 1; j < TN; ++j) above = fminf(above, fabsf(acc[i][j][4 * q + e]) - col_limit[j]);
        again |= above < limits[e];
      }
      __builtin_amdgcn_sched_barrier(0);  // the sums leave no registers for more limits at a time
    }
  if (again) doubt->again = 1;
  __syncthreads();
  if (!doubt->again) return 0;

  // Seldom reached, so what matters of this code is that it stays out of the way.
  const int64_t row0 = int64_t(at.tile_m) * C::BM, col0 = int64_t(at.tile_n) * C::BN;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int row = row_at + 32 * i, col = col_at + 32 * j;
      uint32_t found = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const hv4 limits = *reinterpret_cast<const hv4*>(row_limits + 32 * i + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (half_doubtful(acc[i][j][4 * q + e], limits[e], col_limits[32 * j])) found |= 1u << (4 * q + e);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (col0 + col >= g.n) found = 0;
#pragma unroll 1
      for (uint32_t f = found; f; f &= f - 1) {
        const int bit = __ffs(int(f)) - 1;
        if (row0 + row + bit / 4 * 8 + bit % 4 >= g.m) found &= ~(1u << bit);
      }
      note_doubts(doubt, found, uint32_t(row) << 16 | uint32_t(col), 8 << 16, 1 << 16);
    }
  __syncthreads();
  const int count = doubt->count;
  if (count > kHalfList) return count;
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    const uint32_t where = doubt->at[i];
    const int64_t row = row0 + (where >> 16), col = col0 + (where & 0xffff);
    const float sum = whole_sum<C::THREADS>(a, b, row, col, doubt->shares);
    if (threadIdx.x == 0) doubt->value[i] = ldexpf(sum, half_exponent(g.a_top[row]) + half_exponent(g.b_top[col]));
  }
  __syncthreads();
  return count;
}

// Calls f(row, column, values) for every four consecutive columns of rows of the wave's blocks
// (i, j): values [j] are block column j's at columns column + 32 j of the tile (so a lane
// has the same place of every block).  Of scaled sums the powers of two are taken out and the
// first `patches` of the list put in their places.  Through a wave-private LDS tile of 16
// rows (LDS requests of one wave complete in order).
template <class C, bool SCALED, class F>
__device__ __forceinline__ void half_out(const HalfArgs& g, const HalfItem& at, char* smem, const hv16 (&acc)[C::TN], int i,
                                         const hi4 (&eb)[C::TN], int patches, F&& f) {
  constexpr int TM = C::TM, TN = C::TN, PITCH = 32 * TN + 4;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int li = lane & 31, lh = lane >> 5, c4 = 4 * (lane & 7);
  float* w = reinterpret_cast<float*>(smem) + wave * (16 * PITCH);
  const HalfDoubt* doubt = half_doubt<C>(smem);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 8; ++r) w[((r / 4) * 8 + lh * 4 + r % 4) * PITCH + j * 32 + li] = acc[j][8 * half + r];
    if (SCALED && lane < patches) {
      const int r = int(doubt->at[lane] >> 16) - (wm * TM + i) * 32 - half * 16, c = int(doubt->at[lane] & 0xffff) - wn * TN * 32;
      if (r >= 0 && r < 16 && c >= 0 && c < TN * 32) w[r * PITCH + c] = doubt->value[lane];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1  // the code that a tile passes through once has to leave the K loop's in the instruction cache
    for (int q = 0; q < 2; ++q) {
      const int rr = q * 8 + (lane >> 3);
      const int row = at.tile_m * C::BM + (wm * TM + i) * 32 + half * 16 + rr;
      const int ea = SCALED ? half_exponent(g.a_top[row]) : 0;
      hv4 v[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        v[j] = *reinterpret_cast<const hv4*>(w + rr * PITCH + j * 32 + c4);
        if constexpr (SCALED)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = ldexpf(v[j][e], -(ea + eb[j][e]));
      }
      f(row, c4, v);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// A tile's product, f called with its sums as half_out does.
template <class C, class A, class B, class F>
__device__ __forceinline__ void half_product(const HalfArgs& g, const HalfItem& at, char* smem, const A& a, const B& b, F&& f) {
  static_assert(2 * C::STAGE >= C::NW * 16 * (32 * C::TN + 4) * 4, "the wave tiles fit");
  hi4 eb[C::TN];
  {
    hv16 acc[C::TM][C::TN];
    const int again = half_tile<C>(g, at, smem, acc, a, b);
    if (again <= kHalfList) {
      const int col = at.tile_n * C::BN + (threadIdx.x >> 6) % C::WN * C::TN * 32 + 4 * (threadIdx.x & 7);
#pragma unroll
      for (int j = 0; j < C::TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) eb[j][e] = half_exponent(g.b_top[col + j * 32 + e]);
#pragma unroll
      for (int i = 0; i < C::TM; ++i) half_out<C, true>(g, at, smem, acc[i], i, eb, again, f);
      return;
    }
  }
#pragma unroll 1
  for (int i = 0; i < C::TM; ++i) {
    hv16 acc[C::TN];
    whole_blocks<C>(a, b, int64_t(at.tile_m) * C::BM, int64_t(at.tile_n) * C::BN, i, smem, acc);
    half_out<C, false>(g, at, smem, acc, i, eb, 0, f);
    __syncthreads();
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
using HalfMid = HalfCfg<4, 2, 1, 2, 4>;   // 128 x 128, 8 waves of 32 x 64, two a CU
using HalfFlat = HalfCfg<2, 2, 1, 2, 2>;  // 64 x 128, 4 waves of 32 x 64, three a CU

// kHalfTiles is what these types are.
template <class C>
constexpr bool half_is(int cfg) {
  return kHalfTiles[cfg].bm == C::BM && kHalfTiles[cfg].bn == C::BN && kHalfTiles[cfg].threads == C::THREADS;
}
static_assert(half_is<HalfBig>(0) && half_is<HalfMid>(1) && half_is<HalfFlat>(2));
static_assert(HalfBig::TN == 2 && HalfMid::TN == 2 && HalfFlat::TN == 2);

// Calls f with the configuration's type.
template <class F>
int with_half_cfg(int cfg, F&& f) {
  switch (cfg) {
    case 0: return f(HalfBig{});
    case 1: return f(HalfMid{});
    default: return f(HalfFlat{});
  }
}

// The launch arguments of a product.
inline HalfArgs half_args(const HalfPanels& a, const HalfPanels& b, int m, int n, int k, int cfg, int splits) {
  const HalfTile& t = kHalfTiles[cfg];
  const int steps = (k + kHalfK - 1) / kHalfK, each = (steps + splits - 1) / splits;
  return {a.panels, b.panels, a.stride, b.stride, m, n, k, steps, a.tops, b.tops, a.marks, b.marks,
          (m + t.bm - 1) / t.bm, (n + t.bn - 1) / t.bn, (steps + each - 1) / each, each};
}
inline uint32_t half_items(const HalfArgs& g) { return uint32_t(int64_t(g.tiles_m) * g.tiles_n * g.splits); }

}  // namespace
}  // namespace lmp_hip
