// Operands of the products on the fp16 matrix cores (gemm_half.hpp): the largest finite
// magnitudes of a matrix's rows and columns, and the panels of its values in two fp16 parts.
//
// Both passes take the matrix from a source, which reads it or forms it from what it is
// made of:
//   int64_t rows; int cols;
//   void load(int64_t row, int unit, hv4 (&v)[2])   eight columns, zeros past the last
//   int column(int unit, int h)                     the first column of v[h]; eight units are 64 columns in some order
//   int place(int col)                              where that column's sum goes, or -1
//   float value(int64_t row, int col)               one value, for sums that are formed again
//
// Bound by memory: a pass reads 4 bytes a value and the second writes 4 for each set of panels.
// w of 1024 x 32768 and x of 4096 x 1024 take 42 us and, with both sets of panels, 79 (151 MB at
// 3.6 TB/s, 453 at 5.7); dz of 4096 x 32768, formed from the logits in both, 167 and 310.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.hpp"
#include "gemm_half.hpp"
#include "half_products.hpp"

namespace lmp_hip {
namespace {

constexpr int kPanelThreads = 256;

// Four values of a row from `col` on, zeros past its n.
__device__ __forceinline__ hv4 load_four(const float* row, int col, int n) {
  if (col + 4 <= n) return *reinterpret_cast<const hv4_any*>(row + col);
  hv4 v = hv4(0.0f);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < n) v[e] = row[col + e];
  return v;
}

// A matrix as it is; with `targets`, zeros for the rows whose target is negative: 0 x infinity
// would be NaN.
struct MatrixSource {
  int64_t rows;
  int cols;
  const float* x;
  int64_t ld;
  const int64_t* targets;
  __device__ __forceinline__ void load(int64_t row, int unit, hv4 (&v)[2]) const {
    v[0] = v[1] = hv4(0.0f);
    if (targets && targets[row] < 0) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) v[h] = load_four(x + row * ld, column(unit, h), cols);
  }
  __device__ __forceinline__ int column(int unit, int h) const { return 8 * unit + 4 * h; }
  __device__ __forceinline__ int place(int col) const { return col; }
  __device__ __forceinline__ float value(int64_t row, int col) const {
    return targets && targets[row] < 0 ? 0.0f : x[row * ld + col];
  }
};

// ------------------------------------------------------------ largest magnitudes

// As integers, magnitudes order as they do as floats.
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t m = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
  return m < 0x7f800000u ? m : 0u;
}

// The largest of the wave's, in lane 63: DPP within rows of 16 lanes, then the rows'
// broadcasts to the next.
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
#define LMP_STEP(ctrl, rows) x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), ctrl, rows, 0xF, false)))
  LMP_STEP(0xB1, 0xF);
  LMP_STEP(0x4E, 0xF);
  LMP_STEP(0x141, 0xF);
  LMP_STEP(0x140, 0xF);
  LMP_STEP(0x142, 0xA);
  LMP_STEP(0x143, 0xC);
#undef LMP_STEP
  return x;
}

// A workgroup's sixteen waves, 2^`wide` of them side by side, take 512 columns each, eight a
// lane, down a strip of rows.  Its rows' and columns' maxima meet in LDS, the workgroups' in
// atomics, none of which depends on an order; the strip's sums go to a row of their own.
constexpr int kTopsThreads = 1024, kTopsRows = 2048;  // a strip's rows at most
template <class S>
struct TopsJob {
  S s;
  uint32_t *row_top, *col_top;  // or null; zeros at first
  float* sums;                  // [strips, sums_ld], or null
  int64_t sums_ld;
  int each, wide, col_blocks;
  int64_t blocks;
  static constexpr int SMEM = (kTopsRows + 2048 + 16 * 512) * 4;
  __device__ __forceinline__ void run(int64_t block, char* smem) const {
    constexpr int kAhead = 4;
    uint32_t* rows = reinterpret_cast<uint32_t*>(smem);
    uint32_t* tops = rows + kTopsRows;
    float* parts = reinterpret_cast<float*>(tops + 2048);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int across = wave & ((1 << wide) - 1), down = wave >> wide, step = 16 >> wide, width = 512 << wide;
    const int64_t strip = block / col_blocks, begin = strip * each;
    const int count = int(min(int64_t(each), s.rows - begin)), col0 = int(block - strip * col_blocks) * width;
    const int unit = col0 / 8 + across * 64 + lane;
    if (row_top)
      for (int i = threadIdx.x; i < count; i += kTopsThreads) rows[i] = 0;
    for (int i = threadIdx.x; i < width; i += kTopsThreads) tops[i] = 0;
    __syncthreads();
    uint32_t top[2][4] = {};
    hv4 sum[2] = {hv4(0.0f), hv4(0.0f)};
    const bool inside = unit * 8 < (s.cols + 7) / 8 * 8;
    for (int row = down; row < count; row += step * kAhead) {
      hv4 v[kAhead][2];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        v[i][0] = v[i][1] = hv4(0.0f);
        if (row + step * i < count && inside) s.load(begin + row + step * i, unit, v[i]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        uint32_t most = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t m = finite_magnitude(v[i][h][e]);
            top[h][e] = max(top[h][e], m);
            most = max(most, m);
          }
          sum[h] = sum[h] + v[i][h];
        }
        if (row_top && row + step * i < count) {
          most = wave_most(most);
          if (lane == 63) atomicMax(rows + row + step * i, most);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = s.column(unit, h) + e - col0;
        if (col_top) atomicMax(tops + at, top[h][e]);
        if (sums) parts[down * width + at] = sum[h][e];
      }
    __syncthreads();
    if (row_top)
      for (int i = threadIdx.x; i < count; i += kTopsThreads) atomicMax(row_top + begin + i, rows[i]);
    for (int i = threadIdx.x; i < width && col0 + i < s.cols; i += kTopsThreads) {
      if (col_top) atomicMax(col_top + col0 + i, tops[i]);
      const int to = sums ? s.place(col0 + i) : -1;
      if (to >= 0) {
        float total = parts[i];
        for (int d = 1; d < step; ++d) total += parts[d * width + i];
        sums[strip * sums_ld + to] = total;
      }
    }
  }
};

// Strips enough to fill the chip: a column's maximum is an atomic a strip, so 256 of them at most unless
// the rows are more than 256 strips hold.
inline int tops_wide(int64_t cols) { return cols > 1024 ? 2 : cols > 512 ? 1 : 0; }
inline int64_t most_strips(Runtime* rt, int64_t rows, int64_t cols) {
  const int64_t width = 512 << tops_wide(cols);
  const int64_t want = std::clamp<int64_t>(int64_t(rt->cu_count) * 2 / ((cols + width - 1) / width), 1, 256);
  return std::max(want, (rows + kTopsRows - 1) / kTopsRows);
}
template <class S>
TopsJob<S> tops_job(Runtime* rt, const S& s, uint32_t* row_top, uint32_t* col_top, float* sums = nullptr) {
  const int wide = tops_wide(s.cols), width = 512 << wide, col_blocks = (s.cols + width - 1) / width;
  const int64_t most = most_strips(rt, s.rows, s.cols);
  const int each = int(std::max<int64_t>((s.rows + most - 1) / most, 64 >> wide));
  return {s, row_top, col_top, sums, s.cols, each, wide, col_blocks, (s.rows + each - 1) / each * col_blocks};
}

// ------------------------------------------------------------------------ panels

// Two values times s into the two parts, packed.  Of what is not finite the second part is NaN
// at worst: such sums are formed again.
__device__ __forceinline__ void half_pair(float x, float y, float s, uint32_t& h, uint32_t& m) {
  const hf2 a = __builtin_convertvector(hv2{x * s, y * s}, hf2);
  hf2 b;
  b.x = _Float16(__builtin_fmaf(x, s, -float(a.x)) * (1 / kHalfSecond));
  b.y = _Float16(__builtin_fmaf(y, s, -float(a.y)) * (1 / kHalfSecond));
  h = __builtin_bit_cast(uint32_t, a);
  m = __builtin_bit_cast(uint32_t, b);
}
__device__ __forceinline__ void put_octet(char* to, const float (&v)[8], float s, uint32_t& marks) {
  uint32_t h[4], m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) half_pair(v[2 * j], v[2 * j + 1], s, h[j], m[j]);
  *reinterpret_cast<hu4*>(to) = hu4{h[0], h[1], h[2], h[3]};
  *reinterpret_cast<hu4*>(to + 1024) = hu4{m[0], m[1], m[2], m[3]};
  bool infinite = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = fabsf(v[j] * s);
    infinite |= !(x < __builtin_huge_valf());
    marks += x < kHalfSmall && v[j] != 0.0f;
  }
  if (infinite) marks |= kHalfInfinite;
}
// Counts add, the mark of a row that is not finite stays.
__device__ __forceinline__ void put_marks(uint32_t* to, uint32_t marks) {
  if (marks & ~kHalfInfinite) atomicAdd(to, marks & ~kHalfInfinite);
  if (marks & kHalfInfinite) atomicOr(to, kHalfInfinite);
}

// Panels of the matrix (`r`: its rows are the panels', its columns K) and of its transpose
// (`c`), by tiles of 64 x 64 through LDS.
template <class S>
struct PackJob {
  S s;
  HalfPanels r, c;  // panels may be null
  int64_t tiles_c, blocks;
  static constexpr int PITCH = 68, SMEM = (64 * PITCH + 128) * 4;
  __device__ __forceinline__ void run(int64_t block, char* smem) const {
    float* t = reinterpret_cast<float*>(smem);
    uint32_t* found = reinterpret_cast<uint32_t*>(t + 64 * PITCH);  // marks of the tile's rows, then of its columns
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tr = block / tiles_c, tc = block - tr * tiles_c;
    const int unit = int(tc) * 8 + threadIdx.x % 8;
    if (threadIdx.x < 128) found[threadIdx.x] = 0;
    hv4 v[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = tr * 64 + threadIdx.x / 8 + 32 * i;
      v[i][0] = v[i][1] = hv4(0.0f);
      if (row < s.rows && unit * 8 < s.cols) s.load(row, unit, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<hv4*>(t + (threadIdx.x / 8 + 32 * i) * PITCH + s.column(unit, h) - int(tc) * 64) = v[i][h];
    __syncthreads();
    float o[8];
    if (r.panels) {
      const float power = power_of(half_exponent(r.tops[tr * 64 + lane]));
      uint32_t marks = 0;
#pragma unroll
      for (int oct = wave; oct < 8; oct += 4) {
        if (tc * 64 + oct * 8 >= (int64_t(s.cols) + 31) / 32 * 32) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = t[lane * PITCH + oct * 8 + j];
        put_octet(r.panels + tr * r.stride + (tc * 8 + oct) * 2048 + lane * 16, o, power, marks);
      }
      put_marks(found + lane, marks);
    }
    if (c.panels) {
      const float power = power_of(half_exponent(c.tops[tc * 64 + lane]));
      uint32_t marks = 0;
#pragma unroll
      for (int oct = wave; oct < 8; oct += 4) {
        if (tr * 64 + oct * 8 >= (s.rows + 31) / 32 * 32) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = t[(oct * 8 + j) * PITCH + lane];
        put_octet(c.panels + tc * c.stride + (tr * 8 + oct) * 2048 + lane * 16, o, power, marks);
      }
      put_marks(found + 64 + lane, marks);
    }
    __syncthreads();
    if (r.panels && threadIdx.x < 64) put_marks(r.marks + tr * 64 + lane, found[lane]);
    if (c.panels && threadIdx.x >= 64 && threadIdx.x < 128) put_marks(c.marks + tc * 64 + lane, found[64 + lane]);
  }
};
// Whole groups of four panels, the rows past the matrix zeros.
template <class S>
PackJob<S> pack_job(const S& s, const HalfPanels& r, const HalfPanels& c) {
  const int64_t tiles_r = r.panels ? (s.rows + 255) / 256 * 4 : (s.rows + 63) / 64;
  const int64_t tiles_c = c.panels ? (int64_t(s.cols) + 255) / 256 * 4 : (int64_t(s.cols) + 63) / 64;
  return {s, r, c, tiles_c, tiles_r * tiles_c};
}

// One launch for jobs of one kind, one after another in the grid.
template <int NT, int SMEM, class... Jobs>
__global__ __launch_bounds__(NT) void panel_jobs(Jobs... jobs) {
  __shared__ __attribute__((aligned(16))) char smem[SMEM];
  int64_t block = blockIdx.x;
  bool done = false;
  const auto turn = [&](const auto& job) {
    if (!done && block < job.blocks) {
      job.run(block, smem);
      done = true;
    }
    block -= job.blocks;
  };
  (turn(jobs), ...);
}
template <int NT, int SMEM, class... Jobs>
int launch_panel_jobs(Runtime* rt, const Jobs&... jobs) {
  const int64_t blocks = (jobs.blocks + ...);
  if (blocks == 0) return LMP_OK;
  if (uint64_t(blocks) > kMaxGridThreads / NT)
    return fail(LMP_ERR_UNSUPPORTED, "split products: more tiles than a grid holds");
  panel_jobs<NT, SMEM><<<dim3(uint32_t(blocks)), dim3(NT), 0, rt->stream>>>(jobs...);
  LMP_LAUNCH_CHECK("panel_jobs");
  return LMP_OK;
}
template <class... S>
int run_panel_jobs(Runtime* rt, const TopsJob<S>&... jobs) {
  return launch_panel_jobs<kTopsThreads, TopsJob<MatrixSource>::SMEM>(rt, jobs...);
}
template <class... S>
int run_panel_jobs(Runtime* rt, const PackJob<S>&... jobs) {
  return launch_panel_jobs<kPanelThreads, PackJob<MatrixSource>::SMEM>(rt, jobs...);
}

}  // namespace
}  // namespace lmp_hip
