// Passes over a matrix in strips of rows: a workgroup takes 1024 columns, four a lane, down
// some rows, and keeps its columns' maxima (and sums) in registers.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "gemm_half.hpp"

namespace lmp_hip {
namespace {

constexpr int kStripThreads = 256, kStripCols = 4 * kStripThreads;

struct StripShape {
  int64_t rows;
  int cols;
  int each;    // rows of a strip
  int strips;  // strips that hold the rows
};

// Rows per strip: enough strips to fill the chip, of 8 to 64 rows: what a strip leaves (a
// maximum per column) is a small part of what it reads.
inline StripShape strips_of(Runtime* rt, size_t rows, size_t cols) {
  const int64_t blocks = (int64_t(cols) + kStripCols - 1) / kStripCols;
  const int64_t want = std::max<int64_t>(1, int64_t(rt->cu_count) * 4 / blocks);
  int64_t each = std::clamp<int64_t>((int64_t(rows) + want - 1) / want, 8, 64);
  each = std::max<int64_t>(each, (int64_t(rows) + 65534) / 65535);
  return {int64_t(rows), int(cols), int(each), int((int64_t(rows) + each - 1) / each)};
}
inline dim3 strip_grid(const StripShape& s) {
  return dim3(uint32_t((int64_t(s.cols) + kStripCols - 1) / kStripCols), uint32_t(s.strips));
}

__device__ __forceinline__ int strip_col() { return int(blockIdx.x) * kStripCols + int(threadIdx.x) * 4; }
__device__ __forceinline__ int64_t strip_begin(const StripShape& s) { return int64_t(blockIdx.y) * s.each; }
__device__ __forceinline__ int64_t strip_end(const StripShape& s) {
  return min(s.rows, (int64_t(blockIdx.y) + 1) * s.each);
}

// Four values of a row from `col` on, zeros past its n.
__device__ __forceinline__ hv4 load_four(const float* row, int col, int n) {
  if (col + 4 <= n) return *reinterpret_cast<const hv4_any*>(row + col);
  hv4 v = hv4(0.0f);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < n) v[e] = row[col + e];
  return v;
}

// As integers, magnitudes order as they do as floats, and NaN is above all.
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

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

// Maxima do not depend on the order they meet in.
__device__ __forceinline__ void raise_row(uint32_t* row_top, uint32_t most) {
  most = wave_most(most);
  if ((threadIdx.x & 63) == 63) atomicMax(row_top, most);
}
__device__ __forceinline__ void raise_cols(uint32_t* col_top, int col, int n, const uint32_t (&top)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < n) atomicMax(col_top + col + e, top[e]);
}

}  // namespace
}  // namespace lmp_hip
