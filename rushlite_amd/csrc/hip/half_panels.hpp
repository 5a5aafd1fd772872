// Operands of the products on the fp16 matrix cores (gemm_half.hpp): the largest finite
// magnitudes of a matrix's rows and columns, and the panels of its values in two fp16 parts.
//
// Both passes take the matrix from a source, which reads it or forms it from what it is
// made of:
//   int64_t rows; int cols;
//   hv4 load(int64_t row, int col)   columns col to col + 3 (col a multiple of 4), zeros past the last
//   int place(int col)               where that column's sum goes, or -1
//
// Bound by memory: a pass reads 4 bytes a value and the second writes 4 for each set of panels.
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
  __device__ __forceinline__ hv4 load(int64_t row, int col) const {
    if (targets && targets[row] < 0) return hv4(0.0f);
    return load_four(x + row * ld, col, cols);
  }
  __device__ __forceinline__ int place(int col) const { return col; }
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

// A workgroup takes 256 columns, four a lane, down a strip of rows, each wave every fourth
// row.  Maxima meet in atomics, which do not depend on their order; sums of the strip's
// columns go to a row of their own.
template <class S>
struct TopsJob {
  S s;
  uint32_t *row_top, *col_top;  // or null; zeros at first
  float* sums;                  // [strips, sums_ld], or null
  int64_t sums_ld;
  int each, col_blocks;
  int64_t blocks;
  __device__ __forceinline__ void run(int64_t block, char* smem) const {
    constexpr int kAhead = 8;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t strip = block / col_blocks;
    const int col = int(block - strip * col_blocks) * 256 + lane * 4;
    const int64_t begin = strip * each, end = min(s.rows, begin + each);
    uint32_t top[4] = {0, 0, 0, 0};
    hv4 sum = hv4(0.0f);
    for (int64_t row = begin + wave; row < end; row += 4 * kAhead) {
      hv4 v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        v[i] = hv4(0.0f);
        if (row + 4 * i < end && col < s.cols) v[i] = s.load(row + 4 * i, col);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t m = finite_magnitude(v[i][e]);
          top[e] = max(top[e], m);
          most = max(most, m);
        }
        sum = sum + v[i];
        if (row_top && row + 4 * i < end) {
          most = wave_most(most);
          if (lane == 63) atomicMax(row_top + row + 4 * i, most);
        }
      }
    }
    uint32_t* tops = reinterpret_cast<uint32_t*>(smem);
    float* parts = reinterpret_cast<float*>(smem) + 1024;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      tops[wave * 256 + lane * 4 + e] = top[e];
      if (sums) parts[wave * 256 + lane * 4 + e] = sum[e];
    }
    __syncthreads();
    const int i = threadIdx.x, mine = col - lane * 4 + i;
    if (mine < s.cols) {
      if (col_top) atomicMax(col_top + mine, max(max(tops[i], tops[256 + i]), max(tops[512 + i], tops[768 + i])));
      const int to = sums ? s.place(mine) : -1;
      if (to >= 0) sums[strip * sums_ld + to] = (parts[i] + parts[256 + i]) + (parts[512 + i] + parts[768 + i]);
    }
  }
};

// Strips enough to fill the chip, of 16 rows at least, and 128 of them at most: a column's
// maximum is an atomic a strip.
inline int64_t most_strips(Runtime* rt, int64_t rows, int64_t cols) {
  const int64_t want = std::clamp<int64_t>(int64_t(rt->cu_count) * 4 / ((cols + 255) / 256), 1, 128);
  return std::min(want, (rows + 15) / 16);
}
template <class S>
TopsJob<S> tops_job(Runtime* rt, const S& s, uint32_t* row_top, uint32_t* col_top, float* sums = nullptr) {
  const int col_blocks = (s.cols + 255) / 256;
  const int64_t most = std::max<int64_t>(most_strips(rt, s.rows, s.cols), 1);
  const int each = int(std::max<int64_t>((s.rows + most - 1) / most, 16));
  return {s, row_top, col_top, sums, s.cols, each, col_blocks, (s.rows + each - 1) / each * col_blocks};
}

// ------------------------------------------------------------------------ panels

// Two values times s into the two parts, packed; an infinity has no second part.
__device__ __forceinline__ void half_pair(float x, float y, float s, uint32_t& h, uint32_t& m) {
  const hf2 a = __builtin_convertvector(hv2{x * s, y * s}, hf2);
  hf2 b;
  b.x = _Float16(__builtin_fmaf(x, s, -float(a.x)));
  b.y = _Float16(__builtin_fmaf(y, s, -float(a.y)));
  h = __builtin_bit_cast(uint32_t, a);
  m = __builtin_bit_cast(uint32_t, b);
  if ((h & 0x7fff) == 0x7c00) m &= 0xffff0000u;
  if ((h & 0x7fff0000) == 0x7c000000) m &= 0xffffu;
}
__device__ __forceinline__ void put_octet(char* to, const float (&v)[8], float s) {
  uint32_t h[4], m[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) half_pair(v[2 * j], v[2 * j + 1], s, h[j], m[j]);
  *reinterpret_cast<hu4*>(to) = hu4{h[0], h[1], h[2], h[3]};
  *reinterpret_cast<hu4*>(to + 1024) = hu4{m[0], m[1], m[2], m[3]};
}

// Panels of the matrix (`r`: its rows are the panels', its columns K) and of its transpose
// (`c`), by tiles of 64 x 64 through LDS.
template <class S>
struct PackJob {
  S s;
  HalfPanels r, c;  // panels may be null
  int64_t tiles_c, blocks;
  static constexpr int PITCH = 68;
  __device__ __forceinline__ void run(int64_t block, char* smem) const {
    float* t = reinterpret_cast<float*>(smem);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tr = block / tiles_c, tc = block - tr * tiles_c;
    hv4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = tr * 64 + threadIdx.x / 16 + 16 * i, col = tc * 64 + threadIdx.x % 16 * 4;
      v[i] = hv4(0.0f);
      if (row < s.rows && col < s.cols) v[i] = s.load(row, int(col));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<hv4*>(t + (threadIdx.x / 16 + 16 * i) * PITCH + threadIdx.x % 16 * 4) = v[i];
    __syncthreads();
    float o[8];
    if (r.panels) {
      const float power = power_of(half_exponent(r.tops[tr * 64 + lane]));
#pragma unroll
      for (int oct = wave; oct < 8; oct += 4) {
        if (tc * 64 + oct * 8 >= (int64_t(s.cols) + 31) / 32 * 32) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = t[lane * PITCH + oct * 8 + j];
        put_octet(r.panels + tr * r.stride + (tc * 8 + oct) * 2048 + lane * 16, o, power);
      }
    }
    if (c.panels) {
      const float power = power_of(half_exponent(c.tops[tc * 64 + lane]));
#pragma unroll
      for (int oct = wave; oct < 8; oct += 4) {
        if (tr * 64 + oct * 8 >= (s.rows + 31) / 32 * 32) break;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = t[(oct * 8 + j) * PITCH + lane];
        put_octet(c.panels + tc * c.stride + (tr * 8 + oct) * 2048 + lane * 16, o, power);
      }
    }
  }
};
// Whole groups of four panels, the rows past the matrix zeros.
template <class S>
PackJob<S> pack_job(const S& s, const HalfPanels& r, const HalfPanels& c) {
  const int64_t tiles_r = r.panels ? (s.rows + 255) / 256 * 4 : (s.rows + 63) / 64;
  const int64_t tiles_c = c.panels ? (int64_t(s.cols) + 255) / 256 * 4 : (int64_t(s.cols) + 63) / 64;
  return {s, r, c, tiles_c, tiles_r * tiles_c};
}

// One launch for two jobs.
struct NoJob {
  int64_t blocks = 0;
  __device__ __forceinline__ void run(int64_t, char*) const {}
};
template <class A, class B>
__global__ __launch_bounds__(kPanelThreads) void panel_jobs(A a, B b) {
  __shared__ __attribute__((aligned(16))) char smem[64 * 68 * 4];
  const int64_t block = blockIdx.x;
  if (block < a.blocks) a.run(block, smem);
  else b.run(block - a.blocks, smem);
}
template <class A, class B>
int run_panel_jobs(Runtime* rt, const A& a, const B& b) {
  const int64_t blocks = a.blocks + b.blocks;
  if (blocks == 0) return LMP_OK;
  if (uint64_t(blocks) > kMaxGridThreads / kPanelThreads)
    return fail(LMP_ERR_UNSUPPORTED, "split products: more tiles than a grid holds");
  panel_jobs<<<dim3(uint32_t(blocks)), dim3(kPanelThreads), 0, rt->stream>>>(a, b);
  LMP_LAUNCH_CHECK("panel_jobs");
  return LMP_OK;
}

}  // namespace
}  // namespace lmp_hip
