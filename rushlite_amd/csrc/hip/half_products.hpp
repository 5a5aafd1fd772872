// What the operators on the fp16 matrix cores share on the host (the tiles are gemm_half.hpp's,
// the operands half_panels.hpp's, the gradient products half_backward.hpp's).
#pragma once

#include <cstddef>
#include <cstdint>

#include "common.hpp"
#include "gemm_plan.hpp"

namespace lmp_hip {

// One operand: its panels of 64 rows, `stride` bytes apart, the bits of its rows' largest finite
// magnitudes, and their marks: how many small values a row has, and whether one is not finite.
struct HalfPanels {
  char* panels;
  int64_t stride;
  uint32_t *tops, *marks;
};

// Whether a layer's products x [rows, in] w [in, width] and their gradients may run there: each
// extent is the K of one of them, whose panel's offsets have to fit 32 bits.
inline bool half_fits(size_t rows, size_t in, size_t width) {
  const size_t most = size_t(1) << 23;
  return rows >= 32 && in >= 32 && width >= 32 && rows < most && in < most && width < most;
}

// Times in us by which an operator weighs these products against the fp32 ones.  Those run at 115
// TFLOP/s forward and 160 for the two gradients together, these at 350, and a pass over
// memory at 4.5 TB/s.
inline double half_saves_forward(double products) { return products * 2 * (1 / 115e6 - 1 / 350e6); }
inline double half_saves_backward(double products) { return products * 4 * (1 / 160e6 - 1 / 350e6); }
inline double pass_time(double bytes) { return bytes / 4.5e6; }

// A workspace in words, each part a multiple of 256 bytes.
struct HalfRoom {
  size_t words = 0;
  size_t take(size_t n) {
    const size_t at = words;
    words += (n + 63) / 64 * 64;
    return at;
  }
};
// Words of a number for each of `n` rows (tiles read whole groups of 256), of an operand's panels
// [rows, k], and bytes from panel to panel.
inline size_t half_tops_words(size_t n) { return (n + 255) / 256 * 256; }
inline size_t half_stride(size_t k) { return (k + kHalfK - 1) / kHalfK * size_t(kHalfStep); }
inline size_t half_panel_words(size_t rows, size_t k) { return (rows + 255) / 256 * half_stride(k); }

// Zeros in `n` words.
int clear_words(Runtime* rt, uint32_t* p, size_t n);
// Zeros in `cols` columns of `rows` rows (the gradients of no rows).
int clear_f32(Runtime* rt, float* p, size_t rows, size_t cols, size_t ld);

}  // namespace lmp_hip
