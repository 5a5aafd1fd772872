// Products on the fp16 matrix cores shared by the operators that use them
// (half_products.hip; the tiles are gemm_half.hpp's).
#pragma once

#include <cstddef>
#include <cstdint>

#include "common.hpp"

namespace lmp_hip {

// Whether a layer's products x [rows, in] w [in, width] and their gradients run there: each
// extent is the K of one of them, and a leading dimension has to let a panel's offsets fit 32
// bits.  Fewer rows are bound by reading the weights, which this reads once more than the fp32
// products (32 x 4096 by 4096 x 16384: 167 us against 55).
inline bool half_fits(size_t rows, size_t in, size_t width, size_t most_ld) {
  return rows >= 128 && in >= 32 && width >= 32 && most_ld < (size_t(1) << 22);
}

// Room for n bits of largest magnitudes: tiles read up to 256 past them.
inline size_t half_tops_room(size_t n) { return (n + 255) / 256 * 256 + 256; }

// Zeros in `n` words.
int clear_words(Runtime* rt, uint32_t* p, size_t n);
// Zeros in `cols` columns of `rows` rows (the gradients of no rows).
int clear_f32(Runtime* rt, float* p, size_t rows, size_t cols, size_t ld);

// The bits of the largest magnitude of each row and of each column (either may be null),
// which start as zeros.  NaN is above infinity.
int half_tops(Runtime* rt, const float* x, size_t rows, size_t cols, size_t ld, uint32_t* row_top,
              uint32_t* col_top);

// dx = d w^T and dw (+)= x^T d of a layer with x [rows, in] and w [in, width], each null
// where it is not wanted, with the largest magnitudes that their products need.
struct HalfBackward {
  size_t rows, in, width;
  const float* d;
  size_t ldd;
  const uint32_t *d_row, *d_col;
  const float* x;
  size_t ldx;
  const uint32_t* x_col;
  const float* w;
  size_t ldw;
  const uint32_t* w_row;
  float* dx;
  size_t lddx;
  float* dw;
  size_t lddw;
  bool dw_accumulate;
};
int half_backward(Runtime* rt, const HalfBackward& b);

}  // namespace lmp_hip
