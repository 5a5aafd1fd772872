// What the operators on the fp16 matrix cores (half_products.hpp) clear.
#include "half_products.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>

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

}  // namespace lmp_hip
