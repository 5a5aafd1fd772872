// Which tiles the sizes of tests/test_gpu_split_products.py take (host code), so that a change of the model cannot leave
// a kernel without a test.
#include <cstdio>
#include <cstdlib>

#include "gemm_plan.hpp"

using namespace lmp_hip;

// Tiles by their height, of the forward product and of both gradients, and the gradients' splits of K.
struct Case {
  int64_t rows, in, width;
  int forward, backward, dw_splits, dx_splits;
};
constexpr Case kCases[] = {
    {423, 1000, 32002, 256, 0, 0, 0},     {423, 1000, 32003, 256, 0, 0, 0},     {2300, 520, 10006, 128, 0, 0, 0},
    {2300, 520, 10007, 128, 128, 1, 6},   {1500, 1100, 2402, 64, 128, 1, 2},    {5003, 600, 2402, 64, 128, 3, 1},
    {5003, 600, 1009, 64, 128, 6, 1},     {1031, 2050, 2002, 64, 64, 1, 1},     {2100, 900, 2003, 64, 64, 1, 1},
    {1005, 2000, 3002, 64, 256, 1, 3},    {8200, 1024, 4160, 128, 256, 3, 1}};

int main() {
  for (const Case& c : kCases) {
    const HalfPlan f = half_plan(256, 0, {c.rows, (c.width + 63) / 64 * 64, c.in, false, 2.0f}, {});
    const HalfPlan b = half_plan(256, int64_t(256) << 20, {c.in, c.width, c.rows, true}, {c.rows, c.in, c.width, true});
    const int forward = kHalfTiles[f.cfg].bm, backward = kHalfTiles[b.cfg].bm;
    if (forward != c.forward || (c.backward && (backward != c.backward || b.splits[0] != c.dw_splits || b.splits[1] != c.dx_splits))) {
      std::printf("%lld x %lld by %lld: %d, %d in %d and %d\n", (long long)c.rows, (long long)c.in, (long long)c.width, forward,
                  backward, b.splits[0], b.splits[1]);
      return 1;
    }
  }
  std::puts("half plan cases ok");
  return 0;
}
