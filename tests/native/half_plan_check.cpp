// How the products of split operands are cut into workgroups (host code): every plan can be launched and keeps to its
// scratch memory, and the modelled makespan is that of items handed out one after another.
#include <cmath>
#include <cstdio>
#include <functional>
#include <queue>
#include <vector>

#include "gemm_plan.hpp"

using namespace lmp_hip;

#define CHECK(c)                                              \
  do {                                                        \
    if (!(c)) {                                               \
      std::printf("line %d: %s\n", __LINE__, #c);             \
      return 1;                                               \
    }                                                         \
  } while (0)

constexpr int64_t kScratch = int64_t(256) << 20;

int plans() {
  const int64_t sizes[] = {1, 32, 33, 128, 255, 1000, 4096, 12608, 100003, (1 << 23) - 1};
  for (int64_t m : sizes)
    for (int64_t n : sizes)
      for (int64_t k : sizes)
        for (bool split : {false, true}) {
          const HalfSize a{m, n, k, split}, b{k, m, n, split};
          for (const HalfSize& second : {HalfSize{}, b}) {
            const HalfPlan p = half_plan(256, kScratch, a, second);
            if (p.cfg < 0) {
              CHECK((m + 63) / 64 * ((n + 127) / 128) * 256 > int64_t(kMaxGridThreads) ||
                    (second.n && (k + 63) / 64 * ((m + 127) / 128) * 256 > int64_t(kMaxGridThreads) / 2));
              continue;
            }
            const HalfTile& t = kHalfTiles[p.cfg];
            int64_t items = 0;
            for (int i = 0; i < 2; ++i) {
              const HalfSize& s = i ? second : a;
              const int64_t steps = (s.k + kHalfK - 1) / kHalfK;
              CHECK(p.splits[i] == 1 || (s.split && steps / p.splits[i] >= 4));
              CHECK(p.splits[i] == 1 || p.splits[i] * s.m * s.n * 4 <= kScratch);
              items += (s.m + t.bm - 1) / t.bm * ((s.n + t.bn - 1) / t.bn) * p.splits[i];
            }
            CHECK(items * t.threads <= int64_t(kMaxGridThreads));
            CHECK(second.n || !p.second_first);
          }
        }
  return 0;
}

int makespans() {
  for (int slots : {1, 2, 7, 256})
    for (int n0 : {0, 1, 5, 200, 256, 700})
      for (int n1 : {0, 1, 3, 255, 513, 1000})
        for (float t0 : {1.0f, 3.5f, 40.0f})
          for (float t1 : {1.0f, 2.25f, 17.0f}) {
            if (n0 + n1 == 0) continue;
            std::priority_queue<float, std::vector<float>, std::greater<float>> free;
            for (int i = 0; i < slots; ++i) free.push(0.0f);
            float want = 0.0f;
            for (int i = 0; i < n0 + n1; ++i) {
              const float end = free.top() + (i < n0 ? t0 : t1);
              free.pop();
              free.push(end);
              want = std::max(want, end);
            }
            const float got = half_makespan(slots, n0, t0, n1, t1);
            if (std::fabs(got - want) > 1e-3f * want) std::printf("%d slots, %d of %g, %d of %g: %g, not %g\n", slots, n0, t0, n1, t1, got, want);
            CHECK(std::fabs(got - want) <= 1e-3f * want);
          }
  return 0;
}

int main() {
  if (plans() || makespans()) return 1;
  std::puts("half plans ok");
  return 0;
}
