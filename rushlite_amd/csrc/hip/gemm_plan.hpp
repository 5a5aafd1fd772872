// How the fp32 GEMMs are cut into workgroups: host code without HIP includes.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <iterator>

#include "fastdiv.hpp"

namespace lmp_hip {

// A grid holds fewer than 2^32 threads per dimension: a dispatch counts them in
// 32 bits, and a longer one-shot launch comes out as what is left modulo 2^32
// (2^33 + 64 threads as a single wave).
constexpr uint64_t kMaxGridThreads = 0xffffffffull;

// `blocks` workgroups over two dimensions of a grid, y past 1 only where x alone
// would have too many threads; block y * x_extent + x may lie past the last one.
struct Grid2 {
  uint32_t x = 1, y = 1;
};
inline Grid2 grid_2d(uint64_t blocks, int threads) {
  const uint64_t most = kMaxGridThreads / uint64_t(threads);
  const uint64_t y = (blocks + most - 1) / most;
  return {uint32_t((blocks + y - 1) / y), uint32_t(y)};
}

// ------------------------------------------------------- products of up to 32 rows

// K split over workgroups, `per_wg` values each; a workgroup's `waves` waves take
// consecutive parts of its range.
struct KSplit {
  int splits = 1, per_wg = 0;
};

// One past the last k of a wave that takes `part` values from `kb` on: at most
// k, and no more than kb for a wave past the end (kb + part may not fit an int).
LMP_HD int k_range_end(int kb, int part, int k) {
  const int left = k - kb;
  return kb + (part < left ? part : left);
}

constexpr int kRowsWaves = 4;

// A workgroup for every 32 of n columns fits a grid.
inline bool rows_fit(int64_t n) {
  return uint64_t(n + 31) / 32 <= kMaxGridThreads / (64 * kRowsWaves);
}

// Rows kernel (B transposed, one workgroup per 32 columns).  A CU holds one
// workgroup, so the split count is the one whose rounds of workgroups take the
// fewest tile steps: a step of the whole chip (4 MiB of B) is about 1 us, as
// are a round's start and end, and folding partials costs about 4.
inline KSplit rows_split(int64_t cus, int64_t n, int64_t k) {
  constexpr int64_t kGrain = 32 * kRowsWaves;
  const int64_t blocks = (n + 31) / 32;
  const int64_t k_tiles = (k + kGrain - 1) / kGrain;  // a wave's tiles, unsplit
  int64_t per = k_tiles, best = INT64_MAX;
  const int64_t max_splits =
      std::max<int64_t>(1, std::min<int64_t>(k_tiles / 2, 2 * cus / blocks));
  for (int64_t s = 1; s <= max_splits; ++s) {
    const int64_t steps = (k_tiles + s - 1) / s;
    const int64_t rounds = (blocks * s + cus - 1) / cus;
    const int64_t cost = rounds * (steps + 1) + (s > 1 ? 4 : 0);
    if (cost < best) {
      best = cost;
      per = steps;
    }
  }
  return {int((k_tiles + per - 1) / per), int(per * kGrain)};
}

constexpr int kDirectWaves = 4;

// Register-direct kernel: `splits` workgroups (0: enough for the CUs) of 64 k or
// more per wave for each of `blocks` column blocks.
inline KSplit direct_split(int64_t cus, int64_t blocks, int64_t k, int64_t splits) {
  constexpr int64_t kGrain = 8 * kDirectWaves;
  const int64_t most = std::max<int64_t>(1, k / (64 * kDirectWaves));
  if (splits <= 0) splits = (cus + blocks - 1) / blocks;
  splits = std::max<int64_t>(1, std::min(splits, most));
  const int64_t per = ((k + splits - 1) / splits + kGrain - 1) / kGrain * kGrain;
  return {int((k + per - 1) / per), int(per)};
}

// ---------------------------------------------- products on the bf16 matrix cores

constexpr int kBf3K = 16;  // k values per step

struct Bf3Plan {
  int cfg = -1;  // index into kBf3Tiles; -1: no launch fits a grid
  int splits = 1;
};

// Time of one 16-wide k step of a workgroup, in us: `alone` on its CU, and
// `shared` per workgroup where several take turns (fitted to a sweep of 66
// products over every tile and split, random operands, on one MI355X: the plan
// takes 0.4% more than the best of the sweep, 8% at worst).  A larger tile moves
// and splits each value fewer times: 4096^3 takes 565-640, 650-680, 710-780,
// 870 and about 980 us on the five, 512 x 1000 x 4096 (K split) 44, 37, 34, 37,
// 38 and 256 x 1024 x 1024 25, 19, 16, 15.5, 14.
// APART: the leading products of a value accumulate apart from the small ones,
// one rounding of the sum a step (six without, which the largest tile's
// accumulators leave no registers for).
struct Bf3Tile {
  int bm, bn, threads;
  bool apart;
  float alone, shared;
};
constexpr Bf3Tile kBf3Tiles[] = {{256, 256, 512, false, 1.78f, 2.4f},
                                 {256, 128, 512, true, 1.07f, 1.45f},
                                 {128, 128, 512, true, 0.61f, 0.75f},
                                 {64, 128, 256, true, 0.475f, 0.441f},
                                 {64, 64, 256, true, 0.26f, 0.252f}};

inline int64_t bf3_tiles(const Bf3Tile& t, int64_t m, int64_t n) {
  return ((m + t.bm - 1) / t.bm) * ((n + t.bn - 1) / t.bn);
}

// Tiles and split of K with the least modelled time: workgroups go round the
// CUs, each takes 4.5 us besides its steps (first loads, C), and a split costs
// a second launch (2 us) and a round trip of the partials (5 TB/s).  The
// partials stay within `scratch` bytes, the fixed workspace, whichever entry
// point is called, so that all of them give the same bits; a split keeps at
// least 64 k.  Launches that a grid cannot hold are left out, and the tile with
// one accumulator where it would not give every CU one: there the fp32 kernels
// split K, and their shorter chains round less than its long one (2048^3: 5.7e-7
// from float64 in two splits, 7.0e-7 here unsplit, 2.7e-7 with sums apart).
inline Bf3Plan bf3_plan(int64_t cus, int64_t scratch, int64_t m, int64_t n, int64_t k) {
  const int64_t steps = (k + kBf3K - 1) / kBf3K, mn = m * n;
  const int64_t most =
      std::min<int64_t>(std::max<int64_t>(1, steps / 4),
                        scratch / int64_t(sizeof(float)) /
                            (mn + n + 8));  // room for column sums, asked for or not
  Bf3Plan plan;
  float best = 0.0f;
  for (int c = 0; c < int(std::size(kBf3Tiles)); ++c) {
    const Bf3Tile& t = kBf3Tiles[c];
    const int64_t tiles = bf3_tiles(t, m, n);
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (s > 1 && (s > most || !t.apart)) break;
      if (!t.apart && tiles < cus) break;
      if (uint64_t(tiles) * uint64_t(s) > kMaxGridThreads / uint64_t(t.threads)) break;
      const float load = float((tiles * s + cus - 1) / cus);
      const float per_step = std::max(t.alone, load * t.shared);
      float us = 4.5f + float((steps + s - 1) / s) * per_step;
      if (s > 1) us += 2.0f + float(s + 1) * float(mn) * (4.0f / 5e6f);
      if (plan.cfg < 0 || us < best) {
        best = us;
        plan.cfg = c;
        plan.splits = s;
      }
      if (tiles * s > 8 * cus) break;  // more splits only add partials
    }
  }
  return plan;
}

// Whether two planned products of `a` and `b` workgroups fit one grid.
inline bool bf3_pair_fits(uint64_t a, uint64_t b, int threads) {
  return a + b <= kMaxGridThreads / uint64_t(threads);
}

// ---------------------------------------------- products on the fp16 matrix cores

constexpr int kHalfK = 32;         // k values per step
constexpr int kHalfStep = 8192;    // bytes of a panel's step: 64 rows, both parts

struct HalfTile {
  int bm, bn, threads, per_cu;
  // Time in us of one 32-wide k step of a workgroup, `alone` on its CU and `shared` per
  // workgroup where several take turns, and of its first loads and its tile's way out.
  float alone, shared, ends;
  float rate;  // TFLOP/s of long products on random operands, where the chip's power holds it back
};
constexpr HalfTile kHalfTiles[] = {{256, 256, 512, 1, 1.52f, 1.52f, 11.0f, 400},
                                   {128, 128, 512, 2, 0.59f, 0.45f, 5.5f, 370},
                                   {64, 128, 256, 3, 0.53f, 0.27f, 4.0f, 345}};

// A product [m, n] over k, none if n is 0; `split`: its K may be.  `ends`: its way out's
// weight against a plain product's.
struct HalfSize {
  int64_t m = 0, n = 0, k = 0;
  bool split = false;
  float ends = 1.0f;
};
// Tiles of one configuration, the splits of K, and which of the two products is launched first.
struct HalfPlan {
  int cfg = -1;  // index into kHalfTiles; -1: no launch fits a grid
  int splits[2] = {1, 1};
  bool second_first = false;
};

// When the slots are done that take n0 items of t0 each and then n1 of t1 as they fall free.
inline float half_makespan(int64_t slots, int64_t n0, float t0, int64_t n1, float t1) {
  const int64_t whole = n0 / slots, late = n0 % slots;
  const float begin = float(whole) * t0, last = late ? begin + t0 : begin;
  if (n1 == 0) return last;
  // Both kinds of slots take turns at t1: the first end of a turn of one of them at which n1 are done.
  const auto done = [&](float end) {
    const int64_t early = int64_t((end - begin) / t1 + 1e-3f), after = std::max<int64_t>(int64_t((end - last) / t1 + 1e-3f), 0);
    return (slots - late) * early + late * after >= n1;
  };
  const auto first = [&](float from, int64_t most) {  // of turns 1 to `most`, the last of which is enough
    int64_t low = 1;
    while (low < most) {
      const int64_t mid = (low + most) / 2;
      if (done(from + float(mid) * t1)) most = mid;
      else low = mid + 1;
    }
    return from + float(low) * t1;
  };
  float end = first(begin, (n1 + slots - late - 1) / (slots - late));
  const int64_t turns = late ? int64_t((end - last) / t1) : 0;
  if (turns >= 1 && done(last + float(turns) * t1)) end = std::min(end, first(last, turns));
  return std::max(end, last);
}

// The configuration, splits and order with the least modelled time; partial sums stay within
// `scratch` bytes and a split keeps at least 128 k.  The time at the rate that the chip's power
// allows (operands of zeros run at 650 TFLOP/s in place of 400) and the makespan at that of a
// chip that is not held back meet in a norm: 768 x 4096 over 12608 in 192 tiles
// of 128 x 128 on 256 CUs takes 243 us, of 206 and 237.
inline HalfPlan half_plan(int64_t cus, int64_t scratch, const HalfSize& a, const HalfSize& b) {
  HalfPlan plan;
  float best = 0.0f;
  const HalfSize* size[2] = {&a, &b};
  for (int c = 0; c < int(std::size(kHalfTiles)); ++c) {
    const HalfTile& t = kHalfTiles[c];
    int64_t tiles[2], steps[2];
    float power = 0.0f;
    for (int i = 0; i < 2; ++i) {
      tiles[i] = (size[i]->m + t.bm - 1) / t.bm * ((size[i]->n + t.bn - 1) / t.bn);
      steps[i] = (size[i]->k + kHalfK - 1) / kHalfK;
      power += float(tiles[i]) * float(steps[i]) * float(t.bm) * float(t.bn) * (2 * kHalfK / (1e6f * t.rate));
    }
    const auto fits = [&](int i, int s) {
      return s == 1 || (size[i]->split && steps[i] / s >= 4 &&
                        int64_t(s) * size[i]->m * size[i]->n <= scratch / int64_t(sizeof(float)));
    };
    constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    for (int s0 : kSplits) {
      if (!fits(0, s0)) break;
      for (int s1 : kSplits) {
        if (!fits(1, s1)) break;
        const int64_t items[2] = {tiles[0] * s0, tiles[1] * s1};
        if (uint64_t(items[0] + items[1]) > kMaxGridThreads / uint64_t(t.threads)) break;
        const int64_t held = std::clamp<int64_t>((items[0] + items[1] + cus - 1) / cus, 1, t.per_cu);
        float each[2], fold = 0.0f;
        for (int i = 0; i < 2; ++i) {
          const int s = i ? s1 : s0;
          const float n = float((steps[i] + s - 1) / s);
          each[i] = std::max(n * float(held) * t.shared, n * t.alone + t.ends * size[i]->ends);
          if (s > 1) fold += 3.0f + float(s + 1) * float(size[i]->m) * float(size[i]->n) * (4.0f / 5e6f);
        }
        for (int order = 0; order < (items[1] ? 2 : 1); ++order) {
          const float span = half_makespan(cus * held, items[order], each[order], items[1 - order], each[1 - order]);
          const float us = std::cbrt(span * span * span + power * power * power) + fold;
          if (plan.cfg < 0 || us < best) {
            best = us;
            plan = {c, {s0, s1}, order == 1};
          }
        }
        if (items[1] > 4 * cus * t.per_cu) break;
      }
      if (tiles[0] * s0 > 4 * cus * t.per_cu) break;
    }
  }
  return plan;
}

}  // namespace lmp_hip
