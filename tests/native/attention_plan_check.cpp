// The work lists of packed attention against a direct count: every visible
// (packed row, key) pair is covered once by the forward items, split rows are
// joined over exactly their parts, and every key and tile is listed once.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>

#include "attention_plan.hpp"

using namespace lmp_hip;

#define CHECK(c) \
  do { if (!(c)) { std::printf("failed: %s (line %d)\n", #c, __LINE__); std::exit(1); } } while (0)

static void check(const std::vector<int64_t>& ql, const std::vector<int64_t>& kl, int64_t heads,
                  int64_t kv_heads, bool causal, int64_t units) {
  const AttnLists a = attn_lists(ql.size(), ql.data(), kl.data(), heads, kv_heads, causal, units);
  const int64_t group = heads / kv_heads;
  int64_t q0 = 0, k0 = 0, qt = 0, kt = 0;
  std::map<int64_t, int> parts_seen, block_parts, key_parts;
  for (size_t s = 0; s < ql.size(); ++s) {
    const int64_t lq = ql[s], lk = kl[s], rows = lq * group;
    std::vector<std::vector<int>> cover(size_t(rows), std::vector<int>(size_t(lk), 0));
    std::vector<std::vector<int>> block_cover(size_t(lq), std::vector<int>(size_t(lk), 0));
    std::vector<int> key_cover(size_t(lk), 0), qb(size_t(lq), 0), kb(size_t(lk), 0);
    for (const AttnItem& it : a.rows) {
      if (it.seq != int(s)) continue;
      CHECK(it.q0 == q0 && it.lq == lq && it.k0 == k0 && it.lk == lk);
      CHECK(it.first % kAttnRows == 0 && it.first < rows && it.qt0 == qt && it.kt0 == kt);
      CHECK(it.key_begin % 16 == 0 && it.key_begin <= it.key_end && it.key_end <= lk);
      CHECK(it.part < a.parts);
      if (it.part >= 0) ++parts_seen[it.part];
      for (int64_t r = it.first; r < std::min<int64_t>(rows, it.first + kAttnRows); ++r)
        for (int64_t k = it.key_begin; k < it.key_end; ++k) ++cover[size_t(r)][size_t(k)];
    }
    if (lq && lk)
      for (int64_t r = 0; r < rows; ++r) {
        const int64_t seen = attn_seen(r / group, lq, lk, causal);
        for (int64_t k = 0; k < lk; ++k) CHECK(cover[size_t(r)][size_t(k)] <= 1 && (k >= seen || cover[size_t(r)][size_t(k)]));
      }
    for (const AttnItem& it : a.keys)
      if (it.seq == int(s))
        for (int64_t k = it.first; k < std::min<int64_t>(lk, it.first + kAttnRows); ++k) ++key_cover[size_t(k)];
    for (int c : key_cover) CHECK(c == 1);
    for (const AttnItem& it : a.q_blocks)
      if (it.seq == int(s)) {
        CHECK(it.first % kAttnSplitRows == 0 && it.first < lq && it.qt0 == qt && it.kt0 == kt);
        CHECK(it.key_begin % kAttnTile == 0 && it.key_begin <= it.key_end && it.key_end <= lk);
        CHECK(it.part < a.q_parts);
        if (it.part >= 0) ++block_parts[it.part];
        for (int64_t q = it.first; q < std::min<int64_t>(lq, it.first + kAttnSplitRows); ++q) {
          if (it.key_begin == 0) ++qb[size_t(q)];
          for (int64_t k = it.key_begin; k < it.key_end; ++k) ++block_cover[size_t(q)][size_t(k)];
        }
      }
    for (int c : qb) CHECK(c == 1);
    for (int64_t q = 0; q < lq; ++q)
      for (int64_t k = 0; k < lk; ++k)
        CHECK(block_cover[size_t(q)][size_t(k)] <= 1 &&
              (k >= attn_seen(q, lq, lk, causal) || block_cover[size_t(q)][size_t(k)]));
    CHECK(a.seqs[s].qt0 == qt && a.seqs[s].kt0 == kt && a.seqs[s].q_tiles == (lq + 31) / 32 &&
          a.seqs[s].k_tiles == (lk + 31) / 32);
    for (const AttnItem& it : a.k_blocks)
      if (it.seq == int(s))
        for (int64_t k = it.first; k < std::min<int64_t>(lk, it.first + kAttnSplitRows); ++k) {
          if (it.key_begin == 0) ++kb[size_t(k)];
          if (it.part >= 0 && k == it.first) ++key_parts[it.part];
        }
    for (int c : kb) CHECK(c == 1);
    // The steps of each block of keys: all of them once, and every query that sees a
    // key of the block is in one of their tiles.
    for (int64_t k = 0; k < lk; k += kAttnSplitRows) {
      const int64_t all = attn_key_steps(k, lq, lk, causal, group), q_count = (lq + kAttnTile - 1) / kAttnTile;
      std::vector<int> step(size_t(all), 0);
      for (const AttnItem& it : a.k_blocks)
        if (it.seq == int(s) && it.first == k)
          for (int64_t i = it.key_begin; i < it.key_end; ++i) ++step.at(size_t(i));
      for (int c : step) CHECK(c == 1);
      for (int64_t q = 0; q < lq; ++q)
        if (attn_seen(q, lq, lk, causal) > k) CHECK(q / kAttnTile > q_count - 1 - all / group);
    }
    for (int64_t q = 0; q < lq; q += kAttnTile, ++qt) {
      CHECK(a.q_tiles[size_t(qt)].at == q0 + q && a.q_tiles[size_t(qt)].rows == std::min<int64_t>(kAttnTile, lq - q));
    }
    for (int64_t k = 0; k < lk; k += kAttnTile, ++kt) {
      CHECK(a.k_tiles[size_t(kt)].at == k0 + k && a.k_tiles[size_t(kt)].rows == std::min<int64_t>(kAttnTile, lk - k));
    }
    q0 += lq;
    k0 += lk;
  }
  CHECK(int64_t(a.q_tiles.size()) == qt && int64_t(a.k_tiles.size()) == kt);
  CHECK(a.queries == q0 && a.key_rows == k0);
  const auto joined = [](const std::vector<AttnJoin>& joins, std::map<int64_t, int>& parts, int64_t count) {
    CHECK(int64_t(parts.size()) == count);
    std::map<int64_t, int> got;
    for (const AttnJoin& j : joins) {
      CHECK(j.parts > 1);
      for (int p = 0; p < j.parts; ++p) ++got[j.part + p];
    }
    CHECK(got.size() == parts.size());
    for (auto [p, n] : got) CHECK(n == 1 && parts[p] == 1);
  };
  joined(a.joins, parts_seen, a.parts);
  joined(a.q_joins, block_parts, a.q_parts);
  joined(a.k_joins, key_parts, a.k_parts);
}

int main() {
  std::mt19937 rng(5);
  check({}, {}, 4, 2, true, 1024);
  check({0}, {0}, 4, 2, true, 1024);
  check({0, 5}, {7, 0}, 4, 2, true, 1024);
  check({1}, {1}, 1, 1, true, 1024);
  check({1, 1, 1}, {8192, 100, 1}, 8, 2, true, 1024);
  check({3}, {5000}, 3, 1, false, 64);
  check({300}, {200}, 2, 1, true, 1024);
  check({129}, {129}, 2, 2, true, 1);
  for (int i = 0; i < 200; ++i) {
    const int n = 1 + int(rng() % 4);
    const int64_t kv = 1 + rng() % 3, heads = kv * (1 + rng() % 5);
    std::vector<int64_t> ql, kl;
    for (int s = 0; s < n; ++s) {
      ql.push_back(rng() % 3 ? 1 + rng() % 200 : rng() % 2);
      kl.push_back(1 + rng() % 700);
    }
    check(ql, kl, heads, kv, rng() % 2, 1 + rng() % 300);
  }
  std::printf("attention lists ok\n");
}
