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
                  int64_t kv_heads, bool causal, int64_t workgroups) {
  const AttnLists a = attn_lists(ql.size(), ql.data(), kl.data(), heads, kv_heads, causal, workgroups);
  const int64_t group = heads / kv_heads;
  int64_t q0 = 0, k0 = 0, qt = 0, kt = 0;
  double pairs = 0;
  std::map<int64_t, int> parts_seen;
  for (size_t s = 0; s < ql.size(); ++s) {
    const int64_t lq = ql[s], lk = kl[s], rows = lq * group;
    std::vector<std::vector<int>> cover(size_t(rows), std::vector<int>(size_t(lk), 0));
    std::vector<int> key_cover(size_t(lk), 0), qb(size_t(lq), 0), kb(size_t(lk), 0);
    for (const AttnItem& it : a.rows) {
      if (it.q0 != q0 || it.lq != lq || it.k0 != k0 || it.lk != lk) continue;
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
        if (r % group == 0) pairs += double(seen);
        for (int64_t k = 0; k < lk; ++k) CHECK(cover[size_t(r)][size_t(k)] <= 1 && (k >= seen || cover[size_t(r)][size_t(k)]));
      }
    for (const AttnItem& it : a.keys)
      if (it.k0 == k0 && it.lk == lk && it.q0 == q0)
        for (int64_t k = it.first; k < std::min<int64_t>(lk, it.first + kAttnRows); ++k) ++key_cover[size_t(k)];
    for (int c : key_cover) CHECK(c == 1);
    for (const AttnItem& it : a.q_blocks)
      if (it.q0 == q0 && it.lq == lq && it.k0 == k0)
        for (int64_t q = it.first; q < std::min<int64_t>(lq, it.first + kAttnSplitRows); ++q) {
          ++qb[size_t(q)];
          CHECK(attn_seen(q, lq, lk, causal) <= it.key_end);
        }
    for (int c : qb) CHECK(c == 1);
    for (const AttnItem& it : a.k_blocks)
      if (it.k0 == k0 && it.lk == lk && it.q0 == q0)
        for (int64_t k = it.first; k < std::min<int64_t>(lk, it.first + kAttnSplitRows); ++k) ++kb[size_t(k)];
    for (int c : kb) CHECK(c == 1);
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
  CHECK(a.queries == q0 && a.key_rows == k0 && a.pairs == pairs);
  CHECK(int64_t(parts_seen.size()) == a.parts);
  std::map<int64_t, int> joined;
  for (const AttnJoin& j : a.joins) {
    CHECK(j.parts > 1);
    for (int p = 0; p < j.parts; ++p) ++joined[j.part + p];
  }
  CHECK(joined.size() == parts_seen.size());
  for (auto [p, n] : joined) CHECK(n == 1 && parts_seen[p] == 1);
}

int main() {
  std::mt19937 rng(5);
  // Distinct lengths identify a sequence by its first rows; empty ones come between.
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
