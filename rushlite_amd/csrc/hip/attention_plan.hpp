// The work lists of a packed attention batch.  Host code, no HIP includes.
#pragma once

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <vector>

namespace lmp_hip {

// Rows of one key head: its `group` query heads' rows of every query, packed
// query by query (row r is query r / group of head kv_head * group + r % group),
// so that the heads that share keys share the reads of them.
constexpr int kAttnRows = 16;   // packed rows, or keys, of a work item of the fp32 kernels
constexpr int kAttnSplitRows = 128;  // queries, or keys, of one of the split-fp16 kernels
constexpr int kAttnTile = 32;   // rows of a tile of the split-fp16 operands

// A run of rows of one sequence; one per key head of it is worked on.
struct AttnItem {
  int32_t q0, k0;      // the sequence's first query and key in the packed rows
  int32_t lq, lk;
  int32_t first;       // first packed row, query or key
  int32_t key_begin, key_end;  // of the forward pass
  int32_t part;        // place of its partial result, or -1 where it is the whole
  int32_t qt0, kt0;    // the sequence's first tile of queries and of keys
};

// Packed rows whose partial results are joined.
struct AttnJoin {
  int32_t q0, lq, first, part, parts;
};

// A tile of the split-fp16 operands: rows at .. at + rows - 1 of the packed rows.
struct AttnTile {
  int32_t at, rows;
};

struct AttnLists {
  std::vector<AttnItem> rows;      // packed query rows, fp32 kernels
  std::vector<AttnItem> keys;      // keys, fp32 kernels
  std::vector<AttnJoin> joins;
  std::vector<AttnItem> q_blocks;  // queries, split kernels
  std::vector<AttnItem> k_blocks;  // keys, split kernels
  std::vector<AttnTile> q_tiles, k_tiles;
  int64_t queries = 0, key_rows = 0, parts = 0;
  double pairs = 0;  // (query, key) pairs the mask leaves, of one head
};

// Keys that query i of a sequence sees: [0, seen).
inline int64_t attn_seen(int64_t i, int64_t lq, int64_t lk, bool causal) {
  return causal ? std::clamp<int64_t>(i + 1 + lk - lq, 0, lk) : lk;
}

// `workgroups`: how many fill the chip well.  The keys of packed rows are split
// over several workgroups where the rows alone are too few, in parts of at least
// kLeastPart keys.
constexpr int64_t kLeastPart = 128;

inline AttnLists attn_lists(size_t sequences, const int64_t* ql, const int64_t* kl, int64_t heads,
                            int64_t kv_heads, bool causal, int64_t workgroups) {
  AttnLists a;
  const int64_t group = heads / kv_heads;
  // The keys of all row tiles, for the length of a part.
  double work = 0;
  int64_t tiles = 0;
  for (size_t s = 0; s < sequences; ++s) {
    const int64_t lq = ql[s], lk = kl[s], rows = lq * group;
    for (int64_t r = 0; r < rows; r += kAttnRows) {
      const int64_t last = std::min(rows, r + kAttnRows) - 1;
      work += double(attn_seen(last / group, lq, lk, causal));
      ++tiles;
    }
    for (int64_t i = 0; i < lq; ++i) a.pairs += double(attn_seen(i, lq, lk, causal));
  }
  int64_t part_keys = INT64_MAX;
  if (tiles * kv_heads < workgroups) {
    part_keys = int64_t(work * double(kv_heads) / double(workgroups));
    part_keys = std::max(kLeastPart, (part_keys + 63) / 64 * 64);
  }
  for (size_t s = 0; s < sequences; ++s) {
    const int64_t lq = ql[s], lk = kl[s], rows = lq * group;
    AttnItem it{int32_t(a.queries), int32_t(a.key_rows), int32_t(lq), int32_t(lk), 0, 0, 0, -1,
                int32_t(a.q_tiles.size()), int32_t(a.k_tiles.size())};
    for (int64_t r = 0; r < rows; r += kAttnRows) {
      const int64_t last = std::min(rows, r + kAttnRows) - 1;
      const int64_t seen = attn_seen(last / group, lq, lk, causal);
      const int64_t parts = std::max<int64_t>(1, part_keys == INT64_MAX ? 1 : (seen + part_keys - 1) / part_keys);
      it.first = int32_t(r);
      if (parts > 1) {
        a.joins.push_back({it.q0, it.lq, it.first, int32_t(a.parts), int32_t(parts)});
        // Parts of nearly equal length, at multiples of 16 keys.
        const int64_t steps = (seen + 15) / 16;
        for (int64_t p = 0; p < parts; ++p) {
          it.key_begin = int32_t(steps * p / parts * 16);
          it.key_end = int32_t(std::min(seen, steps * (p + 1) / parts * 16));
          it.part = int32_t(a.parts++);
          a.rows.push_back(it);
        }
      } else {
        it.key_begin = 0;
        it.key_end = int32_t(seen);
        it.part = -1;
        a.rows.push_back(it);
      }
    }
    it.part = -1;
    it.key_begin = 0;
    it.key_end = it.lk;
    for (int64_t k = 0; k < lk; k += kAttnRows) {
      it.first = int32_t(k);
      a.keys.push_back(it);
    }
    for (int64_t q = 0; q < lq; q += kAttnSplitRows) {
      it.first = int32_t(q);
      it.key_end = int32_t(attn_seen(std::min(lq, q + kAttnSplitRows) - 1, lq, lk, causal));
      a.q_blocks.push_back(it);
    }
    it.key_end = it.lk;
    for (int64_t k = 0; k < lk; k += kAttnSplitRows) {
      it.first = int32_t(k);
      a.k_blocks.push_back(it);
    }
    for (int64_t q = 0; q < lq; q += kAttnTile)
      a.q_tiles.push_back({int32_t(a.queries + q), int32_t(std::min<int64_t>(kAttnTile, lq - q))});
    for (int64_t k = 0; k < lk; k += kAttnTile)
      a.k_tiles.push_back({int32_t(a.key_rows + k), int32_t(std::min<int64_t>(kAttnTile, lk - k))});
    a.queries += lq;
    a.key_rows += lk;
  }
  // Longest first: the last workgroups to start are short ones.
  const auto keys_of = [](const AttnItem& x) { return x.key_end - x.key_begin; };
  const auto longer = [&](const AttnItem& x, const AttnItem& y) { return keys_of(x) > keys_of(y); };
  std::stable_sort(a.rows.begin(), a.rows.end(), longer);
  std::stable_sort(a.q_blocks.begin(), a.q_blocks.end(), longer);
  const auto queries_of = [&](const AttnItem& x) {
    return causal ? x.lq - std::clamp(x.first - (x.lk - x.lq), 0, x.lq) : x.lq;
  };
  const auto more = [&](const AttnItem& x, const AttnItem& y) { return queries_of(x) > queries_of(y); };
  std::stable_sort(a.keys.begin(), a.keys.end(), more);
  std::stable_sort(a.k_blocks.begin(), a.k_blocks.end(), more);
  return a;
}

}  // namespace lmp_hip
