// The work lists of a packed attention batch.  Host code, no HIP includes.
#pragma once

#include <algorithm>
#include <cstdint>
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
  // Keys of packed rows and of queries; of the split kernels' keys, steps over the
  // queries that may see them (attn_key_steps).
  int32_t key_begin, key_end;
  int32_t part;        // place of its partial result, or -1 where it is the whole
  int32_t qt0, kt0;    // the sequence's first tile of queries and of keys
  int32_t seq;
};

// Packed rows whose partial results are joined.
struct AttnJoin {
  int32_t q0, lq, first, part, parts;
};

// A sequence's tiles of queries and of keys.
struct AttnSeq {
  int32_t qt0, q_tiles, kt0, k_tiles;
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
  std::vector<AttnJoin> q_joins;
  std::vector<AttnItem> k_blocks;  // keys, split kernels
  std::vector<AttnJoin> k_joins;   // q0 and lq are those of the keys
  std::vector<AttnSeq> seqs;
  std::vector<AttnTile> q_tiles, k_tiles;
  int64_t queries = 0, key_rows = 0, parts = 0, q_parts = 0, k_parts = 0;
  // (row, key) pairs of one head that the kernels go through: of 16 packed rows up
  // to the last one's last key, and of 128 queries.
  double row_work = 0, block_work = 0;
};

// Keys that query i of a sequence sees: [0, seen).
inline int64_t attn_seen(int64_t i, int64_t lq, int64_t lk, bool causal) {
  return causal ? std::clamp<int64_t>(i + 1 + lk - lq, 0, lk) : lk;
}

// The steps of the split kernels' keys from `first` on: a tile of queries of one
// of the group's heads each, the last tile first, the heads of a tile in turn.
inline int64_t attn_key_steps(int64_t first, int64_t lq, int64_t lk, bool causal, int64_t group) {
  const int64_t tiles = (lq + kAttnTile - 1) / kAttnTile;
  const int64_t from = causal ? std::min(tiles, std::max<int64_t>(0, first - (lk - lq)) / kAttnTile) : 0;
  return (tiles - from) * group;
}

// Rows whose keys are split take parts: emit(begin, end, part) for each.  With a
// `step`, of nearly equal length, at multiples of it; without one, of part_keys, so
// that the parts of different rows go over the same keys together, the last one half
// shorter or longer at most.
template <class Emit>
inline void attn_parts(int64_t seen, int64_t part_keys, int64_t step, int64_t* next_part,
                       Emit&& emit) {
  const int64_t over = step ? part_keys - 1 : part_keys / 2;
  const int64_t parts = seen <= part_keys ? 1 : (seen + over) / part_keys;
  if (parts <= 1) return emit(0, seen, int64_t(-1));
  const int64_t steps = step ? (seen + step - 1) / step : 0;
  for (int64_t p = 0; p < parts; ++p) {
    const int64_t begin = step ? steps * p / parts * step : p * part_keys;
    const int64_t end = step ? steps * (p + 1) / parts * step : begin + part_keys;
    emit(begin, p + 1 == parts ? seen : end, (*next_part)++);
  }
}

// The length of a part that gives about `workgroups` of them, `least` at least;
// no split where the rows alone are as many.
inline int64_t attn_part_keys(double work, int64_t rows, int64_t workgroups, int64_t least) {
  if (rows >= workgroups) return INT64_MAX;
  return std::max(least, int64_t(work / double(workgroups)) / 64 * 64 + 64);
}

// `compute_units` of the chip.  The fp32 kernels hold two workgroups on each and
// are split for three times that, the split kernels' forward two.
constexpr int64_t kLeastPart = 128, kLeastSplitPart = 256, kLeastSteps = 8;

inline AttnLists attn_lists(size_t sequences, const int64_t* ql, const int64_t* kl, int64_t heads,
                            int64_t kv_heads, bool causal, int64_t compute_units) {
  AttnLists a;
  const int64_t group = heads / kv_heads;
  // The keys of all rows, for the length of a part.
  double steps = 0;
  int64_t tiles = 0, blocks = 0;
  for (size_t s = 0; s < sequences; ++s) {
    const int64_t lq = ql[s], lk = kl[s], rows = lq * group;
    for (int64_t r = 0; r < rows; r += kAttnRows, ++tiles)
      a.row_work += kAttnRows * double(attn_seen((std::min(rows, r + kAttnRows) - 1) / group, lq, lk, causal));
    for (int64_t q = 0; q < lq; q += kAttnSplitRows, ++blocks)
      a.block_work += kAttnSplitRows * double(attn_seen(std::min(lq, q + kAttnSplitRows) - 1, lq, lk, causal));
    for (int64_t k = 0; k < lk; k += kAttnSplitRows)
      steps += double(attn_key_steps(k, lq, lk, causal, group));
  }
  const int64_t part_keys = attn_part_keys(a.row_work / kAttnRows * double(kv_heads), tiles * kv_heads,
                                           compute_units * 6, kLeastPart);
  const int64_t block_keys = attn_part_keys(a.block_work / kAttnSplitRows * double(heads), blocks * heads,
                                            compute_units * 2, kLeastSplitPart);
  // The key kernel holds one workgroup on a unit; four parts for each even out the
  // causal mask's long and short ones.
  const int64_t part_steps =
      std::max(kLeastSteps, int64_t(steps * double(kv_heads) / double(compute_units * 4)) + 1);
  for (size_t s = 0; s < sequences; ++s) {
    const int64_t lq = ql[s], lk = kl[s], rows = lq * group;
    AttnItem it{int32_t(a.queries), int32_t(a.key_rows), int32_t(lq), int32_t(lk), 0, 0, 0, -1,
                int32_t(a.q_tiles.size()), int32_t(a.k_tiles.size()), int32_t(s)};
    const auto split = [&](int64_t first, int64_t seen, int64_t keys, int64_t step,
                           int64_t* next_part, std::vector<AttnItem>& items,
                           std::vector<AttnJoin>& joins) {
      it.first = int32_t(first);
      const int64_t before = *next_part;
      attn_parts(seen, keys, step, next_part, [&](int64_t begin, int64_t end, int64_t part) {
        it.key_begin = int32_t(begin);
        it.key_end = int32_t(end);
        it.part = int32_t(part);
        items.push_back(it);
      });
      if (*next_part > before)
        joins.push_back({it.q0, it.lq, it.first, int32_t(before), int32_t(*next_part - before)});
    };
    for (int64_t r = 0; r < rows; r += kAttnRows)
      split(r, attn_seen((std::min(rows, r + kAttnRows) - 1) / group, lq, lk, causal), part_keys,
            16, &a.parts, a.rows, a.joins);
    for (int64_t q = 0; q < lq; q += kAttnSplitRows)
      split(q, attn_seen(std::min(lq, q + kAttnSplitRows) - 1, lq, lk, causal), block_keys,
            0, &a.q_parts, a.q_blocks, a.q_joins);
    it.part = -1;
    it.key_begin = 0;
    it.key_end = it.lk;
    for (int64_t k = 0; k < lk; k += kAttnRows) {
      it.first = int32_t(k);
      a.keys.push_back(it);
    }
    for (int64_t k = 0; k < lk; k += kAttnSplitRows) {
      it.first = int32_t(k);
      const int64_t before = a.k_parts;
      attn_parts(attn_key_steps(k, lq, lk, causal, group), part_steps, 0, &a.k_parts,
                 [&](int64_t begin, int64_t end, int64_t part) {
                   it.key_begin = int32_t(begin);
                   it.key_end = int32_t(end);
                   it.part = int32_t(part);
                   a.k_blocks.push_back(it);
                 });
      if (a.k_parts > before)
        a.k_joins.push_back({it.k0, it.lk, it.first, int32_t(before), int32_t(a.k_parts - before)});
    }
    for (int64_t q = 0; q < lq; q += kAttnTile)
      a.q_tiles.push_back({int32_t(a.queries + q), int32_t(std::min<int64_t>(kAttnTile, lq - q))});
    for (int64_t k = 0; k < lk; k += kAttnTile)
      a.k_tiles.push_back({int32_t(a.key_rows + k), int32_t(std::min<int64_t>(kAttnTile, lk - k))});
    a.seqs.push_back({it.qt0, int32_t(a.q_tiles.size()) - it.qt0, it.kt0,
                      int32_t(a.k_tiles.size()) - it.kt0});
    a.queries += lq;
    a.key_rows += lk;
  }
  // Longest first: the last workgroups to start are short ones.
  const auto keys_of = [](const AttnItem& x) { return x.key_end - x.key_begin; };
  const auto longer = [&](const AttnItem& x, const AttnItem& y) {
    return keys_of(x) != keys_of(y) ? keys_of(x) > keys_of(y) : x.key_begin < y.key_begin;
  };
  std::stable_sort(a.rows.begin(), a.rows.end(), longer);
  std::stable_sort(a.q_blocks.begin(), a.q_blocks.end(), longer);
  const auto queries_of = [&](const AttnItem& x) {
    return causal ? x.lq - std::clamp(x.first - (x.lk - x.lq), 0, x.lq) : x.lq;
  };
  const auto more = [&](const AttnItem& x, const AttnItem& y) { return queries_of(x) > queries_of(y); };
  std::stable_sort(a.keys.begin(), a.keys.end(), more);
  std::stable_sort(a.k_blocks.begin(), a.k_blocks.end(), longer);
  return a;
}

}  // namespace lmp_hip
