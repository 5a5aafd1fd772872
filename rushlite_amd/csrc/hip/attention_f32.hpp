// Packed attention on the fp32 matrix cores: right for every case, and the
// kernels of short batches, single tokens and operands that the split-fp16
// kernels leave out.
//
//   S = c Q K^T (c = scale log2 e), P = 2^(S - lse2), O = P V
//   D = rowsum(dO O), dS = scale P (dO V^T - D), dQ = dS K, dK = dS^T Q, dV = P^T dO
//
// A wave works on 16 packed rows (the query heads that share a key head lie side
// by side, so one read of a key serves all of them) and 16 keys at a time with
// v_mfma_f32_16x16x4_f32.  Its operands come from memory straight into their
// registers: an operand whose rows are contracted over d is read 4 values of d a
// lane ("along"), one contracted over its rows 4 columns a lane ("across"); both
// are 16-byte loads, since the order of a contraction is free.  Scores are formed
// transposed, S^T = K Q^T: a lane then holds 4 keys of one query, which is the
// layout in which P is the next product's operand, and a query's running maximum
// and sum stay in its own lanes.  The waves of a workgroup take the steps of the keys
// (or rows) in turn and join at the end, in a fixed order.
//
// Masked places.  A masked score becomes -inf (P exactly 0) whatever it was, and
// where a step holds masked places the operand that P multiplies may hold an
// infinity or NaN that its row must not see (0 inf = NaN): such values are taken
// out of the product and added to the rows that see them.
//
// Measured: one token of 32 requests, 32 heads of 128 on 8 key heads, up to 8192
// keys (1.11 GB of keys and values): 187 us = 5.9 TB/s and 6 us for the join; with
// ordinary loads, keys read when they are due and a third fewer parts 222 and 12.
// One sequence of 32, 4 heads of 64: 5.6 us.  A batch of prompts multiplies at about
// 77 TFLOP/s forward, half of what the fp32 matrix cores do.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_plan.hpp"

namespace lmp_hip {
namespace {

typedef float a4 __attribute__((ext_vector_type(4)));
typedef float a4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float a2_any __attribute__((ext_vector_type(2), aligned(4)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ a4 mfma_16(float a, float b, a4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool finite(float x) {
  return (__builtin_bit_cast(uint32_t, x) & 0x7fffffffu) < 0x7f800000u;
}
// Over the four lanes that share a column of a 16 x 16 block.
__device__ __forceinline__ float column_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float column_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

struct AttnArgs {
  const AttnItem* items;
  int count, kv_heads, group, dim;
  bool causal;
  const float *q, *k, *v, *g;
  int64_t q_ld, k_ld, v_ld, g_ld;
  float scale;
  const float* lse_in;
  const float* out;    // forward's output
  int64_t out_ld;
  float* delta;        // [query][head]: rowsum(g o), which the rows leave for the keys
  float *o, *lse, *dk;  // o: forward's output or dq; dk with o as dv
  int64_t o_ld, dk_ld;
  float *part, *part_ml;  // [part][kv head][16 rows][dim], [...][16][2]
  // [sequence][key head]: not 0 where the split kernels leave the work to these
  // (attention_split.hpp); null where all of it is theirs.
  const int32_t* marks;
  const int32_t* any_mark;
};

// W values at p, zero from column `end` on.  STREAM: with the nontemporal hint.
template <int W, bool STREAM = false>
__device__ __forceinline__ void load_cols(const float* p, int col, int end, float* out) {
  if (col + W <= end) {
    if constexpr (W == 4) {
      const auto* at = reinterpret_cast<const a4_any*>(p + col);
      const a4_any x = STREAM ? __builtin_nontemporal_load(at) : *at;
      out[0] = x[0]; out[1] = x[1]; out[2] = x[2]; out[3] = x[3];
    } else if constexpr (W == 2) {
      const a2_any x = *reinterpret_cast<const a2_any*>(p + col);
      out[0] = x[0]; out[1] = x[1];
    } else {
      out[0] = p[col];
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) out[j] = col + j < end ? p[col + j] : 0.0f;
  }
}

// ND: blocks of 16 columns.  Across: column j * 16 .. of chunk j / 4 is held
// interleaved, `width` neighbouring columns a lane.
template <int ND>
struct Cols {
  static constexpr int width(int j) { return j / 4 < ND / 4 ? 4 : ND % 4; }
  static __device__ __forceinline__ int at(int j, int m) {
    return 64 * (j / 4) + width(j) * m + j % 4;
  }
};

// 16 columns x ND of one row, 4 a lane group: the operand contracted over d.
template <int ND, bool STREAM = false>
__device__ __forceinline__ void load_along(const float* row, int g, int dim, float (&f)[ND][4]) {
#pragma unroll
  for (int b = 0; b < ND; ++b) load_cols<4, STREAM>(row, 16 * b + 4 * g, dim, f[b]);
}
// One row as the operand contracted over its rows: lane m holds columns at(j, m).
template <int ND, bool STREAM = false>
__device__ __forceinline__ void load_across(const float* row, int m, int dim, float (&f)[ND]) {
#pragma unroll
  for (int c = 0; c < ND / 4; ++c) load_cols<4, STREAM>(row, 64 * c + 4 * m, dim, f + 4 * c);
  constexpr int rest = ND % 4;
  if constexpr (rest != 0)
    load_cols<rest, STREAM>(row, 64 * (ND / 4) + rest * m, dim, f + ND / 4 * 4);
}

template <int ND>
__device__ __forceinline__ a4 product_along(const float (&a)[ND][4], const float (&b)[ND][4]) {
  a4 s = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s = mfma_16(a[i][j], b[i][j], s);
  return s;
}

// acc += rows^T p over 16 rows, p the lane's 4 of them (4 g + r) for its column.
// With `masked`, infinities and NaN of the rows reach only the columns that see
// them: sees(row in 0..15) for the lane's column; row_at(row) is its address.
template <int ND, class Sees, class RowAt>
__device__ __forceinline__ void accumulate(a4 (&acc)[ND], float (&f)[4][ND], const float (&p)[4],
                                           int dim, bool masked, Sees&& sees, RowAt&& row_at) {
  bool odd = false;
  if (masked) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < ND; ++j)
        if (!finite(f[r][j])) {
          odd = true;
          f[r][j] = 0.0f;
        }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j] = mfma_16(f[r][j], p[r], acc[j]);
  if (masked && __any(odd)) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    for (int kk = 0; kk < 16; ++kk) {
      float pk = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = __shfl(p[r], (kk >> 2) * 16 + n);
        pk = (kk & 3) == r ? x : pk;
      }
      const bool s = sees(kk);
      const float* row = row_at(kk);
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int c = Cols<ND>::at(j, 4 * g + r);
          const float x = c < dim ? row[c] : 0.0f;
          if (s && !finite(x)) acc[j][r] += pk * x;
        }
    }
  }
}

// The waves' blocks [column of 16][d], summed in order and handed out:
// put(row, column, 4 values).
template <int ND, int WAVES, class Put>
__device__ __forceinline__ void join_waves(const a4 (&acc)[ND], float* lds, Put&& put) {
  constexpr int PITCH = ND * 16 + 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ND; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      lds[(wave * 16 + n) * PITCH + Cols<ND>::at(j, 4 * g + r)] = acc[j][r];
  __syncthreads();
  constexpr int LANES = WAVES * 4;  // of a row
  const int row = threadIdx.x / LANES;
  for (int c = (threadIdx.x % LANES) * 4; c < ND * 16; c += LANES * 4) {
    a4 s = *reinterpret_cast<const a4*>(lds + row * PITCH + c);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += *reinterpret_cast<const a4*>(lds + (w * 16 + row) * PITCH + c);
    put(row, c, s);
  }
}
__device__ __forceinline__ void store_cols(float* row, int col, int end, a4 x) {
  if (col + 4 <= end) {
    *reinterpret_cast<a4_any*>(row + col) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < end) row[col + j] = x[j];
  }
}

// Whether a (sequence, key head) is another set of kernels' work.
__device__ __forceinline__ bool skipped(const AttnArgs& a, const AttnItem& it, int kv) {
  return a.marks && !a.marks[int64_t(it.seq) * a.kv_heads + kv];
}

// The keys of a step are on their way while the step before it ends, its values
// while its scores are formed.  STREAM: every key is read once.
template <int ND, bool STREAM>
__global__ __launch_bounds__(256) void attention_rows(AttnArgs a) {
  if (a.marks && !*a.any_mark) return;
  __shared__ __attribute__((aligned(16))) float lds[4 * 16 * (ND * 16 + 4)];
  __shared__ float ml[2][4][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  for (int64_t w = blockIdx.x; w < int64_t(a.count) * a.kv_heads; w += gridDim.x) {
    const int kv = int(w % a.kv_heads);
    AttnItem it = a.items[w / a.kv_heads];
    if (skipped(a, it, kv)) continue;
    const int rows = min(kAttnRows, it.lq * a.group - it.first);
    if (a.marks && it.part >= 0) {  // no join follows: a split row's first part takes all its keys
      if (it.key_begin > 0) continue;
      const int last = (it.first + rows - 1) / a.group;
      it.part = -1;
      it.key_end = a.causal ? max(0, min(it.lk, last + 1 + it.lk - it.lq)) : it.lk;
    }
    const int packed = it.first + min(n, rows - 1);
    const int query = packed / a.group, head = kv * a.group + packed % a.group;
    const int limit = min(it.key_end, a.causal ? max(0, query + 1 + it.lk - it.lq) : it.lk);
    float q[ND][4];
    load_along<ND>(a.q + int64_t(it.q0 + query) * a.q_ld + int64_t(head) * a.dim, g, a.dim, q);
    const float c = a.scale * kLog2e;
    const float* k0 = a.k + int64_t(it.k0) * a.k_ld + int64_t(kv) * a.dim;
    const float* v0 = a.v + int64_t(it.k0) * a.v_ld + int64_t(kv) * a.dim;
    a4 acc[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j] = a4{0, 0, 0, 0};
    float top = -__builtin_inff(), sum = 0;
    float k[ND][4];
    const auto load_keys = [&](int kt) {
      load_along<ND, STREAM>(k0 + int64_t(min(kt + n, it.lk - 1)) * a.k_ld, g, a.dim, k);
    };
    const int begin = it.key_begin + wave * 16;
    if (begin < it.key_end) load_keys(begin);
    for (int kt = begin; kt < it.key_end; kt += 64) {
      const auto key = [&](int i) { return min(kt + i, it.lk - 1); };
      float v[4][ND];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        load_across<ND, STREAM>(v0 + int64_t(key(4 * g + r)) * a.v_ld, n, a.dim, v[r]);
      const a4 s = product_along<ND>(k, q);
      if (kt + 64 < it.key_end) load_keys(kt + 64);
      float p[4], best = top;
      bool whole = true;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool seen = kt + 4 * g + r < limit;
        whole = whole && seen;
        p[r] = seen ? s[r] * c : -__builtin_inff();
        best = fmaxf(best, p[r]);
      }
      best = column_max(best);
      const float base = best > -__builtin_inff() ? best : 0.0f;
      const float fade = exp2_of(top - base);  // 0 at the first keys
      top = best;
      sum *= fade;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = exp2_of(p[r] - base);
        sum += p[r];
      }
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[j] *= fade;
      accumulate<ND>(acc, v, p, a.dim, __any(!whole), [&](int i) { return kt + i < limit; },
                     [&](int i) { return v0 + int64_t(key(i)) * a.v_ld; });
    }
    sum = column_sum(sum);
    if (g == 0) {
      ml[0][wave][n] = top;
      ml[1][wave][n] = sum;
    }
    __syncthreads();
    float all = ml[0][0][n];
#pragma unroll
    for (int i = 1; i < 4; ++i) all = fmaxf(all, ml[0][i][n]);
    const float base = all > -__builtin_inff() ? all : 0.0f;
    float total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) total += ml[1][i][n] * exp2_of(ml[0][i][n] - base);
    float mine = exp2_of(top - base);
    if (it.part < 0) mine = total > 0 || total != total ? mine / total : 0.0f;
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j] *= mine;
    const int64_t slot = int64_t(it.part) * a.kv_heads + kv;
    if (wave == 0 && g == 0 && n < rows) {
      if (it.part >= 0) {
        a.part_ml[(slot * 16 + n) * 2] = all;
        a.part_ml[(slot * 16 + n) * 2 + 1] = total;
      } else if (a.lse) {
        a.lse[int64_t(it.q0 + query) * (a.kv_heads * a.group) + head] =
            (base + __builtin_amdgcn_logf(total)) * kLn2;
      }
    }
    join_waves<ND, 4>(acc, lds, [&](int row, int col, a4 x) {
      if (row >= rows) return;
      const int r = it.first + row;
      float* to = it.part >= 0
                      ? a.part + (slot * 16 + row) * a.dim
                      : a.o + int64_t(it.q0 + r / a.group) * a.o_ld +
                            int64_t(kv * a.group + r % a.group) * a.dim;
      store_cols(to, col, a.dim, x);
    });
    __syncthreads();
  }
}

// Joins the parts of ROWS packed rows: 16 lanes a row, 16 rows a workgroup.
template <int ROWS>
__global__ __launch_bounds__(256) void attention_join(AttnArgs a, const AttnJoin* joins, int count) {
  const int64_t work = int64_t(count) * a.kv_heads * (ROWS / 16);
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int64_t item = w / (ROWS / 16);
    const int kv = int(item % a.kv_heads);
    const AttnJoin j = joins[item / a.kv_heads];
    const int rows = min(ROWS, j.lq * a.group - j.first);
    const int row = int(w % (ROWS / 16)) * 16 + (threadIdx.x >> 4);
    if (row >= rows) continue;
    const auto slot = [&](int p) {
      return ((int64_t(j.part) + p) * a.kv_heads + kv) * ROWS + row;
    };
    // The row's 16 lanes look at its parts side by side, then take its columns.
    const int lane = threadIdx.x & 15;
    const auto over_lanes = [](float x, auto&& f) {
      x = f(x, __shfl_xor(x, 1));
      x = f(x, __shfl_xor(x, 2));
      x = f(x, __shfl_xor(x, 4));
      return f(x, __shfl_xor(x, 8));
    };
    float all = -__builtin_inff();
    for (int p = lane; p < j.parts; p += 16) all = fmaxf(all, a.part_ml[slot(p) * 2]);
    all = over_lanes(all, [](float x, float y) { return fmaxf(x, y); });
    const float base = all > -__builtin_inff() ? all : 0.0f;
    float total = 0;
    for (int p = lane; p < j.parts; p += 16)
      total += a.part_ml[slot(p) * 2 + 1] * exp2_of(a.part_ml[slot(p) * 2] - base);
    total = over_lanes(total, [](float x, float y) { return x + y; });
    const float one = total > 0 || total != total ? 1.0f / total : 0.0f;
    const int r = j.first + row, query = r / a.group, head = kv * a.group + r % a.group;
    float* to = a.o + int64_t(j.q0 + query) * a.o_ld + int64_t(head) * a.dim;
    for (int c = lane * 4; c < a.dim; c += 64) {
      a4 s = {0, 0, 0, 0};
#pragma unroll 8
      for (int p = 0; p < j.parts; ++p) {
        float x[4];
        load_cols<4>(a.part + slot(p) * a.dim, c, a.dim, x);
        const float f = exp2_of(a.part_ml[slot(p) * 2] - base);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(f, x[i], s[i]);
      }
      store_cols(to, c, a.dim, s * one);
    }
    if (a.lse && (threadIdx.x & 15) == 0)
      a.lse[int64_t(j.q0 + query) * (a.kv_heads * a.group) + head] =
          (base + __builtin_amdgcn_logf(total)) * kLn2;
  }
}

// A row's lse in base 2; +inf, which makes its P zero, where it sees nothing.
__device__ __forceinline__ float lse2_of(float lse) {
  return lse == -__builtin_inff() ? __builtin_inff() : lse * kLog2e;
}

// The backward workgroups have four waves, or eight where there are few of them:
// half as many steps in turn, at half the workgroups on a compute unit (one
// sequence of 256, 4 heads of 64: 34 us with four, 28 with eight; 16 of 64, 16
// heads of 64: 39 and 52).
template <int ND, int WAVES>
__device__ __forceinline__ void back_rows(const AttnArgs& a, float* lds) {
  constexpr int STEP = WAVES * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  const int heads = a.kv_heads * a.group;
  for (int64_t w = blockIdx.x; w < int64_t(a.count) * a.kv_heads; w += gridDim.x) {
    const int kv = int(w % a.kv_heads);
    const AttnItem it = a.items[w / a.kv_heads];
    if (it.part >= 0 && it.key_begin > 0) continue;  // a split row's first part takes all its keys
    if (skipped(a, it, kv)) continue;
    const int rows = min(kAttnRows, it.lq * a.group - it.first);
    const int packed = it.first + min(n, rows - 1);
    const int query = packed / a.group, head = kv * a.group + packed % a.group;
    const int limit = a.causal ? max(0, query + 1 + it.lk - it.lq) : it.lk;
    const int last = (it.first + rows - 1) / a.group;
    const int key_end = a.causal ? max(0, min(it.lk, last + 1 + it.lk - it.lq)) : it.lk;
    float q[ND][4], go[ND][4];
    load_along<ND>(a.q + int64_t(it.q0 + query) * a.q_ld + int64_t(head) * a.dim, g, a.dim, q);
    load_along<ND>(a.g + int64_t(it.q0 + query) * a.g_ld + int64_t(head) * a.dim, g, a.dim, go);
    const float c = a.scale * kLog2e;
    const float lse2 = lse2_of(a.lse_in[int64_t(it.q0 + query) * heads + head]);
    float delta = 0;
    if (a.marks) {  // the splitting kernel has left it
      delta = a.delta[int64_t(it.q0 + query) * heads + head];
    } else {
#pragma unroll
      for (int b = 0; b < ND; ++b) {
        float o[4];
        load_cols<4>(a.out + int64_t(it.q0 + query) * a.out_ld + int64_t(head) * a.dim,
                     16 * b + 4 * g, a.dim, o);
#pragma unroll
        for (int j = 0; j < 4; ++j) delta = fmaf(go[b][j], o[j], delta);
      }
      delta = column_sum(delta);
      if (wave == 0 && g == 0 && n < rows) a.delta[int64_t(it.q0 + query) * heads + head] = delta;
    }
    const float* k0 = a.k + int64_t(it.k0) * a.k_ld + int64_t(kv) * a.dim;
    const float* v0 = a.v + int64_t(it.k0) * a.v_ld + int64_t(kv) * a.dim;
    a4 acc[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j] = a4{0, 0, 0, 0};
    for (int kt = wave * 16; kt < key_end; kt += STEP) {
      const auto key = [&](int i) { return min(kt + i, it.lk - 1); };
      float k[ND][4], v[ND][4], kc[4][ND];
      load_along<ND>(k0 + int64_t(key(n)) * a.k_ld, g, a.dim, k);
      load_along<ND>(v0 + int64_t(key(n)) * a.v_ld, g, a.dim, v);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        load_across<ND>(k0 + int64_t(key(4 * g + r)) * a.k_ld, n, a.dim, kc[r]);
      const a4 s = product_along<ND>(k, q), dp = product_along<ND>(v, go);
      float ds[4];
      bool whole = true;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool seen = kt + 4 * g + r < limit;
        whole = whole && seen;
        ds[r] = seen ? exp2_of(s[r] * c - lse2) * (dp[r] - delta) * a.scale : 0.0f;
      }
      accumulate<ND>(acc, kc, ds, a.dim, __any(!whole), [&](int i) { return kt + i < limit; },
                     [&](int i) { return k0 + int64_t(key(i)) * a.k_ld; });
    }
    join_waves<ND, WAVES>(acc, lds, [&](int row, int col, a4 x) {
      if (row >= rows) return;
      const int r = it.first + row;
      store_cols(a.o + int64_t(it.q0 + r / a.group) * a.o_ld +
                     int64_t(kv * a.group + r % a.group) * a.dim,
                 col, a.dim, x);
    });
    __syncthreads();
  }
}

template <int ND, int WAVES>
__device__ __forceinline__ void back_keys(const AttnArgs& a, float* lds) {
  constexpr int STEP = WAVES * 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
  const int heads = a.kv_heads * a.group;
  for (int64_t w = blockIdx.x; w < int64_t(a.count) * a.kv_heads; w += gridDim.x) {
    const int kv = int(w % a.kv_heads);
    const AttnItem it = a.items[w / a.kv_heads];
    if (skipped(a, it, kv)) continue;
    const int keys = min(kAttnRows, it.lk - it.first), key = it.first + min(n, keys - 1);
    const int rows = it.lq * a.group, ahead = it.lk - it.lq;
    // The first query that sees the first key here.
    const int from = a.causal ? max(0, it.first - ahead) * a.group / 16 * 16 : 0;
    float k[ND][4], v[ND][4];
    load_along<ND>(a.k + int64_t(it.k0 + key) * a.k_ld + int64_t(kv) * a.dim, g, a.dim, k);
    load_along<ND>(a.v + int64_t(it.k0 + key) * a.v_ld + int64_t(kv) * a.dim, g, a.dim, v);
    const float c = a.scale * kLog2e;
    a4 dk[ND], dv[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) dk[j] = dv[j] = a4{0, 0, 0, 0};
    for (int rt = from + wave * 16; rt < rows; rt += STEP) {
      const auto packed = [&](int i) { return min(rt + i, rows - 1); };
      const auto q_at = [&](int i) {
        const int r = packed(i);
        return a.q + int64_t(it.q0 + r / a.group) * a.q_ld +
               int64_t(kv * a.group + r % a.group) * a.dim;
      };
      const auto g_at = [&](int i) {
        const int r = packed(i);
        return a.g + int64_t(it.q0 + r / a.group) * a.g_ld +
               int64_t(kv * a.group + r % a.group) * a.dim;
      };
      const auto sees = [&](int i) {
        return rt + i < rows && (!a.causal || key <= (rt + i) / a.group + ahead);
      };
      float q[ND][4], go[ND][4];
      load_along<ND>(q_at(n), g, a.dim, q);
      load_along<ND>(g_at(n), g, a.dim, go);
      const a4 s = product_along<ND>(q, k), dp = product_along<ND>(go, v);
      float p[4], ds[4];
      bool whole = true;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 4 * g + r, at = packed(i);
        const int64_t stat =
            int64_t(it.q0 + at / a.group) * heads + kv * a.group + at % a.group;
        const bool seen = sees(i);
        whole = whole && seen;
        p[r] = seen ? exp2_of(s[r] * c - lse2_of(a.lse_in[stat])) : 0.0f;
        ds[r] = seen ? p[r] * (dp[r] - a.delta[stat]) * a.scale : 0.0f;
      }
      const bool masked = __any(!whole);
      float f[4][ND];
#pragma unroll
      for (int r = 0; r < 4; ++r) load_across<ND>(g_at(4 * g + r), n, a.dim, f[r]);
      accumulate<ND>(dv, f, p, a.dim, masked, sees, g_at);
#pragma unroll
      for (int r = 0; r < 4; ++r) load_across<ND>(q_at(4 * g + r), n, a.dim, f[r]);
      accumulate<ND>(dk, f, ds, a.dim, masked, sees, q_at);
    }
    join_waves<ND, WAVES>(dv, lds, [&](int row, int col, a4 x) {
      if (row < keys)
        store_cols(a.o + int64_t(it.k0 + it.first + row) * a.o_ld + int64_t(kv) * a.dim, col, a.dim,
                   x);
    });
    join_waves<ND, WAVES>(dk, lds, [&](int row, int col, a4 x) {
      if (row < keys)
        store_cols(a.dk + int64_t(it.k0 + it.first + row) * a.dk_ld + int64_t(kv) * a.dim, col,
                   a.dim, x);
    });
    __syncthreads();
  }
}

template <int ND, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attention_back_rows(AttnArgs a) {
  __shared__ __attribute__((aligned(16))) float lds[WAVES * 16 * (ND * 16 + 4)];
  back_rows<ND, WAVES>(a, lds);
}
template <int ND, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attention_back_keys(AttnArgs a) {
  __shared__ __attribute__((aligned(16))) float lds[WAVES * 16 * (ND * 16 + 4)];
  back_keys<ND, WAVES>(a, lds);
}
// Both over what the split kernels have left, in one launch: nothing as a rule.
template <int ND>
__global__ __launch_bounds__(256) void attention_back_marked(AttnArgs rows, AttnArgs keys) {
  __shared__ __attribute__((aligned(16))) float lds[4 * 16 * (ND * 16 + 4)];
  if (!*rows.any_mark) return;
  back_rows<ND, 4>(rows, lds);
  back_keys<ND, 4>(keys, lds);
}

}  // namespace
}  // namespace lmp_hip
