// Packed attention on the fp16 matrix cores, each operand split into two fp16
// parts: the kernels of long batches.
//
// Why.  The fp32 MFMAs do 157 TFLOP/s, those of fp16 sixteen times that.  A value
// scaled by a power of two is x = h + l + r with h = fp16(x), l = fp16(x - h) and
// |r| <= 2^-23 |x|, so
//   a b = ah bh + ah bl + al bh + (al bl: at most 2^-22 |a b|, 2^-24.6 rms)
// is three fp16 MFMAs with fp32 accumulation, a sixth of the fp32 form's time, with
// a product's error near that of rounding its operands.
//
// Range.  Operands are split per tile of 32 rows of one head, with the power of
// two that takes the tile's largest magnitude to [2^14, 2^15): values down to
// 2^-17 of it keep both parts whole, smaller ones lose at most 2^-40 of it.  The
// powers of two go into the factors of the scores and weights, which are exact.
// A tile with an infinity or a NaN, with a largest value outside [2^-60, 2^41) or
// with rows more than 2^12 apart is marked, and the sequence's key head is left
// to the fp32 kernels (attention_f32.hpp), which run over the marked ones only (one
// such row of the output gradient: 8192 positions backward 20.8 ms for 3.0).
// Weights take a power of two per row that follows its largest so far: of P times the
// value tile's own in the forward pass, so that a tile of large values which hardly
// weigh leaves the others their digits; of P and dS in the backward pass, per query (dq)
// or key (dk, dv), so that a key that few see keeps its gradient's.
//
// Layout.  A first kernel writes the operands as MFMA fragments: the 16 bytes of
// each lane, a fragment's 64 lanes one after another, so that a workgroup's
// tiles go to LDS by direct loads and every LDS read is 1 KiB in lane order,
// free of conflicts.  "Along" fragments (32 rows x 16 columns) are contracted over
// d; "across" ones (32 columns x 16 rows) over rows, their rows in the order in
// which a lane of the 32 x 32 accumulator holds them: scores are formed so that
// a lane's own values are the next product's operand, and no value changes lanes.
//   forward  S^T = K Q^T,  O^T += V^T P^T          a lane holds one query
//   dq       S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T        one query
//   dk, dv   S = Q K^T,   dP = dO V^T,   dV^T += dO^T P, dK^T += Q^T dS   one key
//
// Measured, one causal sequence of 8192, 16 heads of 128 (key heads of four
// each): forward 0.82 ms = 336 TFLOP/s of fp32 products = 1.01 PFLOP/s of fp16 (0.80 ms
// without the two comparisons a step that keep large scores and large values sound), dq
// 1.18 ms = 1.05, dk and dv 1.72 ms = 0.96, where a library's fp16 product of 8192^3 does
// 1.09 on the same card; the fp32 kernels took 22 ms for all of it.  The matrix
// cores are busy 51, 49 and 44% of the cycles, and the clock falls by a sixth under
// them in a loop of calls: power bounds it as much as the waits at the steps' barriers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "attention_f32.hpp"

namespace lmp_hip {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float s2 __attribute__((ext_vector_type(2)));
typedef float s16 __attribute__((ext_vector_type(16)));
typedef uint32_t w4 __attribute__((ext_vector_type(4)));

constexpr int kIrregular = 1000;  // a marked tile's exponent
constexpr int kZeroTile = -128;   // of a tile of zeros
constexpr int kLeastExponent = -60, kMostExponent = 40, kRowsApart = 12;
// Least power of two that the forward pass counts a row's weighted values in: what it
// loses lies 2^40 below, and its factors keep above float32's smallest normal.
constexpr int kLeastPower = -80;

__device__ __forceinline__ s16 mfma_h(h8 a, h8 b, s16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void lds_load16(const char* src, char* lds) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const float*>(src),
                                   reinterpret_cast<float*>(lds), 16, 0, 0);
}
// This wave's loads have arrived, and then the workgroup's.
__device__ __forceinline__ void tiles_arrived() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
  asm volatile("s_barrier" ::: "memory");
}
// The same, and this wave's LDS accesses are done.
__device__ __forceinline__ void step_begins() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(7 << 4);
  asm volatile("s_barrier" ::: "memory");
}
// This wave's LDS accesses are done, and then the workgroup's.
__device__ __forceinline__ void lds_settled() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (3 << 14));
  asm volatile("s_barrier" ::: "memory");
}
__device__ __forceinline__ float times2(float x, int e) { return __builtin_ldexpf(x, e); }
// The values of the two lanes (n and n + 32) that share a column, in both of
// them.  An asm because the builtin of this instruction gives its first result
// twice; the wait states are those it needs after a VALU write.
__device__ __forceinline__ void both_halves(float x, float& low, float& high) {
  low = high = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(low), "+v"(high));
}
__device__ __forceinline__ float both_max(float x) {
  float low, high;
  both_halves(x, low, high);
  return fmaxf(low, high);
}
__device__ __forceinline__ float both_sum(float x) {
  float low, high;
  both_halves(x, low, high);
  return low + high;
}
// Two values into their parts, packed.
__device__ __forceinline__ void split_two(float x, float y, uint32_t& h, uint32_t& l) {
  const h2 hi = __builtin_convertvector(s2{x, y}, h2);
  h = __builtin_bit_cast(uint32_t, hi);
  l = __builtin_bit_cast(uint32_t, __builtin_convertvector(s2{x - float(hi[0]), y - float(hi[1])}, h2));
}
// The 16 values of an accumulator lane as two fragments of 16 rows each.
struct Halves {
  h8 h[2], l[2];
};
__device__ __forceinline__ Halves split_lane(const float (&x)[16]) {
  Halves out;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    w4 h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a, b;
      split_two(x[8 * u + 2 * i], x[8 * u + 2 * i + 1], a, b);
      h[i] = a;
      l[i] = b;
    }
    out.h[u] = __builtin_bit_cast(h8, h);
    out.l[u] = __builtin_bit_cast(h8, l);
  }
  return out;
}
// Row (of 32) of accumulator value r in the wave's first half; 4 more in the other.
constexpr int row_of(int r) { return 8 * (r >> 2) + (r & 3); }

// ND: blocks of 16 columns; NT: of 32.  Bytes of one tile of one head.
template <int ND>
struct Frag {
  static constexpr int NT = (ND + 1) / 2;
  static constexpr int ALONG = ND * 2048, ACROSS = NT * 4096;
};

struct SplitOperand {
  const float* x;  // of its first head
  int64_t ld;
  const AttnTile* tiles;
  int tile_count, heads;
  float sign;
  char *along, *across;  // fragments [tile][head], or null
  int32_t* exponent;     // [tile][head]
  // With x the output gradient: the forward output and lse, for what the backward
  // kernels read, lse in base 2 (+inf where a row sees nothing or is past its
  // sequence) and delta = rowsum(x out), per tile and head one after another, and
  // delta once more by query and head for the marked ones.  Else null.
  const float* out;
  int64_t out_ld;
  const float* lse;
  float *stats, *delta;
};
struct SplitArgs {
  SplitOperand op[4];
  int count, dim;
  int32_t* any_mark;
};

// One tile of one head per workgroup.
template <int ND>
__global__ __launch_bounds__(256) void attention_split(SplitArgs a) {
  constexpr int NT = Frag<ND>::NT, PITCH = NT * 32 + 4, UNITS = NT * 8;
  __shared__ __attribute__((aligned(16))) float tile[32 * PITCH];
  __shared__ uint32_t row_top[32];
  int64_t w = blockIdx.x;
  if (w == 0 && threadIdx.x == 0) *a.any_mark = 0;
  int which = 0;
  while (which + 1 < a.count && w >= int64_t(a.op[which].tile_count) * a.op[which].heads) {
    w -= int64_t(a.op[which].tile_count) * a.op[which].heads;
    ++which;
  }
  const SplitOperand& op = a.op[which];
  const int head = int(w % op.heads);
  const AttnTile t = op.tiles[w / op.heads];
  if (threadIdx.x < 32) row_top[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * UNITS; i += 256) {
    const int row = i / UNITS, col = i % UNITS * 4;
    float x[4] = {0, 0, 0, 0};
    if (row < t.rows) load_cols<4>(op.x + (int64_t(t.at) + row) * op.ld + int64_t(head) * a.dim, col, a.dim, x);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
    *reinterpret_cast<a4*>(tile + row * PITCH + col) = a4{x[0], x[1], x[2], x[3]};
    if (top) atomicMax(&row_top[row], top);
  }
  __syncthreads();
  uint32_t most = row_top[threadIdx.x & 31], least = most ? most : 0x7fffffffu;
#pragma unroll
  for (int s = 1; s < 32; s *= 2) {
    most = max(most, uint32_t(__shfl_xor(int(most), s)));
    least = min(least, uint32_t(__shfl_xor(int(least), s)));
  }
  const int e = int(most >> 23) - 127, e_least = int(least >> 23) - 127;
  const bool marked = most >= 0x7f800000u ||
                      (most && (e < kLeastExponent || e > kMostExponent || e_least < e - kRowsApart));
  if (threadIdx.x == 0) op.exponent[w] = marked ? kIrregular : most ? e : kZeroTile;
  if (op.out) {  // 8 lanes a row
    const int row = threadIdx.x >> 3;
    const int64_t at = int64_t(t.at) + min(row, t.rows - 1);
    const float* out = op.out + at * op.out_ld + int64_t(head) * a.dim;
    float s = 0;
    for (int c = (threadIdx.x & 7) * 4; c < a.dim; c += 32) {
      float y[4];
      load_cols<4>(out, c, a.dim, y);
      const a4 x = *reinterpret_cast<const a4*>(tile + row * PITCH + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fmaf(x[j], y[j], s);
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    s += __shfl_xor(s, 4);
    if ((threadIdx.x & 7) == 0) {
      const bool there = row < t.rows;
      op.stats[w * 64 + row] = there ? lse2_of(op.lse[at * op.heads + head]) : __builtin_inff();
      op.stats[w * 64 + 32 + row] = there ? s : 0.0f;
      if (there) op.delta[at * op.heads + head] = s;
    }
  }
  if (marked) return;
  const float scale = most ? times2(op.sign, 14 - e) : 0.0f;
  const auto put = [&](char* to, const float (&x)[8]) {
    w4 h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p, q;
      split_two(x[2 * i] * scale, x[2 * i + 1] * scale, p, q);
      h[i] = p;
      l[i] = q;
    }
    *reinterpret_cast<w4*>(to) = h;
    *reinterpret_cast<w4*>(to + 1024) = l;
  };
  if (op.along) {
    char* to = op.along + w * Frag<ND>::ALONG;
    for (int f = threadIdx.x; f < ND * 64; f += 256) {
      const int lane = f & 63, s = f >> 6;
      const float* from = tile + (lane & 31) * PITCH + 16 * s + 8 * (lane >> 5);
      const a4 p = *reinterpret_cast<const a4*>(from), q = *reinterpret_cast<const a4*>(from + 4);
      const float x[8] = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
      put(to + s * 2048 + lane * 16, x);
    }
  }
  if (op.across) {
    char* to = op.across + w * Frag<ND>::ACROSS;
    for (int f = threadIdx.x; f < NT * 128; f += 256) {
      const int lane = f & 63, u = (f >> 6) & 1, m = f >> 7;
      const float* from = tile + (16 * u + 4 * (lane >> 5)) * PITCH + 32 * m + (lane & 31);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = from[(j < 4 ? j : j + 4) * PITCH];
      put(to + (m * 2 + u) * 2048 + lane * 16, x);
    }
  }
}

// Marks the sequences' key heads that have a marked tile of any operand, and
// whether there is one.
__global__ __launch_bounds__(256) void attention_marks(const AttnSeq* seqs, int kv_heads, int group,
                                                      const int32_t* q_exp, const int32_t* k_exp,
                                                      const int32_t* v_exp, const int32_t* g_exp,
                                                      int32_t* marks, int32_t* any_mark) {
  const int kv = int(blockIdx.x % kv_heads);
  const AttnSeq s = seqs[blockIdx.x / kv_heads];
  bool odd = false;
  for (int t = threadIdx.x; t < s.k_tiles; t += 256) {
    const int64_t at = int64_t(s.kt0 + t) * kv_heads + kv;
    odd = odd || k_exp[at] == kIrregular || v_exp[at] == kIrregular;
  }
  for (int t = threadIdx.x; t < s.q_tiles * group; t += 256) {
    const int64_t at = int64_t(s.qt0 + t / group) * kv_heads * group + kv * group + t % group;
    odd = odd || q_exp[at] == kIrregular || (g_exp && g_exp[at] == kIrregular);
  }
  const bool any = __syncthreads_or(odd);
  if (threadIdx.x == 0) {
    marks[blockIdx.x] = any;
    if (any) *any_mark = 1;  // cleared by attention_split
  }
}

struct SplitAttnArgs {
  const AttnItem* items;
  int count, kv_heads, group, dim;
  bool causal;
  float scale_log2e;  // |scale| log2 e; the sign is in q's parts
  float scale;        // |scale| for dk, the scale itself for dq
  const char *q_along, *q_across, *k_along, *k_across, *v_along, *v_across, *g_along, *g_across;
  const int32_t *q_exp, *k_exp, *v_exp, *g_exp;
  const int32_t* marks;  // [sequence][key head]
  const float* stats;  // [query tile][head][lse2 of 32 rows, delta of 32 rows]
  float *o, *lse, *dk;
  int64_t o_ld, dk_ld;
  float *part, *part_ml;  // [part][head][128 rows][dim], [...][128][2]
  int64_t part_dk;        // from dv's parts to dk's
};

// A tile's exponent, through the scalar cache: a vector load would wait for the
// tiles that are on their way to LDS.
__device__ __forceinline__ int exponent_at(const int32_t* exponents, int64_t at) {
  typedef const int32_t __attribute__((address_space(4)))* scalar_ptr;
  const uint32_t low = __builtin_amdgcn_readfirstlane(uint32_t(at));
  const uint32_t high = __builtin_amdgcn_readfirstlane(uint32_t(uint64_t(at) >> 32));
  return reinterpret_cast<scalar_ptr>(
      reinterpret_cast<uintptr_t>(exponents))[int64_t((uint64_t(high) << 32) | low)];
}

// Heads that share keys, on one XCD (consecutive workgroups go round the eight).
__device__ __forceinline__ int head_of(int slot, int heads) {
  return heads % 8 == 0 ? slot % 8 * (heads / 8) + slot / 8 : slot;
}

__device__ __forceinline__ const h8& frag(const char* lds, int index) {
  return *reinterpret_cast<const h8*>(lds + index * 1024 + (threadIdx.x & 63) * 16);
}
template <int ND>
__device__ __forceinline__ void load_own(const char* tile, h8 (&h)[ND], h8 (&l)[ND]) {
#pragma unroll
  for (int s = 0; s < ND; ++s) {
    h[s] = frag(tile, 2 * s);
    l[s] = frag(tile, 2 * s + 1);
  }
}
// Orders the instructions around it as `READS` LDS reads, then `MFMAS` products.
template <int READS, int MFMAS>
__device__ __forceinline__ void reads_then_products() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  __builtin_amdgcn_sched_group_barrier(0x008, MFMAS, 0);
}
// Rows (an LDS tile, along) times the wave's own rows.  The fragments of a step of
// 16 columns are read two steps ahead; left to itself the compiler reads each one
// when it is due and waits for it.  The small terms add up apart from the leading
// ones.
template <int ND>
__device__ __forceinline__ void product(const char* lds, const h8 (&h)[ND], const h8 (&l)[ND],
                                        float (&out)[16]) {
  s16 lead = s16(0.0f), low = s16(0.0f);
#pragma unroll
  for (int s = 0; s < ND; ++s) {
    const h8 ah = frag(lds, 2 * s), al = frag(lds, 2 * s + 1);
    low = mfma_h(al, h[s], low);
    lead = mfma_h(ah, h[s], lead);
    low = mfma_h(ah, l[s], low);
  }
  reads_then_products<4, 0>();
#pragma unroll
  for (int s = 0; s < ND; ++s) reads_then_products<2, 3>();
#pragma unroll
  for (int r = 0; r < 16; ++r) out[r] = lead[r] + low[r];
}
// acc += (an LDS tile, across) times the lane's 32 values: two blocks of columns at
// a time, so that no product waits for the one before it, and their fragments
// read one pair ahead.
template <int NT>
__device__ __forceinline__ void accumulate_tile(const char* lds, const Halves& p, s16 (&acc)[NT]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int m = 0; m < NT; m += 2) {
      constexpr int two = 2;
      h8 ah[two], al[two];
#pragma unroll
      for (int i = 0; i < two && m + i < NT; ++i) {
        ah[i] = frag(lds, ((m + i) * 2 + u) * 2);
        al[i] = frag(lds, ((m + i) * 2 + u) * 2 + 1);
      }
#pragma unroll
      for (int i = 0; i < two && m + i < NT; ++i) acc[m + i] = mfma_h(al[i], p.h[u], acc[m + i]);
#pragma unroll
      for (int i = 0; i < two && m + i < NT; ++i) acc[m + i] = mfma_h(ah[i], p.l[u], acc[m + i]);
#pragma unroll
      for (int i = 0; i < two && m + i < NT; ++i) acc[m + i] = mfma_h(ah[i], p.h[u], acc[m + i]);
    }
  reads_then_products<NT == 1 ? 2 : 4, 0>();
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int m = 0; m < NT; m += 2) {
      if (m + 1 < NT) reads_then_products<4, 6>();
      else reads_then_products<2, 3>();
    }
}
// A lane's column of the transposed result: `row` is its row in memory.
template <int NT>
__device__ __forceinline__ void store_lane(float* row, int dim, int half, const s16 (&acc)[NT],
                                           float factor) {
#pragma unroll
  for (int m = 0; m < NT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 32 * m + 8 * i + 4 * half;
      store_cols(row, col, dim,
                 a4{acc[m][4 * i], acc[m][4 * i + 1], acc[m][4 * i + 2], acc[m][4 * i + 3]} * factor);
    }
}
template <int NT>
__device__ __forceinline__ void scale_acc(s16 (&acc)[NT], float f) {
#pragma unroll
  for (int m = 0; m < NT; ++m) acc[m] *= f;
}

// The pointer in scalar registers (it is the same in every lane).
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t x = reinterpret_cast<uint64_t>(p);
  const uint32_t low = __builtin_amdgcn_readfirstlane(uint32_t(x));
  const uint32_t high = __builtin_amdgcn_readfirstlane(uint32_t(x >> 32));
  return reinterpret_cast<const char*>((uint64_t(high) << 32) | low);
}
// Copies CHUNKS KiB to LDS, the WAVES waves in turn.
template <int CHUNKS, int WAVES = 4>
__device__ __forceinline__ void fetch(const char* src, char* lds, int wave) {
  const char* from = uniform(src + wave * 1024);
  const uint32_t lane = (threadIdx.x & 63) * 16;
#pragma unroll
  for (int i = 0; i < (CHUNKS + WAVES - 1) / WAVES; ++i) {
    if (CHUNKS % WAVES == 0 || i * WAVES + wave < CHUNKS)
      lds_load16(from + i * WAVES * 1024 + lane, lds + (i * WAVES + wave) * 1024);
  }
}

// The power of two that takes a lane's dS or P (times 2^e) below 2^15, following its
// largest value so far; two bits are kept free so that it seldom moves.
struct Follower {
  int f = -1000;
  // Returns the power to apply to x; `acc` follows when f moves.
  template <int NT>
  __device__ __forceinline__ int follow(const float (&x)[16], int e, s16 (&acc)[NT]) {
    float top = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
    top = both_max(top);
    const int need = top > 0 ? __builtin_amdgcn_frexp_expf(top) + e - 15 : -1000;
    if (__any(need > f)) {
      const int next = need > f ? need + 2 : f;
      scale_acc(acc, times2(1.0f, max(f - next, -200)));
      f = next;
    }
    return e - f;
  }
};

template <int ND>
__global__ __launch_bounds__(256, 2) void attention_split_rows(SplitAttnArgs a) {
  constexpr int NT = Frag<ND>::NT, STAGE = Frag<ND>::ALONG + Frag<ND>::ACROSS;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, n = lane & 31, heads = a.kv_heads * a.group;
  const int head = head_of(int(blockIdx.x % heads), heads), kv = head / a.group;
  const AttnItem it = a.items[blockIdx.x / heads];
  const int tile0 = it.key_begin / kAttnTile, tiles = (it.key_end - it.key_begin + 31) / kAttnTile;
  const auto fetch_tile = [&](int t) {
    const int64_t at = int64_t(it.kt0 + tile0 + t) * a.kv_heads + kv;
    char* to = lds + (t & 1) * STAGE;
    fetch<ND * 2>(a.k_along + at * Frag<ND>::ALONG, to, wave);
    fetch<NT * 4>(a.v_across + at * Frag<ND>::ACROSS, to + Frag<ND>::ALONG, wave);
  };
  if (a.marks[int64_t(it.seq) * a.kv_heads + kv]) return;
  if (tiles > 0) fetch_tile(0);
  // A wave's queries; waves past the sequence repeat its last tile and store nothing.
  const int first = it.first + 32 * wave, own = min(first / 32, (it.lq - 1) / 32);
  const bool live = first + n < it.lq;
  const int query = min(first + n, it.lq - 1), last = min(first + 31, it.lq - 1);
  const auto seen_by = [&](int q) {
    return min(it.key_end, a.causal ? max(0, q + 1 + it.lk - it.lq) : it.lk);
  };
  const int limit = seen_by(query), whole = seen_by(min(first, it.lq - 1));
  const int end = first < it.lq ? seen_by(last) : 0;
  const int64_t q_at = int64_t(it.qt0 + own) * heads + head;
  h8 qh[ND], ql[ND];
  load_own<ND>(a.q_along + q_at * Frag<ND>::ALONG, qh, ql);
  const int eq = a.q_exp[q_at];
  s16 acc[NT];
#pragma unroll
  for (int m = 0; m < NT; ++m) acc[m] = s16(0.0f);
  float top = -__builtin_inff(), sum = 0;
  float size = kLeastPower;
  int power = kLeastPower;  // acc is O 2^(29 - power)
  for (int t = 0; t < tiles; ++t) {
    const int64_t at = int64_t(it.kt0 + tile0 + t) * a.kv_heads + kv;
    const int ek = exponent_at(a.k_exp, at), ev = exponent_at(a.v_exp, at);
    tiles_arrived();
    if (t + 1 < tiles) fetch_tile(t + 1);
    const int key0 = (tile0 + t) * kAttnTile;
    if (key0 >= end) continue;
    const char* stage = lds + (t & 1) * STAGE;
    float s[16];
    product<ND>(stage, qh, ql, s);
    if (key0 + 32 > whole) {
      const int seen = limit - key0 - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = row_of(r) < seen ? s[r] : -__builtin_inff();
    }
    float best = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) best = fmaxf(best, s[r]);
    best = both_max(best);
    // Kept above zero: -inf times it stays -inf.
    const float c = fmaxf(times2(a.scale_log2e, ek + eq - 28), 1e-37f);
    const float here = best * c, next = fmaxf(top, here);
    const float base = next > -__builtin_inff() ? next : 0.0f;
    // The tile's weights are up to 2^(here - base), times 2^ev: 2^size follows the row's
    // largest so far and falls with it as the weights fade; `power` lies a bit above it,
    // so that it seldom moves.
    if (__any(next > top || ev > power)) {
      size = fmaxf(fmaxf(size - (next - top), float(ev) + (here - base)), float(kLeastPower));
      const int moved = int(ceilf(size)) + 1;
      sum *= exp2_of(top - base);
      scale_acc(acc, exp2_of(top - base + float(power - moved)));
      top = next;
      power = moved;
    }
    const float lift = times2(1.0f, 15 + ev - power);
    // `base` is a rounded product, off from the one that the fma does not round by half
    // a unit in its last place.  Up to 2^20 that is a factor near 1 which every weight of
    // the row has; past it the weights would leave fp16's range, so the product is
    // rounded here too and the row's best key weighs 1.
    if (__any(fabsf(base) > 0x1p20f)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = s[r] * c - base;
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c, -base);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = exp2_of(s[r]);
      sum += s[r];
      s[r] *= lift;
    }
    accumulate_tile<NT>(stage + Frag<ND>::ALONG, split_lane(s), acc);
  }
  sum = both_sum(sum);
  if (!live) return;
  const float back = times2(1.0f, power - 29);
  if (it.part < 0) {
    store_lane<NT>(a.o + int64_t(it.q0 + query) * a.o_ld + int64_t(head) * a.dim, a.dim, half, acc,
                   sum > 0 ? back / sum : 0.0f);
    if (a.lse && half == 0)
      a.lse[int64_t(it.q0 + query) * heads + head] =
          ((top > -__builtin_inff() ? top : 0.0f) + __builtin_amdgcn_logf(sum)) * kLn2;
  } else {
    const int64_t slot =
        (int64_t(it.part) * heads + head) * kAttnSplitRows + (query - it.first);
    store_lane<NT>(a.part + slot * a.dim, a.dim, half, acc, back);
    if (half == 0) {
      a.part_ml[slot * 2] = top;
      a.part_ml[slot * 2 + 1] = sum;
    }
  }
}

// 16 values of a lane through LDS to the same lane of the wave's partner.
__device__ __forceinline__ void give(char* lds, const float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<a4*>(lds + i * 1024 + (threadIdx.x & 63) * 16) =
        a4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
}
__device__ __forceinline__ void take(const char* lds, float (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const a4 v = *reinterpret_cast<const a4*>(lds + i * 1024 + (threadIdx.x & 63) * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * i + j] = v[j];
  }
}

// The backward kernels pair two waves on a SIMD for 32 queries (or keys): one forms
// the weights P, the other dP, and P goes over through LDS.  One wave for both
// holds all of the SIMD's registers, and its exponentials and splits leave the
// matrix cores idle (39% of the time in use, 1.45 ms for dq of 8192 positions, 16
// heads of 128); paired, each has half, and one wave's arithmetic runs beside the
// other's products.  A step's score products are formed a step ahead of its
// gradient's, so a step has one barrier (dq) or two (dk and dv).
template <int ND, bool WEIGHTS>
__device__ __forceinline__ void split_back_rows_wave(const SplitAttnArgs& a, char* lds) {
  constexpr int NT = Frag<ND>::NT, ALONG = Frag<ND>::ALONG, ACROSS = Frag<ND>::ACROSS;
  // [2][K, V along], [2][K across], [2][pair][P]
  char* const across = lds + 4 * ALONG;
  char* const passed = across + 2 * ACROSS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = wave & 3;
  const int half = lane >> 5, n = lane & 31, heads = a.kv_heads * a.group;
  const int head = head_of(int(blockIdx.x % heads), heads), kv = head / a.group;
  const AttnItem it = a.items[blockIdx.x / heads];
  if (a.marks[int64_t(it.seq) * a.kv_heads + kv]) return;
  const int tile0 = it.key_begin / kAttnTile, tiles = (it.key_end - it.key_begin + 31) / kAttnTile;
  const auto at_of = [&](int t) { return int64_t(it.kt0 + tile0 + t) * a.kv_heads + kv; };
  const auto fetch_along = [&](int t) {
    char* to = lds + (t & 1) * 2 * ALONG;
    fetch<ND * 2, 8>(a.k_along + at_of(t) * ALONG, to, wave);
    fetch<ND * 2, 8>(a.v_along + at_of(t) * ALONG, to + ALONG, wave);
  };
  const auto fetch_across = [&](int t) {
    fetch<NT * 4, 8>(a.k_across + at_of(t) * ACROSS, across + (t & 1) * ACROSS, wave);
  };
  if (tiles > 0) fetch_along(0);
  const int first = it.first + 32 * pair, own = min(first / 32, (it.lq - 1) / 32);
  const int query = min(first + n, it.lq - 1), last = min(first + 31, it.lq - 1);
  const auto seen_by = [&](int q) {
    return min(it.key_end, a.causal ? max(0, q + 1 + it.lk - it.lq) : it.lk);
  };
  const int limit = seen_by(query), whole = seen_by(min(first, it.lq - 1));
  const int end = first < it.lq ? seen_by(last) : 0;
  const int64_t q_at = int64_t(it.qt0 + own) * heads + head;
  h8 oh[ND], ol[ND];
  load_own<ND>((WEIGHTS ? a.q_along : a.g_along) + q_at * ALONG, oh, ol);
  const int e_own = WEIGHTS ? a.q_exp[q_at] : a.g_exp[q_at];
  const float stat = a.stats[q_at * 64 + (WEIGHTS ? 0 : 32) + n];
  s16 acc[NT];
#pragma unroll
  for (int m = 0; m < NT; ++m) acc[m] = s16(0.0f);
  Follower power;
  float x[16];
  // The wave's part of step t's scores: P, given to the partner, or dP - delta.
  const auto scores = [&](int t) {
    const int key0 = (tile0 + t) * kAttnTile;
    if (key0 >= end) return;
    const char* stage = lds + (t & 1) * 2 * ALONG;
    if constexpr (WEIGHTS) {
      const float c = times2(a.scale_log2e, exponent_at(a.k_exp, at_of(t)) + e_own - 28);
      product<ND>(stage, oh, ol, x);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = exp2_of(fmaf(x[r], c, -stat));
      if (key0 + 32 > whole) {
        const int seen = limit - key0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = row_of(r) < seen ? x[r] : 0.0f;
      }
      give(passed + ((t & 1) * 4 + pair) * 4096, x);
    } else {
      const float c = times2(1.0f, exponent_at(a.v_exp, at_of(t)) + e_own - 28);
      product<ND>(stage + ALONG, oh, ol, x);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = fmaf(x[r], c, -stat);
    }
  };
  if (tiles > 0) {
    step_begins();
    if (tiles > 1) fetch_along(1);
    fetch_across(0);
    scores(0);
  }
  for (int t = 0; t < tiles; ++t) {
    step_begins();
    if (t + 2 < tiles) fetch_along(t + 2);
    if (t + 1 < tiles) fetch_across(t + 1);
    if (!WEIGHTS && (tile0 + t) * kAttnTile < end) {
      float p[16];
      take(passed + ((t & 1) * 4 + pair) * 4096, p);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] *= p[r];
      const int up = power.follow(x, exponent_at(a.k_exp, at_of(t)), acc);
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = times2(x[r], up);
      accumulate_tile<NT>(across + (t & 1) * ACROSS, split_lane(x), acc);
    }
    if (t + 1 < tiles) scores(t + 1);
  }
  if (WEIGHTS || first + n >= it.lq) return;
  float* to = it.part < 0 ? a.o + int64_t(it.q0 + query) * a.o_ld + int64_t(head) * a.dim
                          : a.part + ((int64_t(it.part) * heads + head) * kAttnSplitRows +
                                      (query - it.first)) * a.dim;
  store_lane<NT>(to, a.dim, half, acc, times2(a.scale, max(power.f, -200) - 14));
}
template <int ND>
__global__ __launch_bounds__(512, ND <= 4 ? 4 : 2) void attention_split_back_rows(SplitAttnArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  // The first four waves form the weights, their partners the gradients of scores.
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) < 4) split_back_rows_wave<ND, true>(a, lds);
  else split_back_rows_wave<ND, false>(a, lds);
}

template <int ND, bool WEIGHTS>
__device__ __forceinline__ void split_back_keys_wave(const SplitAttnArgs& a, char* lds) {
  constexpr int NT = Frag<ND>::NT, ALONG = Frag<ND>::ALONG, ACROSS = Frag<ND>::ACROSS;
  // [2][q, g along], [2][q, g across], [pair][P]: with heads of 64, half of the
  // compute unit's LDS, so that two workgroups share it.
  char* const across = lds + 4 * ALONG;
  char* const passed = across + 4 * ACROSS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pair = wave & 3;
  const int half = lane >> 5, n = lane & 31, heads = a.kv_heads * a.group;
  const int kv = head_of(int(blockIdx.x % a.kv_heads), a.kv_heads);
  const AttnItem it = a.items[blockIdx.x / a.kv_heads];
  if (a.marks[int64_t(it.seq) * a.kv_heads + kv]) return;
  const int ahead = it.lk - it.lq, q_tiles = (it.lq + 31) / kAttnTile;
  // From the last tile of queries back, the group's heads of a tile in turn: every
  // workgroup of a key head goes the same way, so those that run together read
  // the same tiles through the XCD's L2.
  const auto tile_of = [&](int i) { return q_tiles - 1 - i / a.group; };
  const auto at_of = [&](int i) {
    return int64_t(it.qt0 + tile_of(i)) * heads + kv * a.group + i % a.group;
  };
  const auto fetch_along = [&](int i) {
    char* to = lds + (i & 1) * 2 * ALONG;
    const int64_t at = at_of(i);
    fetch<ND * 2, 8>(a.q_along + at * ALONG, to, wave);
    fetch<ND * 2, 8>(a.g_along + at * ALONG, to + ALONG, wave);
  };
  // Lane n's statistic (lse2 or delta) of the step's query n.
  const auto stats_of = [&](int i) { return a.stats[at_of(i) * 64 + (WEIGHTS ? 0 : 32) + n]; };
  const auto fetch_across = [&](int i) {
    char* to = across + (i & 1) * 2 * ACROSS;
    const int64_t at = at_of(i);
    fetch<NT * 4, 8>(a.q_across + at * ACROSS, to, wave);
    fetch<NT * 4, 8>(a.g_across + at * ACROSS, to + ACROSS, wave);
  };
  const int begin = it.key_begin, end = it.key_end;
  if (begin < end) fetch_along(begin);
  const int first = it.first + 32 * pair, own = min(first / 32, (it.lk - 1) / 32);
  const int key = first + n;
  const int64_t k_at = int64_t(it.kt0 + own) * a.kv_heads + kv;
  h8 oh[ND], ol[ND];
  load_own<ND>((WEIGHTS ? a.k_along : a.v_along) + k_at * ALONG, oh, ol);
  const int e_own = WEIGHTS ? a.k_exp[k_at] : a.v_exp[k_at];
  s16 acc[NT];
#pragma unroll
  for (int m = 0; m < NT; ++m) acc[m] = s16(0.0f);
  Follower power;
  float x[16];
  // Whether a query of step i sees a key of the pair.
  const auto seen = [&](int i) {
    return first < it.lk && (!a.causal || tile_of(i) * kAttnTile + 31 + ahead >= first);
  };
  // The wave's part of step i's scores: P, given to the partner, or dP - delta.
  const auto scores = [&](int i, float stat) {
    if (!seen(i)) return;
    const char* stage = lds + (i & 1) * 2 * ALONG;
    const int query0 = tile_of(i) * kAttnTile;
    product<ND>(stage + (WEIGHTS ? 0 : ALONG), oh, ol, x);
    const float c = WEIGHTS ? times2(a.scale_log2e, exponent_at(a.q_exp, at_of(i)) + e_own - 28)
                            : times2(1.0f, exponent_at(a.g_exp, at_of(i)) + e_own - 28);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int v = __builtin_amdgcn_ds_bpermute(16 * half + 4 * row_of(r),
                                                 __builtin_bit_cast(int, stat));
      x[r] = fmaf(x[r], c, -__builtin_bit_cast(float, v));
    }
    if constexpr (!WEIGHTS) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = exp2_of(x[r]);
    if (a.causal && query0 + ahead < first + 31) {
      const int blind = key - query0 - ahead - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = row_of(r) >= blind ? x[r] : 0.0f;
    }
    give(passed + pair * 4096, x);
  };
  float stat = 0;  // of the step after this one
  if (begin < end) {
    stat = stats_of(begin);
    step_begins();
    const float now = stat;
    if (begin + 1 < end) {
      fetch_along(begin + 1);
      stat = stats_of(begin + 1);
    }
    fetch_across(begin);
    scores(begin, now);
  }
  for (int i = begin; i < end; ++i) {
    step_begins();
    const float next = stat;
    if (i + 2 < end) {
      fetch_along(i + 2);
      stat = stats_of(i + 2);
    }
    if (i + 1 < end) fetch_across(i + 1);
    const char* stage = across + (i & 1) * 2 * ACROSS;
    const bool here = seen(i);
    if constexpr (WEIGHTS) {
      if (here) {
        const int up = power.follow(x, exponent_at(a.g_exp, at_of(i)), acc);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = times2(x[r], up);
        accumulate_tile<NT>(stage + ACROSS, split_lane(x), acc);
      }
      lds_settled();  // the partner has taken P
    } else {
      if (here) {
        float p[16];
        take(passed + pair * 4096, p);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= p[r];
        const int up = power.follow(x, exponent_at(a.q_exp, at_of(i)), acc);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = times2(x[r], up);
      }
      lds_settled();
      if (here) accumulate_tile<NT>(stage, split_lane(x), acc);
    }
    if (i + 1 < end) scores(i + 1, next);
  }
  if (key >= it.lk) return;
  const float factor = times2(WEIGHTS ? 1.0f : a.scale, max(power.f, -200) - 14);
  float* to;
  if (it.part < 0)
    to = (WEIGHTS ? a.o + int64_t(it.k0 + key) * a.o_ld : a.dk + int64_t(it.k0 + key) * a.dk_ld) +
         int64_t(kv) * a.dim;
  else
    to = a.part + (WEIGHTS ? 0 : a.part_dk) +
         ((int64_t(it.part) * a.kv_heads + kv) * kAttnSplitRows + (key - it.first)) * a.dim;
  store_lane<NT>(to, a.dim, half, acc, factor);
}
template <int ND>
__global__ __launch_bounds__(512, ND <= 4 ? 4 : 2) void attention_split_back_keys(SplitAttnArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  // The first four waves form the weights, their partners the gradients of scores.
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) < 4) split_back_keys_wave<ND, true>(a, lds);
  else split_back_keys_wave<ND, false>(a, lds);
}

// The sum of the parts of up to 128 rows of `heads` heads: 16 lanes a row.
struct SumArgs {
  const AttnJoin* joins;
  int count, heads, dim;
  const float* part[2];
  float* out[2];
  int64_t ld[2];
};
__global__ __launch_bounds__(256) void attention_sum(SumArgs a) {
  const int64_t work = int64_t(a.count) * a.heads * (kAttnSplitRows / 16);
  const int which = blockIdx.y;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int64_t item = w / (kAttnSplitRows / 16);
    const int head = int(item % a.heads);
    const AttnJoin j = a.joins[item / a.heads];
    const int row = int(w % (kAttnSplitRows / 16)) * 16 + (threadIdx.x >> 4);
    if (j.first + row >= j.lq) continue;
    for (int c = (threadIdx.x & 15) * 4; c < a.dim; c += 64) {
      a4 s = {0, 0, 0, 0};
#pragma unroll 4
      for (int p = 0; p < j.parts; ++p) {
        float x[4];
        load_cols<4>(a.part[which] +
                         (((int64_t(j.part) + p) * a.heads + head) * kAttnSplitRows + row) * a.dim,
                     c, a.dim, x);
        s += a4{x[0], x[1], x[2], x[3]};
      }
      store_cols(a.out[which] + int64_t(j.q0 + j.first + row) * a.ld[which] + int64_t(head) * a.dim,
                 c, a.dim, s);
    }
  }
}

}  // namespace
}  // namespace lmp_hip
